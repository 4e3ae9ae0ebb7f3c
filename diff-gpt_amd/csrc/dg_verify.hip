// Drafted tokens against the target model's probabilities (dg_verify_drafts): how many of a
// row's drafts stand, and a draw of the token after them, from given random numbers.
//
// Draft i stands iff u q_i(x) < p_i(x); after the first that does not, the token is the first
// maximum of max(p - q, 0) / e over the vocabulary, e being Exp(1) variates: an exponential
// race, which draws from that difference without sums or sorting (a prefix sum of 50000
// probabilities in fp32 would move its borders by more than the small ones are apart).
//
// Rows of logits are read once for their maximum and sum, exponentials in fp32 with the scale
// in two terms (its rounding would shift all of a row's exponents alike), sums in fp64 but for a
// thread's four vectors at a time, 32 exponentials at most, so that the decisions u q < p come
// out as in 64 bits but for a few in 10^7.  fp64 logits are taken as they are, all of it in fp64.
// Then one workgroup or several a row race over the logits of the one row that decides.
//
// Few logits: one launch, a workgroup for each row of the batch.  Otherwise two: the
// statistics of all rows, split where rows are few, and the race, whose parts meet in one
// atomic maximum (its result depends on no order; the statistics' launch clears it; in fp64, whose
// ratios and ids are no 64 bits, each leaves its own) and whose last part writes the row's results.
//
// 64 rows of 6 + 5 of 49999 bf16 logits: statistics 18 us, by HBM and vector instructions; race
// 14 us, a chain of latencies: the rows' statistics, the logits, two atomics.  (26 each with
// loads of single elements where rows start anywhere, the exponents' offset raised with every
// new maximum and the parts of a row's statistics joined by one thread.)
// The same of fp64 logits, 282 MB, both launches 94 us (fp32 39; at temperature 0 58 and 23).
#include "dg_common.h"

#include <algorithm>
#include <cmath>

namespace dg {

constexpr int kMostDrafts = 64;

struct VerifyArgs {
  const void* target;
  int64_t tb, tn;
  const void* draft;  // null: the drafts are certain
  int64_t db, dn;
  const int64_t* tokens;
  const float* uniforms;
  const float* noise;
  int64_t noise_ld;
  const int32_t* counts;
  float scale_hi, scale_lo;  // inverse temperature in log2 units, two terms
  double scale;              // ... in natural ones
  int64_t* accepted;
  int64_t* out_tokens;
  float* out_logprobs;
  int B, N, V;
  int rows;   // of logits for each row of the batch: N + 1 of the target, N of the draft
  int split;  // parts of a row's statistics
  int parts;  // parts of a race
  void* stats;               // (B, rows, split) of VerifyStat
  struct VerifyRace* races;  // (B)
  struct VerifyBest* bests;  // fp64: (B, parts)
};

// The arithmetic of a row of T: fp32 in log2 units, fp64 for fp64.
template <typename T>
struct VerifyAcc {
  using type = float;
};
template <>
struct VerifyAcc<double> {
  using type = double;
};

// Sum of exp(scale (x - top)) over (a part of) a row and the logit of its draft.  top is some
// logit of the row that no other is far above (kAhead), and at temperature 0 its maximum, at
// the id `at`.
template <typename A>
struct VerifyStat {
  double sum;
  A top;
  A drafted;
  int at;
  int pad;
};
struct VerifyRace {
  unsigned long long best;  // the ratio's bits above the complement of its id
  unsigned int done;
  unsigned int pad;
};
// A race's best: its ratio, 0 where none is positive, and the first id that has it.
struct VerifyBest {
  double ratio;
  int id;
  int pad;
};

template <typename T>
__device__ __forceinline__ float logit(T x) {
  return to_f32(x);
}
__device__ __forceinline__ double logit(double x) { return x; }

template <typename A>
__device__ __forceinline__ A no_logit() {
  return -(A)__builtin_huge_valf();
}

// exp(scale d), scale d at most kAhead in log2 units
__device__ __forceinline__ float scaled_exp(const VerifyArgs& a, float d) {
  return __builtin_amdgcn_exp2f(__builtin_fmaf(d, a.scale_hi, d * a.scale_lo));
}
__device__ __forceinline__ double scaled_exp(const VerifyArgs& a, double d) { return ::exp(d * a.scale); }

// s and what follows it in the row, o; the draft's logit stays s's.
template <typename A>
__device__ __forceinline__ void join_stat(const VerifyArgs& a, VerifyStat<A>& s, const VerifyStat<A>& o) {
  const bool up = o.top > s.top || (o.top == s.top && o.at < s.at);
  const A top = o.top > s.top ? o.top : s.top;
  // -inf: nothing yet
  const double f = s.top == no_logit<A>() ? 0.0 : (double)scaled_exp(a, s.top - top);
  const double g = o.top == no_logit<A>() ? 0.0 : (double)scaled_exp(a, o.top - top);
  s.sum = s.sum * f + o.sum * g;
  s.top = top;
  s.at = up ? o.at : s.at;
}

// 16 bytes of a row from any element on, in one load (rows of an odd vocabulary start
// anywhere), so that which thread has a logit, and a row's bits, depend on its id alone.
typedef u32x4_t __attribute__((aligned(2))) u32x4_any_t;

template <typename T, int N>
__device__ __forceinline__ void load_any(const T* p, typename VerifyAcc<T>::type (&z)[N]) {
  constexpr int VE = 16 / (int)sizeof(T);
#pragma unroll
  for (int c = 0; c < N / VE; ++c) {
    const u32x4_t w = reinterpret_cast<const u32x4_any_t*>(p)[c];
    if constexpr (sizeof(T) == 8) {
      __builtin_memcpy(z + c * VE, &w, 16);
    } else {
      RowRegs<T, VE> r;
#pragma unroll
      for (int i = 0; i < 4; ++i) r.w[i] = w[i];
#pragma unroll
      for (int i = 0; i < VE; ++i) z[c * VE + i] = elem<T, VE>(r, i);
    }
  }
}

// log2 of how far an exponential may lie above that of `top` before it is raised (each raise
// costs all lanes of a wave some 40 instructions, a comparison one)
constexpr float kAhead = 16.f;

__device__ __forceinline__ bool far_ahead(const VerifyArgs& a, float d) { return d * a.scale_hi > kAhead; }
__device__ __forceinline__ bool far_ahead(const VerifyArgs& a, double d) {
  return d * a.scale > (double)kAhead * 0.69314718055994530942;
}

// N further logits from id v0 on (-inf for what is not there) into a thread's statistics, whose
// sum is `sum` and, of the latest, `part`.  A NaN makes the sum one, beside logits of -inf alone too.
template <typename A, int N, bool GREEDY>
__device__ __forceinline__ void add_logits(const VerifyArgs& a, const A (&z)[N], int v0, A& top, int& at, double& sum, A& part) {
  const A kNone = no_logit<A>();
  A m = z[0];
#pragma unroll
  for (int i = 1; i < N; ++i) m = __builtin_elementwise_max(m, z[i]);
  if (GREEDY ? m > top : top == kNone ? m > top : far_ahead(a, m - top)) {
    if constexpr (GREEDY) {
#pragma unroll
      for (int i = N - 1; i >= 0; --i)
        if (z[i] == m) at = v0 + i;
    }
    if (top != kNone) {
      const A f = scaled_exp(a, top - m);
      part *= f;
      sum *= (double)f;
    }
    top = m;
  }
  if (top == kNone) {  // nothing yet
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (z[i] != z[i]) part = z[i];
    return;
  }
  A some = (A)0;
#pragma unroll
  for (int i = 0; i < N; ++i) some += scaled_exp(a, z[i] - top);
  part += some;
}

// Thread `tid` of `step`'s part of the statistics of a row's vectors first .. end - 1, and of
// what follows the last whole one where end is past it.  Four vectors are in flight.
template <typename T, bool GREEDY>
__device__ __forceinline__ VerifyStat<typename VerifyAcc<T>::type> row_stat(const VerifyArgs& a, const T* x, int first, int end,
                                                                            int tid, int step) {
  using A = typename VerifyAcc<T>::type;
  constexpr int VE = 16 / (int)sizeof(T), U = 4;
  const int whole = min(end, a.V / VE);
  A top = no_logit<A>(), part = (A)0;
  double sum = 0.0;
  int at = 0x7fffffff, j = first + tid;
  for (; j + (U - 1) * step < whole; j += U * step) {
    A z[U][VE];
#pragma unroll
    for (int u = 0; u < U; ++u) load_any<T, VE>(x + (int64_t)(j + u * step) * VE, z[u]);
#pragma unroll
    for (int u = 0; u < U; ++u) add_logits<A, VE, GREEDY>(a, z[u], (j + u * step) * VE, top, at, sum, part);
    sum += (double)part;
    part = (A)0;
  }
  for (; j < whole; j += step) {
    A z[VE];
    load_any<T, VE>(x + (int64_t)j * VE, z);
    add_logits<A, VE, GREEDY>(a, z, j * VE, top, at, sum, part);
  }
  if (j < end) {  // the row's last, incomplete vector
    A z[VE];
#pragma unroll
    for (int i = 0; i < VE; ++i) {
      z[i] = no_logit<A>();
      if (j * VE + i < a.V) z[i] = logit(x[j * VE + i]);
    }
    add_logits<A, VE, GREEDY>(a, z, j * VE, top, at, sum, part);
  }
  return VerifyStat<A>{sum + (double)part, top, (A)0, at, 0};
}

template <typename T>
__device__ __forceinline__ int row_vectors(const VerifyArgs& a) {
  constexpr int VE = 16 / (int)sizeof(T);
  return (a.V + VE - 1) / VE;
}

__device__ __forceinline__ double wave_max(double v) {
#pragma unroll
  for (int x = 1; x < 64; x <<= 1) {
    const double o = __shfl_xor(v, x, 64);
    v = o > v ? o : v;
  }
  return v;
}
// The lanes' statistics joined, for all of them: one factor a lane, then sums in fp64.
template <typename A>
__device__ __forceinline__ VerifyStat<A> wave_stat(const VerifyArgs& a, VerifyStat<A> s) {
  const A top = wave_max(s.top);
  if (s.top != top) {
    s.sum *= s.top == no_logit<A>() ? 0.0 : (double)scaled_exp(a, s.top - top);
    s.at = 0x7fffffff;
  }
#pragma unroll
  for (int x = 1; x < 64; x <<= 1) {
    s.sum += __shfl_xor(s.sum, x, 64);
    s.at = min(s.at, __shfl_xor(s.at, x, 64));
  }
  s.top = top;
  return s;
}

template <typename T>
__device__ __forceinline__ const T* row_at(const VerifyArgs& a, int64_t b, int r) {
  return r <= a.N ? static_cast<const T*>(a.target) + b * a.tb + r * a.tn
                  : static_cast<const T*>(a.draft) + b * a.db + (r - a.N - 1) * a.dn;
}

__device__ __forceinline__ int drafts_of(const VerifyArgs& a, int64_t b) {
  return min(max(a.counts != nullptr ? a.counts[b] : a.N, 0), a.N);
}

// whether row r of the batch's row b is looked at
__device__ __forceinline__ bool row_used(const VerifyArgs& a, int r, int count) {
  return r <= a.N ? r <= count : r - a.N - 1 < count;
}

// The logit of row r's draft, -inf for one outside the vocabulary.
template <typename T>
__device__ __forceinline__ typename VerifyAcc<T>::type drafted_logit(const VerifyArgs& a, int64_t b, int r, const T* x) {
  using A = typename VerifyAcc<T>::type;
  const int i = r <= a.N ? r : r - a.N - 1;
  if (i >= a.N) return (A)0;
  const int64_t t = a.tokens[b * a.N + i];
  return t >= 0 && t < a.V ? logit(x[t]) : no_logit<A>();
}

template <typename A>
__device__ __forceinline__ double drafted_prob(const VerifyArgs& a, const VerifyStat<A>& s) {
  return (double)scaled_exp(a, s.drafted - s.top) / s.sum;
}

// How many of row b's drafts stand: every wave finds it, lane i for draft i.
template <typename A, bool GREEDY>
__device__ __forceinline__ int standing(const VerifyArgs& a, int64_t b, int count, const VerifyStat<A>* stats, int lane) {
  bool falls = false;
  if (lane < count) {
    const int64_t x = a.tokens[b * a.N + lane];
    if constexpr (GREEDY) {
      falls = x != stats[lane].at || stats[lane].sum != stats[lane].sum;
    } else {
      const double p = drafted_prob(a, stats[lane]);
      const double q = a.draft != nullptr ? drafted_prob(a, stats[a.N + 1 + lane]) : 1.0;
      falls = !((double)a.uniforms[b * a.N + lane] * q < p);  // so does a draft outside the vocabulary
    }
  }
  const uint64_t f = __builtin_amdgcn_ballot_w64(falls);
  return f == 0 ? count : __builtin_ctzll(f);
}

// A race's best so far and its order: the larger ratio, of equal ones the smaller id.  fp32: the
// ratio's bits above the complement of its id, 0 where no ratio is positive.
__device__ __forceinline__ unsigned long long race_best(float ratio, int id) {
  return ratio > 0.f ? (unsigned long long)__float_as_uint(ratio) << 32 | (0xffffffffu - (unsigned)id) : 0ull;
}
__device__ __forceinline__ VerifyBest race_best(double ratio, int id) { return VerifyBest{ratio > 0.0 ? ratio : 0.0, id, 0}; }
__device__ __forceinline__ void race_join(unsigned long long& x, unsigned long long o) { x = o > x ? o : x; }
__device__ __forceinline__ void race_join(VerifyBest& x, const VerifyBest& o) {
  if (o.ratio > x.ratio || (o.ratio == x.ratio && o.id < x.id)) x = o;
}
__device__ __forceinline__ bool race_won(unsigned long long x) { return x != 0; }
__device__ __forceinline__ bool race_won(const VerifyBest& x) { return x.ratio > 0.0; }
__device__ __forceinline__ int best_id(unsigned long long x) { return x == 0 ? 0 : (int)(0xffffffffu - (unsigned)x); }
__device__ __forceinline__ int best_id(const VerifyBest& x) { return race_won(x) ? x.id : 0; }
template <typename A>
using RaceBest = decltype(race_best(A(), 0));

__device__ __forceinline__ float over_noise(float r, float n) { return r * __builtin_amdgcn_rcpf(n); }
__device__ __forceinline__ double over_noise(double r, float n) { return r / (double)n; }

// Thread `tid` of `step`'s best of row `at`'s race over vectors first .. end - 1 (of the
// vocabulary).  rest: the row's draft did not stand.
template <typename T, typename A = typename VerifyAcc<T>::type>
__device__ __forceinline__ RaceBest<A> race(const VerifyArgs& a, int64_t b, int at, bool rest, const VerifyStat<A>& sp,
                                            const VerifyStat<A>& sq, int first, int end, int tid, int step) {
#pragma clang fp contract(off)  // p - q of equal logits is 0, not what rounding one product leaves
  constexpr int VE = 16 / (int)sizeof(T);
  const T* const xp = row_at<T>(a, b, at);
  const bool drawn = a.draft != nullptr && rest;  // uniform over the workgroup
  const T* const xq = drawn ? row_at<T>(a, b, a.N + 1 + at) : xp;
  const int64_t drafted = rest && a.draft == nullptr ? a.tokens[b * a.N + at] : -1;
  const float* const e = a.noise + b * a.noise_ld;
  const A ip = (A)(1.0 / sp.sum), iq = drawn ? (A)(1.0 / sq.sum) : (A)0;
  A best = (A)0;
  int id = 0;
  auto run = [&](A zp, A zq, float n, int v) __attribute__((always_inline)) {
    A r = scaled_exp(a, zp - sp.top) * ip;
    if (drawn) r -= scaled_exp(a, zq - sq.top) * iq;
    if (v == drafted) r = (A)0;
    r = over_noise(r, n);
    if (r > best) {  // ids rise: the first of equals stays
      best = r;
      id = v;
    }
  };
  const int whole = min(end, a.V / VE);
  int j = first + tid;
#pragma unroll 2
  for (; j < whole; j += step) {
    A zp[VE], zq[VE];
    float n[VE < 4 ? 4 : VE];
    load_any<T, VE>(xp + (int64_t)j * VE, zp);
    if (drawn) load_any<T, VE>(xq + (int64_t)j * VE, zq);
    if constexpr (VE >= 4) {
      load_any<float, VE>(e + (int64_t)j * VE, n);
    } else {
#pragma unroll
      for (int i = 0; i < VE; ++i) n[i] = e[j * VE + i];
    }
#pragma unroll
    for (int i = 0; i < VE; ++i) run(zp[i], drawn ? zq[i] : (A)0, n[i], j * VE + i);
  }
  if (j < end)
    for (int v = j * VE; v < a.V; ++v) run(logit(xp[v]), logit(xq[v]), e[v], v);
  return race_best(best, id);
}

__device__ __forceinline__ unsigned long long wave_best(unsigned long long x) {
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) race_join(x, __shfl_xor(x, off, 64));
  return x;
}
__device__ __forceinline__ VerifyBest wave_best(VerifyBest x) {
#pragma unroll
  for (int off = 1; off < 64; off <<= 1)
    race_join(x, VerifyBest{__shfl_xor(x.ratio, off, 64), __shfl_xor(x.id, off, 64), 0});
  return x;
}

// Row b's results but for the token behind the standing drafts, by one wave.
template <typename A>
__device__ __forceinline__ void write_drafts(const VerifyArgs& a, int64_t b, int stands, const VerifyStat<A>* stats, int lane) {
  for (int j = lane; j <= a.N; j += 64) {
    if (j == stands) continue;
    int64_t t = -1;
    float lp = 0.f;
    if (j < stands) {
      t = a.tokens[b * a.N + j];
      lp = (float)((double)(stats[j].drafted - stats[j].top) * a.scale - log(stats[j].sum));
    }
    a.out_tokens[b * (a.N + 1) + j] = t;
    a.out_logprobs[b * (a.N + 1) + j] = lp;
  }
  if (lane == 0) a.accepted[b] = stands;
}

// That token, by one thread.
template <typename T, typename A = typename VerifyAcc<T>::type>
__device__ __forceinline__ void write_token(const VerifyArgs& a, int64_t b, int stands, int token, const VerifyStat<A>& s) {
  const A x = logit(row_at<T>(a, b, stands)[token]);
  a.out_tokens[b * (a.N + 1) + stands] = token;
  a.out_logprobs[b * (a.N + 1) + stands] = (float)((double)(x - s.top) * a.scale - log(s.sum));
}

// One workgroup a row of the batch.
template <typename T, bool GREEDY>
__global__ __launch_bounds__(512) void verify_alone_kernel(const VerifyArgs a) {
  using A = typename VerifyAcc<T>::type;
  __shared__ VerifyStat<A> stats[2 * kMostDrafts + 1];
  __shared__ RaceBest<A> bests[8];
  const int64_t b = blockIdx.x;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int count = drafts_of(a, b);
  for (int r = wv; r < a.rows; r += 8) {
    if (!row_used(a, r, count)) continue;
    const T* x = row_at<T>(a, b, r);
    A drafted = (A)0;
    if (lane == 0) drafted = drafted_logit<T>(a, b, r, x);
    VerifyStat<A> s = wave_stat(a, row_stat<T, GREEDY>(a, x, 0, row_vectors<T>(a), lane, 64));
    s.drafted = drafted;
    if (lane == 0) stats[r] = s;
  }
  __syncthreads();
  const int stands = standing<A, GREEDY>(a, b, count, stats, lane);
  if (wv == 0) write_drafts(a, b, stands, stats, lane);
  if constexpr (GREEDY) {
    if (tid == 0) write_token<T>(a, b, stands, min(stats[stands].at, a.V - 1), stats[stands]);
    return;
  }
  const bool rest = stands < count;
  const VerifyStat<A> sp = stats[stands], sq = a.draft != nullptr && rest ? stats[a.N + 1 + stands] : sp;
  for (int again = 0; again < 2; ++again) {
    const RaceBest<A> mine = wave_best(race<T>(a, b, stands, rest && again == 0, sp, sq, 0, row_vectors<T>(a), tid, 512));
    if (lane == 0) bests[wv] = mine;
    __syncthreads();
    RaceBest<A> best = bests[0];
#pragma unroll
    for (int i = 1; i < 8; ++i) race_join(best, bests[i]);
    if (race_won(best) || !rest || again == 1) {  // the same in all threads
      if (tid == 0) write_token<T>(a, b, stands, best_id(best), sp);
      return;
    }
    __syncthreads();  // nothing left of the difference: the target's row itself
  }
}

// Statistics of one part of one row of logits a workgroup.
template <typename T, bool GREEDY>
__global__ __launch_bounds__(256) void verify_stat_kernel(const VerifyArgs a) {
  using A = typename VerifyAcc<T>::type;
  __shared__ VerifyStat<A> waves[4];
  const int part = (int)(blockIdx.x % (unsigned)a.split);
  const unsigned br = blockIdx.x / (unsigned)a.split;
  const int64_t b = br / (unsigned)a.rows;
  const int r = (int)(br - (unsigned)b * (unsigned)a.rows);
  if (r == 0 && part == 0 && threadIdx.x == 0) a.races[b] = VerifyRace{0ull, 0u, 0u};
  if (!row_used(a, r, drafts_of(a, b))) return;  // whole workgroups
  const T* x = row_at<T>(a, b, r);
  A drafted = (A)0;
  if (part == 0 && threadIdx.x == 0) drafted = drafted_logit<T>(a, b, r, x);
  const int n = row_vectors<T>(a);
  const int per = (n + a.split - 1) / a.split;
  const int first = min(part * per, n), end = min(first + per, n);
  const VerifyStat<A> s = wave_stat(a, row_stat<T, GREEDY>(a, x, first, end, (int)threadIdx.x, 256));
  if ((threadIdx.x & 63) == 0) waves[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x != 0) return;
  VerifyStat<A> all = waves[0];
  for (int i = 1; i < 4; ++i) join_stat(a, all, waves[i]);
  all.drafted = drafted;
  static_cast<VerifyStat<A>*>(a.stats)[(int64_t)br * a.split + part] = all;
}

// One part of one row's race a workgroup; the last to end writes the row's results.
template <typename T, bool GREEDY>
__global__ __launch_bounds__(512) void verify_race_kernel(const VerifyArgs a) {
  using A = typename VerifyAcc<T>::type;
  __shared__ VerifyStat<A> stats[2 * kMostDrafts + 1];
  __shared__ RaceBest<A> bests[8];
  __shared__ bool again;
  const int64_t b = blockIdx.x / (unsigned)a.parts;
  const int part = (int)(blockIdx.x - (unsigned)b * (unsigned)a.parts);
  const int tid = threadIdx.x, lane = tid & 63;
  const int wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int count = drafts_of(a, b);
  if (a.split == 1) {
    for (int r = tid; r < a.rows; r += 512)
      if (row_used(a, r, count)) stats[r] = static_cast<const VerifyStat<A>*>(a.stats)[b * a.rows + r];
  } else {  // a wave a row, a lane a part
    for (int r = wv; r < a.rows; r += 8) {
      if (!row_used(a, r, count)) continue;
      const VerifyStat<A>* const s = static_cast<const VerifyStat<A>*>(a.stats) + (b * a.rows + r) * a.split;
      VerifyStat<A> all{0.0, no_logit<A>(), (A)0, 0x7fffffff, 0};
      if (lane < a.split) all = s[lane];
      const A drafted = __shfl(all.drafted, 0, 64);
      all = wave_stat(a, all);
      all.drafted = drafted;
      if (lane == 0) stats[r] = all;
    }
  }
  __syncthreads();
  const int stands = standing<A, GREEDY>(a, b, count, stats, lane);
  if (part == 0 && wv == 0) write_drafts(a, b, stands, stats, lane);
  if constexpr (GREEDY) {
    if (tid == 0) write_token<T>(a, b, stands, min(stats[stands].at, a.V - 1), stats[stands]);
    return;
  }
  const bool rest = stands < count;
  const VerifyStat<A> sp = stats[stands], sq = a.draft != nullptr && rest ? stats[a.N + 1 + stands] : sp;
  const int nv = row_vectors<T>(a);
  const int per = (nv + a.parts - 1) / a.parts;
  const int v0 = min(part * per, nv), v1 = min(v0 + per, nv);
  auto block_best = [&](bool less, int from, int to) {
    const RaceBest<A> mine = wave_best(race<T>(a, b, stands, less, sp, sq, from, to, tid, 512));
    if (lane == 0) bests[wv] = mine;
    __syncthreads();
    RaceBest<A> best = bests[0];
#pragma unroll
    for (int i = 1; i < 8; ++i) race_join(best, bests[i]);
    __syncthreads();
    return best;
  };
  RaceBest<A> best = block_best(rest, v0, v1);
  if (tid == 0) {
    // the parts' best, by whom it does not matter; the last to have added its own goes on
    bool end = true;
    if (a.parts > 1) {
      VerifyBest* const all = a.bests + b * a.parts;
      if constexpr (sizeof(A) == 8) all[part] = best;
      else __hip_atomic_fetch_max(&a.races[b].best, best, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      end = __hip_atomic_fetch_add(&a.races[b].done, 1u, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT) == (unsigned)a.parts - 1;
      if (end) {
        if constexpr (sizeof(A) == 8) {
          for (int i = 0; i < a.parts; ++i) race_join(best, all[i]);
        } else {
          best = __hip_atomic_load(&a.races[b].best, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
      }
    }
    const bool none = !race_won(best) && rest;
    again = end && none;
    if (end && !none) write_token<T>(a, b, stands, best_id(best), sp);
  }
  __syncthreads();
  if (!again) return;
  // nothing left of the difference: the target's row itself
  best = block_best(false, 0, nv);
  if (tid == 0) write_token<T>(a, b, stands, best_id(best), sp);
}

namespace {

// Logits that a wave of verify_alone_kernel goes through, up to which one workgroup does all of a
// row of the batch: of few rows, and of so many that the others' launches fill the chip too.
// us in one launch / two (8 waves, each with every eighth row of logits), rows of the batch x
// rows of logits x V: 64 x 9 x 1000 9.0 / 9.5; 64 x 9 x 2000 10.5 / 9.9; 16 x 3 x 5400
// 10.5 / 11.2; 16 x 3 x 11000 15.8 / 11.5; 8 x 1 x 16000 15.6 / 10.5; 256 x 9 x 2000
// 10.2 / 12.2; 512 x 9 x 4000 18.5 / 21.3 (a second launch is 2 us of the host's as well).
constexpr int64_t kAlone = 6144, kAloneMany = 8192, kManyRows = 256;

struct VerifyShape {
  bool alone;
  int rows, split, parts;
  size_t stat_bytes, race_bytes, ws_bytes;
};

VerifyShape verify_shape(int64_t B, int N, int64_t V, int64_t dtype) {
  VerifyShape t{};
  t.rows = 2 * N + 1;
  t.alone = (t.rows + 7) / 8 * V <= (B < kManyRows ? kAlone : kAloneMany);
  t.split = t.parts = 1;
  if (t.alone) return t;
  // about two workgroups a CU, of 2048 logits at least
  t.split = (int)std::max<int64_t>(1, std::min<int64_t>({(512 + B * t.rows - 1) / (B * t.rows), V / 2048, 64}));
  t.parts = (int)std::max<int64_t>(1, std::min<int64_t>({(256 + B - 1) / B, V / 2048, 64}));
  t.stat_bytes = (size_t)B * t.rows * t.split * (dtype == DG_F64 ? sizeof(VerifyStat<double>) : sizeof(VerifyStat<float>));
  t.race_bytes = (size_t)B * sizeof(VerifyRace);
  t.ws_bytes = t.stat_bytes + t.race_bytes;
  if (dtype == DG_F64) t.ws_bytes += (size_t)B * t.parts * sizeof(VerifyBest);
  return t;
}

template <typename T>
int launch_verify(const VerifyArgs& a, const VerifyShape& t, bool greedy, hipStream_t s) {
  const dim3 block(512);
  if (t.alone) {
    const dim3 grid((unsigned)a.B);
    if (greedy) hipLaunchKernelGGL((verify_alone_kernel<T, true>), grid, block, 0, s, a);
    else hipLaunchKernelGGL((verify_alone_kernel<T, false>), grid, block, 0, s, a);
    return check_launch("verify_alone_kernel");
  }
  const dim3 rows((unsigned)((int64_t)a.B * a.rows * a.split));
  if (greedy) hipLaunchKernelGGL((verify_stat_kernel<T, true>), rows, dim3(256), 0, s, a);
  else hipLaunchKernelGGL((verify_stat_kernel<T, false>), rows, dim3(256), 0, s, a);
  if (const int rc = check_launch("verify_stat_kernel")) return rc;
  const dim3 grid((unsigned)((int64_t)a.B * a.parts));
  if (greedy) hipLaunchKernelGGL((verify_race_kernel<T, true>), grid, block, 0, s, a);
  else hipLaunchKernelGGL((verify_race_kernel<T, false>), grid, block, 0, s, a);
  return check_launch("verify_race_kernel");
}

}  // namespace
}  // namespace dg

using namespace dg;

extern "C" size_t dg_verify_drafts_workspace_size(const dg_verify_drafts_args* args) {
  if (args == nullptr || args->B <= 0 || args->B > 0x7fffffff || args->N < 0 || args->N > kMostDrafts || args->V <= 0 ||
      args->V > 0x3fffffff)
    return 0;
  return verify_shape(args->B, (int)args->N, args->V, args->dtype).ws_bytes;
}

extern "C" int dg_verify_drafts(const dg_verify_drafts_args* args, void* workspace, size_t workspace_bytes, void* stream) {
  DG_REQUIRE(args != nullptr, DG_EINVAL, "verify_drafts: NULL argument");
  DG_REQUIRE(args->B >= 0 && args->B <= 0x7fffffff, DG_EINVAL, "verify_drafts: negative size or one past 2^31 - 1");
  DG_REQUIRE(args->N >= 0 && args->N <= kMostDrafts, DG_EINVAL, "verify_drafts: %lld drafts a row, 0 to %d", (long long)args->N,
             kMostDrafts);
  const int B = (int)args->B, N = (int)args->N;
  const int64_t V = args->V, dtype = args->dtype;
  const double inv_temperature = args->inv_temperature;
  const void *target = args->target, *draft = args->draft;
  DG_REQUIRE(V >= 1 && V <= 0x3fffffff, DG_EINVAL, "verify_drafts: a vocabulary of %lld, 1 to 2^30 - 1", (long long)V);
  DG_REQUIRE(dtype == DG_F32 || dtype == DG_BF16 || dtype == DG_F16 || dtype == DG_F64, DG_EUNSUPPORTED,
             "verify_drafts: dtype %lld unsupported", (long long)dtype);
  DG_REQUIRE(inv_temperature == 0.0 || (inv_temperature >= 0x1p-100 && inv_temperature <= 0x1p100), DG_EINVAL,
             "verify_drafts: the inverse temperature must be 0 or between 2^-100 and 2^100");
  if (B == 0) return DG_OK;
  const bool greedy = inv_temperature == 0.0;
  DG_REQUIRE(target && args->accepted && args->out_tokens && args->out_logprobs && (N == 0 || args->tokens), DG_EINVAL, "verify_drafts: NULL argument");
  DG_REQUIRE(greedy || (args->noise && (N == 0 || args->uniforms)), DG_EINVAL, "verify_drafts: random numbers missing");
  const int64_t es = dtype_bytes((int)dtype);
  DG_REQUIRE(reinterpret_cast<uintptr_t>(target) % es == 0 && reinterpret_cast<uintptr_t>(draft) % es == 0, DG_EINVAL,
             "verify_drafts: logits not aligned to their element size");
  VerifyArgs a{};
  a.target = target; a.tb = args->t_b; a.tn = args->t_n;
  a.draft = greedy ? nullptr : draft; a.db = args->d_b; a.dn = args->d_n;
  a.tokens = args->tokens; a.uniforms = args->uniforms; a.noise = args->noise; a.noise_ld = args->noise_ld; a.counts = args->counts;
  a.scale = greedy ? 1.0 : inv_temperature;
  const double l2 = a.scale * 1.4426950408889634074;
  // the leading term rounded down, so that the rest is positive and -inf times it still -inf
  a.scale_hi = (float)l2;
  if ((double)a.scale_hi >= l2) a.scale_hi = std::nextafter(a.scale_hi, 0.f);
  a.scale_lo = (float)(l2 - (double)a.scale_hi);
  a.accepted = args->accepted; a.out_tokens = args->out_tokens; a.out_logprobs = args->out_logprobs;
  a.B = B; a.N = N; a.V = (int)V;
  const VerifyShape t = verify_shape(B, N, V, dtype);
  a.rows = a.draft != nullptr ? 2 * N + 1 : N + 1;
  a.split = t.split;
  a.parts = greedy ? 1 : t.parts;
  if (t.ws_bytes > 0) {
    DG_REQUIRE(workspace != nullptr && workspace_bytes >= t.ws_bytes, DG_EWORKSPACE,
               "verify_drafts: a workspace of %zu bytes, %zu needed", workspace_bytes, t.ws_bytes);
    DG_REQUIRE((reinterpret_cast<uintptr_t>(workspace) & 15) == 0, DG_EINVAL, "verify_drafts: workspace not 16-byte aligned");
    a.stats = workspace;
    a.races = reinterpret_cast<VerifyRace*>(static_cast<char*>(workspace) + t.stat_bytes);
    a.bests = reinterpret_cast<VerifyBest*>(static_cast<char*>(workspace) + t.stat_bytes + t.race_bytes);
  }
  DG_REQUIRE((int64_t)B * (2 * N + 1) * t.split <= kMostWorkgroups256 && (int64_t)B * t.parts <= kMostWorkgroups256 / 2,
             DG_EINVAL, "verify_drafts: more than 2^32 - 1 threads");
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (dtype == DG_F64) return launch_verify<double>(a, t, greedy, s);
  if (dtype == DG_F32) return launch_verify<float>(a, t, greedy, s);
  if (dtype == DG_BF16) return launch_verify<bf16_t>(a, t, greedy, s);
  return launch_verify<f16_t>(a, t, greedy, s);
}
