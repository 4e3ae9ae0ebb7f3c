// Drafted tokens against the target model's probabilities (dg_verify_drafts): how many of a
// row's drafts stand, and a draw of the token after them, from given random numbers.
//
// Draft i stands iff u q_i(x) < p_i(x); after the first that does not, the token is the first
// maximum of max(p - q, 0) / e over the vocabulary, e being Exp(1) variates: an exponential
// race, which draws from that difference without sums or sorting (a prefix sum of 50000
// probabilities in fp32 would move its borders by more than the small ones are apart).
//
// Rows of logits are read once for their maximum and sum, exponentials in fp32 with the scale
// in two terms (its rounding would shift all of a row's exponents alike), sums in fp64, so
// that the decisions u q < p come out as in 64 bits but for a few in 10^7.  Then one
// workgroup or several a row race over the logits of the one row that decides.
//
// Few logits (kAlone): one launch, a workgroup for each row of the batch.  Otherwise two: the
// statistics of all rows, split where rows are few, and the race, whose parts meet in one
// atomic maximum (its result depends on no order; the statistics' launch clears it) and whose
// last part writes the row's results.
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
  struct VerifyStat* stats;  // (B, rows, split)
  struct VerifyRace* races;  // (B)
};

// Maximum and sum of exp(scale (x - max)) over (a part of) a row, and its first maximum's id.
struct VerifyStat {
  double sum;
  float top;
  int at;
};
struct VerifyRace {
  unsigned long long best;  // the ratio's bits above the complement of its id
  unsigned int done;
  unsigned int pad;
};

template <typename T>
__device__ __forceinline__ float logit(T x) {
  return to_f32(x);
}
template <>
__device__ __forceinline__ float logit<double>(double x) {
  return (float)x;
}

// exp(scale d), d <= 0
__device__ __forceinline__ float scaled_exp(const VerifyArgs& a, float d) {
  return __builtin_amdgcn_exp2f(__builtin_fmaf(d, a.scale_hi, d * a.scale_lo));
}

__device__ __forceinline__ void join_stat(const VerifyArgs& a, VerifyStat& s, const VerifyStat& o) {
  const bool up = o.top > s.top || (o.top == s.top && o.at < s.at);
  const float top = o.top > s.top ? o.top : s.top;
  // -inf: nothing yet
  const double f = s.top == kNegInf ? 0.0 : (double)scaled_exp(a, s.top - top);
  const double g = o.top == kNegInf ? 0.0 : (double)scaled_exp(a, o.top - top);
  s.sum = s.sum * f + o.sum * g;
  s.top = top;
  s.at = up ? o.at : s.at;
}

// This thread's part of a row's statistics: vectors of 16 bytes from an aligned address at or
// before the row, every `step`-th from `first` on.  A vector holds some of the row, so what
// it reads beside lies in the same 16 bytes.
template <typename T>
__device__ __forceinline__ VerifyStat row_stat(const VerifyArgs& a, const T* x, int first, int end, int step) {
  constexpr int VE = 16 / (int)sizeof(T);
  const int off = (int)((reinterpret_cast<uintptr_t>(x) & 15) / sizeof(T));
  const T* const base = x - off;
  VerifyStat s{0.0, kNegInf, 0x7fffffff};
  float part = 0.f;
  bool odd = false;  // a NaN
  for (int j = first; j < end; j += step) {
    const u32x4_t raw = *reinterpret_cast<const u32x4_t*>(base + (int64_t)j * VE);
    T e[VE];
    __builtin_memcpy(e, &raw, 16);
    const int v0 = j * VE - off;
    float z[VE], top = kNegInf;
#pragma unroll
    for (int i = 0; i < VE; ++i) {
      z[i] = v0 + i >= 0 && v0 + i < a.V ? logit<T>(e[i]) : kNegInf;
      odd = odd || z[i] != z[i];
      top = fmaxf(top, z[i]);
    }
    if (top > s.top) {
#pragma unroll
      for (int i = VE - 1; i >= 0; --i)
        if (z[i] == top) s.at = v0 + i;
      if (s.top != kNegInf) part *= scaled_exp(a, s.top - top);
      s.top = top;
    }
    if (s.top == kNegInf) continue;  // nothing yet
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < VE; ++i) sum += scaled_exp(a, z[i] - s.top);
    part += sum;
  }
  s.sum = odd ? (double)__builtin_nanf("") : (double)part;
  return s;
}

template <typename T>
__device__ __forceinline__ int row_vectors(const VerifyArgs& a, const T* x) {
  constexpr int VE = 16 / (int)sizeof(T);
  const int off = (int)((reinterpret_cast<uintptr_t>(x) & 15) / sizeof(T));
  return (int)(((int64_t)a.V + off + VE - 1) / VE);
}

// The lanes' statistics joined, for all of them: one factor a lane, then sums in fp64.
__device__ __forceinline__ VerifyStat wave_stat(const VerifyArgs& a, VerifyStat s) {
  const float top = wave_max(s.top);
  if (s.top != top) {
    s.sum *= s.top == kNegInf ? 0.0 : (double)scaled_exp(a, s.top - top);
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

template <typename T>
__device__ __forceinline__ double prob_at(const VerifyArgs& a, const T* x, const VerifyStat& s, int v) {
  return exp((double)(logit<T>(x[v]) - s.top) * a.scale) / s.sum;
}

// How many of row b's drafts stand: every wave finds it, lane i for draft i.
template <typename T, bool GREEDY>
__device__ __forceinline__ int standing(const VerifyArgs& a, int64_t b, int count, const VerifyStat* stats, int lane) {
  bool falls = false;
  if (lane < count) {
    const int64_t x = a.tokens[b * a.N + lane];
    if constexpr (GREEDY) {
      falls = x != stats[lane].at;
    } else {
      bool ok = x >= 0 && x < a.V;
      if (ok) {
        const double p = prob_at(a, row_at<T>(a, b, lane), stats[lane], (int)x);
        double q = 1.0;
        if (a.draft != nullptr) q = prob_at(a, row_at<T>(a, b, a.N + 1 + lane), stats[a.N + 1 + lane], (int)x);
        ok = (double)a.uniforms[b * a.N + lane] * q < p;
      }
      falls = !ok;
    }
  }
  const uint64_t f = __builtin_amdgcn_ballot_w64(falls);
  return f == 0 ? count : __builtin_ctzll(f);
}

// A thread's best of row `at`'s race over ids v0 .. v1 - 1, every `step`-th: the ratio's bits
// above the complement of its id, 0 where no ratio is positive.  In a row of drafts left over,
// `any` says whether the difference p - q was positive anywhere.
template <typename T>
__device__ __forceinline__ unsigned long long race(const VerifyArgs& a, int64_t b, int at, bool rest, const VerifyStat& sp,
                                                   const VerifyStat& sq, int v0, int v1, int step) {
#pragma clang fp contract(off)  // p - q of equal logits is 0, not what rounding one product leaves
  const T* const xp = row_at<T>(a, b, at);
  const T* const xq = a.draft != nullptr && rest ? row_at<T>(a, b, a.N + 1 + at) : nullptr;
  const int64_t drafted = rest && a.draft == nullptr ? a.tokens[b * a.N + at] : -1;
  const float* const e = a.noise + b * a.noise_ld;
  const float ip = (float)(1.0 / sp.sum), iq = xq != nullptr ? (float)(1.0 / sq.sum) : 0.f;
  float best = 0.f;
  int id = 0;
#pragma unroll 4
  for (int v = v0; v < v1; v += step) {
    float r = scaled_exp(a, logit<T>(xp[v]) - sp.top) * ip;
    if (xq != nullptr) r -= scaled_exp(a, logit<T>(xq[v]) - sq.top) * iq;
    if (v == drafted) r = 0.f;
    r /= e[v];
    if (r > best) {  // ids rise: the first of equals stays
      best = r;
      id = v;
    }
  }
  return best > 0.f ? (unsigned long long)__float_as_uint(best) << 32 | (0xffffffffu - (unsigned)id) : 0ull;
}

__device__ __forceinline__ unsigned long long wave_best(unsigned long long x) {
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const unsigned long long o = __shfl_xor(x, off, 64);
    x = o > x ? o : x;
  }
  return x;
}

// Row b's results, by one wave: lane j writes place j (and lane 0 the last of 64 drafts).
template <typename T, bool GREEDY>
__device__ __forceinline__ void write_row(const VerifyArgs& a, int64_t b, int stands, int token, const VerifyStat* stats,
                                          int lane) {
  for (int j = lane; j <= a.N; j += 64) {
    int64_t t = -1;
    float lp = 0.f;
    if (j <= stands) {
      t = j < stands ? a.tokens[b * a.N + j] : token;
      const VerifyStat s = stats[j];
      lp = (float)((double)(logit<T>(row_at<T>(a, b, j)[t]) - s.top) * a.scale - log(s.sum));
    }
    a.out_tokens[b * (a.N + 1) + j] = t;
    a.out_logprobs[b * (a.N + 1) + j] = lp;
  }
  if (lane == 0) a.accepted[b] = stands;
}

__device__ __forceinline__ int best_id(unsigned long long best) {
  return best == 0 ? -1 : (int)(0xffffffffu - (unsigned)best);
}

// One workgroup a row of the batch.
template <typename T, bool GREEDY>
__global__ __launch_bounds__(512) void verify_alone_kernel(const VerifyArgs a) {
  __shared__ VerifyStat stats[2 * kMostDrafts + 1];
  __shared__ unsigned long long bests[8];
  const int64_t b = blockIdx.x;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int count = drafts_of(a, b);
  for (int r = wv; r < a.rows; r += 8) {
    if (!row_used(a, r, count)) continue;
    const T* x = row_at<T>(a, b, r);
    const VerifyStat s = wave_stat(a, row_stat<T>(a, x, lane, row_vectors<T>(a, x), 64));
    if (lane == 0) stats[r] = s;
  }
  __syncthreads();
  const int stands = standing<T, GREEDY>(a, b, count, stats, lane);
  if constexpr (GREEDY) {
    if (wv == 0) write_row<T, GREEDY>(a, b, stands, min(stats[stands].at, a.V - 1), stats, lane);
    return;
  }
  const bool rest = stands < count;
  const VerifyStat sp = stats[stands], sq = a.draft != nullptr && rest ? stats[a.N + 1 + stands] : sp;
  for (int again = 0; again < 2; ++again) {
    const unsigned long long mine = wave_best(race<T>(a, b, stands, rest && again == 0, sp, sq, tid, a.V, 512));
    if (lane == 0) bests[wv] = mine;
    __syncthreads();
    unsigned long long best = bests[0];
#pragma unroll
    for (int i = 1; i < 8; ++i) best = bests[i] > best ? bests[i] : best;
    if (best != 0 || !rest || again == 1) {  // the same in all threads
      if (wv == 0) write_row<T, GREEDY>(a, b, stands, max(best_id(best), 0), stats, lane);
      return;
    }
    __syncthreads();  // nothing left of the difference: the target's row itself
  }
}

// Statistics of one part of one row of logits a workgroup.
template <typename T>
__global__ __launch_bounds__(256) void verify_stat_kernel(const VerifyArgs a) {
  __shared__ VerifyStat waves[4];
  const int part = (int)(blockIdx.x % (unsigned)a.split);
  const unsigned br = blockIdx.x / (unsigned)a.split;
  const int64_t b = br / (unsigned)a.rows;
  const int r = (int)(br - (unsigned)b * (unsigned)a.rows);
  if (r == 0 && part == 0 && threadIdx.x == 0) a.races[b] = VerifyRace{0ull, 0u, 0u};
  if (!row_used(a, r, drafts_of(a, b))) return;  // whole workgroups
  const T* x = row_at<T>(a, b, r);
  const int n = row_vectors<T>(a, x);
  const int per = (n + a.split - 1) / a.split;
  const int first = min(part * per, n), end = min(first + per, n);
  const VerifyStat s = wave_stat(a, row_stat<T>(a, x, first + (int)threadIdx.x, end, 256));
  if ((threadIdx.x & 63) == 0) waves[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x != 0) return;
  VerifyStat all = waves[0];
  for (int i = 1; i < 4; ++i) join_stat(a, all, waves[i]);
  a.stats[(int64_t)br * a.split + part] = all;
}

// One part of one row's race a workgroup; the last to end writes the row's results.
template <typename T, bool GREEDY>
__global__ __launch_bounds__(512) void verify_race_kernel(const VerifyArgs a) {
  __shared__ VerifyStat stats[2 * kMostDrafts + 1];
  __shared__ unsigned long long bests[8];
  __shared__ int last;
  const int64_t b = blockIdx.x / (unsigned)a.parts;
  const int part = (int)(blockIdx.x - (unsigned)b * (unsigned)a.parts);
  const int tid = threadIdx.x, lane = tid & 63;
  const int wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int count = drafts_of(a, b);
  for (int r = tid; r < a.rows; r += 512) {
    if (!row_used(a, r, count)) continue;
    const VerifyStat* s = a.stats + (b * a.rows + r) * a.split;
    VerifyStat all = s[0];
    for (int i = 1; i < a.split; ++i) join_stat(a, all, s[i]);
    stats[r] = all;
  }
  __syncthreads();
  const int stands = standing<T, GREEDY>(a, b, count, stats, lane);
  if constexpr (GREEDY) {
    if (wv == 0) write_row<T, GREEDY>(a, b, stands, min(stats[stands].at, a.V - 1), stats, lane);
    return;
  }
  const bool rest = stands < count;
  const VerifyStat sp = stats[stands], sq = a.draft != nullptr && rest ? stats[a.N + 1 + stands] : sp;
  const int per = (a.V + a.parts - 1) / a.parts;
  const int v0 = min(part * per, a.V), v1 = min(v0 + per, a.V);
  auto block_best = [&](bool less, int from, int to) {
    const unsigned long long mine = wave_best(race<T>(a, b, stands, less, sp, sq, from + tid, to, 512));
    if (lane == 0) bests[wv] = mine;
    __syncthreads();
    unsigned long long best = bests[0];
#pragma unroll
    for (int i = 1; i < 8; ++i) best = bests[i] > best ? bests[i] : best;
    __syncthreads();
    return best;
  };
  unsigned long long best = block_best(rest, v0, v1);
  if (a.parts > 1) {
    if (tid == 0) {
      __hip_atomic_fetch_max(&a.races[b].best, best, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      last = __hip_atomic_fetch_add(&a.races[b].done, 1u, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT) == (unsigned)a.parts - 1;
      if (last) bests[0] = __hip_atomic_load(&a.races[b].best, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    __syncthreads();
    if (!last) return;
    best = bests[0];
    __syncthreads();
  }
  // nothing left of the difference: the target's row itself
  if (best == 0 && rest) best = block_best(false, 0, a.V);
  if (wv == 0) write_row<T, GREEDY>(a, b, stands, max(best_id(best), 0), stats, lane);
}

namespace {

// Logits of a row of the batch up to which one workgroup does all of it.
constexpr int64_t kAlone = 16384;

struct VerifyShape {
  bool alone;
  int rows, split, parts;
  size_t stat_bytes, ws_bytes;
};

VerifyShape verify_shape(int64_t B, int N, int64_t V) {
  VerifyShape t{};
  t.rows = 2 * N + 1;
  t.alone = t.rows * V <= kAlone;
  t.split = t.parts = 1;
  if (t.alone) return t;
  // about two workgroups a CU, of 2048 logits at least
  t.split = (int)std::max<int64_t>(1, std::min<int64_t>({(512 + B * t.rows - 1) / (B * t.rows), V / 2048, 64}));
  t.parts = (int)std::max<int64_t>(1, std::min<int64_t>({(256 + B - 1) / B, V / 2048, 64}));
  t.stat_bytes = (size_t)B * t.rows * t.split * sizeof(VerifyStat);
  t.ws_bytes = t.stat_bytes + (size_t)B * sizeof(VerifyRace);
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
  hipLaunchKernelGGL(verify_stat_kernel<T>, dim3((unsigned)((int64_t)a.B * a.rows * a.split)), dim3(256), 0, s, a);
  if (const int rc = check_launch("verify_stat_kernel")) return rc;
  const dim3 grid((unsigned)((int64_t)a.B * a.parts));
  if (greedy) hipLaunchKernelGGL((verify_race_kernel<T, true>), grid, block, 0, s, a);
  else hipLaunchKernelGGL((verify_race_kernel<T, false>), grid, block, 0, s, a);
  return check_launch("verify_race_kernel");
}

}  // namespace
}  // namespace dg

using namespace dg;

extern "C" size_t dg_verify_drafts_workspace_size(int B, int N, int64_t V, int dtype) {
  if (B <= 0 || N < 0 || N > kMostDrafts || V <= 0 || V > 0x3fffffff) return 0;
  return verify_shape(B, N, V).ws_bytes;
}

extern "C" int dg_verify_drafts(int B, int N, int64_t V, int dtype, const void* target, int64_t t_b, int64_t t_n,
                                const void* draft, int64_t d_b, int64_t d_n, const int64_t* tokens,
                                const float* uniforms, const float* noise, int64_t noise_ld, const int32_t* counts,
                                float inv_temperature, int64_t* accepted, int64_t* out_tokens, float* out_logprobs,
                                void* workspace, size_t workspace_bytes, void* stream) {
  DG_REQUIRE(B >= 0, DG_EINVAL, "verify_drafts: negative size");
  DG_REQUIRE(N >= 0 && N <= kMostDrafts, DG_EINVAL, "verify_drafts: %d drafts a row, 0 to %d", N, kMostDrafts);
  DG_REQUIRE(V >= 1 && V <= 0x3fffffff, DG_EINVAL, "verify_drafts: a vocabulary of %lld, 1 to 2^30 - 1", (long long)V);
  DG_REQUIRE(dtype == DG_F32 || dtype == DG_BF16 || dtype == DG_F16 || dtype == DG_F64, DG_EUNSUPPORTED,
             "verify_drafts: dtype %d unsupported", dtype);
  DG_REQUIRE(inv_temperature == 0.f || (inv_temperature >= 0x1p-100f && inv_temperature <= 0x1p100f), DG_EINVAL,
             "verify_drafts: the inverse temperature must be 0 or between 2^-100 and 2^100");
  if (B == 0) return DG_OK;
  const bool greedy = inv_temperature == 0.f;
  DG_REQUIRE(target && accepted && out_tokens && out_logprobs && (N == 0 || tokens), DG_EINVAL, "verify_drafts: NULL argument");
  DG_REQUIRE(greedy || (noise && (N == 0 || uniforms)), DG_EINVAL, "verify_drafts: random numbers missing");
  const int64_t es = dtype_bytes(dtype);
  DG_REQUIRE(reinterpret_cast<uintptr_t>(target) % es == 0 && reinterpret_cast<uintptr_t>(draft) % es == 0, DG_EINVAL,
             "verify_drafts: logits not aligned to their element size");
  VerifyArgs a{};
  a.target = target; a.tb = t_b; a.tn = t_n;
  a.draft = greedy ? nullptr : draft; a.db = d_b; a.dn = d_n;
  a.tokens = tokens; a.uniforms = uniforms; a.noise = noise; a.noise_ld = noise_ld; a.counts = counts;
  a.scale = greedy ? 1.0 : (double)inv_temperature;
  const double l2 = a.scale * 1.4426950408889634074;
  // the leading term rounded down, so that the rest is positive and -inf times it still -inf
  a.scale_hi = (float)l2;
  if ((double)a.scale_hi >= l2) a.scale_hi = std::nextafter(a.scale_hi, 0.f);
  a.scale_lo = (float)(l2 - (double)a.scale_hi);
  a.accepted = accepted; a.out_tokens = out_tokens; a.out_logprobs = out_logprobs;
  a.B = B; a.N = N; a.V = (int)V;
  const VerifyShape t = verify_shape(B, N, V);
  a.rows = a.draft != nullptr ? 2 * N + 1 : N + 1;
  a.split = t.split;
  a.parts = greedy ? 1 : t.parts;
  if (t.ws_bytes > 0) {
    DG_REQUIRE(workspace != nullptr && workspace_bytes >= t.ws_bytes, DG_EWORKSPACE,
               "verify_drafts: a workspace of %zu bytes, %zu needed", workspace_bytes, t.ws_bytes);
    DG_REQUIRE((reinterpret_cast<uintptr_t>(workspace) & 15) == 0, DG_EINVAL, "verify_drafts: workspace not 16-byte aligned");
    a.stats = static_cast<VerifyStat*>(workspace);
    a.races = reinterpret_cast<VerifyRace*>(static_cast<char*>(workspace) + t.stat_bytes);
  }
  DG_REQUIRE((int64_t)B * (2 * N + 1) * t.split <= kMostWorkgroups256 && (int64_t)B * t.parts <= kMostWorkgroups256 / 2,
             DG_EINVAL, "verify_drafts: more than 2^32 - 1 threads");
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (dtype == DG_F64) return launch_verify<double>(a, t, greedy, s);
  if (dtype == DG_F32) return launch_verify<float>(a, t, greedy, s);
  if (dtype == DG_BF16) return launch_verify<bf16_t>(a, t, greedy, s);
  return launch_verify<f16_t>(a, t, greedy, s);
}
