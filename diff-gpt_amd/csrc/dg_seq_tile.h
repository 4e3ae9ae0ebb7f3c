// The kernel of packed, tree and paged attention that takes any shape and type
// (seq_tile_kernel), and the joins of split rows.  Rows of whole 16-byte pieces up to 256
// dims in 16-bit types, 128 in fp32, run on the matrix cores instead (dg_seq_mfma.h).
//
// The kernel here (seq_tile_kernel): 32 rows of a key head by 32 keys at a time, 16 rows
// for head_dim over 256 and 8 where a piece has no more (a decode step): 8, 16 or 32 lanes
// a row, in fp32 (fp64 for fp64 data).  Rows lie in LDS for the whole loop; keys and then
// values pass through it in chunks of 64 dims, read element by element (rows may start
// anywhere) into registers while the chunk before is computed.  For the scores a row's
// lanes have a key each, for the outputs dims each; the probabilities go from one to the
// other through LDS.  A hidden key's score is taken out by selection and its values are
// skipped, so nothing it holds can reach a row.  Bound by LDS reads (five of 16 bytes for
// 16 products a lane).  16 x 512 tokens, 8 heads: head_dim 65 bf16 362 us, 600
// fp32 1.86 ms (22 TFLOP/s), 64 fp64 384; a step over 32 caches of 1900, 8 heads: 65 bf16
// 115 us, 600 fp32 540 (4.3 TB/s), 64 fp64 128 (3.9 TB/s).  One row a wave at a time with a
// running softmax in each lane group took 13.1 ms and 2.2 ms in fp64.
#pragma once

#include <type_traits>

#include "dg_seq.h"

namespace dg {

constexpr float kLog2e = 1.44269504088896340736f;

// arithmetic of a row: fp32 in log2 units, fp64 in natural ones (no fp64 exp2 needed)
template <typename T>
struct SeqAcc {
  using type = float;
  static __device__ __forceinline__ float load(T x) { return to_f32(x); }
  static __device__ __forceinline__ float unit_scale(const SeqArgs& a) { return a.scale_log2; }
  static __device__ __forceinline__ float exp(float x) { return __builtin_amdgcn_exp2f(x); }
  static __device__ __forceinline__ float log(float x) { return __builtin_amdgcn_logf(x); }
  static __device__ __forceinline__ T store(float x) { return from_f32<T>(x); }
};
template <>
struct SeqAcc<double> {
  using type = double;
  static __device__ __forceinline__ double load(double x) { return x; }
  static __device__ __forceinline__ double unit_scale(const SeqArgs& a) {
    // an fp32 rounding of 1/sqrt(D) stands for 1/sqrt(D) itself, as in dg_attention
    const double root = 1.0 / sqrt((double)a.D);
    return a.scale == (float)root ? root : (double)a.scale;
  }
  static __device__ __forceinline__ double exp(double x) { return ::exp(x); }
  static __device__ __forceinline__ double log(double x) { return ::log(x); }
  static __device__ __forceinline__ double store(double x) { return x; }
};

template <typename A>
__device__ __forceinline__ A neg_inf() {
  return -(A)__builtin_huge_valf();
}

// The state of a softmax row, joined with another's: (m, l) <- both, and the factors of
// the two outputs.  -inf stands for "no key yet", whose factor is 0.
template <typename S, typename A>
__device__ __forceinline__ void join_softmax(A& m, A& l, A m2, A l2, A& f1, A& f2) {
  const A mn = m > m2 ? m : m2;
  f1 = m == neg_inf<A>() ? (A)0 : S::exp(m - mn);
  f2 = m2 == neg_inf<A>() ? (A)0 : S::exp(m2 - mn);
  l = l * f1 + l2 * f2;
  m = mn;
}

// N consecutive values in LDS, aligned to their size or to 16 bytes.
template <int N, typename A>
__device__ __forceinline__ void lds_load(const A* p, A (&x)[N]) {
  constexpr int V = N * sizeof(A) > 16 ? 16 / sizeof(A) : N;
  typedef A vec __attribute__((ext_vector_type(V)));
#pragma unroll
  for (int e = 0; e < N; e += V) {
    const vec v = *reinterpret_cast<const vec*>(p + e);
#pragma unroll
    for (int k = 0; k < V; ++k) x[e + k] = v[k];
  }
}

// NCH: chunks of 64 dims there may be; LPR: lanes of a row.
template <typename T, int NCH, int LPR, SeqMode MODE>
__global__ __launch_bounds__(256) void seq_tile_kernel(const SeqArgs a) {
  using S = SeqAcc<T>;
  using A = typename S::type;
  constexpr bool TREE = MODE == kTree, PAGED = MODE >= kPaged;
  constexpr int ROWS = 256 / LPR, KT = 32, KPL = KT / LPR;
  constexpr int VW = LPR == 32 ? 2 : 4, NV = 64 / LPR / VW;  // of a chunk, a lane has dims VW (ln + LPR h) + e
  constexpr int PAD = 16 / (int)sizeof(A);  // rows 4 banks apart
  constexpr int QS = NCH * 64 + PAD, CS = 64 + PAD, PS = KT + PAD;
  __shared__ __attribute__((aligned(16))) A qs[ROWS * QS], kvs[KT * CS], ps[ROWS * PS];
  SeqPiece p;
  if (!seq_piece<MODE>(a, p)) return;  // whole workgroups
  const int tid = threadIdx.x, row = tid / LPR, ln = tid % LPR;
  const bool live = (tid & ~63) / LPR < p.rows;  // the wave has a row
  const int last = p.row0 + p.rows - 1;          // rows past it repeat it and are never stored
  const int r = min(p.row0 + row, last), i = r / a.G;
  const A us = S::unit_scale(a);
  for (int e = tid; e < ROWS * NCH * 64; e += 256) {
    const int er = e / (NCH * 64), d = e % (NCH * 64), rr = min(p.row0 + er, last), ri = rr / a.G;
    const T* qp = static_cast<const T*>(a.q) + p.b * a.qb + (p.q0 + ri) * a.qt + (int64_t)(p.kvh * a.G + rr - ri * a.G) * a.qh;
    qs[er * QS + d] = d < a.D ? S::load(qp[d]) : (A)0;
  }
  const T* kp = static_cast<const T*>(a.k) + (PAGED ? 0 : p.b * a.kb) + p.k0 * a.kt + (int64_t)p.kvh * a.kh;
  const T* vp = static_cast<const T*>(a.v) + (PAGED ? 0 : p.b * a.vb) + p.k0 * a.vt + (int64_t)p.kvh * a.vh;
  // Keys t0 .. of one chunk of dims: into registers, a step ahead of their use, and from
  // there into LDS.  Past the piece's keys the last one stands, hidden from every row; past
  // the head zeros.
  const int sd = tid & 63, sk = tid >> 6;
  T w[KT / 4];
  auto fetch = [&](const T* x, int64_t step, int64_t page, int t0, int c) __attribute__((always_inline)) {
    const T* xd = x + min(64 * c + sd, a.D - 1);
#pragma unroll
    for (int n = 0; n < KT / 4; ++n) {
      const int t = min(t0 + sk + 4 * n, p.kend - 1);
      if constexpr (PAGED) {  // zeros from a page that the pool does not have
        const int id = a.table[p.b * a.table_ld + (t >> a.page_log2)];
        w[n] = T{};
        if (id >= 0 && id < a.pages) w[n] = xd[id * page + (t & ((1 << a.page_log2) - 1)) * step];
      } else {
        w[n] = xd[t * step];
      }
    }
  };
  auto put = [&](int c) __attribute__((always_inline)) {
    const bool in = 64 * c + sd < a.D;
#pragma unroll
    for (int n = 0; n < KT / 4; ++n) kvs[(sk + 4 * n) * CS + sd] = in ? S::load(w[n]) : (A)0;
  };
  const int nch = (a.D + 63) / 64;
  uint64_t mask = 0;
  int end = p.kend, first_open = p.own;
  if constexpr (TREE) {
    mask = tree_mask(a, p.b, i);
  } else {
    end = i + p.off + 1;
    first_open = p.row0 / a.G + p.off + 1;
  }
  A o[NCH][NV][VW], m = neg_inf<A>(), l = (A)0, lc = (A)0;
#pragma unroll
  for (int c = 0; c < NCH; ++c)
#pragma unroll
    for (int h = 0; h < NV; ++h)
#pragma unroll
      for (int e = 0; e < VW; ++e) o[c][h][e] = (A)0;

  if (p.kbeg < p.kend) fetch(kp, a.kt, a.kb, p.kbeg, 0);
  for (int t0 = p.kbeg; t0 < p.kend; t0 += KT) {
    A s[KPL];
#pragma unroll
    for (int j = 0; j < KPL; ++j) s[j] = (A)0;
#pragma unroll 1
    for (int c = 0; c < nch; ++c) {
      __syncthreads();
      put(c);
      __syncthreads();
      if (c + 1 < nch) fetch(kp, a.kt, a.kb, t0, c + 1);
      else fetch(vp, a.vt, a.vb, t0, 0);
      if (live) {
#pragma unroll 4
        for (int d = 0; d < 64; d += 4) {
          A q4[4];
          lds_load(qs + row * QS + 64 * c + d, q4);
#pragma unroll
          for (int j = 0; j < KPL; ++j) {
            A k4[4];
            lds_load(kvs + (ln + LPR * j) * CS + d, k4);
#pragma unroll
            for (int e = 0; e < 4; ++e) s[j] += q4[e] * k4[e];
          }
        }
      }
    }
    bool seen[KPL];
    A top = neg_inf<A>();
#pragma unroll
    for (int j = 0; j < KPL; ++j) {
      const int t = t0 + ln + LPR * j;
      seen[j] = t < end;
      if constexpr (TREE) seen[j] = seen[j] && (t < p.own || ((mask >> ((t - p.own) & 63)) & 1));
      s[j] = seen[j] ? s[j] * us : neg_inf<A>();
      top = s[j] > top ? s[j] : top;
    }
#pragma unroll
    for (int x = 1; x < LPR; x <<= 1) {
      const A other = __shfl_xor(top, x, 64);
      top = other > top ? other : top;
    }
    const A mn = top > m ? top : m;
    const A f = m == neg_inf<A>() ? (A)1 : S::exp(m - mn);  // nothing to rescale yet
    const A base = mn == neg_inf<A>() ? (A)0 : mn;
    m = mn;
    l *= f;
    lc *= f;
    A sum = (A)0;
#pragma unroll
    for (int j = 0; j < KPL; ++j) {
      const A w = S::exp(s[j] - base);  // NaN for a NaN score, and the row with it
      if (seen[j]) sum += w;
      ps[row * PS + ln + LPR * j] = seen[j] ? w : (A)-1;  // the row's own lanes read it, after the barriers below
    }
    add_rounded(l, lc, sum);
    if (f != (A)1) {
#pragma unroll
      for (int c = 0; c < NCH; ++c)
#pragma unroll
        for (int h = 0; h < NV; ++h)
#pragma unroll
          for (int e = 0; e < VW; ++e) o[c][h][e] *= f;
    }
    const bool open = t0 + KT <= first_open;  // every row sees every key of the tile
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
      // A loop that ends early is not unrolled, and o indexed at run time: in scratch memory
      // for 16 rows (16 x 512 tokens, 8 heads of 600, fp32: 2.38 ms so, 1.86 unrolled).  A
      // step's 8 rows have fewer outputs a lane, and unrolled they leave room for two
      // workgroups a CU in place of three (32 caches of 1900, 8 heads of 600: 540 us so, 659).
      if (c >= nch) {
        if constexpr (LPR == 32) break;
        else continue;
      }
      __syncthreads();
      put(c);
      __syncthreads();
      if (c + 1 < nch) fetch(vp, a.vt, a.vb, t0, c + 1);
      else fetch(kp, a.kt, a.kb, t0 + KT, 0);
      if (!live) continue;
      auto add = [&](auto every) __attribute__((always_inline)) {
#pragma unroll 2
        for (int t = 0; t < KT; t += 4) {
          A w4[4];
          lds_load(ps + row * PS + t, w4);
#pragma unroll
          for (int u = 0; u < 4; ++u)
#pragma unroll
            for (int h = 0; h < NV; ++h) {
              A v[VW];
              lds_load(kvs + (t + u) * CS + VW * (ln + LPR * h), v);
#pragma unroll
              for (int e = 0; e < VW; ++e) {
                const A x = o[c][h][e] + w4[u] * v[e];
                o[c][h][e] = every.value || !(w4[u] < (A)0) ? x : o[c][h][e];  // a hidden key adds nothing
              }
            }
        }
      };
      if (open) add(std::true_type{});
      else add(std::false_type{});
    }
  }
  l -= lc;
#pragma unroll
  for (int x = 1; x < LPR; x <<= 1) l += __shfl_xor(l, x, 64);
  if (row >= p.rows) return;
  if (MODE != kPacked && a.nsplit > 1) {
    const int64_t part = ((p.b * a.Hkv + p.kvh) * (int64_t)(a.N * a.G) + r) * a.nsplit + p.split;
    A* wo = static_cast<A*>(a.ws_o) + part * a.D;
#pragma unroll
    for (int c = 0; c < NCH; ++c)
#pragma unroll
      for (int h = 0; h < NV; ++h)
#pragma unroll
        for (int e = 0; e < VW; ++e) {
          const int d = 64 * c + VW * (ln + LPR * h) + e;
          if (d < a.D) wo[d] = o[c][h][e];
        }
    if (ln == 0) {
      A* ml = static_cast<A*>(a.ws_ml) + 2 * part;
      ml[0] = m;
      ml[1] = l;
    }
    return;
  }
  // no key at all: zeros; keys whose scores are all -inf: 0 / 0, as a softmax gives
  const bool none = TREE ? p.own == 0 && mask == 0 : PAGED ? i >= p.count : end <= 0;
  if constexpr (PAGED) {
    if (a.lse != nullptr && ln == 0)
      static_cast<A*>(a.lse)[(p.b * a.Hkv + p.kvh) * (int64_t)(a.N * a.G) + r] =
          none ? (A)__builtin_huge_valf() : m + S::log(l);
  }
  T* yp = static_cast<T*>(a.y) + p.b * a.yb + (p.q0 + i) * a.yt + (int64_t)(p.kvh * a.G + r - i * a.G) * a.yh;
#pragma unroll
  for (int c = 0; c < NCH; ++c)
#pragma unroll
    for (int h = 0; h < NV; ++h)
#pragma unroll
      for (int e = 0; e < VW; ++e) {
        const int d = 64 * c + VW * (ln + LPR * h) + e;
        if (d < a.D) yp[d] = S::store(none ? (A)0 : o[c][h][e] / l);
      }
}

// What the join of row r (token i) needs of its lengths: the cached positions, how many of
// its splits were written, and whether it sees nothing.
template <SeqMode MODE>
__device__ __forceinline__ void seq_join_row(const SeqArgs& a, int64_t b, int len, int i, int r, int& own, int& used,
                                             bool& none) {
  if constexpr (MODE >= kPaged) {
    const PagedRow p = paged_row(a, b, len);
    const int chunk = paged_chunk(a, p);
    own = p.own;
    used = min(a.nsplit, (paged_end(a, p, r) + chunk - 1) / chunk);
    none = i >= p.count;
  } else {
    own = min(max(len, 0), a.Tcap - a.N);
    used = min(a.nsplit, (own + a.N + a.chunk - 1) / a.chunk);
    none = own == 0 && tree_mask(a, b, i) == 0;
  }
}

// The splits of a row joined: WPR wavefronts a row, each over every WPR-th split, lanes
// along the head.  A row's used splits follow from its length, so what the workspace held
// before does not matter.  A split's weight is computed once, by the lane of its number.
template <typename T, int WPR, SeqMode MODE>
__global__ __launch_bounds__(256) void seq_join_kernel(const SeqArgs a, const int64_t nrows) {
  using S = SeqAcc<T>;
  using A = typename S::type;
  __shared__ A part[WPR > 1 ? 3 * kMaxHeadDim : 1];
  const int lane = threadIdx.x & 63;
  const int wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t row = WPR > 1 ? (int64_t)blockIdx.x : (int64_t)blockIdx.x * 4 + wv;
  if (row >= nrows) return;  // WPR > 1: whole workgroups
  const int sub = WPR > 1 ? wv : 0;
  const int R = a.N * a.G;
  const int r = (int)(row % R);
  const int64_t bh = row / R;
  const int kvh = (int)(bh % a.Hkv);
  const int64_t b = bh / a.Hkv;
  const int i = r / a.G, h = kvh * a.G + r % a.G;
  const int len = a.lens != nullptr ? __builtin_amdgcn_readfirstlane(a.lens[b]) : a.len;
  int own, used;
  bool none;
  seq_join_row<MODE>(a, b, len, i, r, own, used, none);
  const A* ml = static_cast<const A*>(a.ws_ml) + 2 * row * a.nsplit;
  const A* wo = static_cast<const A*>(a.ws_o) + row * a.nsplit * a.D;
  A m = neg_inf<A>();
  bool bad = false;
  for (int s = lane; s < used; s += 64) {
    const A ms = ml[2 * s], ls = ml[2 * s + 1];
    bad = bad || ms != ms || ls != ls;  // a NaN score
    m = ms > m ? ms : m;
  }
#pragma unroll
  for (int x = 1; x < 64; x <<= 1) {
    const A m2 = __shfl_xor(m, x, 64);
    m = m2 > m ? m2 : m;
  }
  bad = __builtin_amdgcn_ballot_w64(bad) != 0;
  constexpr int ND = kMaxHeadDim / 64;
  A o[ND], l = (A)0;
#pragma unroll
  for (int c = 0; c < ND; ++c) o[c] = (A)0;
  for (int s0 = 0; s0 < used; s0 += 64) {
    const int s = s0 + lane;
    const A ms = s < used ? ml[2 * s] : neg_inf<A>();
    const A w = ms == neg_inf<A>() ? (A)0 : S::exp(ms - m);
    if (ms != neg_inf<A>()) l += ml[2 * s + 1] * w;
    const int n = min(64, used - s0);
#pragma unroll 4
    for (int t = sub; t < n; t += WPR) {
      const A wt = __shfl(w, t, 64);
#pragma unroll
      for (int c = 0; c < ND; ++c)
        if (64 * c < a.D && lane + 64 * c < a.D) {
          const A x = wo[(int64_t)(s0 + t) * a.D + lane + 64 * c];
          o[c] += wt == (A)0 ? (A)0 : wt * x;  // a split without a key, or of no weight
        }
    }
  }
#pragma unroll
  for (int x = 1; x < 64; x <<= 1) l += __shfl_xor(l, x, 64);
  if constexpr (WPR > 1) {
#pragma unroll
    for (int c = 0; c < ND; ++c)
      if (sub > 0 && lane + 64 * c < a.D) part[(sub - 1) * kMaxHeadDim + lane + 64 * c] = o[c];
    __syncthreads();
    if (sub > 0) return;
#pragma unroll
    for (int c = 0; c < ND; ++c)
#pragma unroll
      for (int w = 0; w < WPR - 1; ++w)
        if (lane + 64 * c < a.D) o[c] += part[w * kMaxHeadDim + lane + 64 * c];
  }
  if constexpr (MODE >= kPaged) {
    if (a.lse != nullptr && lane == 0)
      static_cast<A*>(a.lse)[row] = none ? (A)__builtin_huge_valf() : bad ? (A)__builtin_nanf("") : m + S::log(l);
  }
  T* yp = static_cast<T*>(a.y) + b * a.yb + i * a.yt + (int64_t)h * a.yh;
#pragma unroll
  for (int c = 0; c < ND; ++c)
    if (lane + 64 * c < a.D)
      yp[lane + 64 * c] = S::store(none ? (A)0 : bad ? (A)__builtin_nanf("") : o[c] / l);
}

// log2 of what the sums of a split's exponentials are too large by (SeqMma).
template <typename T>
constexpr float seq_lift() {
  return __is_same(T, f16_t) ? 7.f : 0.f;
}

// The same for the head dims of the matrix-core kernel: a lane reads four elements of a
// split at a time, so that a wave reads 64 / (D / 4) splits at once, and lengths and states
// are in flight together (those of unused splits are read and not looked at).  WPR waves a
// row as above.
template <typename T, int D, int WPR, SeqMode MODE>
__device__ __forceinline__ void seq_join4(const SeqArgs& a, const int64_t nrows, const unsigned block) {
  constexpr int LPS = D / 4, SPW = 64 / LPS;  // lanes a split, splits a wave
  __shared__ float part[WPR > 1 ? (WPR - 1) * D : 1];
  const int lane = threadIdx.x & 63;
  const int wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t row = WPR > 1 ? (int64_t)block : (int64_t)block * 4 + wv;
  if (row >= nrows) return;  // WPR > 1: whole workgroups
  const int sub = WPR > 1 ? wv : 0;
  const int R = a.N * a.G;
  const int64_t bh = row / R;
  const int r = (int)(row - bh * R);
  const int64_t b = bh / a.Hkv;
  const int kvh = (int)(bh - b * a.Hkv);
  const int i = r / a.G, h = kvh * a.G + (r - i * a.G);
  const u32x2_t* ml = static_cast<const u32x2_t*>(a.ws_ml) + row * a.nsplit;
  const float* wo = static_cast<const float*>(a.ws_o) + row * a.nsplit * D;
  u32x2_t first = {0u, 0u};
  if (lane < a.nsplit) first = ml[lane];
  const int len = a.lens != nullptr ? a.lens[b] : a.len;
  int own, used;
  bool none;
  seq_join_row<MODE>(a, b, __builtin_amdgcn_readfirstlane(len), i, r, own, used, none);
  auto state = [&](int s0, float& ms, float& ls) __attribute__((always_inline)) {
    const int s = s0 + lane;
    u32x2_t x = first;
    if (s0 > 0 && s < used) x = ml[s];
    ms = s < used ? __uint_as_float(x[0]) : kNegInf;
    ls = s < used ? __uint_as_float(x[1]) : 0.f;
  };
  float m = kNegInf;
  bool bad = false;
  for (int s0 = 0; s0 < used; s0 += 64) {
    float ms, ls;
    state(s0, ms, ls);
    bad = bad || ms != ms || ls != ls;  // a NaN score
    m = fmaxf(m, ms);
  }
  m = wave_max(m);
  bad = __builtin_amdgcn_ballot_w64(bad) != 0;
  f32x4_t o = {0.f, 0.f, 0.f, 0.f};
  float l = 0.f;
  const int ls4 = lane / LPS, d4 = 4 * (lane % LPS);
  for (int s0 = 0; s0 < used; s0 += 64) {
    float ms, ls;
    state(s0, ms, ls);
    const float w = ms == kNegInf ? 0.f : __builtin_amdgcn_exp2f(ms - m);
    l += ms == kNegInf ? 0.f : ls * w;
    const int n = min(64, used - s0);
#pragma unroll 4
    for (int t0 = sub * SPW; t0 < n; t0 += WPR * SPW) {
      const int t = t0 + ls4;
      const float wt = __shfl(w, t & 63, 64);
      const f32x4_t x = *reinterpret_cast<const f32x4_t*>(wo + (int64_t)(s0 + min(t, n - 1)) * D + d4);
      const bool in = t < n && wt != 0.f;  // a split without a key, or of no weight, adds nothing
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] += in ? wt * x[e] : 0.f;
    }
  }
  l = group_sum_dpp<64>(l);
#pragma unroll
  for (int x = LPS; x < 64; x <<= 1)
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] += __shfl_xor(o[e], x, 64);
  if constexpr (WPR > 1) {
    if (sub > 0 && ls4 == 0) *reinterpret_cast<f32x4_t*>(part + (sub - 1) * D + d4) = o;
    __syncthreads();
    if (sub > 0) return;
#pragma unroll
    for (int w = 0; w < WPR - 1; ++w) o += *reinterpret_cast<const f32x4_t*>(part + w * D + d4);
  }
  if (ls4 != 0) return;
  if constexpr (MODE >= kPaged) {
    constexpr float kLift = seq_lift<T>();
    if (a.lse != nullptr && d4 == 0)
      static_cast<float*>(a.lse)[row] =
          none ? __builtin_huge_valf() : bad ? __builtin_nanf("") : m - kLift + __builtin_amdgcn_logf(l);
  }
  T* yp = static_cast<T*>(a.y) + b * a.yb + i * a.yt + (int64_t)h * a.yh;
  float y[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) y[e] = none ? 0.f : bad ? __builtin_nanf("") : o[e] / l;
  if (d4 < a.D) store_vec<T, 4>(yp + d4, y);
}
template <typename T, int D, int WPR, SeqMode MODE>
__global__ __launch_bounds__(256) void seq_join4_kernel(const SeqArgs a, const int64_t nrows) {
  seq_join4<T, D, WPR, MODE>(a, nrows, blockIdx.x);
}

}  // namespace dg
