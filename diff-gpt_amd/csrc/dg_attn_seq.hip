// Attention over packed sequences (dg_attention_packed) and over a few tokens per cached
// row (dg_attention_tree): the entry points, the host-side plan of packed tiles, the join
// of split rows, and the kernel that takes any shape and type.  Rows of whole 16-byte pieces
// up to 256 dims in 16-bit types, 128 in fp32, run on the matrix cores (dg_attn_seq_mfma.hip).
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
#include "dg_seq.h"

#include <algorithm>
#include <cmath>
#include <exception>
#include <type_traits>
#include <vector>

namespace dg {

constexpr float kLog2e = 1.44269504088896340736f;

// arithmetic of a row: fp32 in log2 units, fp64 in natural ones (no fp64 exp2 needed)
template <typename T>
struct SeqAcc {
  using type = float;
  static __device__ __forceinline__ float load(T x) { return to_f32(x); }
  static __device__ __forceinline__ float unit_scale(const SeqArgs& a) { return a.scale_log2; }
  static __device__ __forceinline__ float exp(float x) { return __builtin_amdgcn_exp2f(x); }
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
template <typename T, int NCH, int LPR, bool TREE>
__global__ __launch_bounds__(256) void seq_tile_kernel(const SeqArgs a) {
  using S = SeqAcc<T>;
  using A = typename S::type;
  constexpr int ROWS = 256 / LPR, KT = 32, KPL = KT / LPR;
  constexpr int VW = LPR == 32 ? 2 : 4, NV = 64 / LPR / VW;  // of a chunk, a lane has dims VW (ln + LPR h) + e
  constexpr int PAD = 16 / (int)sizeof(A);  // rows 4 banks apart
  constexpr int QS = NCH * 64 + PAD, CS = 64 + PAD, PS = KT + PAD;
  __shared__ __attribute__((aligned(16))) A qs[ROWS * QS], kvs[KT * CS], ps[ROWS * PS];
  SeqPiece p;
  if (!seq_piece<TREE>(a, p)) return;  // whole workgroups
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
  const T* kp = static_cast<const T*>(a.k) + p.b * a.kb + p.k0 * a.kt + (int64_t)p.kvh * a.kh;
  const T* vp = static_cast<const T*>(a.v) + p.b * a.vb + p.k0 * a.vt + (int64_t)p.kvh * a.vh;
  // Keys t0 .. of one chunk of dims: into registers, a step ahead of their use, and from
  // there into LDS.  Past the piece's keys the last one stands, hidden from every row; past
  // the head zeros.
  const int sd = tid & 63, sk = tid >> 6;
  T w[KT / 4];
  auto fetch = [&](const T* x, int64_t step, int t0, int c) __attribute__((always_inline)) {
    const T* xd = x + min(64 * c + sd, a.D - 1);
#pragma unroll
    for (int n = 0; n < KT / 4; ++n) w[n] = xd[min(t0 + sk + 4 * n, p.kend - 1) * step];
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

  if (p.kbeg < p.kend) fetch(kp, a.kt, p.kbeg, 0);
  for (int t0 = p.kbeg; t0 < p.kend; t0 += KT) {
    A s[KPL];
#pragma unroll
    for (int j = 0; j < KPL; ++j) s[j] = (A)0;
#pragma unroll 1
    for (int c = 0; c < nch; ++c) {
      __syncthreads();
      put(c);
      __syncthreads();
      if (c + 1 < nch) fetch(kp, a.kt, t0, c + 1);
      else fetch(vp, a.vt, t0, 0);
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
      if (c + 1 < nch) fetch(vp, a.vt, t0, c + 1);
      else fetch(kp, a.kt, t0 + KT, 0);
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
  if (TREE && a.nsplit > 1) {
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
  const bool none = TREE ? p.own == 0 && mask == 0 : end <= 0;
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

// The splits of a row joined: WPR wavefronts a row, each over every WPR-th split, lanes
// along the head.  A row's used splits follow from its length, so what the workspace held
// before does not matter.  A split's weight is computed once, by the lane of its number.
template <typename T, int WPR>
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
  const int own = min(max(len, 0), a.Tcap - a.N);
  const int used = min(a.nsplit, (own + a.N + a.chunk - 1) / a.chunk);
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
  const bool none = own == 0 && tree_mask(a, b, i) == 0;
  T* yp = static_cast<T*>(a.y) + b * a.yb + i * a.yt + (int64_t)h * a.yh;
#pragma unroll
  for (int c = 0; c < ND; ++c)
    if (lane + 64 * c < a.D)
      yp[lane + 64 * c] = S::store(none ? (A)0 : bad ? (A)__builtin_nanf("") : o[c] / l);
}

// The same for the head dims of the matrix-core kernel: a lane reads four elements of a
// split at a time, so that a wave reads 64 / (D / 4) splits at once, and lengths and states
// are in flight together (those of unused splits are read and not looked at).  WPR waves a
// row as above.
template <typename T, int D, int WPR>
__global__ __launch_bounds__(256) void seq_join4_kernel(const SeqArgs a, const int64_t nrows) {
  constexpr int LPS = D / 4, SPW = 64 / LPS;  // lanes a split, splits a wave
  __shared__ float part[WPR > 1 ? (WPR - 1) * D : 1];
  const int lane = threadIdx.x & 63;
  const int wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t row = WPR > 1 ? (int64_t)blockIdx.x : (int64_t)blockIdx.x * 4 + wv;
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
  const int own = min(max(__builtin_amdgcn_readfirstlane(len), 0), a.Tcap - a.N);
  const int used = min(a.nsplit, (own + a.N + a.chunk - 1) / a.chunk);
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
  const bool none = own == 0 && tree_mask(a, b, i) == 0;
  T* yp = static_cast<T*>(a.y) + b * a.yb + i * a.yt + (int64_t)h * a.yh;
  float y[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) y[e] = none ? 0.f : bad ? __builtin_nanf("") : o[e] / l;
  if (d4 < a.D) store_vec<T, 4>(yp + d4, y);
}

namespace {

template <typename T, int WPR>
void launch_join4(const SeqArgs& a, dim3 grid, int64_t rows, hipStream_t s) {
  const int D = seq_mfma_dim(a.D);
  if (D == 16) hipLaunchKernelGGL((seq_join4_kernel<T, 16, WPR>), grid, dim3(256), 0, s, a, rows);
  else if (D == 32) hipLaunchKernelGGL((seq_join4_kernel<T, 32, WPR>), grid, dim3(256), 0, s, a, rows);
  else if (D == 64) hipLaunchKernelGGL((seq_join4_kernel<T, 64, WPR>), grid, dim3(256), 0, s, a, rows);
  else if (D == 128) hipLaunchKernelGGL((seq_join4_kernel<T, 128, WPR>), grid, dim3(256), 0, s, a, rows);
  else hipLaunchKernelGGL((seq_join4_kernel<T, 256, WPR>), grid, dim3(256), 0, s, a, rows);
}

template <typename T, bool TREE>
int launch_tile(const SeqArgs& a, dim3 grid, hipStream_t s) {
#define DG_SEQ_TILE(NCH, LPR) hipLaunchKernelGGL((seq_tile_kernel<T, NCH, LPR, TREE>), grid, dim3(256), 0, s, a)
  if (a.rows_per_wg == 32) {
    if (a.D <= 64) DG_SEQ_TILE(1, 8);
    else if (a.D <= 128) DG_SEQ_TILE(2, 8);
    else DG_SEQ_TILE(4, 8);
  } else if (a.rows_per_wg == 16) {
    DG_SEQ_TILE(16, 16);
  } else {
    if (a.D <= 128) DG_SEQ_TILE(2, 32);
    else if (a.D <= 256) DG_SEQ_TILE(4, 32);
    else DG_SEQ_TILE(16, 32);
  }
#undef DG_SEQ_TILE
  return check_launch("seq_tile_kernel");
}

template <bool TREE>
int launch_tile_any(const SeqArgs& a, int dtype, dim3 grid, hipStream_t s) {
  if (dtype == DG_F64) return launch_tile<double, TREE>(a, grid, s);
  if (dtype == DG_F32) return launch_tile<float, TREE>(a, grid, s);
  if (dtype == DG_BF16) return launch_tile<bf16_t, TREE>(a, grid, s);
  return launch_tile<f16_t, TREE>(a, grid, s);
}

// rows of a workgroup of seq_tile_kernel, for so many rows of a key head
int tile_rows(int rows, int D) { return rows <= 8 ? 8 : D <= 256 ? 32 : 16; }

// Splits of a row: enough workgroups to fill the CUs as far as their LDS and registers let
// them share one (256 of 128 KB, as many more as smaller ones fit), and at least so many
// stages each that joining the splits, a launch of its own of some 6 us, costs no more than
// it saves: 8, one where fp32 products make a stage long (16 rows of the batch, 31 tokens
// behind up to 600 keys, 4 heads of 64: 20 us with 4, 15 with 1).  seq_tile_kernel's run up
// to seven a CU and take longer: 2048 of two stages (a step over 32 caches of 1900, 8 heads
// of 64, fp64: 468 us unsplit, 227 so).  us at 256 / 512 / 1024
// workgroups, bf16:
//   rows of 32, head_dim 128 (64 rows, 4 key heads, lengths to 4096)    56.2 / 63.6 / 75.2
//               head_dim  64 (64 rows, 8 key heads, lengths to 1024)    18.0 / 17.9 / 27.7
//           64, head_dim  64 (16 rows, 8 key heads, lengths to 4096)    36.3 / 31.1 / 34.1
//          128, head_dim 128 (16 rows, 4 key heads, lengths to 7168)    75.7 / 57.8 / 51.7
//               head_dim  64 (2 rows, 2 key heads, lengths to 131000)   96.1 / 84.2 / 85.3
constexpr int kMaxSplits = 512;

int tree_chunk(int64_t B, int Hkv, int nrb, int keys, int rows_per_wg, int D, int dtype, bool mfma) {
  const int stage = rows_per_wg <= 32 ? 128 : 64;  // keys, a multiple of every kernel's own
  if (mfma) D = seq_mfma_dim(D);
  const int64_t row_bytes = D * dtype_bytes(dtype);
  const int64_t fill = !mfma ? 2048
                       : rows_per_wg <= 32 ? (row_bytes >= 256 ? 256 : 512)
                       : rows_per_wg == 64 ? (row_bytes >= 512 ? 256 : 512)
                                           : D == 256 ? 512 : D == 128 ? 768 : 1024;
  const int64_t least = !mfma ? 2 : dtype == DG_F32 && D >= 64 ? 1 : 8;
  const int64_t wg = B * Hkv * nrb;
  const int64_t want = (fill + wg - 1) / wg;
  int64_t chunk = std::max<int64_t>((keys + want - 1) / want, (keys + kMaxSplits - 1) / kMaxSplits);
  chunk = std::max<int64_t>((chunk + stage - 1) / stage, least) * stage;
  return (int)std::min<int64_t>(chunk, 0x7fffff00);
}

// Row blocks, splits and workspace of a call.
struct TreeShape {
  int rows_per_wg, nrb, nsplit, chunk;
  size_t o_bytes, ws_bytes;
};

TreeShape tree_shape(int64_t B, int N, int H, int Hkv, int Tcap, int D, int dtype, int rows_per_wg, bool mfma) {
  TreeShape t{};
  const int R = N * (H / Hkv);
  t.rows_per_wg = rows_per_wg;
  t.nrb = (R + rows_per_wg - 1) / rows_per_wg;
  t.chunk = tree_chunk(B, Hkv, t.nrb, Tcap, rows_per_wg, D, dtype, mfma);
  t.nsplit = (int)(((int64_t)Tcap + t.chunk - 1) / t.chunk);
  const size_t acc = dtype == DG_F64 ? 8 : 4;
  const size_t parts = (size_t)B * Hkv * R * t.nsplit;
  if (t.nsplit > 1) {
    t.o_bytes = (parts * (mfma ? seq_mfma_dim(D) : D) * acc + 15) & ~(size_t)15;
    t.ws_bytes = t.o_bytes + parts * 2 * acc;
  }
  return t;
}

bool known_dtype(int dtype) { return dtype == DG_F32 || dtype == DG_BF16 || dtype == DG_F16 || dtype == DG_F64; }

// A bound on the workspace whichever kernel a call takes (the row blocks of each give
// other splits).
size_t tree_workspace(int64_t B, int N, int H, int Hkv, int Tcap, int D, int dtype) {
  size_t most = tree_shape(B, N, H, Hkv, Tcap, D, dtype, tile_rows(N * (H / Hkv), D), false).ws_bytes;
  for (int rows : {32, 64, 128})
    if (D <= 256) most = std::max(most, tree_shape(B, N, H, Hkv, Tcap, D, dtype, rows, true).ws_bytes);
  return most;
}

}  // namespace
}  // namespace dg

using namespace dg;

namespace dg {
namespace {

// The tiles of a batch in launch order.  Workgroup x runs on XCD x mod 8 and takes key head
// h = (x / 8) mod Hkv and entry 8 (x / 8 / Hkv) + (x - h) mod 8 (seq_piece): entry e is of
// list e mod 8, and each key head of a list's sequences has an XCD, and its L2, to itself.
// Sequences go whole to the list with the least work so far, longest first; a long one,
// which would leave lists unequal, tile by tile.  Within a list, windows of sequences whose
// keys stay in an L2 together, and in a window the tiles with the most keys first: every
// CU's share, one workgroup in 32 of its XCD's, then has long and short ones, and the
// launch ends on short ones.  Lists are filled up with empty tiles.
// Batches of few tiles, which run at once, are one window.  us over windows of 1024 / 2048
// / 4096 / 16384 keys, bf16: 512 of 17 - 276, 4 heads of 32, 32.4 / 33.7 / 35.7 / 33.9 (64 x
// 1024 tokens, 8 heads of 64, within 2 %); fp32, 16 x 1000 (128 tiles) in windows of 1024 /
// 2048 / 4096 keys and in one, 278 / 267 / 266 / 207.
constexpr int64_t kWindowKeys = 2048, kOneWindowTiles = 256;

std::vector<dg_packed_tile> plan_tiles(int64_t S, const int64_t* lq, const int64_t* lk, int group) {
  int64_t q0 = 0, k0 = 0;
  struct Seq {
    int64_t q0, k0, lq, lk, work;
  };
  std::vector<Seq> seqs;
  int64_t total = 0;
  for (int64_t s = 0; s < S; ++s) {
    if (lq[s] > 0) {
      const int64_t work = lq[s] * (std::max<int64_t>(0, lk[s] - lq[s] / 2) + 32);
      seqs.push_back(Seq{q0, k0, lq[s], lk[s], work});
      total += work;
    }
    q0 += lq[s];
    k0 += lk[s];
  }
  std::stable_sort(seqs.begin(), seqs.end(), [](const Seq& a, const Seq& b) { return a.work > b.work; });
  struct Entry {
    dg_packed_tile tile;
    int64_t window, keys;
  };
  std::vector<Entry> lists[8];
  int64_t load[8] = {}, held[8] = {}, held_apart = 0, all_tiles = 0;
  for (const Seq& s : seqs) all_tiles += (s.lq * group + kTileRows - 1) / kTileRows;
  const int64_t window_keys = all_tiles <= kOneWindowTiles ? (int64_t)1 << 40 : kWindowKeys;
  auto least = [&]() { return (int)(std::min_element(load, load + 8) - load); };
  for (const Seq& s : seqs) {
    const int64_t rows = s.lq * group, tiles = (rows + kTileRows - 1) / kTileRows;
    const bool apart = s.work > total / 32;
    int at = least();
    // sequences that are apart come first
    const int64_t window =
        window_keys > kWindowKeys ? 0 : apart ? held_apart / window_keys - ((int64_t)1 << 40) : held[at] / window_keys;
    (apart ? held_apart : held[at]) += s.lk;
    for (int64_t t = tiles - 1; t >= 0; --t) {  // a sequence's last queries see the most keys
      const int64_t r = t * kTileRows, n = std::min<int64_t>(kTileRows, rows - r);
      const int64_t keys = std::max<int64_t>(0, (r + n - 1) / group + s.lk - s.lq + 1);
      if (apart) at = least();
      lists[at].push_back(Entry{dg_packed_tile{(int32_t)s.q0, (int32_t)s.lq, (int32_t)s.k0, (int32_t)s.lk, (int32_t)r,
                                               (int32_t)n, {0, 0}},
                                window, keys});
      load[at] += keys + 32;
    }
  }
  size_t most = 0;
  for (auto& l : lists) {
    std::stable_sort(l.begin(), l.end(), [](const Entry& a, const Entry& b) {
      return a.window != b.window ? a.window < b.window : a.keys > b.keys;
    });
    most = std::max(most, l.size());
  }
  std::vector<dg_packed_tile> out(8 * most, dg_packed_tile{});
  for (size_t i = 0; i < most; ++i)
    for (int c = 0; c < 8; ++c)
      if (i < lists[c].size()) out[8 * i + c] = lists[c][i].tile;
  return out;
}

}  // namespace
}  // namespace dg

extern "C" int dg_packed_plan(int64_t S, const int64_t* lq, const int64_t* lk, int group, dg_packed_tile* tiles,
                              int64_t cap, int64_t* counts) {
  DG_REQUIRE(S >= 0 && group >= 1 && cap >= 0, DG_EINVAL, "packed_plan: negative size or group");
  DG_REQUIRE(counts != nullptr && (S == 0 || (lq != nullptr && lk != nullptr)) && (cap == 0 || tiles != nullptr),
             DG_EINVAL, "packed_plan: NULL argument");
  int64_t nq = 0, nk = 0, n = 0;
  for (int64_t s = 0; s < S; ++s) {
    DG_REQUIRE(lq[s] >= 0 && lk[s] >= 0, DG_EINVAL, "packed_plan: sequence %lld has a negative length", (long long)s);
    DG_REQUIRE(lq[s] <= kMostPositions / group, DG_EINVAL, "packed_plan: sequence %lld has more than 2^30 rows", (long long)s);
    DG_REQUIRE(lk[s] <= kMostPositions, DG_EINVAL, "packed_plan: sequence %lld has more than 2^30 keys", (long long)s);
    nq += lq[s];
    nk += lk[s];
    DG_REQUIRE(nq <= 0x7fffffff && nk <= 0x7fffffff, DG_EINVAL, "packed_plan: more than 2^31 - 1 rows");
    n += (lq[s] * group + kTileRows - 1) / kTileRows;
    DG_REQUIRE(n <= 0x7fffffff / 8, DG_EINVAL, "packed_plan: more than 2^28 tiles");
  }
  try {
    const std::vector<dg_packed_tile> plan = plan_tiles(S, lq, lk, group);
    counts[0] = (int64_t)plan.size();
    counts[1] = n;
    counts[2] = 0;
    for (const dg_packed_tile& t : plan) counts[2] = std::max<int64_t>(counts[2], t.rows);
    if (tiles == nullptr) return DG_OK;
    DG_REQUIRE(cap >= (int64_t)plan.size(), DG_EINVAL, "packed_plan: room for %lld tiles, %lld needed", (long long)cap,
               (long long)plan.size());
    std::copy(plan.begin(), plan.end(), tiles);
    return DG_OK;
  } catch (const std::exception& e) {
    set_error("packed_plan: %s", e.what());
    return DG_EWORKSPACE;
  }
}

extern "C" int dg_attention_packed(int64_t Nq, int64_t Nk, int H, int Hkv, int D, int dtype, const void* q, int64_t q_t,
                                   int64_t q_h, const void* k, int64_t k_t, int64_t k_h, const void* v, int64_t v_t,
                                   int64_t v_h, void* y, int64_t y_t, int64_t y_h, float scale,
                                   const dg_packed_tile* tiles, const int64_t counts[3], void* stream) {
  DG_REQUIRE(Nq >= 0 && Nk >= 0 && H >= 0, DG_EINVAL, "attention_packed: negative size");
  DG_REQUIRE(known_dtype(dtype), DG_EUNSUPPORTED, "attention_packed: dtype %d unsupported", dtype);
  DG_REQUIRE(D >= 1 && D <= kMaxHeadDim, DG_EUNSUPPORTED, "attention_packed: head_dim %d outside [1, %d]", D, kMaxHeadDim);
  DG_REQUIRE(Hkv >= 1 && H % Hkv == 0, DG_EINVAL, "attention_packed: %d query heads on %d key heads", H, Hkv);
  DG_REQUIRE(scale > 0.f && std::isfinite(scale * kLog2e), DG_EINVAL, "attention_packed: the scale must be positive and below 2^127");
  DG_REQUIRE(counts != nullptr, DG_EINVAL, "attention_packed: NULL argument");
  DG_REQUIRE(counts[0] >= 0 && counts[0] <= 0x7fffffff && counts[0] % 8 == 0 && counts[1] >= 0 && counts[1] <= counts[0] &&
                 counts[2] >= 0 && counts[2] <= kTileRows,
             DG_EINVAL, "attention_packed: counts (%lld, %lld, %lld) are not dg_packed_plan's", (long long)counts[0],
             (long long)counts[1], (long long)counts[2]);
  if (Nq == 0 || H == 0 || counts[1] == 0 || counts[2] == 0) return DG_OK;  // no tile
  DG_REQUIRE(q && y && tiles && (Nk == 0 || (k && v)), DG_EINVAL, "attention_packed: NULL argument");
  SeqArgs a{};
  a.q = q; a.k = k; a.v = v; a.y = y;
  a.qt = q_t; a.qh = q_h; a.kt = k_t; a.kh = k_h;
  a.vt = v_t; a.vh = v_h; a.yt = y_t; a.yh = y_h;
  a.H = H; a.Hkv = Hkv; a.G = H / Hkv; a.D = D;
  a.scale = scale;
  a.scale_log2 = scale * kLog2e;
  a.tiles = tiles;
  a.nq = Nq; a.nk = Nk;
  a.nsplit = 1;
  const bool mfma = seq_mfma_applicable(a, dtype, false);
  a.rows_per_wg = mfma ? seq_mfma_packed_rows(counts, Hkv, D) : tile_rows((int)counts[2], D);
  a.nrb = (int)((counts[2] + a.rows_per_wg - 1) / a.rows_per_wg);
  const int64_t blocks = counts[0] * Hkv;
  DG_REQUIRE(blocks <= kMostWorkgroups256 && blocks * a.nrb <= kMostWorkgroups256, DG_EINVAL,
             "attention_packed: more than 2^24 - 1 workgroups (tiles times key heads)");
  hipStream_t s = static_cast<hipStream_t>(stream);
  const dim3 grid((unsigned)(blocks * a.nrb));
  return mfma ? launch_seq_mfma_packed(a, dtype, grid, s) : launch_tile_any<false>(a, dtype, grid, s);
}

extern "C" size_t dg_attention_tree_workspace_size(int B, int N, int H, int Hkv, int Tcap, int D, int dtype) {
  if (B <= 0 || N <= 0 || N > 64 || H <= 0 || Hkv <= 0 || H % Hkv || Tcap < N || Tcap > kMostPositions || D <= 0) return 0;
  return tree_workspace(B, N, H, Hkv, Tcap, D, dtype);
}

extern "C" int dg_attention_tree(int B, int N, int H, int Hkv, int Tcap, int D, int dtype, const void* q,
                                 const dg_stride3* q_st, const void* k_cache, const dg_stride3* kc_st,
                                 const void* v_cache, const dg_stride3* vc_st, void* y, const dg_stride3* y_st,
                                 float scale, int len, const int32_t* lens, const int64_t* masks, int64_t mask_b,
                                 void* workspace, size_t workspace_bytes, void* stream) {
  DG_REQUIRE(B >= 0 && H >= 0, DG_EINVAL, "attention_tree: negative size");
  DG_REQUIRE(known_dtype(dtype), DG_EUNSUPPORTED, "attention_tree: dtype %d unsupported", dtype);
  DG_REQUIRE(D >= 1 && D <= kMaxHeadDim, DG_EUNSUPPORTED, "attention_tree: head_dim %d outside [1, %d]", D, kMaxHeadDim);
  DG_REQUIRE(N >= 1 && N <= 64, DG_EINVAL, "attention_tree: %d tokens a row, 1 to 64", N);
  DG_REQUIRE(Tcap >= N, DG_EINVAL, "attention_tree: the cache holds %d positions, %d tokens", Tcap, N);
  DG_REQUIRE(Tcap <= kMostPositions, DG_EINVAL, "attention_tree: a cache of more than 2^30 positions");
  DG_REQUIRE(Hkv >= 1 && H % Hkv == 0, DG_EINVAL, "attention_tree: %d query heads on %d key heads", H, Hkv);
  DG_REQUIRE(H / Hkv <= 0x7fffff, DG_EINVAL, "attention_tree: %d heads a group", H / Hkv);
  DG_REQUIRE(scale > 0.f && std::isfinite(scale * kLog2e), DG_EINVAL, "attention_tree: the scale must be positive and below 2^127");
  DG_REQUIRE(lens != nullptr || (len >= 0 && len <= Tcap - N), DG_EINVAL,
             "attention_tree: %d cached positions and %d tokens in a cache of %d", len, N, Tcap);
  if (B == 0 || H == 0) return DG_OK;
  DG_REQUIRE(q && k_cache && v_cache && y && q_st && kc_st && vc_st && y_st, DG_EINVAL, "attention_tree: NULL argument");
  SeqArgs a{};
  a.q = q; a.k = k_cache; a.v = v_cache; a.y = y;
  a.qb = q_st->b; a.qt = q_st->t; a.qh = q_st->h;
  a.kb = kc_st->b; a.kt = kc_st->t; a.kh = kc_st->h;
  a.vb = vc_st->b; a.vt = vc_st->t; a.vh = vc_st->h;
  a.yb = y_st->b; a.yt = y_st->t; a.yh = y_st->h;
  a.H = H; a.Hkv = Hkv; a.G = H / Hkv; a.D = D;
  a.scale = scale;
  a.scale_log2 = scale * kLog2e;
  a.B = B; a.N = N; a.Tcap = Tcap;
  a.len = len; a.lens = lens;
  a.masks = masks; a.mask_b = mask_b;
  // 32-row tiles of fp32 products are mostly empty over 8 rows, and long at head_dim over 64:
  // a step over 32 caches of 1900, 8 heads of 128, 155 us there and 127 in seq_tile_kernel,
  // 64 of up to 4000, 16 heads on 4, 285 and 221; 4 of 140, 8 heads, 18.8 and 20.6, one of
  // 20000, 4 heads, 41 and 59.
  const bool few = dtype == DG_F32 && D > 64 && N * a.G <= 8 && (int64_t)B * Hkv >= 64;
  const bool mfma = !few && seq_mfma_applicable(a, dtype, true);
  const TreeShape t = tree_shape(B, N, H, Hkv, Tcap, D, dtype, mfma ? seq_mfma_tree_rows(B, N * a.G, Hkv, Tcap, D, dtype) : tile_rows(N * a.G, D), mfma);
  a.rows_per_wg = t.rows_per_wg; a.nrb = t.nrb; a.nsplit = t.nsplit; a.chunk = t.chunk;
  // seq_mfma_tree_rows takes 128 for fewer than 256 tiles over more than 300000 / 255 keys, of
  // which a split has at most a half: that kernel knows no other way
  DG_REQUIRE(!mfma || t.rows_per_wg < 128 || t.nsplit > 1, DG_EUNSUPPORTED, "attention_tree: 128 rows unsplit");
  if (t.nsplit > 1) {
    DG_REQUIRE(workspace != nullptr && workspace_bytes >= t.ws_bytes, DG_EWORKSPACE,
               "attention_tree: a workspace of %zu bytes, %zu needed", workspace_bytes, t.ws_bytes);
    DG_REQUIRE((reinterpret_cast<uintptr_t>(workspace) & 15) == 0, DG_EINVAL, "attention_tree: workspace not 16-byte aligned");
    a.ws_o = workspace;
    a.ws_ml = static_cast<char*>(workspace) + t.o_bytes;
  }
  // a row's waves read its splits in turn: four of them where there are many and rows few
  const int64_t rows = (int64_t)B * H * N;
  const bool many = t.nsplit >= 16 && rows <= 4096;
  const int64_t groups = t.nsplit == 1 ? 0 : many ? rows : (rows + 3) / 4;
  const int64_t blocks = ((int64_t)B * Hkv * t.nsplit + 7) / 8 * 8 * t.nrb;
  DG_REQUIRE(blocks <= kMostWorkgroups256 && groups <= kMostWorkgroups256, DG_EINVAL,
             "attention_tree: more than 2^24 - 1 workgroups");
  hipStream_t s = static_cast<hipStream_t>(stream);
  const int rc = mfma ? launch_seq_mfma_tree(a, dtype, (unsigned)blocks, s)
                      : launch_tile_any<true>(a, dtype, dim3((unsigned)blocks), s);
  if (rc != DG_OK || t.nsplit == 1) return rc;
  const dim3 grid((unsigned)groups);
#define DG_JOIN(T)                                                                         \
  do {                                                                                     \
    if (many) hipLaunchKernelGGL((seq_join_kernel<T, 4>), grid, dim3(256), 0, s, a, rows); \
    else hipLaunchKernelGGL((seq_join_kernel<T, 1>), grid, dim3(256), 0, s, a, rows);      \
  } while (0)
#define DG_JOIN4(T)                                          \
  do {                                                       \
    if (many) launch_join4<T, 4>(a, grid, rows, s);          \
    else launch_join4<T, 1>(a, grid, rows, s);               \
  } while (0)
  if (mfma) {
    if (dtype == DG_F32) DG_JOIN4(float);
    else if (dtype == DG_BF16) DG_JOIN4(bf16_t);
    else DG_JOIN4(f16_t);
  } else {
    if (dtype == DG_F64) DG_JOIN(double);
    else if (dtype == DG_F32) DG_JOIN(float);
    else if (dtype == DG_BF16) DG_JOIN(bf16_t);
    else DG_JOIN(f16_t);
  }
#undef DG_JOIN
#undef DG_JOIN4
  return check_launch("seq_join_kernel");
}
