// A cache in pages: new keys and values into the rows' pages, rotated and normalised
// (dg_paged_append), and rows cut to their newest positions and those of the largest weights
// (dg_paged_evict).
//
// paged_append_kernel.  y = r / sqrt(mean(r^2) + eps), r the pairs of a head turned by their
// position's angle: both in fp32 (fp64) registers, eps that type's, one rounding as y is stored.  (The cache of
// one length, dg_rope.hip, rounds r to the data's type first, as the reference does; once is
// nearer to the exact value, bf16 1.7e-3 of it, and no dearer.)  LPR lanes share a head, 16 bytes
// each; they take HPT heads of a token, whose loads are in flight together and whose angles
// are read once.  Bound by HBM where tokens are many (24 x 700 tokens, 24 heads of 128, bf16:
// 30.5 us, 172 MB; 40.5 with 64-bit products for every head's address, the angles unpacked for
// each and a correctly rounded root), by the launch where they are few.
//
// paged_select_kernel.  The m-th largest weight of a row by its bits: three passes of 11, 11
// and 10 over an order-preserving integer, counted in LDS, then one that ranks what is above
// it and the first of those that equal it.  One workgroup a (row, key head), each wave with a
// stretch of the positions, so that ranks come from ballots and one exchange.  Bound by the
// passes' latencies: 64 (row, key head)s of up to 8100 positions 14.5 us, 128 of up to 200 6.7 (21.9 and
// 12.5 with all weights read anew and ranks summed thread by thread).
// paged_move_kernel then copies the kept positions, 16 bytes a thread (2000 of each of the
// 64's, 128 dims in bf16, 131 MB, 23.5 us, 5.6 TB/s: HBM).
#include "dg_paged.h"

#include <float.h>

#include <algorithm>

namespace dg {

struct AppendArgs {
  const void* src[3];  // q, k, v
  int64_t sb[3], st[3];
  void* dst[3];  // q_out, the pages' k and v
  int64_t db[3], dt[3];
  int sh[3], dh[3];  // from head to head, bytes
  const void* freqs;
  int64_t freqs_ld, freqs_rows;
  const int32_t* table;
  int64_t table_ld, pages;
  const int32_t* lens;
  const int32_t* counts;
  const int32_t* positions;
  int64_t items;
  int N, H, Hkv, D, cap, page_log2, groups, qknorm;
};

// N values of T as raw words: VEC by 16-byte accesses, 8 bytes of them by one of 8 (an fp32
// table's angles of two fp64 dims), p aligned to them; or one by one those below `n`.
template <typename T, int N, bool VEC>
__device__ __forceinline__ void load_some(const T* p, uint32_t (&w)[N * sizeof(T) / 4], int n) {
  constexpr int BYTES = N * (int)sizeof(T);
  if constexpr (VEC && BYTES == 8) {
    const u32x2_t x = *reinterpret_cast<const u32x2_t*>(p);
    w[0] = x[0];
    w[1] = x[1];
  } else if constexpr (VEC) {
    static_assert(BYTES % 16 == 0, "all of the values are loaded");
#pragma unroll
    for (int c = 0; c < BYTES / 16; ++c) {
      const u32x4_t x = reinterpret_cast<const u32x4_t*>(p)[c];
#pragma unroll
      for (int i = 0; i < 4; ++i) w[4 * c + i] = x[i];
    }
  } else {
    T e[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      e[i] = T{};
      if (i < n) e[i] = p[i];
    }
    __builtin_memcpy(w, e, sizeof(e));
  }
}
template <typename T, int N, bool VEC>
__device__ __forceinline__ void store_some(T* p, const uint32_t (&w)[N * sizeof(T) / 4], int n) {
  if constexpr (VEC) {
    static_assert(N * sizeof(T) % 16 == 0, "all of the values are stored");
#pragma unroll
    for (int c = 0; c < N * (int)sizeof(T) / 16; ++c)
      reinterpret_cast<u32x4_t*>(p)[c] = u32x4_t{w[4 * c], w[4 * c + 1], w[4 * c + 2], w[4 * c + 3]};
  } else {
    T e[N];
    __builtin_memcpy(e, w, sizeof(e));
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (i < n) p[i] = e[i];
  }
}

// Pair i of the raw words in the arithmetic's type, and back.
template <typename T>
struct AppendAcc {
  using type = float;
  static constexpr float kEps = FLT_EPSILON;
  __device__ static void load(const uint32_t* w, int i, float& x, float& y) {
    if constexpr (sizeof(T) == 4) {
      x = __uint_as_float(w[2 * i]);
      y = __uint_as_float(w[2 * i + 1]);
    } else {
      RowRegs<T, 2> r;
      r.w[0] = w[i];
      x = elem<T, 2>(r, 0);
      y = elem<T, 2>(r, 1);
    }
  }
  __device__ static void store(uint32_t* w, int i, float x, float y) {
    if constexpr (sizeof(T) == 4) {
      w[2 * i] = __float_as_uint(x);
      w[2 * i + 1] = __float_as_uint(y);
    } else {
      w[i] = pack_pair<T>(x, y);
    }
  }
};
template <>
struct AppendAcc<double> {
  using type = double;
  static constexpr double kEps = DBL_EPSILON;
  __device__ static void load(const uint32_t* w, int i, double& x, double& y) {
    __builtin_memcpy(&x, w + 4 * i, 8);
    __builtin_memcpy(&y, w + 4 * i + 2, 8);
  }
  __device__ static void store(uint32_t* w, int i, double x, double y) {
    __builtin_memcpy(w + 4 * i, &x, 8);
    __builtin_memcpy(w + 4 * i + 2, &y, 8);
  }
};

// 1 / sqrt(x), x > 0
__device__ __forceinline__ double inv_sqrt(double x) { return 1.0 / sqrt(x); }
__device__ __forceinline__ float inv_sqrt(float x) {
  // the hardware's, off by a step at most, and Newton's step behind it (a correctly rounded root
  // and quotient are forty instructions of every head)
  const float y = __builtin_amdgcn_rsqf(x);
  return y == 0.f ? y : __builtin_fmaf(__builtin_fmaf(-x * y, y, 1.0f), 0.5f * y, y);  // 0 for infinity
}

template <int LPR>
__device__ __forceinline__ float lanes_sum(float x) {
  return group_sum_dpp<LPR>(x);
}
template <int LPR>
__device__ __forceinline__ double lanes_sum(double x) {
#pragma unroll
  for (int off = 1; off < LPR; off <<= 1) x += __shfl_xor(x, off, 64);
  return x;
}

// EPL consecutive dims a lane and piece, LPR lanes a head, NCK pieces, HPT heads of a token.
template <typename T, typename FT, int EPL, int LPR, int NCK, int HPT, bool VEC>
__global__ __launch_bounds__(256) void paged_append_kernel(const AppendArgs a) {
  using S = AppendAcc<T>;
  using A = typename S::type;
  constexpr int W = EPL * (int)sizeof(T) / 4, FW = EPL * (int)sizeof(FT) / 4;
  const int sub = threadIdx.x % LPR;
  const uint32_t item = blockIdx.x * (256u / LPR) + threadIdx.x / LPR;  // below 2^31
  if (item >= a.items) return;  // whole lane groups; no barriers follow
  const uint32_t token = item / (uint32_t)a.groups;
  // heads h0, h0 + groups, ..: neighbouring lane groups have neighbouring heads at a time
  const int h0 = (int)(item - token * (uint32_t)a.groups);
  const int64_t b = token / (uint32_t)a.N;
  const int n = (int)(token - (uint32_t)b * (uint32_t)a.N);
  const int heads = a.H + 2 * a.Hkv;

  // The token's heads, which no length decides where to read.  Where tokens are many, those
  // that are not there are not read all the same (24 x 700 tokens, three quarters of them there,
  // 24 heads of 128: 44.8 us read, 41.6 not, before the rest was as it is).
  bool read = true;
  if constexpr (HPT > 1) {
    if (a.counts != nullptr) read = n < a.counts[b];
  }
  // head h's first element, of three tensors one after the other
  auto at = [&](const char* q, const char* k, const char* v, const int (&step)[3], int h) __attribute__((always_inline)) {
    const bool is_q = h < a.H, is_k = h < a.H + a.Hkv;
    const char* base = is_q ? q : is_k ? k : v;
    const int hw = is_q ? h : is_k ? h - a.H : h - a.H - a.Hkv;
    const int by = is_q ? step[0] : is_k ? step[1] : step[2];
    return base + (int64_t)hw * by;
  };
  const char *xq, *xk, *xv;
  {
    const int64_t es = (int64_t)sizeof(T);
    xq = static_cast<const char*>(a.src[0]) + (b * a.sb[0] + n * a.st[0]) * es;
    xk = static_cast<const char*>(a.src[1]) + (b * a.sb[1] + n * a.st[1]) * es;
    xv = static_cast<const char*>(a.src[2]) + (b * a.sb[2] + n * a.st[2]) * es;
  }
  uint32_t x[HPT][NCK][W];
#pragma unroll
  for (int j = 0; j < HPT; ++j) {
    const T* p = reinterpret_cast<const T*>(at(xq, xk, xv, a.sh, min(h0 + a.groups * j, heads - 1)));
#pragma unroll
    for (int c = 0; c < NCK; ++c) {
      const int d = EPL * (sub + LPR * c);
#pragma unroll
      for (int e = 0; e < W; ++e) x[j][c][e] = 0u;
      if (d < a.D && read) load_some<T, EPL, VEC>(p + d, x[j][c], a.D - d);
    }
  }
  const int len = a.lens[b];
  const int own = min(max(len, 0), a.cap);
  const int count = min(max(a.counts != nullptr ? a.counts[b] : a.N, 0), min(a.N, a.cap - own));
  const bool there = n < count;
  const int slot = own + n;
  const int64_t pos = (int64_t)(a.positions != nullptr ? a.positions[b] : own) + n;
  const bool known = pos >= 0 && pos < a.freqs_rows;
  int id = -1;
  if (there) id = a.table[b * a.table_ld + (slot >> a.page_log2)];
  const bool held = id >= 0 && id < a.pages;
  const int in_page = slot & ((1 << a.page_log2) - 1);
  A co[NCK][EPL / 2], si[NCK][EPL / 2];
#pragma unroll
  for (int c = 0; c < NCK; ++c) {
    const int d = EPL * (sub + LPR * c);
    uint32_t cs[FW];
#pragma unroll
    for (int e = 0; e < FW; ++e) cs[e] = 0u;
    if (d < a.D) load_some<FT, EPL, VEC>(static_cast<const FT*>(a.freqs) + (known ? pos : 0) * a.freqs_ld + d, cs, a.D - d);
#pragma unroll
    for (int e = 0; e < EPL / 2; ++e) {
      typename AppendAcc<FT>::type cx, sx;
      AppendAcc<FT>::load(cs, e, cx, sx);
      co[c][e] = cx;
      si[c][e] = sx;
    }
  }
  const char *yq, *yk, *yv;
  {
    const int64_t es = (int64_t)sizeof(T), page = held ? id : 0;
    yq = static_cast<const char*>(a.dst[0]) + (b * a.db[0] + n * a.dt[0]) * es;
    yk = static_cast<const char*>(a.dst[1]) + (page * a.db[1] + in_page * a.dt[1]) * es;
    yv = static_cast<const char*>(a.dst[2]) + (page * a.db[2] + in_page * a.dt[2]) * es;
  }

#pragma unroll
  for (int j = 0; j < HPT; ++j) {
    const int h = h0 + a.groups * j;
    if (h >= heads) break;  // the same in all of the group's lanes
    if (h < a.H + a.Hkv) {
      A y[NCK][EPL], ss = (A)0;
#pragma unroll
      for (int c = 0; c < NCK; ++c)
#pragma unroll
        for (int e = 0; e < EPL; e += 2) {
          A re, im;
          S::load(x[j][c], e / 2, re, im);
          y[c][e] = re * co[c][e / 2] - im * si[c][e / 2];
          y[c][e + 1] = re * si[c][e / 2] + im * co[c][e / 2];
          ss += y[c][e] * y[c][e] + y[c][e + 1] * y[c][e + 1];
        }
      A f = (A)1;
      if (a.qknorm) f = inv_sqrt(lanes_sum<LPR>(ss) * (A)(1.0 / a.D) + S::kEps);
      if (!known) f = (A)__builtin_nanf("");
#pragma unroll
      for (int c = 0; c < NCK; ++c)
#pragma unroll
        for (int e = 0; e < EPL; e += 2) S::store(x[j][c], e / 2, there ? y[c][e] * f : (A)0, there ? y[c][e + 1] * f : (A)0);
    }
    if (h >= a.H && !held) continue;
    T* o = reinterpret_cast<T*>(const_cast<char*>(at(yq, yk, yv, a.dh, h)));
#pragma unroll
    for (int c = 0; c < NCK; ++c) {
      const int d = EPL * (sub + LPR * c);
      if (d < a.D) store_some<T, EPL, VEC>(o + d, x[j][c], a.D - d);
    }
  }
}

struct EvictArgs {
  const float* weights;
  int64_t wb, wh;
  const int32_t* table;
  int64_t table_ld, pages;
  const int32_t* to;
  int64_t to_ld, to_cap;
  const int32_t* lens;
  int32_t* new_lens;
  float* new_weights;
  int32_t* kept;
  const char* k;
  const char* v;
  int64_t kb, kt, kh, vb, vt, vh;  // bytes
  int Hkv, cap, keep, recent, page_log2, pieces;
  int64_t items;
};

// Larger for larger weights: the order of the bits, zeros of both signs alike, NaN above all.
__device__ __forceinline__ uint32_t weight_key(float w) {
  if (w != w) return 0xffffffffu;
  const uint32_t u = __float_as_uint(w + 0.0f);
  return u >> 31 ? ~u : u | 0x80000000u;
}

constexpr int kSelectBins = 2048;
constexpr uint32_t kZeroKey = 0x80000000u;

// KPT weights a thread in registers, for rows of at most THREADS * KPT positions; 0: read anew
// in every pass.
template <int THREADS, int KPT>
__global__ __launch_bounds__(THREADS) void paged_select_kernel(const EvictArgs a) {
  constexpr int WAVES = THREADS / 64, BPT = kSelectBins / THREADS;
  __shared__ uint32_t hist[kSelectBins];
  __shared__ uint32_t totals[WAVES];
  __shared__ uint32_t found[3];
  __shared__ int above[WAVES], equal[WAVES];
  const int64_t bh = blockIdx.x;
  const int64_t b = bh / a.Hkv;
  const int h = (int)(bh - b * a.Hkv);
  const int tid = threadIdx.x, lane = tid & 63;
  const int wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int len = min(max(a.lens[b], 0), a.cap);
  int32_t* const kept = a.kept + bh * a.keep;
  if (len <= a.keep) {
    for (int j = tid; j < a.keep; j += THREADS) kept[j] = j < len ? j : -1;
    return;  // whole workgroups, before any barrier
  }
  const int old = len - a.recent;
  const int m = a.keep - a.recent;  // below old
  const float* const w = a.weights + b * a.wb + (int64_t)h * a.wh;

  // a wave's stretch of the positions, in whole 64
  const int per = ((old + 63) / 64 + WAVES - 1) / WAVES * 64;
  const int t0 = min(wv * per, old), t1 = min(t0 + per, old);
  uint32_t keys[KPT > 0 ? KPT : 1];
  if constexpr (KPT > 0) {
#pragma unroll
    for (int i = 0; i < KPT; ++i) {
      const int t = t0 + 64 * i + lane;
      keys[i] = t < t1 ? weight_key(w[t]) : 0u;
    }
  }
  for (int j = tid; j < a.recent; j += THREADS) kept[m + j] = old + j;
  if (m == 0) return;
  // f(position, key, whether it is one) for each 64 of the stretch
  auto each = [&](auto f) __attribute__((always_inline)) {
    if constexpr (KPT > 0) {
#pragma unroll
      for (int i = 0; i < KPT; ++i) {
        const int t = t0 + 64 * i;
        if (t < t1) f(t + lane, keys[i], t + lane < t1);
      }
    } else {
      for (int t = t0; t < t1; t += 64) {
        const bool in = t + lane < t1;
        f(t + lane, in ? weight_key(w[t + lane]) : 0u, in);
      }
    }
  };

  // the m-th largest key's leading bits (mask): all that are left share them, and `need` of
  // those are taken
  uint32_t prefix = 0, mask = 0, need = (uint32_t)m;
  for (int pass = 0; pass < 3; ++pass) {
    const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0;
    const uint32_t bins = pass == 2 ? 1024 : 2048;
#pragma unroll
    for (int i = 0; i < BPT; ++i) hist[tid + THREADS * i] = 0;
    __syncthreads();
    each([&](int, uint32_t key, bool in) __attribute__((always_inline)) {
      in = in && (key & mask) == prefix;
      const uint32_t bin = (key >> shift) & (bins - 1);
      // many positions may share one value, zero above all: those are counted at once
      const uint64_t zeros = __builtin_amdgcn_ballot_w64(in && key == kZeroKey);
      if (zeros != 0 && lane == 0) atomicAdd(&hist[(kZeroKey >> shift) & (bins - 1)], (uint32_t)__builtin_popcountll(zeros));
      if (in && key != kZeroKey) atomicAdd(&hist[bin], 1u);
    });
    __syncthreads();
    // the bin that holds the need-th largest: thread i has BPT bins from the top down
    uint32_t n[BPT], mine = 0;
#pragma unroll
    for (int i = 0; i < BPT; ++i) {
      n[i] = hist[kSelectBins - 1 - (BPT * tid + i)];
      mine += n[i];
    }
    uint32_t upto = mine;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      const uint32_t x = __shfl_up(upto, off, 64);
      if (lane >= off) upto += x;
    }
    if (lane == 63) totals[wv] = upto;
    __syncthreads();
    for (int i = 0; i < wv; ++i) upto += totals[i];
    if (upto >= need && upto - mine < need) {  // one thread
      uint32_t c = upto - mine;
#pragma unroll
      for (int i = 0; i < BPT; ++i) {
        if (c < need && c + n[i] >= need) {
          found[0] = (uint32_t)(kSelectBins - 1 - (BPT * tid + i));
          found[1] = c;
          found[2] = n[i];
        }
        c += n[i];
      }
    }
    __syncthreads();
    prefix |= found[0] << shift;
    mask |= (bins - 1) << shift;
    need -= found[1];
    if (found[2] == need) break;  // all of the bin are taken
    // the next pass writes found behind a barrier that all reach after reading it here
  }

  // positions above the m-th largest weight, and the first `need` that equal it
  int na = 0, ne = 0;
  each([&](int, uint32_t key, bool in) __attribute__((always_inline)) {
    na += __builtin_popcountll(__builtin_amdgcn_ballot_w64(in && (key & mask) > prefix));
    ne += __builtin_popcountll(__builtin_amdgcn_ballot_w64(in && (key & mask) == prefix));
  });
  if (lane == 0) {
    above[wv] = na;
    equal[wv] = ne;
  }
  __syncthreads();
  int at = 0, eq = 0;
  for (int i = 0; i < wv; ++i) {
    at += above[i];
    eq += equal[i];
  }
  at += min(eq, (int)need);
  const uint64_t below = (1ull << lane) - 1;
  each([&](int t, uint32_t key, bool in) __attribute__((always_inline)) {
    const uint64_t es = __builtin_amdgcn_ballot_w64(in && (key & mask) == prefix);
    const bool take = in && ((key & mask) > prefix ||
                             ((key & mask) == prefix && eq + __builtin_popcountll(es & below) < (int)need));
    const uint64_t ts = __builtin_amdgcn_ballot_w64(take);
    if (take) kept[at + __builtin_popcountll(ts & below)] = t;
    at += __builtin_popcountll(ts);
    eq += __builtin_popcountll(es);
  });
}

// One piece of U of one kept position of a key head a thread; the first piece's thread has
// its weight, and those of the places behind the kept ones.
template <typename U>
__global__ __launch_bounds__(256) void paged_move_kernel(const EvictArgs a) {
  const uint32_t item = blockIdx.x * 256u + threadIdx.x;  // below 2^32
  if (item >= a.items) return;
  const uint32_t at = item / (uint32_t)a.pieces;  // (b, h, j)
  const int piece = (int)(item - at * (uint32_t)a.pieces);
  const int64_t bh = at / (uint32_t)a.to_cap;
  const int j = (int)(at - (uint32_t)bh * (uint32_t)a.to_cap);
  const int64_t b = (uint32_t)bh / (uint32_t)a.Hkv;
  const int h = (int)(bh - b * a.Hkv);
  // by one thread a row, here: the selection is through with the lengths, which these may replace
  if (j == 0 && h == 0 && piece == 0) a.new_lens[b] = min(min(max(a.lens[b], 0), a.cap), a.keep);
  const int t = j < a.keep ? a.kept[bh * a.keep + j] : -1;
  if (piece == 0) a.new_weights[at] = t < 0 ? 0.f : a.weights[b * a.wb + (int64_t)h * a.wh + t];
  if (t < 0) return;
  const int64_t src = a.table[b * a.table_ld + (t >> a.page_log2)];
  const int64_t dst = a.to[b * a.to_ld + (j >> a.page_log2)];
  if (dst < 0 || dst >= a.pages) return;
  const int mask = (1 << a.page_log2) - 1;
  U xk{}, xv{};
  if (src >= 0 && src < a.pages) {
    xk = *reinterpret_cast<const U*>(a.k + src * a.kb + (t & mask) * a.kt + h * a.kh + piece * (int)sizeof(U));
    xv = *reinterpret_cast<const U*>(a.v + src * a.vb + (t & mask) * a.vt + h * a.vh + piece * (int)sizeof(U));
  }
  *reinterpret_cast<U*>(const_cast<char*>(a.k) + dst * a.kb + (j & mask) * a.kt + h * a.kh + piece * (int)sizeof(U)) = xk;
  *reinterpret_cast<U*>(const_cast<char*>(a.v) + dst * a.vb + (j & mask) * a.vt + h * a.vh + piece * (int)sizeof(U)) = xv;
}

namespace {

template <typename T, typename FT, int EPL, int LPR, int NCK, int HPT, bool VEC>
int launch_append(AppendArgs& a, int64_t tokens, hipStream_t s) {
  a.groups = (a.H + 2 * a.Hkv + HPT - 1) / HPT;
  a.items = tokens * a.groups;
  constexpr int PER = 256 / LPR;
  const int64_t blocks = (a.items + PER - 1) / PER;
  DG_REQUIRE(blocks <= kMostWorkgroups256, DG_EINVAL, "paged_append: more than 2^24 - 1 workgroups");
  hipLaunchKernelGGL((paged_append_kernel<T, FT, EPL, LPR, NCK, HPT, VEC>), dim3((unsigned)blocks), dim3(256), 0, s, a);
  return check_launch(VEC ? "paged_append_kernel" : "paged_append_any_kernel");
}

template <typename T, typename FT>
int append_pick(AppendArgs& a, bool vec, int64_t tokens, hipStream_t s) {
  constexpr int EPL = 16 / (int)sizeof(T);
  // one head a lane group where tokens are few, four where their loads are to be in flight
  // together; us one / four, by heads of all tokens: 1536 of 128 3.3 / 4.4, 24576 of 64
  // 3.9 / 4.6, 98304 of 64 8.3 / 6.5, 403200 of 128 42.2 / 36.6
  const bool few = tokens * (a.H + 2 * a.Hkv) <= 32768;
  if (!vec) {
    if (a.D <= 128) return launch_append<T, FT, 2, 64, 1, 1, false>(a, tokens, s);
    return launch_append<T, FT, 2, 64, 8, 1, false>(a, tokens, s);
  }
  const int lanes = a.D / EPL;
#define DG_APPEND(LPR)                                                                 \
  if (lanes <= LPR)                                                                    \
  return few ? launch_append<T, FT, EPL, LPR, 1, 1, true>(a, tokens, s)                \
             : launch_append<T, FT, EPL, LPR, 1, 4, true>(a, tokens, s)
  DG_APPEND(2);
  DG_APPEND(4);
  DG_APPEND(8);
  DG_APPEND(16);
  DG_APPEND(32);
  DG_APPEND(64);
#undef DG_APPEND
  return launch_append<T, FT, EPL, 64, kMaxHeadDim / EPL / 64, 1, true>(a, tokens, s);
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace
}  // namespace dg

using namespace dg;

extern "C" int dg_paged_append(const dg_paged_append_args* args, void* stream) {
  DG_REQUIRE(args != nullptr, DG_EINVAL, "paged_append: NULL argument");
  DG_REQUIRE(int_size(args->B) && int_size(args->N) && args->H >= 0 && args->Hkv >= 0, DG_EINVAL,
             "paged_append: negative size or one past 2^31 - 1");
  DG_REQUIRE(args->H <= 0xffff && args->Hkv <= 0xffff, DG_EINVAL, "paged_append: more than 65535 heads");
  DG_REQUIRE(args->D >= 2 && args->D % 2 == 0 && args->D <= kMaxHeadDim, DG_EUNSUPPORTED,
             "paged_append: head_dim %lld, even ones from 2 to %d", (long long)args->D, kMaxHeadDim);
  DG_REQUIRE(known_dtype(args->dtype), DG_EUNSUPPORTED, "paged_append: dtype %lld unsupported", (long long)args->dtype);
  const int B = (int)args->B, N = (int)args->N, H = (int)args->H, Hkv = (int)args->Hkv, D = (int)args->D, dtype = (int)args->dtype;
  const int64_t freqs_dtype = args->freqs_dtype, freqs_ld = args->freqs_ld, freqs_rows = args->freqs_rows;
  const void *q = args->q, *k = args->k, *v = args->v, *freqs = args->freqs;
  const dg_paged_rows* rows = &args->rows;
  DG_REQUIRE(freqs_dtype == DG_F32 || freqs_dtype == dtype, DG_EUNSUPPORTED,
             "paged_append: freqs dtype must be fp32 or equal to the data dtype");
  if (B == 0 || N == 0 || H + Hkv == 0) return DG_OK;
  AppendArgs a{};
  if (const int rc = check_paged_rows("paged_append", rows, true, &a.page_log2)) return rc;
  DG_REQUIRE(H == 0 || (q && args->q_out), DG_EINVAL, "paged_append: NULL argument");
  DG_REQUIRE(Hkv == 0 || (k && v), DG_EINVAL, "paged_append: NULL argument");
  DG_REQUIRE(freqs && freqs_rows >= 1 && freqs_ld >= 0, DG_EINVAL, "paged_append: freqs table required");
  static const dg_stride3 none = {0, 0, 0};
  const void* src[3] = {q, k, v};
  const dg_stride3* sst[3] = {H ? &args->q_st : &none, Hkv ? &args->k_st : &none, Hkv ? &args->v_st : &none};
  void* dst[3] = {args->q_out, rows->k, rows->v};
  const dg_stride3* dst_st[3] = {H ? &args->qo_st : &none, &rows->k_st, &rows->v_st};
  const int64_t es = dtype_bytes(dtype), fes = dtype_bytes((int)freqs_dtype);
  bool vec = D * es % 16 == 0 && aligned16(freqs) && freqs_ld * fes % 16 == 0;
  for (int w = 0; w < 3; ++w) {
    a.src[w] = src[w];
    a.sb[w] = sst[w]->b; a.st[w] = sst[w]->t;
    a.dst[w] = dst[w];
    a.db[w] = dst_st[w]->b; a.dt[w] = dst_st[w]->t;
    const bool one = (w == 0 ? H : Hkv) == 1;
    const int64_t sh = one ? 0 : sst[w]->h, dh = one ? 0 : dst_st[w]->h, far = ((int64_t)1 << 31) / es;
    DG_REQUIRE(sh > -far && sh < far && dh > -far && dh < far, DG_EINVAL, "paged_append: heads 2^31 bytes apart or more");
    a.sh[w] = (int)(sh * es);
    a.dh[w] = (int)(dh * es);
    vec = vec && aligned16(src[w]) && aligned16(dst[w]);
    for (int64_t x : {a.sb[w], a.st[w], sh, a.db[w], a.dt[w], dh}) vec = vec && x * es % 16 == 0;
  }
  a.freqs = freqs; a.freqs_ld = freqs_ld; a.freqs_rows = freqs_rows;
  a.table = rows->table; a.table_ld = rows->table_ld; a.pages = rows->pages;
  a.lens = rows->lens; a.counts = rows->counts; a.positions = args->positions;
  a.N = N; a.H = H; a.Hkv = Hkv; a.D = D;
  a.cap = (int)(rows->width * rows->page);
  a.qknorm = (args->flags & DG_QKNORM) ? 1 : 0;
  const int64_t tokens = (int64_t)B * N;
  DG_REQUIRE(tokens <= 0x7fffffff, DG_EINVAL, "paged_append: more than 2^24 - 1 workgroups");
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (dtype == DG_F64)
    return freqs_dtype == DG_F32 ? append_pick<double, float>(a, vec, tokens, s) : append_pick<double, double>(a, vec, tokens, s);
  if (dtype == DG_F32) return append_pick<float, float>(a, vec, tokens, s);
  if (dtype == DG_BF16)
    return freqs_dtype == DG_F32 ? append_pick<bf16_t, float>(a, vec, tokens, s) : append_pick<bf16_t, bf16_t>(a, vec, tokens, s);
  return freqs_dtype == DG_F32 ? append_pick<f16_t, float>(a, vec, tokens, s) : append_pick<f16_t, f16_t>(a, vec, tokens, s);
}

extern "C" int dg_paged_evict(const dg_paged_evict_args* args, void* stream) {
  DG_REQUIRE(args != nullptr, DG_EINVAL, "paged_evict: NULL argument");
  DG_REQUIRE(int_size(args->B) && int_size(args->Hkv) && args->Hkv >= 1, DG_EINVAL, "paged_evict: bad size");
  DG_REQUIRE(args->D >= 1 && args->D <= kMaxHeadDim, DG_EUNSUPPORTED, "paged_evict: head_dim %lld outside [1, %d]",
             (long long)args->D, kMaxHeadDim);
  DG_REQUIRE(known_dtype(args->dtype), DG_EUNSUPPORTED, "paged_evict: dtype %lld unsupported", (long long)args->dtype);
  DG_REQUIRE(args->keep >= 1 && args->keep <= kMostPositions && args->recent >= 0 && args->recent <= args->keep, DG_EINVAL,
             "paged_evict: keep %lld positions, %lld of them the last", (long long)args->keep, (long long)args->recent);
  const int B = (int)args->B, Hkv = (int)args->Hkv, D = (int)args->D, dtype = (int)args->dtype;
  const int keep = (int)args->keep, recent = (int)args->recent;
  const int64_t to_ld = args->to_ld, to_width = args->to_width;
  const dg_paged_rows* rows = &args->rows;
  const float* weights = args->weights;
  const int32_t* to = args->to;
  if (B == 0) return DG_OK;
  EvictArgs a{};
  if (const int rc = check_paged_rows("paged_evict", rows, true, &a.page_log2)) return rc;
  DG_REQUIRE(weights && to && args->new_lens && args->new_weights && args->kept, DG_EINVAL, "paged_evict: NULL argument");
  DG_REQUIRE(to_width >= 1 && to_width <= kMostPositions / rows->page && keep <= to_width * rows->page, DG_EINVAL,
             "paged_evict: %d positions into %lld pages of %lld", keep, (long long)to_width, (long long)rows->page);
  const int64_t es = dtype_bytes(dtype);
  a.weights = weights; a.wb = args->w_b; a.wh = args->w_h;
  a.table = rows->table; a.table_ld = rows->table_ld; a.pages = rows->pages;
  a.to = to; a.to_ld = to_ld; a.to_cap = to_width * rows->page;
  a.lens = rows->lens;
  a.new_lens = args->new_lens; a.new_weights = args->new_weights; a.kept = args->kept;
  a.k = static_cast<const char*>(rows->k); a.v = static_cast<const char*>(rows->v);
  a.kb = rows->k_st.b * es; a.kt = rows->k_st.t * es; a.kh = rows->k_st.h * es;
  a.vb = rows->v_st.b * es; a.vt = rows->v_st.t * es; a.vh = rows->v_st.h * es;
  a.Hkv = Hkv; a.cap = (int)(rows->width * rows->page); a.keep = keep; a.recent = recent;
  // the widest accesses that rows, heads and pages allow
  int64_t unit = 16;
  for (int64_t x : {(int64_t)reinterpret_cast<uintptr_t>(a.k), (int64_t)reinterpret_cast<uintptr_t>(a.v), a.kb, a.kt, a.kh, a.vb,
                    a.vt, a.vh, D * es})
    while (x % unit != 0) unit >>= 1;
  DG_REQUIRE(unit >= es, DG_EINVAL, "paged_evict: pages not aligned to their element size");
  a.pieces = (int)(D * es / unit);
  DG_REQUIRE((int64_t)B * Hkv <= 0xffffffffll / 1024, DG_EINVAL, "paged_evict: more than 2^32 - 1 threads");
  a.items = (int64_t)B * Hkv * a.to_cap * a.pieces;
  const int64_t blocks = (a.items + 255) / 256;
  DG_REQUIRE(blocks <= kMostWorkgroups256, DG_EINVAL, "paged_evict: more than 2^32 - 1 threads");
  hipStream_t s = static_cast<hipStream_t>(stream);
  const dim3 heads((unsigned)(B * Hkv));
  // weights in registers as far as they fit, few by few waves; us so / read anew, rows x positions:
  // 128 x 200 7.7 / 8.2, 64 x 2000 10.6 / 9.6, 64 x 8000 16.3 / 18.7, 64 x 16000 22.9 / 28.2,
  // 256 x 60000 133 / 173 (this launch and a small move)
  if (a.cap <= 2048) hipLaunchKernelGGL((paged_select_kernel<256, 8>), heads, dim3(256), 0, s, a);
  else if (a.cap <= 16384) hipLaunchKernelGGL((paged_select_kernel<1024, 16>), heads, dim3(1024), 0, s, a);
  else if (a.cap <= 65536) hipLaunchKernelGGL((paged_select_kernel<1024, 64>), heads, dim3(1024), 0, s, a);
  else hipLaunchKernelGGL((paged_select_kernel<1024, 0>), heads, dim3(1024), 0, s, a);
  if (const int rc = check_launch("paged_select_kernel")) return rc;
  const dim3 grid((unsigned)blocks);
  if (unit == 16) hipLaunchKernelGGL(paged_move_kernel<u32x4_t>, grid, dim3(256), 0, s, a);
  else if (unit == 8) hipLaunchKernelGGL(paged_move_kernel<u32x2_t>, grid, dim3(256), 0, s, a);
  else if (unit == 4) hipLaunchKernelGGL(paged_move_kernel<uint32_t>, grid, dim3(256), 0, s, a);
  else hipLaunchKernelGGL(paged_move_kernel<uint16_t>, grid, dim3(256), 0, s, a);
  return check_launch("paged_move_kernel");
}
