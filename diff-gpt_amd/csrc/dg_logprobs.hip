// Log probabilities of given tokens, entropy and the most likely alternatives
// (dg_token_logprobs), reading the logits once.
//
// With m the row's maximum, s the sum of e^(x - m) and t that of (x - m) e^(x - m):
// log p(id) = x[id] - m - log s, and the entropy is log s - t / s.
//
//   V <= 256, up to 16 alternatives (lp_small_kernel): 16 lanes a row, its logits in
//     registers.  Each lane sorts its 16 as (value, inverted id) integers and the lanes'
//     lists meet in four bitonic merges over DPP: no round per alternative.
//   longer rows (lp_row_kernel): 64 to 1024 threads a row, its logits in registers up to
//     32768, in 16-bit types 65536; beyond, each 16 bytes' maximum in registers up to 262144
//     and 524288, so that only those which hold candidates are read again.  The row's k-th
//     largest logit is at least the k-th largest of 64 maxima over disjoint parts of it,
//     which a bit-by-bit selection finds; the few logits from that bound on (about 64 (1/64 +
//     1/63 + ...), k terms: k + k^2 / 128 for small k, 300 for 64) go to LDS and are ranked
//     there by counting.  Where they overflow the buffer (256 logits for a row of one wave,
//     which half the rows do at 64 alternatives), the k-th largest of those it holds is the
//     next bound, and the row is looked through again (4096 x 4096 fp32 with 64 alternatives
//     66 us; one alternative after the other 2012).  Ties in number beyond the buffer are
//     taken in id order from the row; what neither takes (NaN among the first k, long
//     staircases of ties) goes one alternative after the other.
//   fp64: a wavefront a row, one pass per alternative.
//
// Bound by the vector ALU next to HBM: a logit takes some 10 operations (two unpackings,
// maximum, difference, exp2 at a quarter of the rate, two sums).  35328 x 256 bf16 with 8
// alternatives 13.2 us (26 MB: 5 us of HBM; sorting is half the operations), 2048 x 49999
// bf16 with 20 64 us (205 MB, 3.2 TB/s), 35000 x 1024 fp32 57 us (2.5 TB/s), 500 x 131072
// fp32 53 us (262 MB, 4.9 TB/s).
#include "dg_common.h"

namespace dg {

struct LogprobArgs {
  const void* x;
  int64_t ld, M, V;
  const int64_t* ids;
  void* logprob;
  void* entropy;
  int top;
  void* top_logprob;
  int64_t* top_ids;
};

// 16 bytes at any element's address: rows of an odd vocabulary start anywhere, and which
// thread holds a logit must not depend on where (the sums' order, so a row's bits, would)
typedef unsigned int u32x4_any_t __attribute__((ext_vector_type(4), aligned(2)));
__device__ __forceinline__ u32x4_t load16(const void* p) { return *reinterpret_cast<const u32x4_any_t*>(p); }

constexpr float kLog2e = 1.44269504088896340736f;

// (value descending, id ascending, NaN last) order of two logits
template <typename A>
__device__ __forceinline__ bool comes_before(A v1, int64_t i1, A v2, int64_t i2) {
  if (v1 != v1) return v2 != v2 && i1 < i2;
  return v2 != v2 || v1 > v2 || (v1 == v2 && i1 < i2);
}

// One logit's part of s and t.  A logit of -inf (or one so far below m that the
// difference overflows) adds 0 to both; NaN, and m = +-inf, make s NaN.
__device__ __forceinline__ void add_logit(float x, float m, float& s, float& t) {
  const float z = x - m;
  const float e = __builtin_amdgcn_exp2f(z * kLog2e);
  s += e;
  t = __builtin_fmaf(fmaxf(z, -1e30f), e, t);
}

// The given token's logit; NaN for an id outside the row.
template <typename T>
__device__ __forceinline__ float given_logit(const LogprobArgs& a, const T* x, int64_t id) {
  return id < 0 || id >= a.V ? __builtin_nanf("") : to_f32(x[id]);
}

// log p(id) and the entropy of a row, by one lane
__device__ __forceinline__ void store_row_stats(const LogprobArgs& a, int64_t row, float given, float m, float logs, float s,
                                                float t) {
  static_cast<float*>(a.logprob)[row] = given - m - logs;
  if (a.entropy != nullptr) static_cast<float*>(a.entropy)[row] = logs - t / s;
}

// ---------------------------------------------------------------------------
// V <= 256: 16 lanes a row
// ---------------------------------------------------------------------------

// (value, id) as an integer that sorts by value, then by descending id: larger comes first.
// 0 is no logit at all; NaN ranks below -inf.
template <typename T>
struct LpKey {
  using type = uint32_t;  // 16 bits of value, 16 of id
  static __device__ __forceinline__ uint32_t make(T v, int id) {
    const float f = to_f32(v) + 0.f;  // -0 ranks as 0
    uint32_t u;                       // the value's bits in the upper half
    if constexpr (__is_same(T, bf16_t)) u = __float_as_uint(f);
    else u = (uint32_t)from_f32<T>(f).bits << 16;
    u ^= (uint32_t)((int)u >> 31) | 0x80000000u;
    u = f != f ? 0u : u;
    return (u & 0xffff0000u) | (0xffffu - (uint32_t)id);
  }
  static __device__ __forceinline__ int id(uint32_t k) { return 0xffff - (int)(k & 0xffffu); }
  static __device__ __forceinline__ float value(uint32_t k) {
    const uint32_t u = k >> 16;
    T v;
    v.bits = (uint16_t)((u & 0x8000u) ? u & 0x7fffu : ~u);
    return to_f32(v);
  }
};
template <>
struct LpKey<float> {
  using type = uint64_t;
  static __device__ __forceinline__ uint64_t make(float v, int id) {
    const uint32_t b = __float_as_uint(v + 0.f);
    const uint32_t u = (b & 0x80000000u) ? ~b : b | 0x80000000u;
    return ((uint64_t)(v != v ? 0u : u) << 32) | (0xffffffffu - (uint32_t)id);
  }
  static __device__ __forceinline__ int id(uint64_t k) { return (int)(0xffffffffu - (uint32_t)k); }
  static __device__ __forceinline__ float value(uint64_t k) {
    const uint32_t u = (uint32_t)(k >> 32);
    return __uint_as_float((u & 0x80000000u) ? u & 0x7fffffffu : ~u);
  }
};

template <int CTRL>
__device__ __forceinline__ uint32_t dpp_key(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xF, 0xF, true);  // every lane has a partner
}
template <int CTRL>
__device__ __forceinline__ uint64_t dpp_key(uint64_t v) {
  return (uint64_t)dpp_key<CTRL>((uint32_t)v) | ((uint64_t)dpp_key<CTRL>((uint32_t)(v >> 32)) << 32);
}

__device__ __forceinline__ void order_keys(uint32_t& hi, uint32_t& lo) {
  const uint32_t h = max(hi, lo), l = min(hi, lo);
  hi = h;
  lo = l;
}
__device__ __forceinline__ void order_keys(uint64_t& hi, uint64_t& lo) {
  const bool swap = lo > hi;
  const uint64_t h = swap ? lo : hi, l = swap ? hi : lo;
  hi = h;
  lo = l;
}

// Batcher's odd-even merge sort, descending
template <int N, typename K>
__device__ __forceinline__ void sort_keys(K* v) {
#pragma unroll
  for (int p = 1; p < N; p *= 2)
#pragma unroll
    for (int k = p; k >= 1; k /= 2)
#pragma unroll
      for (int j = k % p; j + k < N; j += 2 * k)
#pragma unroll
        for (int i = 0; i < k; ++i)
          if (i + j + k < N && (i + j) / (2 * p) == (i + j + k) / (2 * p)) order_keys(v[i + j], v[i + j + k]);
}
// a bitonic sequence, descending
template <int N, typename K>
__device__ __forceinline__ void sort_bitonic(K* v) {
#pragma unroll
  for (int w = N / 2; w >= 1; w /= 2)
#pragma unroll
    for (int i = 0; i < N; ++i)
      if ((i & w) == 0) order_keys(v[i], v[i + w]);
}
// the N first of two sorted lists of N, the other one the partner lane's
template <int N, int CTRL, typename K>
__device__ __forceinline__ void merge_lists(K* v) {
  K m[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const K other = dpp_key<CTRL>(v[N - 1 - i]);
    m[i] = v[i] > other ? v[i] : other;
  }
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = m[i];
  sort_bitonic<N>(v);
}

// maximum over 16 consecutive lanes
__device__ __forceinline__ float max16(float v) {
  v = fmaxf(v, dpp<kDppQuadXor1>(v));
  v = fmaxf(v, dpp<kDppQuadXor2>(v));
  v = fmaxf(v, dpp<kDppHalfMirror>(v));
  return fmaxf(v, dpp<kDppMirror>(v));
}

// KP: the length of the lists, 0 where no alternatives are asked for.  VEC: rows of whole
// 16-byte vectors.
template <typename T, int KP, bool VEC>
__global__ __launch_bounds__(256) void lp_small_kernel(const LogprobArgs a) {
  using Key = LpKey<T>;
  using K = typename Key::type;
  constexpr int VE = VEC ? 16 / (int)sizeof(T) : 1;  // logits of a load
  constexpr int NV = 16 / VE;
  const int lane = threadIdx.x & 15;
  const int64_t r0 = (int64_t)blockIdx.x * 16 + (threadIdx.x >> 4);
  const int64_t row = r0 < a.M ? r0 : a.M - 1;  // rows past the last repeat it, unstored
  const T* x = static_cast<const T*>(a.x) + row * a.ld;
  const int V = (int)a.V;
  T v[16];
#pragma unroll
  for (int c = 0; c < NV; ++c) {
    const int i0 = (16 * c + lane) * VE;
    if constexpr (VEC) {
      u32x4_t w = {0u, 0u, 0u, 0u};
      if (i0 < V) w = load16(x + i0);
      __builtin_memcpy(&v[c * VE], &w, 16);
    } else {
      v[c] = i0 < V ? x[i0] : T{};
    }
  }
  float m = kNegInf;
#pragma unroll
  for (int i = 0; i < 16; ++i)
    if ((16 * (i / VE) + lane) * VE < V) m = fmaxf(m, to_f32(v[i]));
  m = max16(m);
  float s = 0.f, t = 0.f;
#pragma unroll
  for (int i = 0; i < 16; ++i)
    if ((16 * (i / VE) + lane) * VE < V) add_logit(to_f32(v[i]), m, s, t);
  s = group_sum_dpp<16>(s);
  t = group_sum_dpp<16>(t);
  const float logs = logf(s);
  if (lane == 0 && r0 < a.M) store_row_stats(a, row, given_logit(a, x, a.ids[row]), m, logs, s, t);
  if constexpr (KP > 0) {
    K k[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int id = (16 * (i / VE) + lane) * VE + i % VE;
      k[i] = id < V ? Key::make(v[i], id) : (K)0;
    }
    if constexpr (KP == 8) {
      sort_keys<8>(k);
      sort_keys<8>(k + 8);
      K f[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) f[i] = k[i] > k[15 - i] ? k[i] : k[15 - i];
#pragma unroll
      for (int i = 0; i < 8; ++i) k[i] = f[i];
      sort_bitonic<8>(k);
    } else {
      sort_keys<16>(k);
    }
    merge_lists<KP, kDppQuadXor1>(k);
    merge_lists<KP, kDppQuadXor2>(k);
    merge_lists<KP, kDppHalfMirror>(k);
    merge_lists<KP, kDppMirror>(k);
    K mine = k[0];
#pragma unroll
    for (int i = 1; i < KP; ++i) mine = lane == i ? k[i] : mine;
    if (lane < a.top && r0 < a.M) {
      a.top_ids[row * a.top + lane] = Key::id(mine);
      static_cast<float*>(a.top_logprob)[row * a.top + lane] = Key::value(mine) - m - logs;
    }
  }
}

// ---------------------------------------------------------------------------
// 64 to 1024 threads a row
// ---------------------------------------------------------------------------

// Integers that sort as the values of T do, 16-bit ones in the upper half, and back.
template <typename T>
__device__ __forceinline__ uint32_t sort_bits(float v) {
  uint32_t u;
  if constexpr (sizeof(T) == 4) u = __float_as_uint(v);
  else u = (uint32_t)from_f32<T>(v).bits << 16;  // v is a value of T
  return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}
template <typename T>
__device__ __forceinline__ float from_sort_bits(uint32_t u) {
  const uint32_t bits = (u & 0x80000000u) ? u & 0x7fffffffu : ~u;
  if constexpr (sizeof(T) == 4) {
    return __uint_as_float(bits);
  } else {
    T r;
    r.bits = (uint16_t)(bits >> 16);
    return to_f32(r);
  }
}

// The k-th largest (k from 1) of the wave's 64 values, NaN-free: bit by bit.
template <typename T>
__device__ __forceinline__ float kth_largest(float v, int k) {
  constexpr int BITS = 8 * (int)sizeof(T);
  const uint32_t u = sort_bits<T>(v);
  uint64_t alive = ~0ull;
  uint32_t kth = 0;
#pragma unroll
  for (int b = 31; b >= 32 - BITS; --b) {
    const uint64_t ones = __builtin_amdgcn_ballot_w64((u >> b) & 1u) & alive;
    const int n = __builtin_popcountll(ones);
    if (n >= k) {
      alive = ones;
      kth |= 1u << b;
    } else {
      k -= n;
      alive &= ~ones;
    }
  }
  return from_sort_bits<T>(kth);
}

// The k-th largest of n values in LDS, NaN-free, the same way: the largest number that k
// of them reach.
template <typename T>
__device__ __forceinline__ float kth_largest_of(const float* v, int n, int k, int lane) {
  uint32_t kth = 0;
#pragma unroll 1
  for (int b = 31; b >= 32 - 8 * (int)sizeof(T); --b) {
    const uint32_t trial = kth | (1u << b);
    int reach = 0;
#pragma unroll 4
    for (int c = 0; c < n; c += 64)
      reach += __builtin_popcountll(__builtin_amdgcn_ballot_w64(c + lane < n && sort_bits<T>(v[min(c + lane, n - 1)]) >= trial));
    if (reach >= k) kth = trial;
  }
  return from_sort_bits<T>(kth);
}

// A row's logits as its threads hold (HELD) or read them: its 16-byte vectors, the thread's j-th one
// vector j * NT + tid, and at most one of the logits behind them.  Where a thread has
// none it holds -inf and an id of V or more.
template <typename T, int NT, int NV, bool HELD>
struct LpRow {
  static constexpr int VE = 16 / (int)sizeof(T);
  static constexpr uint32_t kNone = sizeof(T) == 4 ? 0xff800000u : __is_same(T, bf16_t) ? 0xff80ff80u : 0xfc00fc00u;
  const T* x;
  int V, nvec, tid;
  int extra;  // id of the single logit
  float single;
  u32x4_t raw[HELD ? NV : 1];

  T single_raw;

  __device__ __forceinline__ u32x4_t vector(int i) const {
    u32x4_t w = {kNone, kNone, kNone, kNone};
    if (i < nvec) w = load16(x + (int64_t)i * VE);
    return w;
  }
  // The loads, without a branch around any but where the row has no vector at all: those
  // of vectors behind the last re-read it.  `row` is the same for the wave.
  __device__ __forceinline__ void start(const T* row, int v, int t) {
    x = row;
    V = v;
    tid = t;
    nvec = V / VE;
    extra = tid < V - nvec * VE ? nvec * VE + tid : V;
    single_raw = x[min(extra, V - 1)];
    if constexpr (HELD) {
      int at = tid;
      asm volatile("" : "+v"(at));  // the offsets are worked out for each row, not kept
      if (NT > 64 || nvec > 0) {  // the larger workgroups' rows always have one
#pragma unroll
        for (int j = 0; j < NV; ++j)
          raw[j] = load16(reinterpret_cast<const char*>(x) + 16u * (uint32_t)min(j * NT + at, nvec - 1));
      }
    }
  }
  // they have arrived
  __device__ __forceinline__ void arrive() {
    single = extra < V ? to_f32(single_raw) : kNegInf;
    if constexpr (HELD) {
#pragma unroll
      for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) raw[j][e] = j * NT + tid < nvec ? raw[j][e] : kNone;
    }
  }
  // The words as they are, unpacked anew by each pass: kept unpacked they would take
  // twice the registers.
  __device__ __forceinline__ void forget_unpacked() {
    if constexpr (HELD) {
#pragma unroll
      for (int j = 0; j < NV; ++j) asm volatile("" : "+v"(raw[j]));
    }
  }
  // f(the logits of a vector, the first one's id, its number) over the thread's vectors,
  // the wave's lanes together
  template <typename F>
  __device__ __forceinline__ void vectors(F f) const {
    auto vec = [&](const u32x4_t& w, int i, int j) __attribute__((always_inline)) {
      T e[VE];
      __builtin_memcpy(e, &w, 16);
      float v[VE];
#pragma unroll
      for (int c = 0; c < VE; ++c) v[c] = to_f32(e[c]);
      int id = i * VE;
      asm volatile("" : "+v"(id));  // comparisons with ids are made where they are used, not kept
      f(v, id, j);
    };
    if constexpr (HELD) {
      const int wave0 = __builtin_amdgcn_readfirstlane(tid & ~63);
#pragma unroll
      for (int j = 0; j < NV; ++j)
        if (j * NT + wave0 < nvec) vec(raw[j], j * NT + tid, j);
    } else {
      for (int i = tid; (i & ~63) < nvec; i += NT) vec(vector(i), i, 0);
    }
  }
};

// LDS of a row's threads
template <int NW, int CAP>
struct LpShared {
  float part[NW][64];                 // the lanes' maxima
  float wmax[NW], sum[NW], tsum[NW];  // m, s and t of the waves' parts
  int count;                          // candidates
  float best_v[NW];                   // a round's first logit of each wave
  int best_i[NW];
  float cand_v[CAP];
  int cand_i[CAP];
};

// Threads of a row meet here, as far as LDS goes: loads of the next row stay in flight.
// One wave needs no barrier.
template <int NT>
__device__ __forceinline__ void lp_sync() {
  if constexpr (NT > 64) {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
  } else {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
  }
}

// Waves a SIMD that the registers must allow: two rows of 1024 threads on a CU, whose loads
// and arithmetic then overlap, as long as a thread's logits leave room (2048 x 49999 bf16:
// one row on a CU 95 us, one with the next one's loads in flight 87, two 68).
template <typename T, int NT, int NV, bool HELD>
constexpr int lp_row_waves() {
  return NT >= 512 && NV <= (HELD ? 8 : 32) ? 8 : 4;
}

// NT threads a row, which meet twice: when every wave's part of the softmax is known, and
// when the candidates are collected.  Workgroups of 256 threads at least (several rows
// where NT is 64).
template <typename T, int NT, int NV, bool HELD>
__global__ __launch_bounds__(NT < 256 ? 256 : NT, (lp_row_waves<T, NT, NV, HELD>())) void lp_row_kernel(const LogprobArgs a) {
  constexpr int NW = NT / 64, RPB = NT < 256 ? 256 / NT : 1, CAP = NT == 64 ? 256 : 1024;
  constexpr int kRounds = 8;  // times a bound is raised at most: each leaves some top / CAP of too many
  constexpr int VE = 16 / (int)sizeof(T);
  __shared__ LpShared<NW, CAP> sh_all[RPB];
  LpShared<NW, CAP>& sh = sh_all[RPB == 1 ? 0 : threadIdx.x / NT];
  const int tid = threadIdx.x % NT, lane = tid & 63;
  const int wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int64_t row = (int64_t)blockIdx.x * RPB + (RPB == 1 ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x / NT));
  if (row >= a.M) return;  // RPB > 1: whole waves, which share no barrier
  const T* x = static_cast<const T*>(a.x) + row * a.ld;
  const int top = a.top;
  const int64_t given_id = a.ids[row];
  LpRow<T, NT, NV, HELD> r;
  r.start(x, (int)a.V, tid);
  const float given = given_logit(a, x, given_id);
  if (tid == 0) sh.count = 0;
  r.arrive();

  auto vec_max = [](const float(&v)[VE]) __attribute__((always_inline)) {
    float x0 = v[0];
#pragma unroll
    for (int c = 1; c < VE; ++c) x0 = fmaxf(x0, v[c]);
    return x0;
  };
  auto about = [](float& s1, float& t1, float m1, float m2) __attribute__((always_inline)) {
    const float d = m1 - m2;  // <= 0; where it overflows, or the factor vanishes, nothing is left
    const float f = __builtin_amdgcn_exp2f(d * kLog2e);
    t1 = f == 0.f ? 0.f : f * __builtin_fmaf(d, s1, t1);
    s1 = f * s1;
  };
  constexpr bool ONCE = !HELD && NV > 1;
  constexpr float kLowest = -3.402823466e38f;
  float vmax[NV];  // each vector's maximum
#pragma unroll
  for (float& x0 : vmax) x0 = kNegInf;
  const float single_max = fmaxf(r.single, kNegInf);  // a NaN is no maximum
  float mine = single_max;
  // s and t of the thread's logits about its own maximum, then of the wave's about the wave's
  // (-inf alone: about the lowest number, which leaves s at 0)
  float own = fmaxf(mine, kLowest);
  float s = 0.f, t = 0.f;
  if constexpr (ONCE) {
    // kU vectors in flight, each one's logits about the maximum so far
    constexpr int kU = 4;
    const int wave0 = __builtin_amdgcn_readfirstlane(tid & ~63);
#pragma unroll
    for (int g = 0; g < NV / kU; ++g) {
      if (g * kU * NT + wave0 >= r.nvec) break;
      u32x4_t w[kU];
#pragma unroll
      for (int u = 0; u < kU; ++u) w[u] = load16(x + (int64_t)min((g * kU + u) * NT + tid, r.nvec - 1) * VE);
#pragma unroll
      for (int u = 0; u < kU; ++u) {
        const int j = g * kU + u;
        T e[VE];
        float v[VE];
        __builtin_memcpy(e, &w[u], 16);
#pragma unroll
        for (int c = 0; c < VE; ++c) v[c] = j * NT + tid < r.nvec ? to_f32(e[c]) : kNegInf;
        vmax[j] = vec_max(v);
        const float high = fmaxf(own, vmax[j]);
        about(s, t, own, high);
        own = high;
#pragma unroll
        for (int c = 0; c < VE; ++c) add_logit(v[c], own, s, t);
      }
    }
#pragma unroll
    for (const float x0 : vmax) mine = fmaxf(mine, x0);
    if (r.extra < r.V) add_logit(r.single, own, s, t);
  } else {
    r.vectors([&](const float(&v)[VE], int, int j) __attribute__((always_inline)) {
      const float x0 = vec_max(v);
      if constexpr (HELD) vmax[j] = x0;
      mine = fmaxf(mine, x0);
    });
    r.forget_unpacked();
    own = fmaxf(mine, kLowest);
    if (r.extra < r.V) add_logit(r.single, own, s, t);
    r.vectors([&](const float(&v)[VE], int, int) __attribute__((always_inline)) {
#pragma unroll
      for (int c = 0; c < VE; ++c) add_logit(v[c], own, s, t);
    });
    r.forget_unpacked();
  }
  float m = wave_max(own);
  about(s, t, own, m);
  s = group_sum_dpp<64>(s);
  t = group_sum_dpp<64>(t);
  float part = mine;
  if constexpr (NW > 1) {
    sh.part[wv][lane] = mine;
    if (lane == 0) {
      sh.wmax[wv] = m;
      sh.sum[wv] = s;
      sh.tsum[wv] = t;
    }
    lp_sync<NT>();
    // every wave joins the waves' parts, a lane each
    const int w = lane & (NW - 1);
    const float mw = sh.wmax[w];
    s = sh.sum[w];
    t = sh.tsum[w];
    m = wave_max(mw);
    about(s, t, mw, m);
    s = group_sum_dpp<NW>(s);
    t = group_sum_dpp<NW>(t);
    part = sh.part[0][lane];
#pragma unroll
    for (int v = 1; v < NW; ++v) part = fmaxf(part, sh.part[v][lane]);
  }
  const float logs = wave_max(part) == kNegInf ? __builtin_nanf("") : logf(s);
  if (tid == 0) store_row_stats(a, row, given, m, logs, s, t);
  if (top == 0) return;
  if constexpr (NW == 1) lp_sync<NT>();

  int64_t* ids = a.top_ids + row * top;
  float* lps = static_cast<float*>(a.top_logprob) + row * top;
  float bound = kth_largest<T>(part, top);
  // a logit that passes, into LDS as far as there is room; the wave's lanes together
  auto offer = [&](bool in, float v, int id) __attribute__((always_inline)) {
    const uint64_t b = __builtin_amdgcn_ballot_w64(in);
    if (b != 0) {
      int at = 0;
      if (lane == 0) at = atomicAdd(&sh.count, __builtin_popcountll(b));
      at = __builtin_amdgcn_readfirstlane(at);
      at += __builtin_amdgcn_mbcnt_hi((uint32_t)(b >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)b, 0));
      if (in && at < CAP) {
        sh.cand_v[at] = v;
        sh.cand_i[at] = id;
      }
    }
  };
  auto rank = [&](int n) __attribute__((always_inline)) {
    if constexpr (NW == 1) {
      // one wave compares many with each other for long (n^2 / 64 times): the first `top` of
      // them, and their ties, move to the front
      if (n > 128) {
        const float last = kth_largest_of<T>(sh.cand_v, n, top, lane);
        int kept = 0;
        for (int c = 0; c < n; c += 64) {
          const float v = sh.cand_v[min(c + lane, n - 1)];
          const int id = sh.cand_i[min(c + lane, n - 1)];
          const bool in = c + lane < n && v >= last;
          const uint64_t b = __builtin_amdgcn_ballot_w64(in);
          lp_sync<NT>();  // everyone has read its own
          if (in) {
            const int at = kept + __builtin_amdgcn_mbcnt_hi((uint32_t)(b >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)b, 0));
            sh.cand_v[at] = v;
            sh.cand_i[at] = id;
          }
          kept += __builtin_popcountll(b);
        }
        lp_sync<NT>();
        n = kept;
      }
    }
    for (int c = tid; c < n; c += NT) {
      const float v = sh.cand_v[c];
      const int id = sh.cand_i[c];
      int before = 0;
      for (int o = 0; o < n; ++o) before += comes_before(sh.cand_v[o], sh.cand_i[o], v, id) ? 1 : 0;
      if (before < top) {
        ids[before] = id;
        lps[before] = v - m - logs;
      }
    }
  };
  if (__builtin_amdgcn_ballot_w64(single_max >= bound) != 0) offer(r.single >= bound && r.extra < r.V, r.single, r.extra);
  if constexpr (ONCE) {
    // the few vectors that hold one are read again
    uint64_t holds = 0;
#pragma unroll
    for (int j = 0; j < NV; ++j) holds |= (uint64_t)(__builtin_amdgcn_ballot_w64(vmax[j] >= bound) != 0) << j;
    for (; holds != 0; holds &= holds - 1) {
      const int i = __builtin_ctzll(holds) * NT + tid;
      const u32x4_t w = r.vector(i);
      T e[VE];
      __builtin_memcpy(e, &w, 16);
#pragma unroll
      for (int c = 0; c < VE; ++c) offer(to_f32(e[c]) >= bound && i < r.nvec, to_f32(e[c]), i * VE + c);
    }
  } else {
    r.vectors([&](const float(&v)[VE], int id, int j) __attribute__((always_inline)) {
      float most;
      if constexpr (HELD) most = vmax[j];
      else most = vec_max(v);
      if (__builtin_amdgcn_ballot_w64(most >= bound) == 0) return;  // the lanes' vectors hold none
#pragma unroll
      for (int c = 0; c < VE; ++c) offer(v[c] >= bound && id < r.V, v[c], id + c);
    });
  }
  lp_sync<NT>();
  int n = sh.count;
  if (n >= top && n <= CAP) {
    rank(n);
    return;
  }
  // From here on the row is read from memory again.  Too many: those at hand give a higher
  // bound; where they are ties with the one before, those above it are taken, and of those
  // equal to it the first in id order.
  const bool enough = n >= top;
  for (int round = 0;; ++round) {
    const float higher = enough && round < kRounds ? kth_largest_of<T>(sh.cand_v, CAP, top, lane) : bound;
    const bool ties = !(higher > bound);
    bound = higher;
    auto passes = [&](float v) __attribute__((always_inline)) { return ties ? v > bound : v >= bound; };
    lp_sync<NT>();  // everyone has read the count and the candidates
    if (tid == 0) sh.count = 0;
    lp_sync<NT>();
    if (__builtin_amdgcn_ballot_w64(passes(single_max)) != 0) offer(passes(r.single) && r.extra < r.V, r.single, r.extra);
#pragma unroll 1
    for (int i = tid; (i & ~63) < r.nvec; i += NT) {
      const u32x4_t w = r.vector(i);
      T e[VE];
      __builtin_memcpy(e, &w, 16);
#pragma unroll
      for (int c = 0; c < VE; ++c) offer(passes(to_f32(e[c])) && i < r.nvec, to_f32(e[c]), i * VE + c);
    }
    lp_sync<NT>();
    n = sh.count;
    if (ties || n <= CAP) break;
  }
  if (enough && n <= CAP) {
    rank(n);
    // after ties fewer than the first may have come; otherwise this finds none to add
    if (wv == 0) {
      int at = n;
      for (int v0 = 0; v0 < r.V && at < top; v0 += 64) {
        const bool in = v0 + lane < r.V && to_f32(x[min(v0 + lane, r.V - 1)]) == bound;
        const uint64_t b = __builtin_amdgcn_ballot_w64(in);
        const int mine = at + __builtin_amdgcn_mbcnt_hi((uint32_t)(b >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)b, 0));
        if (in && mine < top) {
          ids[mine] = v0 + lane;
          lps[mine] = bound - m - logs;
        }
        at += __builtin_popcountll(b);
      }
    }
    return;
  }
  // one alternative after the other
  float pv = 0.f;
  int pi = -1;
  for (int j = 0; j < top; ++j) {
    float bv = 0.f;
    int bi = r.V;
    auto take = [&](float v2, int i2, bool in) __attribute__((always_inline)) {
      in = in && i2 < r.V && (bi == r.V || comes_before(v2, i2, bv, bi));
      bv = in ? v2 : bv;
      bi = in ? i2 : bi;
    };
    for (int id = tid; id < r.V; id += NT) {
      const float v = to_f32(x[id]);
      take(v, id, pi < 0 || comes_before(pv, pi, v, id));
    }
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const float v2 = __shfl_xor(bv, o, 64);
      const int i2 = __shfl_xor(bi, o, 64);
      take(v2, i2, true);
    }
    if constexpr (NW > 1) {
      lp_sync<NT>();
      if (lane == 0) {
        sh.best_v[wv] = bv;
        sh.best_i[wv] = bi;
      }
      lp_sync<NT>();
#pragma unroll
      for (int w = 0; w < NW; ++w) take(sh.best_v[w], sh.best_i[w], true);
    }
    pv = bv;
    pi = bi;
    if (tid == 0) {
      ids[j] = bi;
      lps[j] = bv - m - logs;
    }
  }
}

// ---------------------------------------------------------------------------
// fp64: a wavefront a row
// ---------------------------------------------------------------------------

// m, s, t of a part of the row, joined with another part's
__device__ __forceinline__ void join_part(double& m, double& s, double& t, double m2, double s2, double t2) {
  const double ninf = -__builtin_huge_val();
  const double mn = m > m2 ? m : m2;
  if (mn == ninf) {  // neither holds a probability; a NaN stays in s
    s += s2;
    return;
  }
  // a part at -inf has s = 0 (or NaN) and no t; one whose factor vanishes, the difference
  // of two finite logits may overflow, adds nothing
  const double d1 = m - mn, d2 = m2 - mn;
  const double f1 = exp(d1), f2 = exp(d2);
  t = (f1 == 0 ? 0 : f1 * (t + d1 * s)) + (f2 == 0 ? 0 : f2 * (t2 + d2 * s2));
  s = (m == ninf ? s : f1 * s) + (m2 == ninf ? s2 : f2 * s2);
  m = mn;
}

__global__ __launch_bounds__(256) void lp_f64_kernel(const LogprobArgs a) {
  const double ninf = -__builtin_huge_val();
  const int lane = threadIdx.x & 63;
  const int64_t row = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (row >= a.M) return;
  const double* x = static_cast<const double*>(a.x) + row * a.ld;
  double m = ninf, s = 0, t = 0;
  for (int64_t v = lane; v < a.V; v += 64) {
    const double z = x[v];
    if (z == ninf) continue;
    if (z != z) {
      s = z;
      continue;
    }
    join_part(m, s, t, z, 1, 0);
  }
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const double m2 = __shfl_xor(m, o, 64), s2 = __shfl_xor(s, o, 64), t2 = __shfl_xor(t, o, 64);
    join_part(m, s, t, m2, s2, t2);
  }
  const double logs = m == ninf ? __builtin_nan("") : log(s);
  if (lane == 0) {
    const int64_t id = a.ids[row];
    static_cast<double*>(a.logprob)[row] = id < 0 || id >= a.V ? __builtin_nan("") : x[id] - m - logs;
    if (a.entropy != nullptr) static_cast<double*>(a.entropy)[row] = logs - t / s;
  }
  double pv = 0;
  int64_t pi = -1;
  for (int j = 0; j < a.top; ++j) {
    double bv = 0;
    int64_t bi = a.V;
    for (int64_t v = lane; v < a.V; v += 64) {
      const double z = x[v];
      if (pi >= 0 && !comes_before(pv, pi, z, v)) continue;
      if (bi == a.V || comes_before(z, v, bv, bi)) {
        bv = z;
        bi = v;
      }
    }
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const double v2 = __shfl_xor(bv, o, 64);
      const int64_t i2 = __shfl_xor((long long)bi, o, 64);
      if (i2 < a.V && (bi == a.V || comes_before(v2, i2, bv, bi))) {
        bv = v2;
        bi = i2;
      }
    }
    pv = bv;
    pi = bi;
    if (lane == 0) {
      a.top_ids[row * a.top + j] = bi;
      static_cast<double*>(a.top_logprob)[row * a.top + j] = bv - m - logs;
    }
  }
}

namespace {

// A launch has 2^32 - 1 threads at most.
bool rows_fit(int64_t M, int rows, int threads) { return (M + rows - 1) / rows <= 0xffffffffll / threads; }
#define DG_LP_MANY "token_logprobs: %lld rows are more than one launch takes"

template <typename T>
int launch_logprobs(const LogprobArgs& a, hipStream_t s) {
  constexpr int VE = 16 / (int)sizeof(T);
  const bool vec = a.V % VE == 0;
  if (a.V <= 256 && a.top <= 16) {
    DG_REQUIRE(rows_fit(a.M, 16, 256), DG_EINVAL, DG_LP_MANY, (long long)a.M);
    const dim3 grid((unsigned)((a.M + 15) / 16));
#define DG_LP(KP)                                                                                    \
  do {                                                                                               \
    if (vec) hipLaunchKernelGGL((lp_small_kernel<T, KP, true>), grid, dim3(256), 0, s, a);           \
    else hipLaunchKernelGGL((lp_small_kernel<T, KP, false>), grid, dim3(256), 0, s, a);              \
  } while (0)
    if (a.top == 0) DG_LP(0);
    else if (a.top <= 8) DG_LP(8);
    else DG_LP(16);
#undef DG_LP
    return check_launch("lp_small_kernel");
  }
  // The least threads that hold the row, 16 to 64 logits each.  More threads a row gain
  // little where rows are few (256 x 4000, 64 -> 1024 threads: 9.7 -> 8.2 us) and lose
  // elsewhere (512 x 2000: 8.6 -> 11.0).
#define DG_LP_ROW(NT, PER)                                                                                           \
  do {                                                                                                               \
    constexpr int kRows = (NT) < 256 ? 256 / (NT) : 1;                                                               \
    DG_REQUIRE(rows_fit(a.M, kRows, (NT) < 256 ? 256 : (NT)), DG_EINVAL, DG_LP_MANY, (long long)a.M);                \
    hipLaunchKernelGGL((lp_row_kernel<T, (NT), (PER) / VE, true>), dim3((unsigned)((a.M + kRows - 1) / kRows)),      \
                       dim3((NT) < 256 ? 256 : (NT)), 0, s, a);                                                      \
    return check_launch("lp_row_kernel_" #NT);                                                                       \
  } while (0)
  if (a.V <= 16 * 64) DG_LP_ROW(64, 16);
  if (a.V <= 32 * 64) DG_LP_ROW(64, 32);
  if (a.V <= 64 * 64) DG_LP_ROW(64, 64);
  if (a.V <= 32 * 256) DG_LP_ROW(256, 32);
  if (a.V <= 64 * 256) DG_LP_ROW(256, 64);
  if (a.V <= 64 * 512) DG_LP_ROW(512, 64);
  if constexpr (sizeof(T) == 2)
    if (a.V <= 64 * 1024) DG_LP_ROW(1024, 64);
#undef DG_LP_ROW
  // Longer rows are read once, as far as the vectors' maxima fit, and the vectors that hold
  // candidates again: fp32 from 32769 logits on, 16-bit types from 65537.  us held in 1024
  // threads' registers, or read three times, / read once: 500 x 65000 fp32 38 / 33, 500 x
  // 131072 bf16 47 / 37, fp32 112 / 53, 300 x 200000 fp32 107 / 44; 500 x 31000 fp32 21 / 23,
  // 2048 x 49999 bf16 66 / 80.
  DG_REQUIRE(rows_fit(a.M, 1, 1024), DG_EINVAL, DG_LP_MANY, (long long)a.M);
#define DG_LP_LONG(NV, NAME)                                                                                \
  do {                                                                                                      \
    hipLaunchKernelGGL((lp_row_kernel<T, 1024, (NV), false>), dim3((unsigned)a.M), dim3(1024), 0, s, a);    \
    return check_launch(NAME);                                                                              \
  } while (0)
  if (a.V / VE <= 32 * 1024) DG_LP_LONG(32, "lp_once_kernel");
  if (a.V / VE <= 64 * 1024) DG_LP_LONG(64, "lp_once_kernel");
  DG_LP_LONG(1, "lp_long_kernel");
#undef DG_LP_LONG
}

}  // namespace
}  // namespace dg

using namespace dg;

extern "C" int dg_token_logprobs(int64_t M, int64_t V, int dtype, const void* x, int64_t x_ld, const int64_t* ids,
                                 void* logprob, void* entropy, int top, void* top_logprob, int64_t* top_ids,
                                 void* stream) {
  DG_REQUIRE(M >= 0 && V >= 1, DG_EINVAL, "token_logprobs: %lld rows of %lld logits", (long long)M, (long long)V);
  DG_REQUIRE(dtype == DG_F32 || dtype == DG_BF16 || dtype == DG_F16 || dtype == DG_F64, DG_EUNSUPPORTED,
             "token_logprobs: dtype %d unsupported", dtype);
  DG_REQUIRE(top >= 0 && top <= 64 && top <= V, DG_EINVAL, "token_logprobs: top %d outside [0, min(V, 64)]", top);
  DG_REQUIRE(V <= 0x3fffffff && M <= 0x7fffffff, DG_EINVAL, "token_logprobs: too many logits or rows");
  if (M == 0) return DG_OK;
  DG_REQUIRE(x && ids && logprob && (top == 0 || (top_logprob && top_ids)), DG_EINVAL, "token_logprobs: NULL argument");
  const LogprobArgs a{x, x_ld, M, V, ids, logprob, entropy, top, top_logprob, top_ids};
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (dtype == DG_F64) {
    DG_REQUIRE(rows_fit(M, 4, 256), DG_EINVAL, DG_LP_MANY, (long long)M);
    hipLaunchKernelGGL(lp_f64_kernel, dim3((unsigned)((M + 3) / 4)), dim3(256), 0, s, a);
    return check_launch("lp_f64_kernel");
  }
  if (dtype == DG_F32) return launch_logprobs<float>(a, s);
  if (dtype == DG_BF16) return launch_logprobs<bf16_t>(a, s);
  return launch_logprobs<f16_t>(a, s);
}
