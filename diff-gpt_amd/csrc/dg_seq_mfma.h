// Packed attention, token trees over a cache and attention over a cache in pages on the matrix
// cores: bf16 and fp16 at head_dim up to 256, fp32 up to 128, rows of whole 16-byte pieces
// (dg_seq_tile.h has the kernel for every other shape).  D here is 16, 32, 64, 128 or 256: a head of fewer
// dims is computed as one of the next of these, its missing pieces zeros (16 x 512 tokens, 8 heads of
// 80: bf16 32 us, fp32 139; in seq_tile_kernel 385 and 340).
//
// A workgroup is WAVES wavefronts over one key head of one sequence: RT tiles of 32
// (query, head of the group) rows by KS = WAVES / RT groups of keys.  With few rows (RT 1:
// a decode step, a small tree) the waves split the keys and join their softmax states at
// the end; with many (RT 4: a prompt) they share each key tile.  Keys stream through two
// LDS stages per group, copied there straight from global memory (buffer_load_dwordx4 ...
// lds) while the stage before is computed: K and V rows with their 16-byte pieces
// XOR-swizzled.  Both products are transposed so that a lane's statistics belong to one row:
//
//   S^T (32 keys x 32 rows) = K Q^T     K from LDS, Q^T in registers for the whole loop
//   O^T (D x 32 rows)      += V^T P^T   P^T is S^T's accumulator registers as they are
//
// 16-bit data: v_mfma_f32_32x32x16_{bf16,f16}, V^T through the transposing LDS read;
// probabilities go into the second product as two terms of the data's type, 16 bits (bf16)
// and 20 (fp16) of them, so that an output is rounded once, as it is stored.  One term was
// 1.4 - 1.5 times as far from the exact result (bf16 2.3e-3 of it, now 1.6e-3), and faster:
// us, one term / two: 6 sequences of up to 7168 tokens, 16 heads on 4 of 128, bf16 490 / 652;
// 64 of 100 - 2048, 8 heads of 64, 192 / 237; 16 trees of 24 over up to 7168, 16 heads on 4 of
// 128, 43 / 51; one token for each of 64 caches of up to 4096 the same.
// fp32: v_mfma_f32_32x32x2_f32 throughout.  Lane l (half hh =
// l / 32) holds, in register r of a 32x32 block, row 8 (r / 4) + 4 hh + r % 4 of column
// l % 32, its row of the batch.
//
// The exponent's offset is a whole number of log2 units, raised only where the row's own
// maximum outgrows it by more than kLazyLog2 (an offset that followed the neighbours' would
// move the grid on which the exponents are rounded): rescaling by a power of two is exact,
// and a row's bits depend on no other row of its tile.  Scores are masked
// only in key blocks that some row of the wave sees part of; values there that are not
// finite are kept out of the product (clean_stage).
//
// Bound by the softmax's vector instructions beside the matrix cores' for prompts (38 cycles
// of a SIMD for 64 scores: fused product, exp2 at a quarter of the rate, sum, maximum, and
// three instructions for the two terms of a probability), by HBM for few rows.  bf16: 6 sequences of up to 7168
// tokens, 16 heads on 4 of 128, 660 us (720 TFLOP/s; vector ALU 56 % busy, matrix cores
// 58 %); 64 of 100 - 2048, 8 heads of 64, 221 us (500 TFLOP/s; 70 %, 39 %); one token for
// each of 64 caches of up to 4096, 16 heads on 4 of 128, 53 us (269 MB, 5.1 TB/s), in pages of
// 64 positions 56; 16 chunks of 256 - 512 tokens behind 1000 - 7168, in pages of 16, 370 (640
// TFLOP/s; 46 % and 46 %).
// Not kept: the K fragments of a block in flight together, two chains for the row sums, 168
// registers at head_dim 64, raised wave priority around the products (each within 2 %);
// outputs checked for values that are not finite at the end and the piece done again (5 %
// slower), the look at V shared between the waves (even).
#pragma once

#include "dg_prefill.h"
#include "dg_seq.h"

namespace dg {

typedef __attribute__((__vector_size__(8 * sizeof(__bf16)))) __bf16 sbf16x8_t;
typedef __attribute__((__vector_size__(8 * sizeof(_Float16)))) _Float16 sf16x8_t;
typedef unsigned short u16x2_t __attribute__((ext_vector_type(2)));

// Two probabilities as pairs of T, the leading bits and the rest.  The leading ones are cut
// off, not rounded, and the rest of one that is not 0 never vanishes (its last bit stays), so
// both are positive and a value of +-inf times either is +-inf, never 0 * inf.
struct ProbPairs {
  uint32_t high, low;
};

template <typename T>
struct SeqMma;
template <>
struct SeqMma<bf16_t> {
  using vec8 = sbf16x8_t;
  static constexpr uint32_t kExp = 0x7f80u;
  static constexpr float kLift = 0.f;
  __device__ static ProbPairs split(float a, float b) {
    constexpr float kPast = 1.0f + 0x1p-23f;
    const uint32_t ua = __float_as_uint(a), ub = __float_as_uint(b);
    const float la = __builtin_fmaf(a, kPast, -__uint_as_float(ua & 0xffff0000u));
    const float lb = __builtin_fmaf(b, kPast, -__uint_as_float(ub & 0xffff0000u));
    return {__builtin_amdgcn_perm(ub, ua, 0x07060302u), pack_pair<bf16_t>(la, lb)};
  }
  __device__ static floatx16_t mma(vec8 a, vec8 b, floatx16_t c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
};
template <>
struct SeqMma<f16_t> {
  using vec8 = sf16x8_t;
  static constexpr uint32_t kExp = 0x7c00u;
  // fp16's steps end at 2^-24, and a long row's faint keys count: weights are 2^7 times what
  // they are in the other types, from 2^7 (a row's largest) to 2^15 at most (kLazyLog2)
  static constexpr float kLift = 7.f;
  __device__ static ProbPairs split(float a, float b) {
    const uint32_t h = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(a, b));
    float la, lb;  // a, b less their halves of h, one instruction each
    asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel_hi:[1,0,0]" : "=v"(la) : "v"(h), "v"(a));
    asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "=v"(lb) : "v"(h), "v"(b));
    const u16x2_t l = __builtin_bit_cast(u16x2_t, __builtin_amdgcn_cvt_pkrtz(la, lb));
    uint32_t ones = 0x00010001u;
    asm("" : "+s"(ones));  // the minimum of unknown numbers: one v_pk_min_u16, no comparisons
    const u16x2_t some = __builtin_elementwise_min(__builtin_bit_cast(u16x2_t, h), __builtin_bit_cast(u16x2_t, ones));
    return {h, __builtin_bit_cast(uint32_t, __builtin_elementwise_max(l, some))};
  }
  __device__ static floatx16_t mma(vec8 a, vec8 b, floatx16_t c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
  }
};
template <>
struct SeqMma<float> {
  using vec8 = float;  // unused
  static constexpr uint32_t kExp = 0x7f800000u;
  static constexpr float kLift = 0.f;
};

// Workgroup shapes.  Two stages of K and V for every key group: up to 128 KB of LDS (one
// workgroup a CU, 64 KB of keys in flight) where the waves split the keys.
template <typename T, int D, int RT>
struct SeqCfg {
  static constexpr int ES = (int)sizeof(T);
  static constexpr int WAVES = (D * ES >= 512 && RT == 1) ? 2 : 4;
  static constexpr int KS = WAVES / RT;
  // 32-key blocks of a stage
  static constexpr int MB = RT == 4 ? (ES == 2 && D == 64 ? 2 : 1) : D * ES <= 64 ? 2 : 1;
  static constexpr int BN = 32 * MB;
  static constexpr int PPR = D * ES / 16;        // 16-byte pieces of a row
  static constexpr int RPD = 64 / PPR;           // rows a wave-wide copy covers
  static constexpr int NDMA = BN / RPD;          // copies of a K (or V) tile
  static constexpr int TILE = BN * D;            // elements
  static constexpr int NC = D / 16;              // 16-bit: contraction steps of S^T
  static constexpr int QC = D / 2;               // fp32: ... of two dims
  static constexpr int NB = D < 32 ? 1 : D / 32; // 32-row blocks of O^T (D = 16 fills half of one)
  static constexpr int JOIN = (NB * 16 + 2) * 64;  // floats of a wave's state
  static_assert(NDMA >= 1 && KS >= 1, "tile split");
  // the joined states and the outputs reuse the stages: writers alternate between the two
  static_assert((((KS - 1) * RT + 1) / 2) * JOIN * 4 <= KS * 2 * TILE * ES, "joined states fit a stage");
  static_assert(ES == 4 || ((RT + 1) / 2) * 32 * D <= KS * 2 * TILE, "outputs fit a stage");
  // workgroups a CU that the registers must allow (fp32 at head_dim 64, 64 x 512 tokens: four
  // spill, 215 us; three 180.  bf16 at 256, 16 x 512, 8 heads, one term of each probability: two
  // spill, 148; one 76)
  static constexpr int WGS = RT == 4 ? (ES == 4 ? (D <= 32 ? 4 : D == 64 ? 3 : 2) : D <= 64 ? 4 : D == 128 ? 3 : 1) : (D * ES <= 128 ? 2 : 1);
};

template <int PPR, int ES>
__device__ __forceinline__ int seq_swz(int r) {
  if constexpr (ES == 4) return r & (PPR >= 16 ? 15 : PPR - 1);
  else if constexpr (PPR == 8) return ((r & 2) << 1) | ((r >> 2) & 3);
  else if constexpr (PPR >= 16) return ((r & 3) << 2) | ((r >> 2) & 3);
  else if constexpr (PPR == 4) return (r >> 2) & 3;
  else return 0;
}

template <typename T, int D, int RT>
constexpr int seq_threads() {
  return 64 * SeqCfg<T, D, RT>::WAVES;
}
template <typename T, int D, int RT>
constexpr int seq_wgs_per_cu() {
  return SeqCfg<T, D, RT>::WGS;
}

// 16 bytes of zeros in device memory: what a copy reads in place of a position that is not there.
__device__ const u32x4_t kZeros16 = {0u, 0u, 0u, 0u};

template <typename T, int D, int RT, SeqMode MODE>
__global__ __launch_bounds__((seq_threads<T, D, RT>()), (seq_wgs_per_cu<T, D, RT>()))
void seq_mfma_kernel(const SeqArgs a) {
  using C = SeqCfg<T, D, RT>;
  using M = SeqMma<T>;
  using vec8 = typename M::vec8;
  constexpr int ES = C::ES, KS = C::KS, MB = C::MB, BN = C::BN, PPR = C::PPR, NB = C::NB, TILE = C::TILE;
  constexpr bool F32 = ES == 4, TREE = MODE == kTree, PAGED = MODE >= kPaged;
  constexpr float kNone = kNegInf;

  __shared__ __attribute__((aligned(16))) T kv0[KS * 2 * TILE];
  __shared__ __attribute__((aligned(16))) T kv1[KS * 2 * TILE];

  SeqPiece pc;
  if (!seq_piece<MODE>(a, pc)) return;  // whole workgroups, before any barrier
  const int lane = threadIdx.x & 63;
  const int wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int rt = wv % RT, kg = wv / RT;
  const int hh = lane >> 5, r32 = lane & 31;

  // the lane's row: rows past the piece's repeat its last one and are never stored
  const int wrow = pc.row0 + 32 * rt, rend = pc.row0 + pc.rows;
  const bool live = wrow < rend;
  const int row = min(wrow + r32, rend - 1);
  const int qi = row / a.G, qg = row - qi * a.G;
  const int head = pc.kvh * a.G + qg;
  // keys below `open` every row of the wave sees, from `wend` on none does; below
  // `first_open` every row of the workgroup
  int open, wend, first_open;
  uint64_t mask = 0;
  if constexpr (TREE) {
    open = first_open = pc.own;
    wend = pc.kend;
    mask = tree_mask(a, pc.b, qi);
  } else {
    first_open = pc.row0 / a.G + pc.off + 1;
    open = min(wrow, rend - 1) / a.G + pc.off + 1;
    wend = min(wrow + 31, rend - 1) / a.G + pc.off + 1;
  }
  if constexpr (PAGED) wend = min(wend, pc.kend);  // a split's keys may end before
  if (!live) wend = 0;

  const T* kp = static_cast<const T*>(a.k) + pc.b * a.kb + pc.k0 * a.kt + (int64_t)pc.kvh * a.kh;
  const T* vp = static_cast<const T*>(a.v) + pc.b * a.vb + pc.k0 * a.vt + (int64_t)pc.kvh * a.vh;

  // ---- global -> LDS copy of a stage's keys -----------------------------------------
  // The RT waves of a key group share its copies: lane l of copy i fills slot l % PPR of
  // row l / PPR of rows i * RPD ..  The buffer resource ends behind the piece's last key:
  // rows past it read as zeros.
  int ko[(C::NDMA + RT - 1) / RT], vo[(C::NDMA + RT - 1) / RT];
#pragma unroll
  for (int n = 0; n < (PAGED ? 0 : (C::NDMA + RT - 1) / RT); ++n) {
    const int r = (n * RT + rt) * C::RPD + lane / PPR;
    const int piece = (lane % PPR) ^ seq_swz<PPR, ES>(r);
    // pieces past the head: out of range of any resource, which makes them zeros
    const bool in = 16 * piece < a.D * ES;
    ko[n] = in ? r * (int)a.kt * ES + 16 * piece : (int)0x80000000u;
    vo[n] = in ? r * (int)a.vt * ES + 16 * piece : (int)0x80000000u;
  }
  // Where the piece's keys span less than 2^31 bytes, one resource serves all stages, the
  // stage's start in the scalar offset.
  const int64_t kstep_b = a.kt * ES, vstep_b = a.vt * ES;  // bytes from key to key
  const int nkeys = max(0, pc.kend - pc.kbeg);
  const int row_b = a.D * ES;
  const bool near = nkeys * max(kstep_b, vstep_b) + row_b < ((int64_t)1 << 31);
  const T* const kp0 = kp + (int64_t)pc.kbeg * a.kt;
  const T* const vp0 = vp + (int64_t)pc.kbeg * a.vt;
  const __amdgpu_buffer_rsrc_t krs0 = __builtin_amdgcn_make_buffer_rsrc(
      const_cast<T*>(kp0), 0, near && nkeys > 0 ? (int)((nkeys - 1) * kstep_b + row_b) : 0, kBufferWord3);
  const __amdgpu_buffer_rsrc_t vrs0 = __builtin_amdgcn_make_buffer_rsrc(
      const_cast<T*>(vp0), 0, near && nkeys > 0 ? (int)((nkeys - 1) * vstep_b + row_b) : 0, kBufferWord3);
  auto copy_from = [&](T* st, __amdgpu_buffer_rsrc_t krs, __amdgpu_buffer_rsrc_t vrs, int ks0, int vs0)
      __attribute__((always_inline)) {
    T* const ks = st + kg * 2 * TILE;
#pragma unroll
    for (int n = 0; n < (C::NDMA + RT - 1) / RT; ++n) {
      const int i = n * RT + rt;
      if (C::NDMA % RT != 0 && i >= C::NDMA) break;  // wave-uniform
      lds_copy16_buf(krs, ko[n], ks0, ks + i * C::RPD * D);
      lds_copy16_buf(vrs, vo[n], vs0, ks + TILE + i * C::RPD * D);
    }
  };
  // Paged: lane j holds the page of key j of the stage to be copied next, loaded a stage ahead
  // and not looked at before (a comparison beside the load would wait for it, and with it for
  // the stage's copies).
  int ids = -1;
  auto fetch_ids = [&](int k0) __attribute__((always_inline)) {
    ids = a.table[pc.b * a.table_ld + (min(k0 + lane, pc.kend - 1) >> a.page_log2)];
  };
  // kPaged: rows of GR keys, which a page holds whole, have one resource, that of nothing for a
  // page the pool lacks.  Rows past the piece's last key are copied too: hidden from all.
  // (us, an address for every lane / so: one token for each of 64 caches of up to 4096, 16 heads
  // on 4 of 128, bf16, pages of 64, 68 / 56; 16 of 256 - 512 behind 1000 - 7168, pages of 16, 511 / 473.)
  constexpr int GR = paged_granule(D, ES), NC1 = (C::NDMA + RT - 1) / RT;
  uint32_t page_b = 0, key_b = 0, npages = 0;
  const char *kbase = nullptr, *vbase = nullptr;
  if constexpr (MODE == kPaged) {
    page_b = (uint32_t)(a.kb * ES);
    key_b = (uint32_t)(a.kt * ES);
    npages = (uint32_t)a.pages;
    kbase = reinterpret_cast<const char*>(static_cast<const T*>(a.k) + (int64_t)pc.kvh * a.kh);
    vbase = reinterpret_cast<const char*>(static_cast<const T*>(a.v) + (int64_t)pc.kvh * a.vh);
#pragma unroll
    for (int n = 0; n < NC1; ++n) {
      const int r = (n * RT + rt) * C::RPD + lane / PPR;
      const int piece = (lane % PPR) ^ seq_swz<PPR, ES>(r);
      const int in_gr = RT == 1 ? r % GR : lane / PPR;
      ko[n] = 16 * piece < a.D * ES ? in_gr * (int)key_b + 16 * piece : (int)0x80000000u;
    }
  }
  auto copy_whole = [&](T* st, int k0) __attribute__((always_inline)) {
    T* const ks = st + kg * 2 * TILE;
    const int gr_b = (GR - 1) * (int)key_b + a.D * ES;
    __amdgpu_buffer_rsrc_t rk, rv;
#pragma unroll
    for (int n = 0; n < NC1; ++n) {
      const int i = n * RT + rt;
      if (C::NDMA % RT != 0 && i >= C::NDMA) break;  // wave-uniform
      if (RT > 1 || n * C::RPD % GR == 0) {
        const uint32_t id = (uint32_t)__builtin_amdgcn_readlane(ids, i * C::RPD);
        const uint32_t slot = (uint32_t)(k0 + i * C::RPD) & ((1u << a.page_log2) - 1);
        const uint64_t off = (uint64_t)min(id, npages - 1) * page_b + slot * key_b;
        const int bytes = id < npages ? gr_b : 0;
        rk = __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(kbase + off), 0, bytes, kBufferWord3);
        rv = __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(vbase + off), 0, bytes, kBufferWord3);
      }
      lds_copy16_buf(rk, ko[n], 0, ks + i * C::RPD * D);
      lds_copy16_buf(rv, ko[n], 0, ks + TILE + i * C::RPD * D);
    }
  };
  // kPagedAny: every lane has an address, that of kZeros16 for what is not there.
  auto copy_pages = [&](T* st, int k0) __attribute__((always_inline)) {
    T* const ks = st + kg * 2 * TILE;
    const T* const kh = static_cast<const T*>(a.k) + (int64_t)pc.kvh * a.kh;
    const T* const vh = static_cast<const T*>(a.v) + (int64_t)pc.kvh * a.vh;
#pragma unroll
    for (int n = 0; n < (C::NDMA + RT - 1) / RT; ++n) {
      const int i = n * RT + rt;
      if (C::NDMA % RT != 0 && i >= C::NDMA) break;  // wave-uniform
      const int r = i * C::RPD + lane / PPR;
      const int e = ((lane % PPR) ^ seq_swz<PPR, ES>(r)) * (16 / ES);
      const int id = __shfl(ids, r, 64);
      const int slot = (k0 + r) & ((1 << a.page_log2) - 1);
      const bool in = id >= 0 && id < a.pages && k0 + r < pc.kend && e < a.D;
      const void* const kz = in ? static_cast<const void*>(kh + id * a.kb + slot * a.kt + e) : &kZeros16;
      const void* const vz = in ? static_cast<const void*>(vh + id * a.vb + slot * a.vt + e) : &kZeros16;
      lds_copy16(kz, ks + i * C::RPD * D);
      lds_copy16(vz, ks + TILE + i * C::RPD * D);
    }
  };
  auto copy_stage = [&](T* st, int k0) __attribute__((always_inline)) {
    if constexpr (PAGED) {
      if constexpr (MODE == kPaged) copy_whole(st, k0);
      else copy_pages(st, k0);
      fetch_ids(k0 + KS * BN);
      return;
    }
    const int rel = k0 - pc.kbeg;
    if (near && rel < nkeys) {
      copy_from(st, krs0, vrs0, rel * (int)kstep_b, rel * (int)vstep_b);
    } else {  // far, or a group's stage behind the last key: zeros
      const int left = min(BN, nkeys - rel);
      const int kn = left <= 0 ? 0 : (int)((left - 1) * kstep_b) + row_b;
      const int vn = left <= 0 ? 0 : (int)((left - 1) * vstep_b) + row_b;
      copy_from(st, __builtin_amdgcn_make_buffer_rsrc(const_cast<T*>(kp0 + rel * a.kt), 0, kn, kBufferWord3),
                __builtin_amdgcn_make_buffer_rsrc(const_cast<T*>(vp0 + rel * a.vt), 0, vn, kBufferWord3), 0, 0);
    }
  };
  // this wave's copies have landed; the waves of a group also wait for each other
  auto stage_ready = [&]() __attribute__((always_inline)) {
    __builtin_amdgcn_s_waitcnt(0);
    if constexpr (RT > 1) __builtin_amdgcn_s_barrier();
  };

  // ---- the rows ----------------------------------------------------------------------
  const T* qp = static_cast<const T*>(a.q) + pc.b * a.qb + (pc.q0 + qi) * a.qt + (int64_t)head * a.qh;
  vec8 qf[F32 ? C::QC : C::NC];
  if constexpr (F32) {
#pragma unroll
    for (int m = 0; m < C::QC / 4; ++m) {
      const int d = C::QC * hh + 4 * m;
      const f32x4_t x = *reinterpret_cast<const f32x4_t*>(qp + min(d, a.D - 4));
#pragma unroll
      for (int e = 0; e < 4; ++e) qf[4 * m + e] = d < a.D ? x[e] : 0.f;
    }
  } else {
#pragma unroll
    for (int c = 0; c < C::NC; ++c) {
      const int d = 16 * c + 8 * hh;
      const u32x4_t x = *reinterpret_cast<const u32x4_t*>(qp + min(d, a.D - 8));
      qf[c] = __builtin_bit_cast(vec8, d < a.D ? x : u32x4_t{0u, 0u, 0u, 0u});
    }
  }

  const int kstep = KS * BN;
  const int kfirst = pc.kbeg + kg * BN;  // this group's first stage
  const int nstage = (pc.kend - pc.kbeg + kstep - 1) / kstep;
  if constexpr (PAGED) {
    if (nstage > 0) fetch_ids(kfirst);  // pc.kend is 1 at least
  }
  if (nstage > 0) copy_stage(kv0, kfirst);

  floatx16_t o[NB];
#pragma unroll
  for (int nb = 0; nb < NB; ++nb)
#pragma unroll
    for (int r = 0; r < 16; ++r) o[nb][r] = 0.f;
  // the exponent's offset (log2 units, whole) and this lane's sum, whose last addition's
  // rounding is lc
  float mo = kNone, l = 0.f, lc = 0.f;

  // per-lane parts of the transposing reads of V (16-bit)
  const int g16 = lane >> 4, t16 = lane & 15;
  int voff[2][NB];
  if constexpr (!F32) {
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int r = 8 * u + 4 * (g16 >> 1) + (t16 >> 2);
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
        const int col = (32 * nb + 16 * (g16 & 1) + 4 * (t16 & 3)) & (D - 1);  // D = 16: both halves read its dims
        voff[u][nb] = r * D + 8 * ((col >> 3) ^ seq_swz<PPR, ES>(r)) + (col & 7);
      }
    }
  }
  const int kswz = seq_swz<PPR, ES>(r32);

  // which of the 32 keys from kb on this lane's row sees
  auto visible = [&](int kb) __attribute__((always_inline)) -> uint32_t {
    if constexpr (TREE) {
      const int d = pc.own - kb;
      if (d >= 32) return ~0u;
      if (d >= 0) return (uint32_t)(((uint64_t)mask << d) | ((1ull << d) - 1));
      return -d >= 64 ? 0u : (uint32_t)(mask >> -d);
    } else {
      const int lim = qi + pc.off - kb;
      return lim < 0 ? 0u : lim >= 31 ? ~0u : (2u << lim) - 1;
    }
  };
  // A value that is not finite, in a key block that some row sees only part of, would reach
  // the others as 0 * inf.  Where a stage that crosses `first_open` holds one, it is added
  // to the outputs of the rows that see its key, and leaves the tile.  Rare, and out of the
  // products' way; the waves that share tiles take the same path.
  auto not_finite = [](uint32_t bits) __attribute__((always_inline)) { return (bits & M::kExp) == M::kExp; };
  auto finite_tile = [&](const T* vs) __attribute__((always_inline)) -> bool {
    const u32x4_t* p = reinterpret_cast<const u32x4_t*>(vs);
    bool fine = true;
    if constexpr (F32) {
      uint32_t top = 0;
#pragma unroll 4
      for (int i = 0; i < TILE * ES / 1024; ++i) {
        const u32x4_t w = p[64 * i + lane];
#pragma unroll
        for (int e = 0; e < 4; ++e) top = max(top, w[e] & 0x7fffffffu);
      }
      fine = top < M::kExp;
    } else {
      u16x2_t top = {0, 0};
#pragma unroll 4
      for (int i = 0; i < TILE * ES / 1024; ++i) {
        const u32x4_t w = p[64 * i + lane];
#pragma unroll
        for (int e = 0; e < 4; ++e)
          top = __builtin_elementwise_max(top, __builtin_bit_cast(u16x2_t, w[e] & 0x7fff7fffu));
      }
      fine = top[0] < M::kExp && top[1] < M::kExp;
    }
    return __builtin_amdgcn_ballot_w64(!fine) == 0;
  };
  auto clean_stage = [&](T* st, int t) __attribute__((always_inline)) {
    const int s0 = pc.kbeg + t * kstep;
    if (s0 + kstep <= first_open) return;
    bool fine = true;
    if constexpr (RT == 1) {
      fine = finite_tile(st + kg * 2 * TILE + TILE);
    } else {
#pragma unroll
      for (int g = 0; g < KS; ++g) fine = finite_tile(st + g * 2 * TILE + TILE) && fine;
    }
    if (fine) return;
    T* const vs = st + kg * 2 * TILE + TILE;
#pragma unroll 1
    for (int j = 0; j < BN; ++j) {
      bool sees = (visible(s0 + kg * BN + (j & ~31)) >> (j & 31)) & 1u;
      // a paged split's last stage may go past its keys, into the next one's: not its own
      if constexpr (PAGED) sees = sees && s0 + kg * BN + j < pc.kend;
      const int ksw = seq_swz<PPR, ES>(j);
#pragma unroll
      for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int r = 0; r < (D == 16 ? 8 : 16); ++r) {
          constexpr int EPP = 16 / ES;
          const int i = 8 * (r >> 2) + 4 * hh + (r & 3);
          const int d = F32 ? NB * i + nb : 32 * nb + i;
          const float x = to_f32(vs[j * D + EPP * ((d / EPP) ^ ksw) + d % EPP]);
          if (sees && !(__builtin_fabsf(x) < __builtin_huge_valf())) o[nb][r] += x;
        }
    }
    if constexpr (RT > 1) __syncthreads();  // everyone has added
    u32x4_t* const p = reinterpret_cast<u32x4_t*>(vs);
#pragma unroll 1
    for (int i = 0; i < TILE * ES / 1024; ++i) {
      u32x4_t w = p[64 * i + lane];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if constexpr (F32) {
          if (not_finite(w[e])) w[e] = 0u;
        } else {
          if (not_finite(w[e])) w[e] &= 0xffff0000u;
          if (not_finite(w[e] >> 16)) w[e] &= 0x0000ffffu;
        }
      }
      p[64 * i + lane] = w;
    }
    if constexpr (RT > 1) {
      __syncthreads();
    } else {
      __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
      __builtin_amdgcn_wave_barrier();
      __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    }
  };

  auto compute = [&](const T* st, int k0) __attribute__((always_inline)) {
    const T* Ks = st + kg * 2 * TILE;
    const T* Vs = Ks + TILE;
    floatx16_t s[MB];
    // a block past the wave's last key has zeros for K: no product, no weight
#pragma unroll
    for (int mb = 0; mb < MB; ++mb) {
#pragma unroll
      for (int r = 0; r < 16; ++r) s[mb][r] = 0.f;
      if constexpr (F32) {
        const float* krow = reinterpret_cast<const float*>(Ks) + (32 * mb + r32) * D;
#pragma unroll
        for (int p = 0; p < C::QC / 4; ++p) {
          const f32x4_t kf = *reinterpret_cast<const f32x4_t*>(krow + 4 * (((PPR / 2) * hh + p) ^ kswz));
#pragma unroll
          for (int e = 0; e < 4; ++e)
            s[mb] = __builtin_amdgcn_mfma_f32_32x32x2f32(kf[e], qf[4 * p + e], s[mb], 0, 0, 0);
        }
      } else {
#pragma unroll
        for (int c = 0; c < C::NC; ++c) {
          const u32x4_t kf = *reinterpret_cast<const u32x4_t*>(Ks + (32 * mb + r32) * D + 8 * ((2 * c + hh) ^ kswz));
          s[mb] = M::mma(__builtin_bit_cast(vec8, kf), qf[c], s[mb]);
        }
      }
    }
#pragma unroll
    for (int mb = 0; mb < MB; ++mb) {
      const int kb = k0 + 32 * mb;
      if (kb + 32 > open) {
        if constexpr (TREE) {
          const uint32_t vis = visible(kb) >> (4 * hh);
#pragma unroll
          for (int r = 0; r < 16; ++r)
            if (!((vis >> (8 * (r >> 2) + (r & 3))) & 1u)) s[mb][r] = kNone;
        } else {
          const int lim = qi + pc.off - kb - 4 * hh;
#pragma unroll
          for (int r = 0; r < 16; ++r)
            if (8 * (r >> 2) + (r & 3) > lim) s[mb][r] = kNone;
        }
      }
    }
    if constexpr (PAGED && RT == 1) {
      if (a.scores != nullptr && pc.row0 + r32 < rend) {
        float* const so = a.scores + ((pc.b * a.Hkv + pc.kvh) * (int64_t)(a.N * a.G) + row) * a.scores_ld + k0 + 4 * hh;
#pragma unroll
        for (int mb = 0; mb < MB; ++mb)
#pragma unroll
          for (int g = 0; g < 4; ++g)
            *reinterpret_cast<f32x4_t*>(so + 32 * mb + 8 * g) =
                f32x4_t{s[mb][4 * g], s[mb][4 * g + 1], s[mb][4 * g + 2], s[mb][4 * g + 3]};
      }
    }
    float mt = s[0][0];
#pragma unroll
    for (int mb = 0; mb < MB; ++mb)
#pragma unroll
      for (int r = mb == 0 ? 1 : 0; r < 16; ++r) mt = fmaxf(mt, s[mb][r]);
    mt = half_pair_max(mt) * a.scale_log2;
    const bool raise = mt > mo + kLazyLog2;  // the row's own affair, whatever its neighbours' scores
    if (__builtin_amdgcn_ballot_w64(raise) != 0) {
      const float mn = raise ? __builtin_floorf(mt) : mo;
      // no key before: l is 0, and o what clean_stage added
      const float f = mo == kNone ? 1.f : __builtin_amdgcn_exp2f(mo - mn);
      mo = mn;
      l *= f;
      lc *= f;
#pragma unroll
      for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[nb][r] *= f;
    }
    // sums and outputs of all a row's parts are lifted alike
    const float moff = mo == kNone ? 0.f : mo - M::kLift;  // no key yet: every score here is -inf
#pragma unroll
    for (int mb = 0; mb < MB; ++mb) {
      const T* vb = Vs + 32 * mb * D;
      float sum = 0.f;
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        s[mb][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[mb][r], a.scale_log2, -moff));
        sum += s[mb][r];
      }
      add_rounded(l, lc, sum);
      if constexpr (F32) {
#pragma unroll
        for (int c = 0; c < 16; ++c) {
          const int key = 8 * (c >> 2) + 4 * hh + (c & 3);
          const float* vrow = reinterpret_cast<const float*>(vb) + key * D;
          const int ksw = seq_swz<PPR, ES>(key);
          float vf[NB];
          if constexpr (D == 16) {
            vf[0] = vrow[4 * (((r32 & 15) >> 2) ^ ksw) + (r32 & 3)];
          } else if constexpr (D == 32) {
            vf[0] = vrow[4 * ((r32 >> 2) ^ ksw) + (r32 & 3)];
          } else if constexpr (D == 64) {
            const u32x2_t x = *reinterpret_cast<const u32x2_t*>(vrow + 4 * ((r32 >> 1) ^ ksw) + 2 * (r32 & 1));
            vf[0] = __uint_as_float(x[0]);
            vf[1] = __uint_as_float(x[1]);
          } else {
            const f32x4_t x = *reinterpret_cast<const f32x4_t*>(vrow + 4 * (r32 ^ ksw));
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) vf[nb] = x[nb];
          }
#pragma unroll
          for (int nb = 0; nb < NB; ++nb) o[nb] = __builtin_amdgcn_mfma_f32_32x32x2f32(vf[nb], s[mb][c], o[nb], 0, 0, 0);
        }
      } else {
        vec8 ph[2], pl[2];
#pragma unroll
        for (int c2 = 0; c2 < 2; ++c2) {
          ProbPairs w[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) w[i] = M::split(s[mb][8 * c2 + 2 * i], s[mb][8 * c2 + 2 * i + 1]);
          ph[c2] = __builtin_bit_cast(vec8, u32x4_t{w[0].high, w[1].high, w[2].high, w[3].high});
          pl[c2] = __builtin_bit_cast(vec8, u32x4_t{w[0].low, w[1].low, w[2].low, w[3].low});
        }
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
          for (int c2 = 0; c2 < 2; ++c2) {
            const uint2 lo = lds_read_tr16(vb + 16 * c2 * D + voff[0][nb]);
            const uint2 hi = lds_read_tr16(vb + 16 * c2 * D + voff[1][nb]);
            const vec8 vf = __builtin_bit_cast(vec8, u32x4_t{lo.x, lo.y, hi.x, hi.y});
            o[nb] = M::mma(vf, ph[c2], o[nb]);
            o[nb] = M::mma(vf, pl[c2], o[nb]);
          }
      }
    }
  };

  stage_ready();
  for (int t = 0; t < nstage; t += 2) {
    const int k0 = kfirst + t * kstep;
    if (t + 1 < nstage) copy_stage(kv1, k0 + kstep);
    clean_stage(kv0, t);
    if (k0 < wend) compute(kv0, k0);
    stage_ready();  // stage 1 filled; every wave is done with stage 0
    if (t + 1 >= nstage) break;
    if (t + 2 < nstage) copy_stage(kv0, k0 + 2 * kstep);
    clean_stage(kv1, t + 1);
    if (k0 + kstep < wend) compute(kv1, k0 + kstep);
    stage_ready();
  }
  l = half_pair_sum(l - lc);

  // ---- the key groups' states joined ---------------------------------------------------
  if constexpr (KS > 1) {
    __syncthreads();
    auto slot = [&](int w) __attribute__((always_inline)) {
      return reinterpret_cast<float*>((w & 1) ? kv1 : kv0) + (w >> 1) * C::JOIN;
    };
    if (kg > 0) {
      float* f = slot((kg - 1) * RT + rt);
#pragma unroll
      for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int r = 0; r < 16; ++r) f[(16 * nb + r) * 64 + lane] = o[nb][r];
      f[NB * 16 * 64 + lane] = mo;
      f[(NB * 16 + 1) * 64 + lane] = l;
    }
    __syncthreads();
    if (kg > 0) return;
#pragma unroll
    for (int g = 1; g < KS; ++g) {
      const float* f = slot((g - 1) * RT + rt);
      const float m2 = f[NB * 16 * 64 + lane], l2 = f[(NB * 16 + 1) * 64 + lane];
      const float mn = fmaxf(mo, m2);
      const float f1 = mo == kNone ? 0.f : __builtin_amdgcn_exp2f(mo - mn);
      const float f2 = m2 == kNone ? 0.f : __builtin_amdgcn_exp2f(m2 - mn);
      mo = mn;
      // a state without a key has zeros; l takes a NaN along
      l = l * f1 + l2 * f2;
#pragma unroll
      for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[nb][r] = o[nb][r] * f1 + f[(16 * nb + r) * 64 + lane] * f2;
    }
    // the outputs go through the same LDS: reads above come first
    if constexpr (!F32) __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  }
  if (!live) return;

  // ---- the result ----------------------------------------------------------------------
  const bool stored = wrow + r32 < rend;
  if ((TREE && RT == 4) || (MODE != kPacked && a.nsplit > 1)) {  // 128 rows of a tree are always split
    const int64_t part = ((pc.b * a.Hkv + pc.kvh) * (int64_t)(a.N * a.G) + row) * a.nsplit + pc.split;
    if (stored) {
      float* wo = static_cast<float*>(a.ws_o) + part * D;
      if constexpr (F32 && NB > 1) {
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int d = NB * (8 * (r >> 2) + 4 * hh + (r & 3));
#pragma unroll
          for (int nb = 0; nb < NB; ++nb) wo[d + nb] = o[nb][r];
        }
      } else {
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
          for (int g = 0; g < (D == 16 ? 2 : 4); ++g)
            *reinterpret_cast<f32x4_t*>(wo + 32 * nb + 8 * g + 4 * hh) =
                f32x4_t{o[nb][4 * g], o[nb][4 * g + 1], o[nb][4 * g + 2], o[nb][4 * g + 3]};
      }
      if (hh == 0) {
        float* ml = static_cast<float*>(a.ws_ml) + 2 * part;
        ml[0] = mo;
        ml[1] = l;
      }
    }
    return;
  }
  // no key at all: zeros; keys whose scores are all -inf: 0 / 0, as a softmax gives
  const bool none = TREE ? pc.own == 0 && mask == 0 : PAGED ? qi >= pc.count : qi + pc.off < 0;
  if constexpr (PAGED) {
    if (a.lse != nullptr && stored && hh == 0)
      static_cast<float*>(a.lse)[(pc.b * a.Hkv + pc.kvh) * (int64_t)(a.N * a.G) + row] =
          none ? __builtin_huge_valf() : mo - M::kLift + __builtin_amdgcn_logf(l);
  }
  const float inv = none ? 0.f : 1.0f / l;
  if constexpr (F32) {
    if (!stored) return;
    float* yp = static_cast<float*>(a.y) + pc.b * a.yb + (pc.q0 + qi) * a.yt + (int64_t)head * a.yh;
    // register 4g + e of block nb is dim NB (8 g + 4 hh + e) + nb
#pragma unroll
    for (int g = 0; g < (D == 16 ? 2 : 4); ++g) {
      float w[4 * NB];
#pragma unroll
      for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) w[NB * e + nb] = none ? 0.f : o[nb][4 * g + e] * inv;
#pragma unroll
      for (int x = 0; x < NB; ++x) {
        const int d = NB * (8 * g + 4 * hh) + 4 * x;
        if (d < a.D) *reinterpret_cast<f32x4_t*>(yp + d) = f32x4_t{w[4 * x], w[4 * x + 1], w[4 * x + 2], w[4 * x + 3]};
      }
    }
  } else {
    // through LDS, so that a store writes whole rows; the wave's own rows, no barrier
    constexpr int RPS = 64 / PPR;  // rows a wave-wide store covers
    T* stg = ((rt & 1) ? kv1 : kv0) + (rt >> 1) * 32 * D;
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
      for (int g = 0; g < (D == 16 ? 2 : 4); ++g) {
        const uint32_t w0 = none ? 0u : pack_pair<T>(o[nb][4 * g] * inv, o[nb][4 * g + 1] * inv);
        const uint32_t w1 = none ? 0u : pack_pair<T>(o[nb][4 * g + 2] * inv, o[nb][4 * g + 3] * inv);
        const int sl = (4 * nb + g) ^ (r32 & (PPR - 1));
        *reinterpret_cast<u32x2_t*>(stg + r32 * D + 8 * sl + 4 * hh) = u32x2_t{w0, w1};
      }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    const int piece = lane % PPR;
#pragma unroll
    for (int p = 0; p < 32 / RPS; ++p) {
      const int r = p * RPS + lane / PPR;
      const u32x4_t w = *reinterpret_cast<const u32x4_t*>(stg + r * D + 8 * (piece ^ (r & (PPR - 1))));
      const int rr = wrow + r;
      if (rr < rend && 8 * piece < a.D) {
        const int i = rr / a.G, h = pc.kvh * a.G + (rr - i * a.G);
        T* yp = static_cast<T*>(a.y) + pc.b * a.yb + (pc.q0 + i) * a.yt + (int64_t)h * a.yh;
        *reinterpret_cast<u32x4_t*>(yp + 8 * piece) = w;
      }
    }
  }
}

}  // namespace dg
