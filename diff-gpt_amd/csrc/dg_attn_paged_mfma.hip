// Attention over a cache in pages on the matrix cores: the launches of seq_mfma_kernel's
// paged form (dg_seq_mfma.h), and the weights that each position was given.
//
// paged_weights_kernel: w[t] += sum over the rows r of one key head of exp2(s_rt - lse_r), with
// lse the attention's own.  A wave holds 32 positions' keys in registers for the whole loop,
// and tiles of 32 rows pass through LDS, a stage ahead, shared by its four waves:
//
//   S (32 rows x 32 keys) = Q K^T    Q from LDS, K in registers
//
// so that a lane's 16 scores belong to one position and add up where they are; the two
// halves of a wave meet at the end.  No atomics: a position belongs to one wave.  8 x 200
// tokens behind 500 - 4000 positions, 8 heads of 64 on 8, fp16: 11 us, the attention before it
// 32.8 (vector ALU 27 % busy, matrix cores 4 %: bound by the latencies of a workgroup: its keys
// and then its stages of rows in turn).  Many rows: by the exponentials, a fused product, an
// exp2 at a quarter of the rate and a sum each where nothing is hidden; 8 x 256 behind 1260 -
// 4000, 16 heads on 4 of 128, 50 us, 56 with every score masked (two tiles a stage, which 64 dims
// in 16 bits have, took 48 there, but left 4 waves a SIMD of 5: 64 x 5 tokens 33 -> 34.5).
#include "dg_paged.h"
#include "dg_seq_mfma.h"

namespace dg {

template <typename T, int D>
__global__ __launch_bounds__(256, D * sizeof(T) <= 256 ? 5 : 3) void paged_weights_kernel(const SeqArgs a, const PagedWeights w) {
  using C = SeqCfg<T, D, 4>;
  using M = SeqMma<T>;
  using vec8 = typename M::vec8;
  constexpr bool F32 = C::ES == 4;
  constexpr int ES = C::ES, PPR = C::PPR, RPD = C::RPD, ROWS = D * ES <= 128 ? 64 : 32, NDMA = ROWS / RPD;
  __shared__ __attribute__((aligned(16))) T qs[2][ROWS * D];
  __shared__ __attribute__((aligned(16))) float ls[2][ROWS];

  // workgroup x runs on XCD x mod 8: the key blocks of a key head follow each other there and
  // share its rows
  const unsigned t8 = blockIdx.x >> 3;
  const int blk = (int)(t8 % (unsigned)w.blocks);
  const int64_t u = (int64_t)(t8 / (unsigned)w.blocks) * 8 + (blockIdx.x & 7u);
  const int64_t b = u / a.Hkv;
  const int kvh = (int)(u - b * a.Hkv);
  if (b >= a.B) return;  // the grid is rounded up
  const PagedRow pr = paged_row(a, b, __builtin_amdgcn_readfirstlane(a.lens[b]));
  const int total = pr.own + pr.count, nrows = pr.count * a.G;
  if (nrows == 0) return;  // whole workgroups, before any barrier
  const int lane = threadIdx.x & 63, hh = lane >> 5, r32 = lane & 31;
  const int wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  for (int64_t k0 = (int64_t)blk * kWeightKeys; k0 < total; k0 += (int64_t)w.blocks * kWeightKeys) {
    const int kb = (int)k0;
    const int t = kb + 32 * wv + r32;  // this lane's position

    // rows are (token, head of the group) pairs; position t is seen from row `from` on
    const int64_t from64 = (int64_t)(t - pr.own) * a.G;
    const int from = t >= total ? nrows : (int)max(from64, (int64_t)0);
    // the rows that all of the wave's positions are seen from
    const int last = kb + 32 * wv + 31;
    const int all_from = last >= total ? nrows : (int)max((int64_t)(last - pr.own) * a.G, (int64_t)0);
    // the first tile that any position of the workgroup is seen from
    const int first = max(kb - pr.own, 0) * a.G / 32 * 32;

    const T* const qb = static_cast<const T*>(a.q) + b * a.qb + (int64_t)kvh * a.G * a.qh;
    const float* const lse = static_cast<const float*>(a.lse) + (b * a.Hkv + kvh) * (int64_t)(a.N * a.G);
    auto copy_rows = [&](int st, int row0) __attribute__((always_inline)) {
#pragma unroll
      for (int n = 0; n < (NDMA + 3) / 4; ++n) {
        const int i = 4 * n + wv;
        if (NDMA % 4 != 0 && i >= NDMA) break;  // wave-uniform
        if (row0 + i * RPD / 32 * 32 >= nrows) break;  // tiles without a row are not computed
        const int r = i * RPD + lane / PPR, row = row0 + r;
        const int e = ((lane % PPR) ^ seq_swz<PPR, ES>(r)) * (16 / ES);
        const int qi = row / a.G;
        const bool in = row < nrows && e < a.D;
        const void* p = in ? static_cast<const void*>(qb + qi * a.qt + (int64_t)(row - qi * a.G) * a.qh + e) : &kZeros16;
        lds_copy16(p, qs[st] + i * RPD * D);
      }
    };
    auto row_lse = [&](int row0) __attribute__((always_inline)) {
      const int row = row0 + (int)threadIdx.x;
      return threadIdx.x < ROWS && row < nrows ? lse[row] : __builtin_huge_valf();
    };

    copy_rows(0, first);
    const float head = row_lse(first);
    vec8 kf[F32 ? C::QC : C::NC];
    int id = -1;
    if (t < total) id = a.table[b * a.table_ld + (t >> a.page_log2)];
    const bool there = id >= 0 && id < a.pages;
    const T* const kp = static_cast<const T*>(a.k) + (there ? id : 0) * a.kb + (int64_t)kvh * a.kh +
                        (t & ((1 << a.page_log2) - 1)) * a.kt;
    if constexpr (F32) {
#pragma unroll
      for (int m = 0; m < C::QC / 4; ++m) {
        const int d = C::QC * hh + 4 * m;
        f32x4_t x = {0.f, 0.f, 0.f, 0.f};
        if (there && d < a.D) x = *reinterpret_cast<const f32x4_t*>(kp + d);
#pragma unroll
        for (int e = 0; e < 4; ++e) kf[4 * m + e] = x[e];
      }
    } else {
#pragma unroll
      for (int c = 0; c < C::NC; ++c) {
        const int d = 16 * c + 8 * hh;
        u32x4_t x = {0u, 0u, 0u, 0u};
        if (there && d < a.D) x = *reinterpret_cast<const u32x4_t*>(kp + d);
        kf[c] = __builtin_bit_cast(vec8, x);
      }
    }

    const int kswz = seq_swz<PPR, ES>(r32);
    float acc = 0.f, accc = 0.f;
    int st = 0;
    if (threadIdx.x < ROWS) ls[0][threadIdx.x] = head;
    for (int stage0 = first; stage0 < nrows; stage0 += ROWS, st ^= 1) {
      __builtin_amdgcn_s_waitcnt(0);
      __syncthreads();  // stage st filled; every wave is done with the other
      float next = 0.f;
      if (stage0 + ROWS < nrows) {
        copy_rows(st ^ 1, stage0 + ROWS);
        next = row_lse(stage0 + ROWS);
      }
#pragma unroll
      for (int tile = 0; tile < ROWS / 32; ++tile) {
        const int row0 = stage0 + 32 * tile;
        if (row0 >= nrows) break;  // the same in all waves
        const T* const Q = qs[st] + 32 * tile * D;
        floatx16_t s;
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] = 0.f;
        if constexpr (F32) {
#pragma unroll
          for (int p = 0; p < C::QC / 4; ++p) {
            const f32x4_t qf = *reinterpret_cast<const f32x4_t*>(reinterpret_cast<const float*>(Q) + r32 * D + 4 * (((PPR / 2) * hh + p) ^ kswz));
#pragma unroll
            for (int e = 0; e < 4; ++e) s = __builtin_amdgcn_mfma_f32_32x32x2f32(qf[e], kf[4 * p + e], s, 0, 0, 0);
          }
        } else {
#pragma unroll
          for (int c = 0; c < C::NC; ++c) {
            const u32x4_t qf = *reinterpret_cast<const u32x4_t*>(Q + r32 * D + 8 * ((2 * c + hh) ^ kswz));
            s = M::mma(__builtin_bit_cast(vec8, qf), kf[c], s);
          }
        }
        // lane l, register r: row 8 (r / 4) + 4 hh + r % 4 of the tile
        const int lo = from - row0 - 4 * hh, hi = nrows - row0 - 4 * hh;
        float sum = 0.f;
        if (row0 >= all_from && row0 + 32 <= nrows) {  // nothing hidden
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            const f32x4_t l4 = *reinterpret_cast<const f32x4_t*>(&ls[st][32 * tile + 8 * g + 4 * hh]);
#pragma unroll
            for (int e = 0; e < 4; ++e) sum += __builtin_amdgcn_exp2f(__builtin_fmaf(s[4 * g + e], a.scale_log2, -l4[e]));
          }
          add_rounded(acc, accc, sum);
          continue;
        }
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const f32x4_t l4 = *reinterpret_cast<const f32x4_t*>(&ls[st][32 * tile + 8 * g + 4 * hh]);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int r = 8 * g + e;
            const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s[4 * g + e], a.scale_log2, -l4[e]));
            sum += r >= lo && r < hi ? p : 0.f;
          }
        }
        add_rounded(acc, accc, sum);
      }
      // written here, not where it is loaded: that would wait for the copies
      if (threadIdx.x < ROWS) ls[st ^ 1][threadIdx.x] = next;
    }
    acc = half_pair_sum(acc - accc);
    if (hh == 0 && t < total) {
      float* const o = w.out + b * w.wb + (int64_t)kvh * w.wh + t;
      *o += acc;
    }
    __syncthreads();  // every wave is done with the rows before the next block's come
  }
}

namespace {

template <typename T, int D, int RT>
int launch_paged(const SeqArgs& a, dim3 grid, hipStream_t s) {
  const dim3 block(64 * SeqCfg<T, D, RT>::WAVES);
  const int64_t es = (int64_t)sizeof(T), page = (int64_t)1 << a.page_log2, far = (int64_t)1 << 31;
  if (page >= paged_granule(D, (int)es) && a.kb == a.vb && a.kt == a.vt && a.kb >= 0 && a.kb * es < far && page * a.kt * es < far) {
    hipLaunchKernelGGL((seq_mfma_kernel<T, D, RT, kPaged>), grid, block, 0, s, a);
    return check_launch(RT == 1 ? "seq_mfma_paged_32" : RT == 2 ? "seq_mfma_paged_64" : "seq_mfma_paged_128");
  }
  hipLaunchKernelGGL((seq_mfma_kernel<T, D, RT, kPagedAny>), grid, block, 0, s, a);
  return check_launch(RT == 1 ? "seq_mfma_paged_any_32" : RT == 2 ? "seq_mfma_paged_any_64" : "seq_mfma_paged_any_128");
}

template <typename T, int RT>
int launch_paged_d(const SeqArgs& a, dim3 grid, hipStream_t s) {
  const int D = seq_mfma_dim(a.D);
  if (D == 16) return launch_paged<T, 16, RT>(a, grid, s);
  if (D == 32) return launch_paged<T, 32, RT>(a, grid, s);
  if (D == 64) return launch_paged<T, 64, RT>(a, grid, s);
  if (D == 128) return launch_paged<T, 128, RT>(a, grid, s);
  if constexpr (sizeof(T) == 2) return launch_paged<T, 256, RT>(a, grid, s);
  return DG_EUNSUPPORTED;
}

template <typename T>
int launch_paged_t(const SeqArgs& a, dim3 grid, hipStream_t s) {
  if (a.rows_per_wg == 32) return launch_paged_d<T, 1>(a, grid, s);
  if (a.rows_per_wg == 64) return launch_paged_d<T, 2>(a, grid, s);
  return launch_paged_d<T, 4>(a, grid, s);
}

template <typename T>
int launch_weights(const SeqArgs& a, const PagedWeights& w, dim3 grid, hipStream_t s) {
  const int D = seq_mfma_dim(a.D);
  if (D == 16) hipLaunchKernelGGL((paged_weights_kernel<T, 16>), grid, dim3(256), 0, s, a, w);
  else if (D == 32) hipLaunchKernelGGL((paged_weights_kernel<T, 32>), grid, dim3(256), 0, s, a, w);
  else if (D == 64) hipLaunchKernelGGL((paged_weights_kernel<T, 64>), grid, dim3(256), 0, s, a, w);
  else if (D == 128) hipLaunchKernelGGL((paged_weights_kernel<T, 128>), grid, dim3(256), 0, s, a, w);
  else if constexpr (sizeof(T) == 2) hipLaunchKernelGGL((paged_weights_kernel<T, 256>), grid, dim3(256), 0, s, a, w);
  return check_launch("paged_weights_kernel");
}

}  // namespace

int launch_seq_mfma_paged(const SeqArgs& a, int dtype, unsigned blocks, hipStream_t s) {
  if (dtype == DG_F32) return launch_paged_t<float>(a, dim3(blocks), s);
  if (dtype == DG_BF16) return launch_paged_t<bf16_t>(a, dim3(blocks), s);
  return launch_paged_t<f16_t>(a, dim3(blocks), s);
}

int launch_paged_weights_mfma(const SeqArgs& a, const PagedWeights& w, int dtype, unsigned blocks, hipStream_t s) {
  if (dtype == DG_F32) return launch_weights<float>(a, w, dim3(blocks), s);
  if (dtype == DG_BF16) return launch_weights<bf16_t>(a, w, dim3(blocks), s);
  return launch_weights<f16_t>(a, w, dim3(blocks), s);
}

}  // namespace dg
