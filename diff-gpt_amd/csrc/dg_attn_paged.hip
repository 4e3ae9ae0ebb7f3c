// Attention over a cache in pages (dg_paged_attention): the entry point, the split of long
// rows, the forms of any shape and type of the attention (seq_tile_kernel's, dg_seq_tile.h) and
// of the positions' weights (paged_weights_any_kernel), and the joins.  Rows of whole 16-byte
// pieces up to 256 dims in 16-bit types, 128 in fp32, run on the matrix cores
// (dg_attn_paged_mfma.hip).
#include "dg_paged.h"
#include "dg_seq_tile.h"

#include <algorithm>
#include <cmath>

namespace dg {

// Rows of a key head up to which, and bytes in all, the attention leaves its scores.
constexpr int64_t kScoreRows = 8, kScoreBytes = 64 << 20;

// w[t] += sum over the rows r of one key head of exp(s_rt - lse_r), 64 positions a workgroup
// by 32 rows at a time: a thread has one position and every fourth row, keys and rows pass
// through LDS in chunks of 64 dims.
template <typename T>
__global__ __launch_bounds__(256) void paged_weights_any_kernel(const SeqArgs a, const PagedWeights w) {
  using S = SeqAcc<T>;
  using A = typename S::type;
  constexpr int KT = 64, RT = 32, RPT = RT / 4, CS = 65;
  __shared__ A ks[KT * CS], qs[RT * 64], part[4 * KT];
  const int blk = (int)(blockIdx.x % (unsigned)w.blocks);
  const int64_t u = blockIdx.x / (unsigned)w.blocks;
  const int64_t b = u / a.Hkv;
  const int kvh = (int)(u - b * a.Hkv);
  const PagedRow pr = paged_row(a, b, __builtin_amdgcn_readfirstlane(a.lens[b]));
  const int total = pr.own + pr.count, nrows = pr.count * a.G;
  if (nrows == 0) return;  // whole workgroups
  const int tid = threadIdx.x, key = tid & 63, sub = tid >> 6;
  for (int64_t k0 = (int64_t)blk * KT; k0 < total; k0 += (int64_t)w.blocks * KT) {
    const int kb = (int)k0, t = kb + key;
    const int from = t >= total ? nrows : (int)max((int64_t)(t - pr.own) * a.G, (int64_t)0);
    const int first = max(kb - pr.own, 0) * a.G / RT * RT;
    const T* const qb = static_cast<const T*>(a.q) + b * a.qb + (int64_t)kvh * a.G * a.qh;
    const T* const kh = static_cast<const T*>(a.k) + (int64_t)kvh * a.kh;
    const A* const lse = static_cast<const A*>(a.lse) + (b * a.Hkv + kvh) * (int64_t)(a.N * a.G);
    const A us = S::unit_scale(a);
    A acc = (A)0, rest = (A)0;
    for (int row0 = first; row0 < nrows; row0 += RT) {
      A s[RPT];
#pragma unroll
      for (int j = 0; j < RPT; ++j) s[j] = (A)0;
      for (int d0 = 0; d0 < a.D; d0 += 64) {
        __syncthreads();
        for (int e = tid; e < KT * 64; e += 256) {
          const int kt = kb + e / 64, d = d0 + e % 64;
          A x = (A)0;
          if (kt < total && d < a.D) {
            const int id = a.table[b * a.table_ld + (kt >> a.page_log2)];
            if (id >= 0 && id < a.pages) x = S::load(kh[id * a.kb + (kt & ((1 << a.page_log2) - 1)) * a.kt + d]);
          }
          ks[e / 64 * CS + e % 64] = x;
        }
        for (int e = tid; e < RT * 64; e += 256) {
          const int row = row0 + e / 64, d = d0 + e % 64, qi = row / a.G;
          qs[e] = row < nrows && d < a.D ? S::load(qb[qi * a.qt + (int64_t)(row - qi * a.G) * a.qh + d]) : (A)0;
        }
        __syncthreads();
        for (int d = 0; d < 64; ++d) {
          const A k = ks[key * CS + d];
#pragma unroll
          for (int j = 0; j < RPT; ++j) s[j] += k * qs[(sub + 4 * j) * 64 + d];
        }
      }
      A sum = (A)0;
#pragma unroll
      for (int j = 0; j < RPT; ++j) {
        const int row = row0 + sub + 4 * j;
        if (row >= from && row < nrows) sum += S::exp(s[j] * us - lse[row]);
      }
      add_rounded(acc, rest, sum);
    }
    part[sub * KT + key] = acc - rest;
    __syncthreads();
    if (sub == 0 && t < total) {
      float* const o = w.out + b * w.wb + (int64_t)kvh * w.wh + t;
      *o = (float)((A)*o + ((part[key] + part[KT + key]) + (part[2 * KT + key] + part[3 * KT + key])));
    }
    __syncthreads();
  }
}

// order[0 ..] = the rows of the batch by how many positions their tokens see, the most first:
// where more workgroups than run at once take their turns, the launch then ends on short
// ones.  Ranks by counting, at most kOrdered rows.  us as they come / so, with this launch:
// 16 rows of 256 - 512 tokens behind 1000 - 7168, 16 heads on 4 of 128, 425 / 372; 48 of up to
// 300 behind up to 3000, 8 on 2 of 64, 86 / 67; a token behind each of 48 of 100 - 4096, 16 on 4
// of 128, in two splits, 46.7 / 41.3, of 256 223 / 222; 16 alike 417 / 420.
constexpr int kOrdered = 1024;

__global__ __launch_bounds__(kOrdered) void paged_order_kernel(const SeqArgs a, int32_t* order) {
  __shared__ int keys[kOrdered];
  const int b = threadIdx.x;
  int key = -1;
  if (b < a.B) {
    const int own = min(max(a.lens[b], 0), a.Tcap);
    const int count = min(max(a.counts != nullptr ? a.counts[b] : a.N, 0), min(a.N, a.Tcap - own));
    key = count > 0 ? own + count : 0;
  }
  keys[b] = key;
  __syncthreads();
  if (b >= a.B) return;
  int rank = 0;
  for (int j = 0; j < a.B; ++j) rank += keys[j] > key || (keys[j] == key && j < b);
  order[rank] = b;
}

// The same from the scores that the attention left (a.scores), four positions a thread: where
// few rows share a position, their scores are a fraction of its key.  48 rows of a step, 4 rows a
// key head of 128 dims, up to 4096 positions: 5.1 us in place of the 19.9 of paged_weights_kernel.
// JOINED: the rows' sums are in a.lse; otherwise their splits' are joined here, as seq_join4 does.
template <bool JOINED>
__device__ __forceinline__ void paged_scores(const SeqArgs& a, const PagedWeights& w, const float lift, const unsigned block) {
  __shared__ float sums[kScoreRows];
  const int64_t bh = block / (unsigned)w.blocks;
  const int blk = (int)(block - (unsigned)bh * (unsigned)w.blocks);
  const int64_t b = bh / a.Hkv;
  const int kvh = (int)(bh - b * a.Hkv);
  const PagedRow pr = paged_row(a, b, __builtin_amdgcn_readfirstlane(a.lens[b]));
  const int total = pr.own + pr.count, nrows = pr.count * a.G;
  if (nrows == 0 || blk * 1024 >= total) return;  // whole workgroups
  if constexpr (!JOINED) {
    const int lane = threadIdx.x & 63, chunk = paged_chunk(a, pr);
    for (int r = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); r < nrows; r += 4) {
      const u32x2_t* const ml = static_cast<const u32x2_t*>(a.ws_ml) + (bh * (a.N * a.G) + r) * a.nsplit;
      const int used = min(a.nsplit, (paged_end(a, pr, r) + chunk - 1) / chunk);
      float m = kNegInf, l = 0.f;
      bool bad = false;
      for (int s = lane; s < used; s += 64) {
        const float ms = __uint_as_float(ml[s][0]);
        bad = bad || ms != ms || __uint_as_float(ml[s][1]) != __uint_as_float(ml[s][1]);
        m = fmaxf(m, ms);
      }
      m = wave_max(m);
      bad = __builtin_amdgcn_ballot_w64(bad) != 0;
      for (int s = lane; s < used; s += 64) {
        const float ms = __uint_as_float(ml[s][0]);
        l += ms == kNegInf ? 0.f : __uint_as_float(ml[s][1]) * __builtin_amdgcn_exp2f(ms - m);
      }
      l = group_sum_dpp<64>(l);
      if (lane == 0) sums[r] = bad ? __builtin_nanf("") : m - lift + __builtin_amdgcn_logf(l);
    }
    __syncthreads();
  }
  for (int64_t t64 = 4 * (blk * (int64_t)256 + threadIdx.x); t64 < total; t64 += (int64_t)1024 * w.blocks) {
    const int t = (int)t64;
    const int64_t row = bh * (a.N * a.G);
    const float* const lse = JOINED ? static_cast<const float*>(a.lse) + row : sums;
    const float* const s = a.scores + row * a.scores_ld + t;
    f32x4_t sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int r = 0; r < nrows; ++r) {
      // a position that the row's tile was not run over lies behind what the row sees
      const int seen = pr.own + r / a.G;
      if (t > seen) continue;
      const f32x4_t x = *reinterpret_cast<const f32x4_t*>(s + r * a.scores_ld);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(x[e], a.scale_log2, -lse[r]));
        sum[e] += t + e <= seen ? p : 0.f;
      }
    }
    float* const o = w.out + b * w.wb + (int64_t)kvh * w.wh + t;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (t + e < total) o[e] += sum[e];
  }
}
__global__ __launch_bounds__(256) void paged_scores_kernel(const SeqArgs a, const PagedWeights w) {
  paged_scores<true>(a, w, 0.f, blockIdx.x);
}
// The outputs of split rows joined by the first `joins` workgroups, the weights from their scores
// by the others, in one launch (48 x 1 token behind 100 - 4096, 16 heads on 4 of 128, two
// launches / one: 59.6 / 58.1 us with the attention).
template <typename T, int D, int WPR>
__global__ __launch_bounds__(256) void paged_join_scores_kernel(const SeqArgs a, const int64_t nrows, const unsigned joins,
                                                                const PagedWeights w) {
  if (blockIdx.x < joins) seq_join4<T, D, WPR, kPaged>(a, nrows, blockIdx.x);
  else paged_scores<false>(a, w, seq_lift<T>(), blockIdx.x - joins);
}

namespace {

template <typename T>
int launch_tile(const SeqArgs& a, dim3 grid, hipStream_t s) {
#define DG_PAGED_TILE(NCH, LPR) hipLaunchKernelGGL((seq_tile_kernel<T, NCH, LPR, kPaged>), grid, dim3(256), 0, s, a)
  if (a.rows_per_wg == 32) {
    if (a.D <= 64) DG_PAGED_TILE(1, 8);
    else if (a.D <= 128) DG_PAGED_TILE(2, 8);
    else DG_PAGED_TILE(4, 8);
  } else if (a.rows_per_wg == 16) {
    DG_PAGED_TILE(16, 16);
  } else {
    if (a.D <= 128) DG_PAGED_TILE(2, 32);
    else if (a.D <= 256) DG_PAGED_TILE(4, 32);
    else DG_PAGED_TILE(16, 32);
  }
#undef DG_PAGED_TILE
  return check_launch("seq_tile_paged");
}

// scores: workgroups of the weights from scores (0: none)
template <typename T, int D, int WPR>
void launch_join4(const SeqArgs& a, unsigned joins, int64_t rows, const PagedWeights& w, unsigned scores, hipStream_t s) {
  if (scores > 0)
    hipLaunchKernelGGL((paged_join_scores_kernel<T, D, WPR>), dim3(joins + scores), dim3(256), 0, s, a, rows, joins, w);
  else
    hipLaunchKernelGGL((seq_join4_kernel<T, D, WPR, kPaged>), dim3(joins), dim3(256), 0, s, a, rows);
}

template <typename T, int WPR>
void launch_join4_dim(const SeqArgs& a, unsigned joins, int64_t rows, const PagedWeights& w, unsigned scores, hipStream_t s) {
  const int D = seq_mfma_dim(a.D);
  if (D == 16) launch_join4<T, 16, WPR>(a, joins, rows, w, scores, s);
  else if (D == 32) launch_join4<T, 32, WPR>(a, joins, rows, w, scores, s);
  else if (D == 64) launch_join4<T, 64, WPR>(a, joins, rows, w, scores, s);
  else if (D == 128) launch_join4<T, 128, WPR>(a, joins, rows, w, scores, s);
  else launch_join4<T, 256, WPR>(a, joins, rows, w, scores, s);
}

template <typename T>
int launch_join(const SeqArgs& a, bool mfma, bool many, unsigned joins, int64_t rows, const PagedWeights& w, unsigned scores,
                hipStream_t s) {
  if constexpr (sizeof(T) < 8) {
    if (mfma) {
      if (many) launch_join4_dim<T, 4>(a, joins, rows, w, scores, s);
      else launch_join4_dim<T, 1>(a, joins, rows, w, scores, s);
      return check_launch(scores > 0 ? "paged_join_scores_kernel" : "seq_join4_paged");
    }
  }
  if (many) hipLaunchKernelGGL((seq_join_kernel<T, 4, kPaged>), dim3(joins), dim3(256), 0, s, a, rows);
  else hipLaunchKernelGGL((seq_join_kernel<T, 1, kPaged>), dim3(joins), dim3(256), 0, s, a, rows);
  return check_launch("seq_join_paged");
}

// Rows of a workgroup.  Few (token, head) rows as a tree's.  Many: 32 where all such workgroups
// run at once, unless heads of 128 dims have many keys in all to read; 128 where there are so
// many tiles that 64 would read the keys too often (a packed batch's rule, half as many
// tiles again, since rows rarely have all of their tokens).  us with 32 / 64 / 128 rows and the
// splits of each that are best, rows x tokens behind up to so many keys, heads on key heads:
//   8 x 200, 4000, 8 / 8 of 64 36.3 / 43.5 / 44.0; 12 x 40, 2000, 8 / 2 of 64 16.8 / 22 / 30;
//   1 x 300, 30000, 8 / 2 of 64 54 / 73 / 87; 48 x 300, 3000, 8 / 2 of 64 131 / 107 / 139;
//   1 x 512, 7000, 16 / 4 of 128 78 / 64 / 70; 30 x 200, 600, 16 / 4 of 128 134 / 55 / 43;
//   16 x 512, 7168, 16 / 4 of 128 499 / 293 / 276
int mfma_rows(int64_t B, int64_t rows, int Hkv, int keys, int D, int dtype) {
  if (rows <= 128) return seq_mfma_tree_rows(B, (int)rows, Hkv, keys, D, dtype);
  const bool wide = seq_mfma_dim(D) * dtype_bytes(dtype) > 128;
  const int64_t tiles = B * Hkv * ((rows + 127) / 128);
  if (B * Hkv * ((rows + 31) / 32) <= (wide ? 256 : 512) && !(wide && tiles * keys > 300000)) return 32;
  return tiles <= (D > 64 ? 576 : 960) ? 64 : 128;
}

constexpr int kMaxSplits = 512;

enum PagedKernel { kTileKernel, kMfmaKernel, kVecKernel };

// Row blocks, splits and workspace of a call.
struct PagedShape {
  int rows_per_wg, nrb, nsplit, chunk, rb_groups, rb_each;
  int64_t blocks;
  bool ordered, ranked;  // the longest rows first: by paged_order_kernel, by each wave
  int64_t scores_ld;
  size_t o_bytes, lse_at, scores_at, order_at, ws_bytes;
};

// Nanoseconds that a workgroup takes for 128 keys, about (each alone on its CU, or as many as
// fit).
int64_t stage_ns(int D, int dtype, int rows_per_wg) {
  if (dtype == DG_F32) {
    if (D == 128) return rows_per_wg == 128 ? 17000 : 8800;
    return (D == 64 ? 2900 : D == 32 ? 2200 : 1100) * (rows_per_wg / 32);
  }
  return (D <= 32 ? 450 : D == 64 ? 700 : D == 128 ? 1000 : 2000) * (rows_per_wg / 32);
}

// The number of splits of a row of `longest` keys that ends first: a round, or so many and a
// quarter, of `fill` workgroups at once of its share of the keys each, and from two splits
// on the join, a launch of its own (8 us beside what the partial results take to write and
// read).  us measured, keys, heads on key heads, rows a workgroup, by splits 1 / 2 / 4 / 8:
//   1 x 512 tokens, 7000, 16 / 4 of 128, 64      123 / 78 / 64 / 73
//   4 x 100, 8000, 8 / 8 of 128, 32             53.7 / 37 / 45 / 54
//   8 x 200, 4000, 8 / 8 of 64, 32              36.3 / 43 / 51 / 51
//   6 x 237, 5580, 2 / 2 of 16, 32              21.7 / 18 / 16 / 19
//   5 x 25, 13386, fp32, 24 / 6 of 80, 64       909 / 464 / 246 / 198
int best_splits(int64_t wg, int64_t rows, int64_t longest, int64_t chunk, int64_t fill, int D, int64_t ns, bool few, bool scored) {
  const int64_t whole = longest * ns / 128;
  auto percent = [&](int64_t n) { return n <= fill ? 100 : 100 * n / fill + 25; };
  int best = 1;
  int64_t least = percent(wg) * whole / 100;
  const int64_t most = std::min<int64_t>(longest / chunk, kMaxSplits);
  for (int k = 2; k <= most && wg * k <= 4 * fill; ++k) {
    const int64_t cost = percent(wg * k) * whole / (100 * k) + 8000 + rows * k * D * 8 / 3000;
    if (cost < least) {
      least = cost;
      best = k;
    }
  }
  // One tile of rows a key head (few) and long rows (2048 positions on, whatever their type and dims):
  // as many splits as run at once, which the model, whose join is a busy chip's, finds too dear where
  // positions are cheap.  us as above / so, rows alike within two: 1 token behind 2100, 4 / 4 of 16 11.4 / 8.3, of 32
  // 13.4 / 8.7; 8 of them 12.1 / 10.0, 13.5 / 11.0; of 64 and 128 dims, and behind 4100, the same
  if (few && longest >= 2048 && 2 * wg <= fill) best = std::max(best, (int)std::min<int64_t>(fill / wg, most));
  // Rows are rarely all as long as the longest, so that two splits pay before they run at once, but
  // only where a launch behind the attention is there anyway, that of the weights from scores
  // (scored).  us as above / in two, a token a row behind, with weights:
  //   48 of 100 - 4096, 16 / 4 of 128 77 / 68, of 2000 - 4096 88 / 85; 40 of 100 - 2048, 12 / 4 41.7 / 37.2;
  //   100 of 50 - 2500, 8 / 2 of 64 35.3 / 32.5; 200 of 100 - 3001, 4 / 2 57.2 / 56.4; rows alike lose,
  //   48 of 4000, 16 / 4 of 128 100 / 106, and shorter ones, 48 of 100 - 1500 36.8 / 39.1
  // the same without weights:
  //   61 / 58, 68 / 73; 34.5 / 34.3; 25.5 / 25.5; 43.4 / 47.8; 78 / 91
  if (scored && longest >= 2048 && wg < fill && 2 * wg > fill) best = std::max<int>(best, std::min<int64_t>(2, most));
  return best;
}

PagedShape paged_shape(int64_t B, int N, int H, int Hkv, int D, int dtype, int64_t longest, int64_t cap, int weights,
                       int rows_per_wg, PagedKernel kernel) {
  const bool mfma = kernel != kTileKernel, vec = kernel == kVecKernel;
  PagedShape t{};
  const int64_t R = (int64_t)N * (H / Hkv);
  t.rows_per_wg = rows_per_wg;
  t.nrb = (int)((R + rows_per_wg - 1) / rows_per_wg);
  const int Dm = mfma ? seq_mfma_dim(D) : D;
  const int64_t row_bytes = Dm * dtype_bytes(dtype);
  const int64_t fill = !mfma ? 2048
                       : vec ? 1024
                       : rows_per_wg <= 32 ? (row_bytes >= 256 ? 256 : 512)
                       : rows_per_wg == 64 ? (row_bytes >= 512 ? 256 : 512)
                                           : Dm == 256 ? 512 : Dm == 128 ? 768 : 1024;
  const int64_t wg = std::max<int64_t>(1, B * Hkv * t.nrb);
  const int64_t ns = vec ? 1200 + Dm * R * 3 : mfma ? stage_ns(Dm, dtype, rows_per_wg) : 0;
  // fewest keys of a split: in fp32, where a stage of 128 takes as long as the join, that; us with
  // 256 / 128, fp32: 7 x 5 tokens behind 1200 - 2500, 6 heads on 3 of 128, 39.6 / 32.0; 1 x 30,
  // 8000, 4 on 4 of 128 39.8 / 30.8; 3 x 8, 700, 4 on 4 of 64 17.2 / 15.0
  t.chunk = kernel == kMfmaKernel && dtype == DG_F32 && Dm >= 64 ? 128 : 256;
  const int64_t ld = (cap + 255) / 256 * 256;
  const bool scored = weights && mfma && rows_per_wg == 32 && R <= kScoreRows && B * Hkv * R * ld * 4 <= kScoreBytes;
  t.nsplit = mfma ? best_splits(wg, B * Hkv * R, longest, t.chunk, fill, Dm, ns, R <= 32, scored)
                  : (int)std::max<int64_t>(1, std::min<int64_t>({(fill + wg - 1) / wg, longest / 256, kMaxSplits}));
  // every XCD has work: the row blocks of few (b, key head, split) go to several, in groups
  const int64_t units = B * Hkv * t.nsplit;
  t.rb_groups = (int)std::max<int64_t>(1, std::min<int64_t>(t.nrb, (64 + units - 1) / units));
  t.rb_each = (t.nrb + t.rb_groups - 1) / t.rb_groups;
  t.blocks = (units * t.rb_groups + 7) / 8 * 8 * t.rb_each;
  const bool turns = B > 1 && longest >= 1024 && t.blocks > fill;
  t.ranked = turns && B <= kRankedRows;
  t.ordered = turns && !t.ranked && B <= kOrdered;
  const size_t acc = dtype == DG_F64 ? 8 : 4;
  const size_t parts = (size_t)(B * Hkv * R) * t.nsplit;
  if (t.nsplit > 1) {
    t.o_bytes = (parts * Dm * acc + 15) & ~(size_t)15;
    t.ws_bytes = t.o_bytes + ((parts * 2 * acc + 15) & ~(size_t)15);
  }
  t.lse_at = t.ws_bytes;
  if (weights) t.ws_bytes += ((size_t)(B * Hkv * R) * acc + 15) & ~(size_t)15;
  t.scores_at = t.ws_bytes;
  if (scored) {
    t.scores_ld = ld;
    t.ws_bytes += (size_t)(B * Hkv * R * ld * 4);
  }
  t.order_at = t.ws_bytes;
  if (t.ordered) t.ws_bytes += (size_t)B * sizeof(int32_t);
  return t;
}

int tile_rows(int64_t rows, int D) { return rows <= 8 ? 8 : D <= 256 ? 32 : 16; }

}  // namespace

int check_paged_rows(const char* what, const dg_paged_rows* r, bool need_v, int* log2) {
  DG_REQUIRE(r != nullptr && r->k && (r->v || !need_v) && r->table && r->lens, DG_EINVAL, "%s: NULL argument", what);
  DG_REQUIRE(r->pages >= 1 && r->pages <= 0x7fffffff, DG_EINVAL, "%s: %lld pages", what, (long long)r->pages);
  DG_REQUIRE(r->page >= 1 && r->page <= kMostPositions && (r->page & (r->page - 1)) == 0, DG_EINVAL,
             "%s: a page of %lld positions, not a power of two", what, (long long)r->page);
  DG_REQUIRE(r->width >= 1 && r->width <= kMostPositions / r->page, DG_EINVAL,
             "%s: a table of %lld pages of %lld positions, 1 to 2^30 positions", what, (long long)r->width, (long long)r->page);
  *log2 = 0;
  while (((int64_t)1 << *log2) < r->page) ++*log2;
  return DG_OK;
}

}  // namespace dg

using namespace dg;

namespace dg {
namespace {

// A call looked over: its kernel's arguments and how it runs.
struct PagedCall {
  SeqArgs a;
  PagedShape t;
  PagedKernel kernel;
  bool empty;
};

int paged_call(const dg_paged_attention_args* args, PagedCall* c) {
  DG_REQUIRE(args != nullptr, DG_EINVAL, "paged_attention: NULL argument");
  DG_REQUIRE(int_size(args->B) && int_size(args->N) && int_size(args->H), DG_EINVAL,
             "paged_attention: negative size or one past 2^31 - 1");
  DG_REQUIRE(known_dtype(args->dtype), DG_EUNSUPPORTED, "paged_attention: dtype %lld unsupported", (long long)args->dtype);
  DG_REQUIRE(args->D >= 1 && args->D <= kMaxHeadDim, DG_EUNSUPPORTED, "paged_attention: head_dim %lld outside [1, %d]",
             (long long)args->D, kMaxHeadDim);
  DG_REQUIRE(args->Hkv >= 1 && args->Hkv <= 0x7fffffff && args->H % args->Hkv == 0, DG_EINVAL,
             "paged_attention: %lld query heads on %lld key heads", (long long)args->H, (long long)args->Hkv);
  const int64_t R = args->N * (args->H / args->Hkv);
  DG_REQUIRE(args->B * args->Hkv <= kMostWorkgroups256, DG_EINVAL, "paged_attention: more than 2^24 - 1 workgroups");
  DG_REQUIRE(R <= kMostPositions, DG_EINVAL, "paged_attention: a row of more than 2^30 (token, head) rows");
  const float scale = (float)args->scale;
  DG_REQUIRE(scale > 0.f && std::isfinite(scale * kLog2e), DG_EINVAL, "paged_attention: the scale must be positive and below 2^127");
  *c = PagedCall{};
  c->empty = args->B == 0 || args->N == 0 || args->H == 0;
  if (c->empty) return DG_OK;
  const int B = (int)args->B, N = (int)args->N, H = (int)args->H, Hkv = (int)args->Hkv, D = (int)args->D, dtype = (int)args->dtype;
  const dg_paged_rows* rows = &args->rows;
  SeqArgs& a = c->a;
  if (const int rc = check_paged_rows("paged_attention", rows, true, &a.page_log2)) return rc;
  DG_REQUIRE(args->q && args->y, DG_EINVAL, "paged_attention: NULL argument");
  const int64_t cap = rows->width * rows->page;
  DG_REQUIRE(args->longest >= 1 && args->longest <= cap, DG_EINVAL, "paged_attention: longest %lld, the table covers %lld positions",
             (long long)args->longest, (long long)cap);
  a.q = args->q; a.k = rows->k; a.v = rows->v; a.y = args->y;
  a.qb = args->q_st.b; a.qt = args->q_st.t; a.qh = args->q_st.h;
  a.kb = rows->k_st.b; a.kt = rows->k_st.t; a.kh = rows->k_st.h;
  a.vb = rows->v_st.b; a.vt = rows->v_st.t; a.vh = rows->v_st.h;
  a.yb = args->y_st.b; a.yt = args->y_st.t; a.yh = args->y_st.h;
  a.H = H; a.Hkv = Hkv; a.G = H / Hkv; a.D = D;
  a.scale = scale;
  a.scale_log2 = scale * kLog2e;
  a.B = B; a.N = N; a.Tcap = (int)cap;
  a.lens = rows->lens; a.counts = rows->counts;
  a.table = rows->table; a.table_ld = rows->table_ld; a.pages = rows->pages;
  // fp32 heads of up to 256 dims are looked at as if of 64, up to 128 of which the matrix cores take
  SeqArgs narrow = a;
  narrow.D = std::min(D, 64);
  const bool pieces = D <= 256 && D % 4 == 0 && seq_mfma_applicable(narrow, dtype, true);
  c->kernel = dtype == DG_F32 && R <= paged_vec_rows(D) && pieces ? kVecKernel
              : seq_mfma_applicable(a, dtype, true)      ? kMfmaKernel
                                                         : kTileKernel;
  const int rows_per_wg = c->kernel == kVecKernel    ? 32
                          : c->kernel == kMfmaKernel ? mfma_rows(B, R, Hkv, (int)args->longest, D, dtype)
                                                     : tile_rows(R, D);
  c->t = paged_shape(B, N, H, Hkv, D, dtype, args->longest, cap, args->weights != nullptr, rows_per_wg, c->kernel);
  const PagedShape& t = c->t;
  a.rows_per_wg = t.rows_per_wg; a.nrb = t.nrb; a.nsplit = t.nsplit; a.chunk = t.chunk;
  a.rb_groups = t.rb_groups; a.rb_each = t.rb_each;
  a.ranked = t.ranked;
  return DG_OK;
}

}  // namespace
}  // namespace dg

extern "C" size_t dg_paged_attention_workspace_size(const dg_paged_attention_args* args) {
  PagedCall c;
  return paged_call(args, &c) == DG_OK ? c.t.ws_bytes : 0;
}

extern "C" int dg_paged_attention(const dg_paged_attention_args* args, void* workspace, size_t workspace_bytes, void* stream) {
  PagedCall c;
  if (const int rc = paged_call(args, &c)) return rc;
  if (c.empty) return DG_OK;
  SeqArgs& a = c.a;
  const PagedShape& t = c.t;
  const bool mfma = c.kernel != kTileKernel, vec = c.kernel == kVecKernel;
  const int B = a.B, Hkv = a.Hkv, dtype = (int)args->dtype;
  const int64_t R = (int64_t)a.N * a.G, cap = a.Tcap;
  float* const weights = args->weights;
  if (t.ws_bytes > 0) {
    DG_REQUIRE(workspace != nullptr && workspace_bytes >= t.ws_bytes, DG_EWORKSPACE,
               "paged_attention: a workspace of %zu bytes, %zu needed", workspace_bytes, t.ws_bytes);
    DG_REQUIRE((reinterpret_cast<uintptr_t>(workspace) & 15) == 0, DG_EINVAL, "paged_attention: workspace not 16-byte aligned");
    a.ws_o = workspace;
    a.ws_ml = static_cast<char*>(workspace) + t.o_bytes;
    if (weights != nullptr) a.lse = static_cast<char*>(workspace) + t.lse_at;
    if (t.scores_ld > 0) {
      a.scores = reinterpret_cast<float*>(static_cast<char*>(workspace) + t.scores_at);
      a.scores_ld = t.scores_ld;
    }
    if (t.ordered) a.order = reinterpret_cast<int32_t*>(static_cast<char*>(workspace) + t.order_at);
  }
  const int64_t nrows = (int64_t)B * Hkv * R;
  const bool many = t.nsplit >= 16 && nrows <= 4096;
  const int64_t groups = t.nsplit == 1 ? 0 : many ? nrows : (nrows + 3) / 4;
  const int64_t blocks = t.blocks;
  PagedWeights w{weights, args->w_b, args->w_h, 0};
  const bool scored = t.scores_ld > 0, wmfma = mfma && (dtype != DG_F32 || a.D <= 128);
  const int wkeys = scored ? 1024 : wmfma ? kWeightKeys : 64;
  w.blocks = (int)((args->longest + wkeys - 1) / wkeys);
  const int64_t wblocks = weights == nullptr ? 0 : wmfma && !scored ? ((int64_t)B * Hkv + 7) / 8 * 8 * w.blocks : (int64_t)B * Hkv * w.blocks;
  DG_REQUIRE(blocks <= kMostWorkgroups256 && groups + wblocks <= kMostWorkgroups256, DG_EINVAL,
             "paged_attention: more than 2^24 - 1 workgroups");
  hipStream_t s = static_cast<hipStream_t>(stream);
  const dim3 grid((unsigned)blocks), wgrid((unsigned)wblocks);
  int rc;
  if (t.ordered) {
    hipLaunchKernelGGL(paged_order_kernel, dim3(1), dim3(kOrdered), 0, s, a, const_cast<int32_t*>(a.order));
    if ((rc = check_launch("paged_order_kernel")) != DG_OK) return rc;
  }
  if (vec) rc = launch_paged_vec(a, (unsigned)blocks, s);
  else if (mfma) rc = launch_seq_mfma_paged(a, dtype, (unsigned)blocks, s);
  else if (dtype == DG_F64) rc = launch_tile<double>(a, grid, s);
  else if (dtype == DG_F32) rc = launch_tile<float>(a, grid, s);
  else if (dtype == DG_BF16) rc = launch_tile<bf16_t>(a, grid, s);
  else rc = launch_tile<f16_t>(a, grid, s);
  if (rc == DG_OK && t.nsplit > 1) {
    const unsigned joins = (unsigned)groups, scores = scored ? (unsigned)wblocks : 0;
    if (dtype == DG_F64) rc = launch_join<double>(a, mfma, many, joins, nrows, w, scores, s);
    else if (dtype == DG_F32) rc = launch_join<float>(a, mfma, many, joins, nrows, w, scores, s);
    else if (dtype == DG_BF16) rc = launch_join<bf16_t>(a, mfma, many, joins, nrows, w, scores, s);
    else rc = launch_join<f16_t>(a, mfma, many, joins, nrows, w, scores, s);
  }
  if (rc != DG_OK || weights == nullptr) return rc;
  if (scored && t.nsplit > 1) return DG_OK;  // with the join
  if (scored) {
    hipLaunchKernelGGL(paged_scores_kernel, wgrid, dim3(256), 0, s, a, w);
    return check_launch("paged_scores_kernel");
  }
  if (wmfma) return launch_paged_weights_mfma(a, w, dtype, (unsigned)wblocks, s);
  if (dtype == DG_F64) hipLaunchKernelGGL(paged_weights_any_kernel<double>, wgrid, dim3(256), 0, s, a, w);
  else if (dtype == DG_F32) hipLaunchKernelGGL(paged_weights_any_kernel<float>, wgrid, dim3(256), 0, s, a, w);
  else if (dtype == DG_BF16) hipLaunchKernelGGL(paged_weights_any_kernel<bf16_t>, wgrid, dim3(256), 0, s, a, w);
  else hipLaunchKernelGGL(paged_weights_any_kernel<f16_t>, wgrid, dim3(256), 0, s, a, w);
  return check_launch("paged_weights_any_kernel");
}
