// Packed attention and token trees over a cache on the matrix cores: the choice of workgroup
// shapes and the launches of seq_mfma_kernel (dg_seq_mfma.h).
#include "dg_seq_mfma.h"

namespace dg {

namespace {

// Rows of a tree's workgroup, 32 RT, that seq_mfma_tree_rows chooses from.
constexpr bool tree_has_shape(int D, int RT, bool f32) { return RT == 1 || (f32 ? RT == 2 && D == 128 : D >= 64); }

template <typename T, int D, int RT, SeqMode MODE>
int launch_seq(const SeqArgs& a, dim3 grid, hipStream_t s) {
  hipLaunchKernelGGL((seq_mfma_kernel<T, D, RT, MODE>), grid, dim3(64 * SeqCfg<T, D, RT>::WAVES), 0, s, a);
  return check_launch(MODE == kTree ? (RT == 1 ? "seq_mfma_tree_32" : RT == 2 ? "seq_mfma_tree_64" : "seq_mfma_tree_128")
                           : (RT == 1 ? "seq_mfma_packed_32" : RT == 2 ? "seq_mfma_packed_64" : "seq_mfma_packed_128"));
}

template <typename T, int RT, SeqMode MODE>
int launch_seq_d(const SeqArgs& a, dim3 grid, hipStream_t s) {
  constexpr bool kF32 = sizeof(T) == 4;
#define DG_SEQ_D(DIM)                                  \
  if constexpr (MODE == kPacked || tree_has_shape(DIM, RT, kF32)) \
    if (seq_mfma_dim(a.D) == DIM) return launch_seq<T, DIM, RT, MODE>(a, grid, s)
  DG_SEQ_D(16);
  DG_SEQ_D(32);
  DG_SEQ_D(64);
  DG_SEQ_D(128);
  if constexpr (!kF32) DG_SEQ_D(256);
#undef DG_SEQ_D
  return DG_EUNSUPPORTED;
}

template <int RT, SeqMode MODE>
int launch_seq_t(const SeqArgs& a, int dtype, dim3 grid, hipStream_t s) {
  if (dtype == DG_F32) return launch_seq_d<float, RT, MODE>(a, grid, s);
  if (dtype == DG_BF16) return launch_seq_d<bf16_t, RT, MODE>(a, grid, s);
  return launch_seq_d<f16_t, RT, MODE>(a, grid, s);
}

}  // namespace

// 16-bit types up to 256 dims, fp32 up to 128, rows of whole 16-byte pieces aligned to them, and
// a stage's rows (up to 64) within 2^31 bytes of each other.
bool seq_mfma_applicable(const SeqArgs& a, int dtype, bool tree) {
  if (dtype == DG_F64 || a.D > (dtype == DG_F32 ? 128 : 256) || a.D * dtype_bytes(dtype) % 16 != 0) return false;
  const int64_t es = dtype_bytes(dtype);
  auto rows = [&](const void* p, int64_t b, int64_t t, int64_t h) {
    return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && (!tree || b * es % 16 == 0) && t * es % 16 == 0 && h * es % 16 == 0;
  };
  const int64_t most = ((int64_t)1 << 31) / (64 * es) - a.D;
  if (a.kt < 0 || a.vt < 0 || a.kt > most || a.vt > most) return false;
  return rows(a.q, a.qb, a.qt, a.qh) && rows(a.k, a.kb, a.kt, a.kh) && rows(a.v, a.vb, a.vt, a.vh) &&
         rows(a.y, a.yb, a.yt, a.yh);
}

// Rows of a tree's workgroup.  32 (the waves split the keys) spread a row's keys over the
// most waves; 64 and 128 read them fewer times.  us with 32 / 64 / 128 rows, "rows of the
// batch x (token, head) rows", lengths up to, key heads:
//   head_dim <= 32, every one tried:  bf16 16 x 60, 600, 4: 8.7 / 13.8 / 18.1; fp32 32 x 60,
//     2000, 4: 29.9 / 30.6 / 30.8; 64 x 64, 4000, 8: 113 / 147 / 147
//   fp32 head_dim 64: 3 x 152, 140, 1: 11.8 / 14.2 / 18; 64 x 256, 3000, 4: 288 / 294 / 417
//     head_dim 128: 32 x 48, 2000, 4: 148 / 105 / 105; 2 x 256, 20000, 2: 188 / 118 / 137
//   16-bit, few keys in all: head_dim 64 16 x 60, 600, 4: 10.8 / 16.2 / 19.2, head_dim 128
//     4 x 152, 1500, 4: 20.9 / 19.9 / 27.9, 32 x 96, 2000, 4: 42.4 / 41.4 / 41.5; many:
//     head_dim 64 4 x 128, 70000, 8: 140 / 143 / 125, head_dim 128 16 x 96, 7168, 4: 79.7 /
//     53.5 / 54.3
//   64 rows fill the chip, no splits: 64 x 256, 4000, 4: head_dim 64 108 / 104 / 128,
//     head_dim 128 240 / 175 / 207
int seq_mfma_tree_rows(int64_t B, int rows, int Hkv, int keys, int D, int dtype) {
  if (rows <= 32 || D <= 32) return 32;
  if (dtype == DG_F32) return D <= 64 ? 32 : 64;
  const int64_t tiles = B * Hkv * ((rows + 127) / 128);
  if (tiles * keys <= 300000) return 32;
  return rows <= 64 || tiles >= 256 ? 64 : 128;
}

int launch_seq_mfma_tree(const SeqArgs& a, int dtype, unsigned blocks, hipStream_t s) {
  const dim3 grid(blocks);
  if (a.rows_per_wg == 32) return launch_seq_t<1, kTree>(a, dtype, grid, s);
  if (a.rows_per_wg == 64) return launch_seq_t<2, kTree>(a, dtype, grid, s);
  return launch_seq_t<4, kTree>(a, dtype, grid, s);
}

// A tile goes to one workgroup of 128 rows, to two of 64 that split the keys in two, or to
// four of 32 that split them in four: the more where tiles are few, since a workgroup
// walks its keys one stage after the other, and never fewer than fill the rows.  us with
// 32 / 64 / 128 rows, tiles times key heads in brackets, bf16:
//   head_dim  64: 8 x 512 tokens [256] 21.1 / 16.7 / 18.0, 16 [512] 35.7 / 22.1 / 22.2,
//     32 [1024] 59.6 / 34.3 / 28.1; 6 x 2048 [768] 88.6 / 71.2 / 70.8; 48 chunks of up to
//     300 behind up to 3000 keys, groups of 4 [436] 60.8 / 51.3 / 68.4, 64 [550] 86.5 /
//     81.8 / 83.0
//   head_dim 256: 2 x 512 [64] 26.6 / 29.9 / 42.7, 2 x 2048 in groups of 2 [256] 167 / 121 /
//     129, 16 x 512 [512] 157 / 104 / 85.5
//   head_dim 128: 1 x 3584 in groups of 2 [448] 156 / 105 / 123, 2 x 2048 [512] 129 / 81 / 79
int seq_mfma_packed_rows(const int64_t counts[3], int Hkv, int D) {
  const int64_t tiles = counts[1] * Hkv;
  if (counts[2] <= 32 || tiles <= 64) return 32;
  return counts[2] <= 64 || tiles <= (D > 64 ? 384 : 640) ? 64 : 128;
}

int launch_seq_mfma_packed(const SeqArgs& a, int dtype, dim3 grid, hipStream_t s) {
  if (a.rows_per_wg == 32) return launch_seq_t<1, kPacked>(a, dtype, grid, s);
  if (a.rows_per_wg == 64) return launch_seq_t<2, kPacked>(a, dtype, grid, s);
  return launch_seq_t<4, kPacked>(a, dtype, grid, s);
}

}  // namespace dg
