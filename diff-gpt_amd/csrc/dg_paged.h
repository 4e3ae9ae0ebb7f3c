// Shared by the entry points over a cache in pages (dg_paged.hip, dg_attn_paged.hip,
// dg_attn_paged_mfma.hip).
#pragma once

#include "dg_seq.h"

namespace dg {

inline bool int_size(int64_t n) { return n >= 0 && n <= 0x7fffffff; }
inline bool known_dtype(int64_t dtype) { return dtype == DG_F32 || dtype == DG_BF16 || dtype == DG_F16 || dtype == DG_F64; }

// What every entry point asks of a dg_paged_rows; *log2 receives that of its page.
int check_paged_rows(const char* what, const dg_paged_rows* r, bool need_v, int* log2);

// dg_attn_paged_mfma.hip: attention of workgroups of 32, 64 or 128 (token, head) rows, and the
// positions' weights, for shapes that seq_mfma_applicable takes.
int launch_seq_mfma_paged(const SeqArgs& a, int dtype, unsigned blocks, hipStream_t s);

// dg_attn_paged_vec.hip: up to so many fp32 (token, head) rows of a key head of up to 256 dims,
// in 16-byte pieces.  us there / on the matrix cores (which take no more than 128 dims), 64 rows
// of the batch, 4 key heads, 2000 positions, by rows of a key head:
//   head_dim  16: 1 17.7 / 27.1, 2 19.7 / 27.0, 4 29.9 / 27.3
//             64: 1 44.7 / 53.9, 2 46.0 / 54.1, 4 57.2 / 53.7
//            128: 1 98.0 / 173, 4 111 / 169, 8 235 / 171 (4 of 500: 1 14.6 / 27.7, 4 30.8 / 27.7)
constexpr int paged_vec_rows(int D) { return D <= 64 ? 2 : D <= 128 ? 4 : 8; }
int launch_paged_vec(const SeqArgs& a, unsigned blocks, hipStream_t s);

// The weights' arguments: a.q, a.k, the table and lengths as for the attention, a.lse its
// result; a.nrb is unused.
struct PagedWeights {
  float* out;
  int64_t wb, wh;
  int blocks;  // workgroups of a (b, key head), which take key blocks in turn
};
constexpr int kWeightKeys = 128;  // positions of a workgroup
int launch_paged_weights_mfma(const SeqArgs& a, const PagedWeights& w, int dtype, unsigned blocks, hipStream_t s);

}  // namespace dg
