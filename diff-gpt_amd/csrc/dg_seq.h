// Launch arguments shared by the kernels of packed attention, of token trees over a cache and
// of attention over a cache in pages (dg_seq_tile.h: any shape; dg_seq_mfma.h: 16-bit and fp32
// data at head_dim up to 256 and 128, in rows of whole 16-byte pieces).
//
// These operators reduce to one piece of work: the rows of one key head, where the
// rows are the (query, head of the group) pairs r = i * G + g of a sequence, over a
// range of that sequence's keys.  Heads of a group so share every key they read, and
// a few queries still fill a tile of rows.
#pragma once

#include "dg_common.h"

namespace dg {

// packed: whole sequences one after the other; tree: up to 64 tokens a row over its cache,
// each with a mask; paged: any number of tokens a row, each seeing what lies before it, over
// a cache in pages (kPagedAny: of any size and strides, where kPaged asks for pages of
// paged_granule positions at least and the same strides, within 2^31 bytes, for keys and values)
enum SeqMode { kPacked, kTree, kPaged, kPagedAny };

struct SeqArgs {
  const void* q;
  const void* k;
  const void* v;
  void* y;
  int64_t qb, qt, qh;
  int64_t kb, kt, kh;
  int64_t vb, vt, vh;
  int64_t yb, yt, yh;
  int H, Hkv, G, D;
  float scale;       // the softmax scale
  float scale_log2;  // ... * log2(e)
  // packed: tiles of rows, and the rows q and k hold in all
  const dg_packed_tile* tiles;
  int64_t nq, nk;
  // tree: rows of the batch, tokens a row, positions a cache page holds
  int B, N, Tcap;
  int len;              // cached positions, where lens is null
  const int32_t* lens;  // (B)
  const int64_t* masks; // bit m of masks[b * mask_b + n]: token n sees token m; null: the earlier ones and itself
  int64_t mask_b;
  int rows_per_wg;  // rows of a workgroup
  int nrb;          // row blocks of a (b, key head); packed: workgroups of a tile
  int nsplit;       // key splits of a row (1: y is written)
  int chunk;        // keys of a split
  // nsplit > 1: unnormalised outputs (nsplit, D) and (maximum, sum) pairs (nsplit, 2) of row
  // (b * Hkv + key head) * N * G + r
  void* ws_o;
  void* ws_ml;
  // paged: position t of row b lies in page table[b * table_ld + (t >> page_log2)] of `pages`,
  // kb / vb elements apart; `lens` cached positions and `counts` (null: N) tokens behind them.
  // Tcap positions a table row covers; `chunk` is the fewest keys of a split.
  const int32_t* table;
  int64_t table_ld, pages;
  int page_log2;
  const int32_t* counts;
  const int32_t* order;  // the rows of the batch, longest first (null: as they are, or ranked)
  bool ranked;           // the longest rows first, of kRankedRows at most, found by each wave
  int rb_groups, rb_each;  // row blocks of a (b, key head, split) that share an XCD, and how many such groups
  // the scores of R rows, unscaled, -inf for hidden ones: (B, Hkv, R, scores_ld), where not null
  // (workgroups of 32 rows on the matrix cores)
  float* scores;
  int64_t scores_ld;
  // log2 (fp64: natural logarithm) of the sum of a row's exponentials, +inf for rows that see
  // nothing, where not null
  void* lse;
};

constexpr int kTileRows = 128;  // most rows of a packed tile
// most rows, and keys, of a sequence: positions a stage further on stay within 32 bits
constexpr int64_t kMostPositions = (int64_t)1 << 30;
constexpr unsigned kAtOnce = 1536;  // workgroups that start with the launch, about

// A workgroup's piece: the rows row0 .. row0 + rows - 1 of a sequence of `nrows` rows,
// over keys [kbeg, kend).  Query i sees key t iff t < own, or t < own + 64 and bit
// t - own of its mask; packed and paged: iff t <= i + off.
struct SeqPiece {
  int row0, rows;  // of the sequence's (query, head) rows
  int kbeg, kend;
  int off;         // packed: Lk - Lq; paged: own
  int own;         // tree, paged: the cached positions
  int count;       // paged: the row's tokens; those behind see nothing
  int64_t b;       // tree, paged: the row of the batch; packed: 0
  int64_t q0, k0;  // packed: the sequence's first rows in q and k
  int kvh, split;
};

// The cached positions and new tokens of a paged row, whatever its lengths say within what
// its table covers.
struct PagedRow {
  int own, count;
};
__device__ __forceinline__ PagedRow paged_row(const SeqArgs& a, int64_t b, int len) {
  PagedRow r;
  r.own = min(max(len, 0), a.Tcap);
  const int count = a.counts != nullptr ? __builtin_amdgcn_readfirstlane(a.counts[b]) : a.N;
  r.count = min(max(count, 0), min(a.N, a.Tcap - r.own));
  return r;
}
// Keys of each of its splits: as even as whole 128s allow, so that rows of every length are split
// as far as the launch has splits, and never fewer than a.chunk.  A stage of the matrix-core
// kernel has up to 256 keys (32 rows of up to 64 bytes a key), in key blocks that a split has
// whole or not at all.
__device__ __forceinline__ int paged_chunk(const SeqArgs& a, const PagedRow& r) {
  const int even = (r.own + r.count + a.nsplit - 1) / a.nsplit;
  return max(a.chunk, (even + 127) & ~127);
}
// The nth row of the batch by how many positions its tokens see, in whole 64s, the most first,
// and its lengths: a lane has a row, whose rank every wave counts for itself (0.3 us of each
// workgroup; a launch that ranks is 4 us of the call: 48 x 1 token behind 100 - 4096, 16 heads
// on 4 of 128, with weights, 62.6 / 59.6, 64 of 8 on 8 without 115.8 / 113.9).
constexpr int kRankedRows = 64;
__device__ __forceinline__ int paged_nth(const SeqArgs& a, int nth, PagedRow& r) {
  const int lane = threadIdx.x & 63, b = min(lane, a.B - 1);
  const int own = min(max(a.lens[b], 0), a.Tcap);
  const int count = min(max(a.counts != nullptr ? a.counts[b] : a.N, 0), min(a.N, a.Tcap - own));
  const int key = lane < a.B ? ((count > 0 ? own + count : 0) & ~63) | (63 - lane) : -1;
  int rank = 0;
  for (int j0 = 0; j0 < a.B; j0 += 8)
#pragma unroll
    for (int j = 0; j < 8; ++j) rank += __builtin_amdgcn_readlane(key, j0 + j) > key;
  const int at = __builtin_ctzll(__builtin_amdgcn_ballot_w64(lane < a.B && rank == nth));
  r.own = __builtin_amdgcn_readlane(own, at);
  r.count = __builtin_amdgcn_readlane(count, at);
  return at;
}
// The keys that the row block with (query, head) row `row` sees; 0 where it has no token.
__device__ __forceinline__ int paged_end(const SeqArgs& a, const PagedRow& r, int row) {
  const int row0 = row / a.rows_per_wg * a.rows_per_wg;
  if (row0 / a.G >= r.count) return 0;
  return r.own + min(r.count, (min(row0 + a.rows_per_wg, a.N * a.G) - 1) / a.G + 1);
}

// The piece of this workgroup; false where there is nothing to do.  Nothing a table or
// a length in device memory says takes an access outside q, k, v and y: tiles that do
// not lie inside them are left out, lengths beyond the cache are taken as its end.
template <SeqMode MODE>
__device__ __forceinline__ bool seq_piece(const SeqArgs& a, SeqPiece& p) {
  if constexpr (MODE >= kPaged) {
    // workgroup x runs on XCD x mod 8: groups of row blocks, which read the same keys, follow
    // each other there, the last rows first, which see the most
    const unsigned t = blockIdx.x >> 3;
    const unsigned each = t % (unsigned)a.rb_each;
    unsigned u = t / (unsigned)a.rb_each * 8 + (blockIdx.x & 7u);
    const int rb = a.nrb - 1 - (int)(u % (unsigned)a.rb_groups * (unsigned)a.rb_each + each);
    u /= (unsigned)a.rb_groups;
    p.split = (int)(u % (unsigned)a.nsplit);
    u /= (unsigned)a.nsplit;
    p.kvh = (int)(u % (unsigned)a.Hkv);
    u /= (unsigned)a.Hkv;
    if (rb < 0 || u >= (unsigned)a.B) return false;  // the grid is rounded up
    PagedRow r;
    if (a.ranked) {
      p.b = paged_nth(a, (int)u, r);
    } else {
      p.b = a.order != nullptr ? __builtin_amdgcn_readfirstlane(a.order[u]) : (int)u;
      r = paged_row(a, p.b, __builtin_amdgcn_readfirstlane(a.lens[p.b]));
    }
    p.row0 = rb * a.rows_per_wg;
    p.rows = min(a.rows_per_wg, a.N * a.G - p.row0);
    p.q0 = p.k0 = 0;
    p.own = p.off = r.own;
    p.count = r.count;
    const int chunk = paged_chunk(a, r);
    const int end = paged_end(a, r, p.row0);
    p.kbeg = p.split * chunk;  // below 2^31: fewer than a split more than the keys
    p.kend = min(end, p.kbeg + chunk);
    // the first split of unsplit rows that see nothing has their zeros to write
    return p.kbeg < p.kend || a.nsplit == 1;
  } else if constexpr (MODE == kTree) {
    // workgroup x runs on XCD x mod 8: the row blocks of a split, which read the same
    // keys, follow each other there
    const unsigned t = blockIdx.x >> 3;
    const int rb = (int)(t % (unsigned)a.nrb);
    int64_t u = (int64_t)(t / (unsigned)a.nrb) * 8 + (blockIdx.x & 7u);
    p.split = (int)(u % a.nsplit);
    u /= a.nsplit;
    p.kvh = (int)(u % a.Hkv);
    p.b = u / a.Hkv;
    if (p.b >= a.B) return false;  // the grid is rounded up
    const int len = a.lens != nullptr ? __builtin_amdgcn_readfirstlane(a.lens[p.b]) : a.len;
    p.row0 = rb * a.rows_per_wg;
    p.rows = min(a.rows_per_wg, a.N * a.G - p.row0);
    p.off = 0;
    p.q0 = p.k0 = 0;
    p.own = min(max(len, 0), a.Tcap - a.N);
    p.kbeg = p.split * a.chunk;
    p.kend = min(p.own + a.N, p.kbeg + a.chunk);
    return p.kbeg < p.kend;
  } else {
    // Position u of the XCD's workgroups: a tile's parts follow each other, they share its
    // keys.  Where all run at once every other 32 of them, one for each CU, are taken in
    // reverse, so that no CU gets each time the most of 32 falling numbers of keys.
    // 48 chunks of up to 300 queries behind up to 3000 keys, fp16, head_dim 64 in groups
    // of 4: 59.9 us, reversed 56.4; 71 of 150 behind 1500, bf16, head_dim 128 51.2, 49.7.
    // (Reversed with four times as many workgroups: 689 -> 712.)
    unsigned u = blockIdx.x >> 3;
    if (gridDim.x <= kAtOnce && (u & 32u) != 0 && (u | 31u) < gridDim.x >> 3) u ^= 31u;
    const unsigned part = u % (unsigned)a.nrb;
    u /= (unsigned)a.nrb;
    // which entry: dg_packed_plan's lists, an XCD further for each key head
    const unsigned slot = u / (unsigned)a.Hkv;
    p.kvh = (int)(u - slot * (unsigned)a.Hkv);
    dg_packed_tile t = a.tiles[8 * (int64_t)slot + ((blockIdx.x - (unsigned)p.kvh) & 7u)];
    t.q0 = __builtin_amdgcn_readfirstlane(t.q0);
    t.lq = __builtin_amdgcn_readfirstlane(t.lq);
    t.k0 = __builtin_amdgcn_readfirstlane(t.k0);
    t.lk = __builtin_amdgcn_readfirstlane(t.lk);
    t.row0 = __builtin_amdgcn_readfirstlane(t.row0);
    t.rows = __builtin_amdgcn_readfirstlane(t.rows);
    p.split = 0;
    p.b = 0;
    p.own = 0;
    if (t.lq <= 0 || t.lk < 0 || t.q0 < 0 || t.k0 < 0 || (int64_t)t.q0 + t.lq > a.nq || (int64_t)t.k0 + t.lk > a.nk)
      return false;
    if (t.row0 < 0 || t.rows <= 0 || t.rows > kTileRows || (int64_t)t.row0 + t.rows > (int64_t)t.lq * a.G) return false;
    // the workgroup's part of the tile
    t.row0 += (int)part * a.rows_per_wg;
    t.rows = min(a.rows_per_wg, t.rows - (int)part * a.rows_per_wg);
    if (t.rows <= 0) return false;
    p.row0 = t.row0;
    p.rows = t.rows;
    p.off = t.lk - t.lq;
    p.q0 = t.q0;
    p.k0 = t.k0;
    p.kbeg = 0;
    // the keys that the tile's last query sees
    p.kend = max(0, (t.row0 + t.rows - 1) / a.G + p.off + 1);
    return true;
  }
}

// sum += x, with what rounding added to the sum the time before taken out of x first (Kahan,
// "Further remarks on reducing truncation errors", 1965).  A row's weights are added one
// small number after the other to a sum that one key may dominate: without it, 100000 keys
// that are 2^25 times less likely than one other leave 0.1 % of the row's weight out.
template <typename A>
__device__ __forceinline__ void add_rounded(A& sum, A& rounding, A x) {
  const A y = x - rounding;
  const A s = sum + y;
  rounding = (s - sum) - y;
  sum = s;
}

// The tokens of the tree that token n of row b sees.
__device__ __forceinline__ uint64_t tree_mask(const SeqArgs& a, int64_t b, int n) {
  const uint64_t all = a.N >= 64 ? ~0ull : (1ull << a.N) - 1;
  if (a.masks == nullptr) return n >= 63 ? ~0ull : (2ull << n) - 1;
  return (uint64_t)a.masks[b * a.mask_b + n] & all;
}

// Positions that the matrix-core kernels copy from one page at a time: eight, or the rows that a
// wave's 64 pieces of 16 bytes cover.
constexpr int paged_granule(int D, int es) { return 1024 / (D * es) > 8 ? 1024 / (D * es) : 8; }

// The head_dim that the matrix-core kernels and their workspaces round D (up to 256) up to.
constexpr int seq_mfma_dim(int D) { return D <= 16 ? 16 : D <= 32 ? 32 : D <= 64 ? 64 : D <= 128 ? 128 : 256; }

// dg_attn_seq_mfma.hip: whether it takes the shape, the rows of a tree's workgroup over so
// many (token, head) rows and of a packed tile's, and its launches
bool seq_mfma_applicable(const SeqArgs& a, int dtype, bool tree);
int seq_mfma_tree_rows(int64_t B, int rows, int Hkv, int keys, int D, int dtype);
int seq_mfma_packed_rows(const int64_t counts[3], int Hkv, int D);
int launch_seq_mfma_packed(const SeqArgs& a, int dtype, dim3 grid, hipStream_t s);
int launch_seq_mfma_tree(const SeqArgs& a, int dtype, unsigned blocks, hipStream_t s);

}  // namespace dg
