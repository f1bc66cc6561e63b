// Attention of a few query rows per sequence over the paged cache, where a row
// sees part of it: the decode step with a sliding window and first tokens, the
// decode step over an 8-bit cache, and the verification of a tree of drafted
// tokens. The argument block and what a row sees.
#pragma once

#include <cmath>

#include "cache8.h"

namespace tsa {

struct RowsArgs {
  void* out;
  const void* q;
  const void* kc;
  const void* vc;
  const float* ks;  // 8-bit caches: scales (NB, Hkv, BS), else null
  const float* vs;
  const int32_t* bt;
  const int32_t* lens;   // (B) tokens of each sequence that are not drafted ones
  const int32_t* cu;     // trees: (B + 1) ranges of the packed rows, else null (row s is sequence s's)
  const uint32_t* mask;  // trees: 32-bit words of the rows' node masks
  int64_t o_sr, o_sh, o_sd, q_sr, q_sh, q_sd;
  int64_t kc_b, kc_h, kc_s, kc_d, vc_b, vc_h, vc_s, vc_d;
  int64_t ks_b, ks_h, ks_s, vs_b, vs_h, vs_s;
  int64_t bt_s0, bt_s1, len_s, cu_s, mask_s;  // (mask_s in 32-bit words)
  int64_t NB, N;      // pages; packed rows
  int32_t B, Hq, Hkv, G, BS, max_blocks, D;
  int32_t T;          // trees: rows of a sequence that are computed; else 1
  int32_t words;      // trees: 32-bit words of a row's mask
  int32_t window;     // the last tokens a row sees (0: all)
  int32_t sinks;      // the first tokens that stay visible
  int32_t S;          // splits of a unit's tokens (0: the stream)
  int32_t NW;         // waves of the stream
  int32_t out8;       // output rows are unit-stride, in 8-byte pieces
  int32_t RT, RB, per_split;  // trees: 32-row tiles of a workgroup, row blocks of a unit, most 32-key blocks of a split
  int32_t order;              // trees: workgroups take the sequences by length (TreeOrder)
  // The matrix-core forms: page strides in bytes, and the tiles (16 tokens) of a
  // page as a multiplier and a shift (tiles_of_page).
  uint32_t k_page, v_page, ks_page, vs_page, page_mul, page_shift;
  float scale_log2;
  float* part;        // their partials
  int32_t* pref;      // the stream: tile pairs before each sequence
};

constexpr float kNegInfR = -INFINITY;

// tile / (BS / 16) for tiles below 2^23 (tables hold less than 2^27 tokens):
// (tile * mul) >> (23 + shift) with shift = ceil(log2 d), mul = ceil(2^(23 +
// shift) / d), whose error, less than d <= 2^shift in 2^(23 + shift), stays
// below a unit of 1 / d for tiles below 2^23.
__host__ __device__ __forceinline__ uint32_t page_of_tile(uint32_t tile, uint32_t mul, uint32_t shift) {
  return static_cast<uint32_t>((static_cast<uint64_t>(tile) * mul) >> (23 + shift));
}
inline void page_div(int64_t block_size, uint32_t& mul, uint32_t& shift) {
  const uint64_t d = static_cast<uint64_t>(block_size) / 16;
  shift = 0;
  while ((uint64_t{1} << shift) < d) ++shift;
  mul = static_cast<uint32_t>(((uint64_t{1} << (23 + shift)) + d - 1) / d);
}
inline void set_page_div(RowsArgs& a) { page_div(a.BS, a.page_mul, a.page_shift); }

// A sequence's tokens: ctx of the cache's, then the drafted nodes at positions
// ctx .. ctx + nodes - 1; end is past the last that its block table holds. rows
// of q/out start at row0 (nodes of them). lo: first token of the window.
struct SeqRange {
  int ctx, nodes, end, lo;
  int64_t row0;
};
__device__ __forceinline__ SeqRange seq_of(const RowsArgs& a, int s) {
  SeqRange r;
  const int64_t cap = a.NB > 0 ? static_cast<int64_t>(a.max_blocks) * a.BS : 0;
  int64_t len = a.lens[s * a.len_s];
  len = len < 0 ? 0 : len > cap ? cap : len;
  if (a.cu) {
    int64_t r0 = a.cu[s * a.cu_s], r1 = a.cu[(s + 1) * a.cu_s];
    r0 = r0 < 0 ? 0 : r0 > a.N ? a.N : r0;
    r1 = r1 < r0 ? r0 : r1 > a.N ? a.N : r1;
    const int64_t held = 32 * static_cast<int64_t>(a.words), n = r1 - r0 < held ? r1 - r0 : held;  // (those a mask names)
    r.row0 = r0;
    r.nodes = static_cast<int>(n < a.T ? n : a.T);
    r.end = static_cast<int>(len + n < cap ? len + n : cap);
  } else {
    r.row0 = s;
    r.nodes = 1;
    r.end = static_cast<int>(len);
  }
  r.ctx = static_cast<int>(len);
  r.lo = a.window > 0 && r.ctx > a.window ? r.ctx - a.window : 0;
  return r;
}

// Sequences of a call whose workgroups take them by length: one a thread of the
// smaller workgroup (two waves). With the order / without, us: trees of 4-16 nodes,
// 32/8 heads, 512-4096 tokens, 64 sequences 123 / 137, 96 177 / 205, 128 241 / 267;
// 128 of 100-2048 122 / 131; of 40-64 nodes, 64/8 heads, 16 of 2000-8192 212 / 227.
constexpr int kTreeOrderSeqs = 128;
// 32-key blocks of a tree's splits: the unit's own, evenly, in fours (a wave each).
__device__ __forceinline__ int tree_per_split(const RowsArgs& a, int nblk) {
  const int even = ((nblk + a.S - 1) / a.S + 3) & ~3;
  return min(a.per_split, max(even, 16));
}

// Host side: the checks of the entry points. k_scale and v_scale are NULL for
// caches of query's dtype; cu_nodes and tree_mask are NULL but for trees.
int check_rows(const tsa_view* out, const tsa_view* query, const tsa_view* k_cache, const tsa_view* v_cache,
               const tsa_view* k_scale, const tsa_view* v_scale, const tsa_view* block_tables, const tsa_view* lens,
               const tsa_view* cu_nodes, const tsa_view* tree_mask, int64_t max_nodes, int64_t window, int64_t sinks,
               double softmax_scale, RowsArgs& a);

constexpr int kRowsMaxSeqs = 4096;  // sequences of one decode launch (the stream's prefix is in LDS)
// The plan of a decode launch on the matrix cores: splits of a unit (0: the
// stream, of `waves` waves) and the workspace, part_bytes of partials and the
// stream's prefix.
struct DecodeRowsPlan {
  int S, waves;
  size_t part_bytes, total;
};
DecodeRowsPlan decode_rows_plan(int64_t B, int64_t Hq, int64_t Hkv, int64_t D, int64_t cap, int64_t window,
                                int64_t sinks);
// paged_rows_unit.hip, paged_rows_stream.hip: the launches (a.S, a.NW, a.part, a.pref set).
int rows_unit_launch(const RowsArgs& a, int dt, int cache_dt, hipStream_t stream, const char* what);
int rows_stream_launch(const RowsArgs& a, int dt, int cache_dt, hipStream_t stream, const char* what);
// paged_rows_tree.hip: the plan of a tree call of at most T nodes a sequence (S 0: too
// many workgroups or rows for it), and the launch.
struct TreeRowsPlan {
  int RT, RB, S, per_split;
  size_t bytes;
};
TreeRowsPlan tree_rows_plan(int64_t B, int64_t T, int64_t Hq, int64_t Hkv, int64_t D, int64_t cap);
int rows_tree_launch(const RowsArgs& a, int dt, hipStream_t stream);

}  // namespace tsa
