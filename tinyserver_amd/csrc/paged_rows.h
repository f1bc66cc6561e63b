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
  int32_t S;          // splits of a unit's tokens
  float scale_log2;
  float* part;        // their partials
};

constexpr float kNegInfR = -INFINITY;

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
    const int64_t n = r1 - r0 < a.T ? r1 - r0 : a.T;
    r.row0 = r0;
    r.nodes = static_cast<int>(n);
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

// Host side: the checks of the entry points. k_scale and v_scale are NULL for
// caches of query's dtype; cu_nodes and tree_mask are NULL but for trees.
int check_rows(const tsa_view* out, const tsa_view* query, const tsa_view* k_cache, const tsa_view* v_cache,
               const tsa_view* k_scale, const tsa_view* v_scale, const tsa_view* block_tables, const tsa_view* lens,
               const tsa_view* cu_nodes, const tsa_view* tree_mask, int64_t max_nodes, int64_t window, int64_t sinks,
               double softmax_scale, RowsArgs& a);

// paged_rows_unit.hip: the decode forms on the matrix cores. Splits of a unit of
// at most max_tiles visible 16-token tiles, and the launch (a.S, a.part set).
int rows_unit_splits(int64_t max_tiles, bool cache8);
int rows_unit_launch(const RowsArgs& a, int dt, int cache_dt, hipStream_t stream, const char* what);

}  // namespace tsa
