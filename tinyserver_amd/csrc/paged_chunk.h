// Attention of a chunk of new tokens a sequence over the paged cache that holds
// them and the tokens before them (tsa_paged_chunk): the argument block, what a row
// sees, and what the entry point calls.
#pragma once

#include <cmath>

#include "paged_rows.h"

namespace tsa {

// What a workgroup's second launch needs of run r: the item that r starts inside of.
struct ChunkSplit {
  int64_t row0;              // packed row of the item's first query
  int32_t kvh, queries;      // its kv head and queries
  int32_t runs;              // runs r .. r + runs - 1 end it; 0: r is not its first cut
};
struct ChunkArgs {
  void* out;
  const void* q;
  const void* kc;
  const void* vc;
  const int32_t* bt;
  const int32_t* ctx;  // (B) tokens of each sequence before its new ones
  const int32_t* cu;   // (B + 1) ranges of the packed new tokens
  int64_t o_sr, o_sh, o_sd, q_sr, q_sh, q_sd;
  int64_t kc_b, kc_h, kc_s, kc_d, vc_b, vc_h, vc_s, vc_d;
  int64_t bt_s0, bt_s1, ctx_s, cu_s;
  int64_t NB, N;  // pages; packed rows
  int32_t B, Hq, Hkv, G, BS, max_blocks, D;
  int32_t T;      // rows of a sequence that are computed, at most
  float scale_log2;
  // The matrix-core form: page strides in bytes, the tiles (16 tokens) of a page as
  // a multiplier and a shift (page_of_tile), whether output rows go in pieces
  // of four; the queries of a row block, the least blocks of a run, whether runs are
  // whole items, and 2^16 / G rounded up (row / G of a row block's 256 at most).
  uint32_t k_page, v_page, page_mul, page_shift;
  int32_t out8, QB, min_run, whole, g_mul;
  // Its workspace: the number of runs, their splits and partial results.
  int32_t* runs;
  ChunkSplit* splits;
  float* part;
};

constexpr float kNegInfC = -INFINITY;

// A sequence's rows row0 .. row0 + n - 1 of q/out stand at positions ctx ..; end:
// past its last token that the block table holds. Row i sees the keys below
// min(ctx + i + 1, end).
struct ChunkSeq {
  int ctx, n, end;
  int64_t row0;
};
__device__ __forceinline__ ChunkSeq chunk_seq(const ChunkArgs& a, int s) {
  ChunkSeq r;
  const int64_t cap = static_cast<int64_t>(a.max_blocks) * a.BS;  // (below 2^27)
  int64_t c = a.ctx[s * a.ctx_s];
  c = c < 0 ? 0 : c > cap ? cap : c;
  int64_t r0 = a.cu[s * a.cu_s], r1 = a.cu[(s + 1) * a.cu_s];
  r0 = r0 < 0 ? 0 : r0 > a.N ? a.N : r0;
  r1 = r1 < r0 ? r0 : r1 > a.N ? a.N : r1;
  const int64_t n = r1 - r0 < a.T ? r1 - r0 : a.T;
  r.ctx = static_cast<int>(c);
  r.n = static_cast<int>(n);
  r.end = static_cast<int>(c + n < cap ? c + n : cap);
  r.row0 = r0;
  return r;
}

// paged_chunk_stream.hip: the plan of a call on the matrix cores (runs 0: sizes past
// its limits) and its launch; paged_chunk_f32.hip: that of float32 calls.
struct ChunkPlan {
  int runs, waves, QB, min_run, whole;
  size_t bytes;
};
ChunkPlan chunk_plan(int64_t B, int64_t N, int64_t T, int64_t Hq, int64_t Hkv, int64_t D, int64_t cap, bool f32);
int chunk_stream_launch(ChunkArgs& a, const ChunkPlan& p, int dt, void* workspace, hipStream_t stream);
int chunk_f32_launch(const ChunkArgs& a, const ChunkPlan& p, hipStream_t stream);

}  // namespace tsa
