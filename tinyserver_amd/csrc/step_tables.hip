// A step's block tables, positions and slots from its requests' lengths
// (tsa_step_tables), new pages taken off a free list.
//
// Request s has ctx_s tokens in the cache and q_s new ones; with pages of BS
// tokens it holds have_s = ceil(ctx_s / BS) of them and needs need_s = ceil((ctx_s +
// q_s) / BS). With exclusive sums Q_s of q and F_s of need - have in batch order:
//   token Q_s + i:  position ctx_s + i, in column (ctx_s + i) / BS of the table;
//   column have_s + i of request s takes free_blocks[num_free - 1 - (F_s + i)].
//
// One launch; what bounds it is its latency (lengths -> sums -> table entry ->
// store). Every workgroup sums all lengths itself, kSeqs at a time, rather than wait
// for another's sums, then takes its own run of tokens (a binary search over the
// sums in LDS) and its own requests' table columns. Measured: 8 requests of one token
// 4.8 us; 512 of 1-128 tokens (33,000 tokens, 512 x 512 columns) 6.9 with 256 tokens and
// a request a workgroup, 12.4 with 1,024 and two.
#include "tsa_common.h"

namespace tsa {

struct StepArgs {
  int32_t *bt, *cu, *seq, *pos, *blk, *slot, *left;  // outputs
  int32_t* tables;
  const int32_t *rows, *ctx, *q, *free_list, *num_free;  // rows, free_list, num_free may be null
  int64_t bt_s0, bt_s1, cu_s, seq_s, pos_s, blk_s, slot_s;
  int64_t t_s0, t_s1, rows_s, ctx_s, q_s, free_s;
  int64_t R, W, T, F;   // table rows and columns, tokens, entries of the free list
  int32_t B, width;
  uint32_t BS;
  bool take;            // pages are taken off the free list
};

constexpr int kStepThreads = 256, kStepPer = 4, kSeqs = kStepThreads * kStepPer;
constexpr int kStepTokens = 256;  // tokens of a workgroup

// Block-wide exclusive sums of x; total: of all threads.
__device__ __forceinline__ uint64_t block_scan(uint64_t x, uint64_t* waves, uint64_t& total) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const uint64_t incl = wave_scan_u64(x);
  if (lane == 63) waves[w] = incl;
  __syncthreads();
  uint64_t before = 0;
  total = 0;
#pragma unroll
  for (int i = 0; i < kStepThreads / 64; ++i) {
    before += i < w ? waves[i] : 0;
    total += waves[i];
  }
  __syncthreads();
  return before + incl - x;
}

__device__ __forceinline__ int32_t clamp31(uint64_t x) { return static_cast<int32_t>(x < 0x7FFFFFFFu ? x : 0x7FFFFFFFu); }

__global__ __launch_bounds__(kStepThreads) void step_tables_kernel(StepArgs a) {
  __shared__ uint64_t waves[kStepThreads / 64];
  __shared__ uint64_t tok_before[kSeqs];  // new tokens before each request of this round
  __shared__ uint64_t page_before[kSeqs];
  __shared__ int32_t s_ctx[kSeqs], s_have[kSeqs], s_need[kSeqs], s_row[kSeqs];
  const int tid = threadIdx.x;
  const uint64_t t0 = uint64_t{blockIdx.x} * kStepTokens, T = static_cast<uint64_t>(a.T);
  const uint64_t t1 = t0 + kStepTokens < T ? t0 + kStepTokens : T;
  int64_t nf = a.F;
  if (a.num_free) {
    nf = *a.num_free;
    nf = nf < 0 ? 0 : nf > a.F ? a.F : nf;
  }
  auto page_of = [&](int64_t row, uint32_t col, uint32_t have, uint64_t before) -> int32_t {
    if (row < 0 || col >= static_cast<uint64_t>(a.W)) return -1;
    if (col < have) return a.tables[row * a.t_s0 + col * a.t_s1];
    const int64_t at = nf - 1 - static_cast<int64_t>(before + (col - have));
    return at >= 0 ? a.free_list[at * a.free_s] : -1;
  };
  uint64_t tok_run = 0, page_run = 0;
  for (int base = 0; base < a.B; base += kSeqs) {
    // ---- This round's requests: lengths, pages, and the sums before each.
    uint32_t q[kStepPer], fresh[kStepPer];
    uint64_t q_sum = 0, f_sum = 0;
#pragma unroll
    for (int i = 0; i < kStepPer; ++i) {
      const int k = tid * kStepPer + i, s = base + k;
      int32_t c = 0, n = 0;
      int64_t row = -1;
      if (s < a.B) {
        c = a.ctx[s * a.ctx_s];
        n = a.q[s * a.q_s];
        row = a.rows ? a.rows[s * a.rows_s] : s;
        if (row >= a.R) row = -1;
      }
      constexpr int kLongest = (1 << 30) - 1;
      const uint32_t cc = c > 0 ? min(c, kLongest) : 0, nn = n > 0 ? min(n, kLongest) : 0;
      const uint32_t W = static_cast<uint32_t>(a.W);
      const uint32_t need = min((cc + nn + a.BS - 1) / a.BS, W);
      const uint32_t have = a.take ? min((cc + a.BS - 1) / a.BS, W) : need;
      q[i] = nn;
      fresh[i] = row < 0 ? 0 : need - have;
      q_sum += nn;
      f_sum += fresh[i];
      s_ctx[k] = static_cast<int32_t>(cc);
      s_have[k] = static_cast<int32_t>(have);
      s_need[k] = static_cast<int32_t>(need);
      s_row[k] = static_cast<int32_t>(row);
    }
    uint64_t q_total, f_total;
    uint64_t qb = tok_run + block_scan(q_sum, waves, q_total), fb = page_run + block_scan(f_sum, waves, f_total);
#pragma unroll
    for (int i = 0; i < kStepPer; ++i) {
      const int k = tid * kStepPer + i, s = base + k;
      tok_before[k] = qb;
      page_before[k] = fb;
      qb += q[i];
      fb += fresh[i];
      if (s < a.B && s % static_cast<int>(gridDim.x) == static_cast<int>(blockIdx.x)) {
        a.cu[(s + 1) * a.cu_s] = clamp31(qb);
        a.seq[s * a.seq_s] = clamp31(uint64_t{static_cast<uint32_t>(s_ctx[k])} + q[i]);
      }
    }
    __syncthreads();
    const int here = min(kSeqs, a.B - base);
    // ---- Tables of every gridDim.x-th request.
    const int first = (static_cast<int>(blockIdx.x) - base % static_cast<int>(gridDim.x) + static_cast<int>(gridDim.x)) %
                      static_cast<int>(gridDim.x);
    for (int k = first; k < here; k += gridDim.x) {
      const int64_t row = s_row[k], s = base + k;
      const uint32_t have = s_have[k], need = s_need[k];
      const uint64_t before = page_before[k];
      for (uint32_t col = tid; col < max(static_cast<uint32_t>(a.width), need); col += kStepThreads) {
        const int32_t page = col < need ? page_of(row, col, have, before) : 0;
        if (col >= have && col < need && row >= 0) a.tables[row * a.t_s0 + col * a.t_s1] = page;
        if (col < static_cast<uint32_t>(a.width)) a.bt[s * a.bt_s0 + col * a.bt_s1] = page;
      }
    }
    // ---- This workgroup's tokens among the round's.
    const uint64_t lo = t0 > tok_run ? t0 : tok_run, hi = t1 < tok_run + q_total ? t1 : tok_run + q_total;
    for (uint64_t t = lo + tid; t < hi; t += kStepThreads) {
      int l = 0, h = here;  // the last request that starts at or before t (those without tokens start with their next)
      while (h - l > 1) {
        const int mid = (l + h) >> 1;
        if (tok_before[mid] <= t) l = mid; else h = mid;
      }
      const uint32_t p = static_cast<uint32_t>(s_ctx[l]) + static_cast<uint32_t>(t - tok_before[l]);
      const uint32_t col = p / a.BS;
      a.pos[t * a.pos_s] = static_cast<int32_t>(p);
      a.slot[t * a.slot_s] = static_cast<int32_t>(p - col * a.BS);
      a.blk[t * a.blk_s] = page_of(s_row[l], col, s_have[l], page_before[l]);
    }
    tok_run += q_total;
    page_run += f_total;
    __syncthreads();
  }
  // ---- Tokens that no request has.
  for (uint64_t t = (t0 > tok_run ? t0 : tok_run) + tid; t < t1; t += kStepThreads) {
    a.pos[t * a.pos_s] = 0;
    a.slot[t * a.slot_s] = -1;
    a.blk[t * a.blk_s] = -1;
  }
  if (blockIdx.x == 0 && tid == 0) {
    a.cu[0] = 0;
    if (a.left) *a.left = static_cast<int32_t>(nf - static_cast<int64_t>(page_run) < INT32_MIN
                                                   ? INT32_MIN : nf - static_cast<int64_t>(page_run));
  }
}

}  // namespace tsa

using namespace tsa;

static int ints(const tsa_view* v, int64_t n, const char* name) {
  TSA_REQUIRE(view_ok(v, 1) && v->dtype == TSA_I32 && v->size[0] == n, "%s must be a 1D int32 tensor of %lld", name,
              (long long)n);
  return TSA_OK;
}

extern "C" int tsa_step_tables(const tsa_view* block_tables, const tsa_view* cu_seqlens, const tsa_view* seq_lens,
                               const tsa_view* positions, const tsa_view* block_mapping, const tsa_view* slot_mapping,
                               const tsa_view* free_left, const tsa_view* tables, const tsa_view* rows,
                               const tsa_view* context_lens, const tsa_view* query_lens, const tsa_view* free_blocks,
                               const tsa_view* num_free, int64_t block_size, void* stream) {
  TSA_REQUIRE(view_ok(tables, 2) && tables->dtype == TSA_I32, "tables must be a 2D int32 tensor (rows, columns)");
  TSA_REQUIRE(view_ok(context_lens, 1) && context_lens->dtype == TSA_I32, "context_lens must be a 1D int32 tensor");
  const int64_t B = context_lens->size[0];
  TSA_REQUIRE(block_size >= 1 && block_size < (int64_t{1} << 27), "block_size must be positive (got %lld)",
              (long long)block_size);
  if (int rc = ints(query_lens, B, "query_lens")) return rc;
  if (rows) {
    if (int rc = ints(rows, B, "rows")) return rc;
  } else {
    TSA_REQUIRE(tables->size[0] >= B, "tables must have a row for each of the %lld requests", (long long)B);
  }
  TSA_REQUIRE(view_ok(block_tables, 2) && block_tables->dtype == TSA_I32 && block_tables->size[0] == B,
              "block_tables must be a 2D int32 tensor (num_seqs, width)");
  if (int rc = ints(cu_seqlens, B + 1, "cu_seqlens")) return rc;
  if (int rc = ints(seq_lens, B, "seq_lens")) return rc;
  TSA_REQUIRE(view_ok(positions, 1), "positions must be a 1D int32 tensor");
  const int64_t T = positions->size[0];
  if (int rc = ints(positions, T, "positions")) return rc;
  if (int rc = ints(block_mapping, T, "block_mapping")) return rc;
  if (int rc = ints(slot_mapping, T, "slot_mapping")) return rc;
  if (free_blocks) {
    TSA_REQUIRE(view_ok(free_blocks, 1) && free_blocks->dtype == TSA_I32, "free_blocks must be a 1D int32 tensor");
    if (num_free) {
      if (int rc = ints(num_free, 1, "num_free")) return rc;
    }
    if (int rc = ints(free_left, 1, "free_left")) return rc;
    TSA_REQUIRE(!num_free || free_left->data != num_free->data, "free_left may not be num_free");
  } else {
    TSA_REQUIRE(!num_free && !free_left, "num_free and free_left go with free_blocks");
  }
  constexpr int64_t kMost = int64_t{1} << 30;
  TSA_UNSUPPORTED(B <= kMost && T <= kMost && tables->size[0] <= kMost && tables->size[1] <= kMost &&
                      block_tables->size[1] <= kMost && (!free_blocks || free_blocks->size[0] <= kMost),
                  "sizes past 2^30 are not implemented");
  StepArgs a{};
  auto p = [](const tsa_view* v) { return v ? static_cast<int32_t*>(v->data) : nullptr; };
  a.bt = p(block_tables); a.cu = p(cu_seqlens); a.seq = p(seq_lens); a.pos = p(positions);
  a.blk = p(block_mapping); a.slot = p(slot_mapping); a.left = p(free_left);
  a.tables = p(tables); a.rows = p(rows); a.ctx = p(context_lens); a.q = p(query_lens);
  a.num_free = p(num_free);
  a.bt_s0 = block_tables->stride[0]; a.bt_s1 = block_tables->stride[1];
  a.cu_s = cu_seqlens->stride[0]; a.seq_s = seq_lens->stride[0]; a.pos_s = positions->stride[0];
  a.blk_s = block_mapping->stride[0]; a.slot_s = slot_mapping->stride[0];
  a.t_s0 = tables->stride[0]; a.t_s1 = tables->stride[1];
  a.rows_s = rows ? rows->stride[0] : 0;
  a.ctx_s = context_lens->stride[0]; a.q_s = query_lens->stride[0];
  if (free_blocks) {
    a.take = true;
    a.free_list = p(free_blocks);
    a.free_s = free_blocks->stride[0];
    a.F = free_blocks->size[0];
  }
  a.R = tables->size[0]; a.W = tables->size[1]; a.T = T;
  a.B = static_cast<int32_t>(B); a.width = static_cast<int32_t>(block_tables->size[1]);
  a.BS = static_cast<uint32_t>(block_size);
  // A workgroup for every kStepTokens tokens, and enough for a few requests each.
  const int64_t by_tokens = (T + kStepTokens - 1) / kStepTokens, by_tables = B < 1024 ? B : 1024;
  const int64_t grid = by_tokens > by_tables ? by_tokens : by_tables;
  step_tables_kernel<<<dim3(static_cast<uint32_t>(grid > 0 ? grid : 1)), dim3(kStepThreads), 0,
                       static_cast<hipStream_t>(stream)>>>(a);
  return check_launch("tsa_step_tables");
}
