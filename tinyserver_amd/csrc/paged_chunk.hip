// Attention of a chunk of new tokens over the paged cache (paged_chunk.h): the
// entry point, and the kernel for every shape.
//
//   out[i, h] = sum_j p_j V_j,  p = softmax_j(q[i, h] . K_j scale),  j <= ctx + i
//
// over one sequence's cache rows j (kv head h / G), whose last ones are the chunk's
// own, stored before the call.
#include "paged_chunk.h"

namespace tsa {

// Any strides, page size and head_dim up to 512: one wave per (row, q-head), fp32
// on the vector units. Lane j scores token base + j of a 64-token run; the run's
// visible tokens then stream V with lanes over dims. Tokens that a row does not see
// are not read.
template <typename T>
__global__ __launch_bounds__(64) void paged_chunk_generic(ChunkArgs a) {
  const int lane = threadIdx.x;
  constexpr int kMaxPerLane = 8;  // D <= 512
  const int64_t items = a.N * a.Hq;
  for (int64_t it = blockIdx.x; it < items; it += gridDim.x) {
    const int h = static_cast<int>(it % a.Hq), kvh = h / a.G, D = a.D;
    const int64_t row = it / a.Hq;
    int lo = 0, hi = a.B;  // the last sequence that starts at or before the row
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (a.cu[mid * a.cu_s] <= row) lo = mid; else hi = mid;
    }
    const int s = lo;
    const ChunkSeq r = chunk_seq(a, s);
    if (row < r.row0 || row >= r.row0 + r.n) continue;
    const int64_t upto = int64_t{r.ctx} + (row - r.row0) + 1;
    const int end = static_cast<int>(upto < r.end ? upto : r.end);
    const T* const qrow = static_cast<const T*>(a.q) + row * a.q_sr + h * a.q_sh;
    const T* const kbase = static_cast<const T*>(a.kc) + kvh * a.kc_h;
    const T* const vbase = static_cast<const T*>(a.vc) + kvh * a.vc_h;
    const int32_t* const bt_row = a.bt + s * a.bt_s0;
    float acc[kMaxPerLane];
#pragma unroll
    for (int i = 0; i < kMaxPerLane; ++i) acc[i] = 0.f;
    float m = kNegInfC, l = 0.f;
    for (int base = 0; base < end; base += 64) {
      const int tok = base + lane;
      bool sees = tok < end;
      int phys = 0, slot = 0;
      float sc = kNegInfC;
      if (sees) {
        const int lb = tok / a.BS;
        phys = bt_row[lb * a.bt_s1];
        slot = tok - lb * a.BS;
        sees = phys >= 0 && phys < a.NB;
      }
      if (sees) {
        float dot = 0.f;
        const T* const kr = kbase + phys * a.kc_b + slot * a.kc_s;
        for (int d = 0; d < D; ++d) dot += to_float(qrow[d * a.q_sd]) * to_float(kr[d * a.kc_d]);
        sc = dot * a.scale_log2;
      }
      float cmax = sc;
      for (int off = 32; off >= 1; off >>= 1) cmax = fmaxf(cmax, __shfl_xor(cmax, off, 64));
      const float m_new = fmaxf(m, cmax), mu = m_new == kNegInfC ? 0.f : m_new;
      const float alpha = fast_exp2(m - mu);
      const float p = fast_exp2(sc - mu);  // (a visible NaN stays one)
      float psum = p;
      for (int off = 32; off >= 1; off >>= 1) psum += __shfl_xor(psum, off, 64);
      l = l * alpha + psum;
#pragma unroll
      for (int i = 0; i < kMaxPerLane; ++i) acc[i] *= alpha;
      for (uint64_t left = __ballot(sees); left; left &= left - 1) {
        const int j = __builtin_ctzll(left);
        const float pj = __shfl(p, j, 64);
        const int64_t pg = __shfl(phys, j, 64), sl = __shfl(slot, j, 64);
        const T* const vr = vbase + pg * a.vc_b + sl * a.vc_s;
#pragma unroll
        for (int i = 0; i < kMaxPerLane; ++i) {
          const int d = lane + 64 * i;
          if (d < D) acc[i] += pj * to_float(vr[d * a.vc_d]);
        }
      }
      m = m_new;
    }
    T* const orow = static_cast<T*>(a.out) + row * a.o_sr + h * a.o_sh;
#pragma unroll
    for (int i = 0; i < kMaxPerLane; ++i) {
      const int d = lane + 64 * i;
      if (d < D) orow[d * a.o_sd] = from_float<T>(l == 0.f ? 0.f : acc[i] / l);
    }
  }
}

template <typename T>
static int launch_generic(const ChunkArgs& a, hipStream_t stream) {
  const int64_t items = a.N * a.Hq;
  paged_chunk_generic<T><<<dim3(static_cast<uint32_t>(items < (1 << 20) ? items : 1 << 20)), dim3(64), 0, stream>>>(a);
  return check_launch("tsa_paged_chunk");
}

// The matrix-core forms: head_dim 64 or 128, pages of whole 16-token tiles, unit-stride
// rows of 16-byte pieces, strides whose offsets within a page fit 31 bits (a page's own
// 32), and in 16 bits a positive scale (their maximum is one of raw scores). Fills what
// they need of a.
static bool takes_mfma(ChunkArgs& a, const tsa_view* out, const tsa_view* query, const tsa_view* k_cache,
                       const tsa_view* v_cache) {
  const bool f32 = query->dtype == TSA_F32;
  if ((a.D != 64 && a.D != 128) || a.BS % 16 || a.max_blocks == 0 || !(f32 || a.scale_log2 > 0.f)) return false;
  if (!rows_vec16(query) || !rows_vec16(k_cache) || !rows_vec16(v_cache)) return false;
  auto fits = [&](int64_t page, int64_t slot) {
    return page >= 0 && page < (int64_t{1} << 31) && slot >= 0 && slot < (int64_t{1} << 30) / a.BS;  // (elements)
  };
  if (!fits(a.kc_b, a.kc_s) || !fits(a.vc_b, a.vc_s)) return false;
  a.k_page = static_cast<uint32_t>(a.kc_b * 2);
  a.v_page = static_cast<uint32_t>(a.vc_b * 2);
  a.out8 = a.o_sd == 1 && a.o_sr % 4 == 0 && a.o_sh % 4 == 0 && reinterpret_cast<uintptr_t>(out->data) % (f32 ? 16 : 8) == 0;
  page_div(a.BS, a.page_mul, a.page_shift);
  return true;
}

// The checks of the entry point.
static int check_chunk(const tsa_view* out, const tsa_view* query, const tsa_view* k_cache, const tsa_view* v_cache,
                       const tsa_view* block_tables, const tsa_view* context_lens, const tsa_view* cu_seqlens,
                       int64_t max_seqlen, double softmax_scale, ChunkArgs& a) {
  TSA_REQUIRE(view_ok(query, 3), "query must be a 3D tensor (num_tokens, num_heads, head_dim)");
  TSA_REQUIRE(view_ok(out, 3), "out must be a 3D tensor shaped like query");
  TSA_REQUIRE(view_ok(k_cache, 4) && view_ok(v_cache, 4),
              "k_cache and v_cache must be 4D tensors (num_blocks, num_kv_heads, block_size, head_dim)");
  TSA_REQUIRE(view_ok(block_tables, 2) && block_tables->dtype == TSA_I32,
              "block_tables must be a 2D int32 tensor (num_seqs, max_num_blocks_per_seq)");
  TSA_REQUIRE(view_ok(context_lens, 1) && context_lens->dtype == TSA_I32, "context_lens must be a 1D int32 tensor");
  const int dt = query->dtype;
  TSA_REQUIRE(is_float_dtype(dt) && out->dtype == dt && k_cache->dtype == dt && v_cache->dtype == dt,
              "query, out, k_cache and v_cache must share one floating dtype (got %s, %s, %s, %s)", dtype_name(dt),
              dtype_name(out->dtype), dtype_name(k_cache->dtype), dtype_name(v_cache->dtype));
  for (int d = 0; d < 3; ++d) TSA_REQUIRE(out->size[d] == query->size[d], "out must have query's shape");
  for (int d = 0; d < 4; ++d) TSA_REQUIRE(k_cache->size[d] == v_cache->size[d], "k_cache and v_cache must match");
  const int64_t N = query->size[0], Hq = query->size[1], D = query->size[2], B = block_tables->size[0];
  const int64_t NB = k_cache->size[0], Hkv = k_cache->size[1], BS = k_cache->size[2];
  TSA_REQUIRE(k_cache->size[3] == D, "cache head_dim %lld != query head_dim %lld", (long long)k_cache->size[3],
              (long long)D);
  TSA_REQUIRE(Hkv > 0 && Hq % Hkv == 0, "num_heads (%lld) must be a multiple of num_kv_heads (%lld)", (long long)Hq,
              (long long)Hkv);
  TSA_REQUIRE(BS > 0, "block_size must be positive");
  TSA_REQUIRE(context_lens->size[0] == B, "block_tables and context_lens must have the same number of rows (%lld and %lld)",
              (long long)B, (long long)context_lens->size[0]);
  TSA_REQUIRE(view_ok(cu_seqlens, 1) && cu_seqlens->dtype == TSA_I32 && cu_seqlens->size[0] == B + 1,
              "cu_seqlens must be a 1D int32 tensor (num_seqs + 1)");
  TSA_REQUIRE(max_seqlen >= 0, "max_seqlen must be non-negative (got %lld)", (long long)max_seqlen);
  TSA_REQUIRE(B < 65536 && Hq < 65536, "num_seqs and num_heads must be below 65536");
  // (each factor is bounded before the product)
  TSA_REQUIRE(BS < (int64_t{1} << 27) && block_tables->size[1] < (int64_t{1} << 27) &&
                  block_tables->size[1] * BS < (int64_t{1} << 27),
              "block table too long");
  TSA_UNSUPPORTED(N < (int64_t{1} << 27), "2^27 and more new tokens are not implemented");
  TSA_UNSUPPORTED(D <= 512, "head_dim %lld > 512 is not implemented", (long long)D);

  a = ChunkArgs{};
  a.out = out->data; a.q = query->data; a.kc = k_cache->data; a.vc = v_cache->data;
  a.bt = static_cast<const int32_t*>(block_tables->data);
  a.ctx = static_cast<const int32_t*>(context_lens->data);
  a.cu = static_cast<const int32_t*>(cu_seqlens->data);
  a.o_sr = out->stride[0]; a.o_sh = out->stride[1]; a.o_sd = out->stride[2];
  a.q_sr = query->stride[0]; a.q_sh = query->stride[1]; a.q_sd = query->stride[2];
  a.kc_b = k_cache->stride[0]; a.kc_h = k_cache->stride[1]; a.kc_s = k_cache->stride[2]; a.kc_d = k_cache->stride[3];
  a.vc_b = v_cache->stride[0]; a.vc_h = v_cache->stride[1]; a.vc_s = v_cache->stride[2]; a.vc_d = v_cache->stride[3];
  a.bt_s0 = block_tables->stride[0]; a.bt_s1 = block_tables->stride[1];
  a.ctx_s = context_lens->stride[0]; a.cu_s = cu_seqlens->stride[0];
  a.NB = NB; a.N = N;
  a.B = static_cast<int32_t>(B); a.Hq = static_cast<int32_t>(Hq); a.Hkv = static_cast<int32_t>(Hkv);
  a.G = static_cast<int32_t>(Hq / Hkv); a.BS = static_cast<int32_t>(BS);
  a.max_blocks = static_cast<int32_t>(NB > 0 ? block_tables->size[1] : 0); a.D = static_cast<int32_t>(D);
  a.T = static_cast<int32_t>(max_seqlen < N ? max_seqlen : N);
  a.scale_log2 = static_cast<float>(softmax_scale * 1.4426950408889634);
  return TSA_OK;
}

}  // namespace tsa

using namespace tsa;

extern "C" int tsa_paged_chunk(const tsa_view* out, const tsa_view* query, const tsa_view* k_cache,
                               const tsa_view* v_cache, const tsa_view* block_tables, const tsa_view* context_lens,
                               const tsa_view* cu_seqlens, int64_t max_seqlen, double softmax_scale, void* workspace,
                               size_t workspace_bytes, void* stream) {
  ChunkArgs a;
  if (int rc = check_chunk(out, query, k_cache, v_cache, block_tables, context_lens, cu_seqlens, max_seqlen,
                           softmax_scale, a))
    return rc;
  if (a.B == 0 || a.T == 0 || a.Hq == 0 || a.D == 0) return TSA_OK;
  const hipStream_t st = static_cast<hipStream_t>(stream);
  if (takes_mfma(a, out, query, k_cache, v_cache)) {
    const ChunkPlan p = chunk_plan(a.B, a.N, a.T, a.Hq, a.Hkv, a.D, int64_t{a.max_blocks} * a.BS,
                                   query->dtype == TSA_F32);
    if (p.runs > 0) {
      TSA_REQUIRE(workspace != nullptr && workspace_bytes >= p.bytes, "workspace of %zu bytes is too small: %zu needed",
                  workspace_bytes, p.bytes);
      TSA_REQUIRE(reinterpret_cast<uintptr_t>(workspace) % 256 == 0, "workspace must be 256-byte aligned");
      return chunk_stream_launch(a, p, query->dtype, workspace, st);
    }
  }
  switch (query->dtype) {
    case TSA_BF16: return launch_generic<bf16_t>(a, st);
    case TSA_F16: return launch_generic<f16_t>(a, st);
    default: return launch_generic<float>(a, st);
  }
}

extern "C" size_t tsa_paged_chunk_workspace_bytes(int64_t num_seqs, int64_t num_tokens, int64_t max_seqlen,
                                                  int64_t num_heads, int64_t num_kv_heads, int64_t head_dim,
                                                  int64_t max_blocks_per_seq, int64_t block_size) {
  if (num_seqs <= 0 || num_tokens <= 0 || max_seqlen <= 0 || num_heads <= 0 || num_kv_heads <= 0 ||
      num_heads % num_kv_heads || num_seqs >= 65536 || num_heads >= 65536 || num_tokens >= (int64_t{1} << 27) ||
      (head_dim != 64 && head_dim != 128) || block_size <= 0 || block_size >= (int64_t{1} << 27) || block_size % 16 ||
      max_blocks_per_seq <= 0 || max_blocks_per_seq >= (int64_t{1} << 27) ||
      max_blocks_per_seq * block_size >= (int64_t{1} << 27))
    return 0;  // (calls of such sizes are refused, have nothing to do, or take no workspace)
  const int64_t cap = max_blocks_per_seq * block_size;
  const size_t f16 = chunk_plan(num_seqs, num_tokens, max_seqlen, num_heads, num_kv_heads, head_dim, cap, false).bytes;
  const size_t f32 = chunk_plan(num_seqs, num_tokens, max_seqlen, num_heads, num_kv_heads, head_dim, cap, true).bytes;
  return f16 > f32 ? f16 : f32;
}
