// Attention of a few query rows per sequence over the paged cache
// (paged_rows.h): windowed decode, decode over 8-bit caches, draft trees. The
// entry points, and the form for what the matrix-core ones do not take
// (paged_rows_unit.h, paged_rows_stream.h; paged_rows_tree.h, paged_rows_tree_lds.h).
#include "paged_rows.h"

namespace tsa {

// Any strides, page size and head_dim up to 512: one wave per (row, q-head),
// fp32 on the vector units. Lane j scores token base + j of a 64-token chunk;
// the chunk's visible tokens then stream V with lanes over dims. Tokens a row
// does not see are not read (for its V) and not scored, whatever they hold.
template <typename T, typename C>
__global__ __launch_bounds__(64) void paged_rows_generic(RowsArgs a) {
  const int lane = threadIdx.x;
  constexpr int kMaxPerLane = 8;  // D <= 512
  const int64_t items = static_cast<int64_t>(a.B) * a.T * a.Hq;
  for (int64_t it = blockIdx.x; it < items; it += gridDim.x) {
    const int h = static_cast<int>(it % a.Hq), node = static_cast<int>(it / a.Hq % a.T);
    const int s = static_cast<int>(it / a.Hq / a.T), kvh = h / a.G, D = a.D;
    const SeqRange r = seq_of(a, s);
    if (node >= r.nodes) continue;
    const int64_t row = r.row0 + node;
    const T* const qrow = static_cast<const T*>(a.q) + row * a.q_sr + h * a.q_sh;
    const C* const kbase = static_cast<const C*>(a.kc) + kvh * a.kc_h;
    const C* const vbase = static_cast<const C*>(a.vc) + kvh * a.vc_h;
    const int32_t* const bt_row = a.bt + s * a.bt_s0;
    float acc[kMaxPerLane];
#pragma unroll
    for (int i = 0; i < kMaxPerLane; ++i) acc[i] = 0.f;
    float m = kNegInfR, l = 0.f;
    // The first tokens' chunks, then the window's (one run where they meet).
    const int first_end = r.lo > 0 ? min(a.sinks, r.lo) : 0;
    for (int base = first_end > 0 ? 0 : r.lo & ~63; base < r.end;
         base = base + 64 < first_end || base + 64 >= r.lo ? base + 64 : r.lo & ~63) {
      const int tok = base + lane;
      bool sees = tok < r.ctx && (tok >= r.lo || tok < first_end);
      if (a.cu && tok >= r.ctx && tok < r.end) {
        const int j = tok - r.ctx;
        sees = (j >> 5) < a.words && ((a.mask[row * a.mask_s + (j >> 5)] >> (j & 31)) & 1);
      }
      int64_t phys = 0, slot = 0;
      float sc = kNegInfR, vscale = 1.f;
      if (sees) {
        const int lb = tok / a.BS;
        phys = bt_row[lb * a.bt_s1];
        slot = tok - lb * a.BS;
        sees = phys >= 0 && phys < a.NB;
      }
      if (sees) {
        float dot = 0.f;
        const C* const kr = kbase + phys * a.kc_b + slot * a.kc_s;
        for (int d = 0; d < D; ++d) dot += to_float(qrow[d * a.q_sd]) * to_float(kr[d * a.kc_d]);
        if constexpr (sizeof(C) == 1) {
          dot *= a.ks[phys * a.ks_b + kvh * a.ks_h + slot * a.ks_s];
          vscale = a.vs[phys * a.vs_b + kvh * a.vs_h + slot * a.vs_s];
        }
        sc = dot * a.scale_log2;
      }
      float cmax = sc;
      for (int off = 32; off >= 1; off >>= 1) cmax = fmaxf(cmax, __shfl_xor(cmax, off, 64));
      const float m_new = fmaxf(m, cmax), mu = m_new == kNegInfR ? 0.f : m_new;
      const float alpha = fast_exp2(m - mu);
      const float p = fast_exp2(sc - mu);  // (a visible NaN stays one)
      float psum = p;
      for (int off = 32; off >= 1; off >>= 1) psum += __shfl_xor(psum, off, 64);
      l = l * alpha + psum;
#pragma unroll
      for (int i = 0; i < kMaxPerLane; ++i) acc[i] *= alpha;
      for (uint64_t left = __ballot(sees); left; left &= left - 1) {
        const int j = __builtin_ctzll(left);
        const float pj = __shfl(sizeof(C) == 1 ? p * vscale : p, j, 64);
        const int64_t pg = __shfl(static_cast<int>(phys), j, 64), sl = __shfl(static_cast<int>(slot), j, 64);
        const C* const vr = vbase + pg * a.vc_b + sl * a.vc_s;
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

template <typename T, typename C>
static int launch_rows(const RowsArgs& a, hipStream_t stream, const char* what) {
  const int64_t items = static_cast<int64_t>(a.B) * a.T * a.Hq;
  paged_rows_generic<T, C><<<dim3(static_cast<uint32_t>(items < (1 << 20) ? items : 1 << 20)), dim3(64), 0, stream>>>(a);
  return check_launch(what);
}

int check_rows(const tsa_view* out, const tsa_view* query, const tsa_view* k_cache, const tsa_view* v_cache,
               const tsa_view* k_scale, const tsa_view* v_scale, const tsa_view* block_tables, const tsa_view* lens,
               const tsa_view* cu_nodes, const tsa_view* tree_mask, int64_t max_nodes, int64_t window, int64_t sinks,
               double softmax_scale, RowsArgs& a) {
  const bool tree = cu_nodes != nullptr;
  const char* const len_name = tree ? "context_lens" : "seq_lens";
  TSA_REQUIRE(view_ok(query, 3), "query must be a 3D tensor (%s, num_heads, head_dim)", tree ? "num_nodes" : "num_seqs");
  TSA_REQUIRE(view_ok(out, 3), "out must be a 3D tensor shaped like query");
  TSA_REQUIRE(view_ok(k_cache, 4) && view_ok(v_cache, 4),
              "k_cache and v_cache must be 4D tensors (num_blocks, num_kv_heads, block_size, head_dim)");
  TSA_REQUIRE(view_ok(block_tables, 2) && block_tables->dtype == TSA_I32,
              "block_tables must be a 2D int32 tensor (num_seqs, max_num_blocks_per_seq)");
  TSA_REQUIRE(view_ok(lens, 1) && lens->dtype == TSA_I32, "%s must be a 1D int32 tensor", len_name);
  const int dt = query->dtype;
  const bool q8 = k_scale != nullptr || v_scale != nullptr;
  TSA_REQUIRE(is_float_dtype(dt) && out->dtype == dt, "query and out must share one floating dtype (got %s/%s)",
              dtype_name(dt), dtype_name(out->dtype));
  if (q8) {
    TSA_REQUIRE(is_cache8_dtype(k_cache->dtype) && v_cache->dtype == k_cache->dtype,
                "k_cache and v_cache must share one 8-bit dtype, e4m3 or int8 (got %s/%s)", dtype_name(k_cache->dtype),
                dtype_name(v_cache->dtype));
    TSA_REQUIRE(view_ok(k_scale, 3) && view_ok(v_scale, 3) && k_scale->dtype == TSA_F32 && v_scale->dtype == TSA_F32,
                "k_scale and v_scale must be 3D float32 tensors (num_blocks, num_kv_heads, block_size)");
    for (int d = 0; d < 3; ++d)
      TSA_REQUIRE(k_scale->size[d] == k_cache->size[d] && v_scale->size[d] == k_cache->size[d],
                  "k_scale and v_scale must have the cache's shape but its head_dim");
  } else {
    TSA_REQUIRE(k_cache->dtype == dt && v_cache->dtype == dt, "query, out, k_cache and v_cache must share one floating dtype");
  }
  for (int d = 0; d < 3; ++d) TSA_REQUIRE(out->size[d] == query->size[d], "out must have query's shape");
  for (int d = 0; d < 4; ++d) TSA_REQUIRE(k_cache->size[d] == v_cache->size[d], "k_cache and v_cache must match");
  const int64_t N = query->size[0], Hq = query->size[1], D = query->size[2], B = block_tables->size[0];
  const int64_t NB = k_cache->size[0], Hkv = k_cache->size[1], BS = k_cache->size[2];
  TSA_REQUIRE(k_cache->size[3] == D, "cache head_dim %lld != query head_dim %lld", (long long)k_cache->size[3],
              (long long)D);
  TSA_REQUIRE(Hkv > 0 && Hq % Hkv == 0, "num_heads (%lld) must be a multiple of num_kv_heads (%lld)", (long long)Hq,
              (long long)Hkv);
  TSA_REQUIRE(BS > 0, "block_size must be positive");
  TSA_REQUIRE(lens->size[0] == B, "block_tables and %s must have the same number of rows (%lld and %lld)", len_name,
              (long long)B, (long long)lens->size[0]);
  if (tree) {
    TSA_REQUIRE(view_ok(cu_nodes, 1) && cu_nodes->dtype == TSA_I32 && cu_nodes->size[0] == B + 1,
                "cu_nodes must be a 1D int32 tensor (num_seqs + 1)");
    TSA_REQUIRE(view_ok(tree_mask, 2) && tree_mask->dtype == TSA_I64 && tree_mask->size[0] == N,
                "tree_mask must be a 2D int64 tensor (num_nodes, words)");
    TSA_REQUIRE(tree_mask->size[1] >= 1 || N == 0, "tree_mask must have at least one word a node");
    TSA_REQUIRE(tree_mask->stride[1] == 1 || tree_mask->size[1] <= 1, "tree_mask's words must be contiguous");
    TSA_UNSUPPORTED(tree_mask->size[1] <= 1024, "trees of more than 65536 nodes are not implemented");
    TSA_REQUIRE(max_nodes >= 0 && max_nodes <= N, "max_nodes (%lld) must be within [0, num_nodes]", (long long)max_nodes);
  } else {
    TSA_REQUIRE(N == B, "block_tables and seq_lens must have num_seqs (%lld) rows", (long long)N);
  }
  TSA_REQUIRE(window >= 0 && sinks >= 0, "window and sinks must be non-negative");
  TSA_REQUIRE(B < 65536 && Hq < 65536, "num_seqs and num_heads must be below 65536");
  // (each factor is bounded before the product)
  TSA_REQUIRE(BS < (int64_t{1} << 27) && block_tables->size[1] < (int64_t{1} << 27) &&
                  block_tables->size[1] * BS < (int64_t{1} << 27),
              "block table too long");
  TSA_UNSUPPORTED(D <= 512, "head_dim %lld > 512 is not implemented", (long long)D);

  a = RowsArgs{};
  a.out = out->data; a.q = query->data; a.kc = k_cache->data; a.vc = v_cache->data;
  a.bt = static_cast<const int32_t*>(block_tables->data);
  a.lens = static_cast<const int32_t*>(lens->data);
  a.o_sr = out->stride[0]; a.o_sh = out->stride[1]; a.o_sd = out->stride[2];
  a.q_sr = query->stride[0]; a.q_sh = query->stride[1]; a.q_sd = query->stride[2];
  a.kc_b = k_cache->stride[0]; a.kc_h = k_cache->stride[1]; a.kc_s = k_cache->stride[2]; a.kc_d = k_cache->stride[3];
  a.vc_b = v_cache->stride[0]; a.vc_h = v_cache->stride[1]; a.vc_s = v_cache->stride[2]; a.vc_d = v_cache->stride[3];
  a.bt_s0 = block_tables->stride[0]; a.bt_s1 = block_tables->stride[1]; a.len_s = lens->stride[0];
  if (q8) {
    a.ks = static_cast<const float*>(k_scale->data);
    a.vs = static_cast<const float*>(v_scale->data);
    a.ks_b = k_scale->stride[0]; a.ks_h = k_scale->stride[1]; a.ks_s = k_scale->stride[2];
    a.vs_b = v_scale->stride[0]; a.vs_h = v_scale->stride[1]; a.vs_s = v_scale->stride[2];
  }
  a.NB = NB; a.N = N;
  a.B = static_cast<int32_t>(B); a.Hq = static_cast<int32_t>(Hq); a.Hkv = static_cast<int32_t>(Hkv);
  a.G = static_cast<int32_t>(Hq / Hkv); a.BS = static_cast<int32_t>(BS);
  a.max_blocks = static_cast<int32_t>(block_tables->size[1]); a.D = static_cast<int32_t>(D);
  a.T = 1;
  if (tree) {
    a.cu = static_cast<const int32_t*>(cu_nodes->data);
    a.cu_s = cu_nodes->stride[0];
    a.mask = static_cast<const uint32_t*>(tree_mask->data);
    a.mask_s = 2 * tree_mask->stride[0];
    a.words = static_cast<int32_t>(2 * tree_mask->size[1]);
    const int64_t most = 32 * int64_t{a.words};  // nodes past the mask's width are not computed either
    a.T = static_cast<int32_t>(max_nodes < most ? max_nodes : most);
  }
  constexpr int64_t kMost = int64_t{1} << 30;  // (past any block table)
  a.window = static_cast<int32_t>(window < kMost ? window : kMost);
  a.sinks = static_cast<int32_t>(sinks < kMost ? sinks : kMost);
  a.scale_log2 = static_cast<float>(softmax_scale * 1.4426950408889634);
  return TSA_OK;
}

// Sequences of one launch: within the stream's prefix, 2^22 workgroups, and
// 2^30 tile pairs (its prefix is 32 bits).
static int64_t decode_rows_chunk(int64_t B, int64_t Hq, int64_t Hkv, int64_t cap) {
  const int64_t units = Hkv * ((Hq / Hkv + 15) / 16), pairs = (cap + 31) / 32 + 1;
  int64_t n = kRowsMaxSeqs < B ? kRowsMaxSeqs : B;
  n = n < (int64_t{1} << 22) / units ? n : (int64_t{1} << 22) / units;
  n = n < (int64_t{1} << 30) / pairs ? n : (int64_t{1} << 30) / pairs;
  return n < 1 ? 1 : n;
}
// The workspace of a decode call: of its full chunks and of the last one.
static size_t decode_rows_bytes(int64_t B, int64_t Hq, int64_t Hkv, int64_t D, int64_t cap, int64_t window,
                                int64_t sinks) {
  const int64_t chunk = decode_rows_chunk(B, Hq, Hkv, cap);
  const size_t full = decode_rows_plan(chunk, Hq, Hkv, D, cap, window, sinks).total;
  const size_t last = B % chunk ? decode_rows_plan(B % chunk, Hq, Hkv, D, cap, window, sinks).total : 0;
  return full > last ? full : last;
}

// The matrix-core forms: 16-bit queries, head_dim 64 or 128, pages of whole
// 16-token tiles, unit-stride rows of 16-byte pieces, and strides whose offsets
// within a page fit 31 bits (a page's own 32). Fills what they need of a.
static bool takes_mfma(RowsArgs& a, const tsa_view* out, const tsa_view* query, const tsa_view* k_cache, const tsa_view* v_cache) {
  if ((query->dtype != TSA_BF16 && query->dtype != TSA_F16) || (a.D != 64 && a.D != 128) || a.BS % 16 || a.NB == 0)
    return false;
  if (!rows_vec16(query) || !rows_vec16(k_cache) || !rows_vec16(v_cache)) return false;
  const int64_t eb = dtype_bytes(k_cache->dtype);
  auto fits = [&](int64_t page, int64_t slot, int64_t bytes) {
    return page >= 0 && page < (int64_t{1} << 32) / bytes && slot >= 0 && slot < (int64_t{1} << 31) / bytes / a.BS;
  };
  if (!fits(a.kc_b, a.kc_s, eb) || !fits(a.vc_b, a.vc_s, eb)) return false;
  if (a.ks && (!fits(a.ks_b, a.ks_s, 4) || !fits(a.vs_b, a.vs_s, 4))) return false;
  a.k_page = static_cast<uint32_t>(a.kc_b * eb);
  a.v_page = static_cast<uint32_t>(a.vc_b * eb);
  a.ks_page = static_cast<uint32_t>(a.ks_b * 4);
  a.vs_page = static_cast<uint32_t>(a.vs_b * 4);
  a.out8 = a.o_sd == 1 && a.o_sr % 4 == 0 && a.o_sh % 4 == 0 && reinterpret_cast<uintptr_t>(out->data) % 8 == 0;
  set_page_div(a);
  return true;
}

static int dispatch_rows(const RowsArgs& a, int dt, int cache_dt, hipStream_t stream, const char* what) {
  if (a.B == 0 || a.T == 0 || a.Hq == 0 || a.D == 0 || a.N == 0) return TSA_OK;
  const bool e4m3 = cache_dt == TSA_E4M3;
  switch (dt) {
    case TSA_BF16:
      return a.ks == nullptr ? launch_rows<bf16_t, bf16_t>(a, stream, what)
             : e4m3          ? launch_rows<bf16_t, e4m3_t>(a, stream, what)
                             : launch_rows<bf16_t, i8_t>(a, stream, what);
    case TSA_F16:
      return a.ks == nullptr ? launch_rows<f16_t, f16_t>(a, stream, what)
             : e4m3          ? launch_rows<f16_t, e4m3_t>(a, stream, what)
                             : launch_rows<f16_t, i8_t>(a, stream, what);
    default:
      return a.ks == nullptr ? launch_rows<float, float>(a, stream, what)
             : e4m3          ? launch_rows<float, e4m3_t>(a, stream, what)
                             : launch_rows<float, i8_t>(a, stream, what);
  }
}

}  // namespace tsa

using namespace tsa;

extern "C" int tsa_paged_decode_window(const tsa_view* out, const tsa_view* query, const tsa_view* k_cache,
                                       const tsa_view* v_cache, const tsa_view* k_scale, const tsa_view* v_scale,
                                       const tsa_view* block_tables, const tsa_view* seq_lens, int64_t window,
                                       int64_t sinks, double softmax_scale, void* workspace, size_t workspace_bytes,
                                       void* stream) {
  RowsArgs a;
  if (int rc = check_rows(out, query, k_cache, v_cache, k_scale, v_scale, block_tables, seq_lens, nullptr, nullptr, 0,
                          window, sinks, softmax_scale, a))
    return rc;
  if (a.B > 0 && a.Hq > 0 && takes_mfma(a, out, query, k_cache, v_cache)) {
    const int64_t cap = int64_t{a.max_blocks} * a.BS, chunk = decode_rows_chunk(a.B, a.Hq, a.Hkv, cap);
    const size_t need = decode_rows_bytes(a.B, a.Hq, a.Hkv, a.D, cap, a.window, a.sinks);
    TSA_REQUIRE(need == 0 || (workspace != nullptr && workspace_bytes >= need),
                "workspace of %zu bytes is too small: %zu needed", workspace_bytes, need);
    TSA_REQUIRE(need == 0 || reinterpret_cast<uintptr_t>(workspace) % 256 == 0, "workspace must be 256-byte aligned");
    const hipStream_t st = static_cast<hipStream_t>(stream);
    for (int64_t b = 0; b < block_tables->size[0]; b += chunk) {  // (one chunk, but for batches past its limits)
      RowsArgs c = a;
      c.B = static_cast<int32_t>(block_tables->size[0] - b < chunk ? block_tables->size[0] - b : chunk);
      c.q = static_cast<const char*>(a.q) + b * a.q_sr * dtype_bytes(query->dtype);
      c.out = static_cast<char*>(a.out) + b * a.o_sr * dtype_bytes(query->dtype);
      c.bt = a.bt + b * a.bt_s0;
      c.lens = a.lens + b * a.len_s;
      const DecodeRowsPlan p = decode_rows_plan(c.B, a.Hq, a.Hkv, a.D, cap, a.window, a.sinks);
      c.S = p.S;
      c.NW = p.waves;
      c.part = static_cast<float*>(workspace);
      c.pref = reinterpret_cast<int32_t*>(static_cast<char*>(workspace) + p.part_bytes);
      if (int rc = p.S > 0 ? rows_unit_launch(c, query->dtype, k_cache->dtype, st, "tsa_paged_decode_window")
                           : rows_stream_launch(c, query->dtype, k_cache->dtype, st, "tsa_paged_decode_window"))
        return rc;
    }
    return TSA_OK;
  }
  return dispatch_rows(a, query->dtype, k_cache->dtype, static_cast<hipStream_t>(stream), "tsa_paged_decode_window");
}

extern "C" int tsa_paged_tree(const tsa_view* out, const tsa_view* query, const tsa_view* k_cache,
                              const tsa_view* v_cache, const tsa_view* block_tables, const tsa_view* context_lens,
                              const tsa_view* cu_nodes, const tsa_view* tree_mask, int64_t max_nodes,
                              double softmax_scale, void* workspace, size_t workspace_bytes, void* stream) {
  RowsArgs a;
  TSA_REQUIRE(cu_nodes != nullptr, "cu_nodes must be a 1D int32 tensor (num_seqs + 1)");
  if (int rc = check_rows(out, query, k_cache, v_cache, nullptr, nullptr, block_tables, context_lens, cu_nodes,
                          tree_mask, max_nodes, 0, 0, softmax_scale, a))
    return rc;
  if (a.B > 0 && a.Hq > 0 && a.T > 0 && a.N > 0 && a.scale_log2 > 0.f && takes_mfma(a, out, query, k_cache, v_cache)) {
    const TreeRowsPlan p = tree_rows_plan(a.B, a.T, a.Hq, a.Hkv, a.D, int64_t{a.max_blocks} * a.BS);
    if (p.S > 0) {
      TSA_REQUIRE(p.bytes == 0 || (workspace != nullptr && workspace_bytes >= p.bytes),
                  "workspace of %zu bytes is too small: %zu needed", workspace_bytes, p.bytes);
      TSA_REQUIRE(p.bytes == 0 || reinterpret_cast<uintptr_t>(workspace) % 256 == 0, "workspace must be 256-byte aligned");
      a.S = p.S; a.RT = p.RT; a.RB = p.RB; a.per_split = p.per_split;
      a.order = a.B > 1 && a.B <= kTreeOrderSeqs && int64_t{a.B} * a.Hkv * a.S * a.RB > 256;  // (more than one workgroup a CU: else a lookup for nothing)
      a.part = static_cast<float*>(workspace);
      return rows_tree_launch(a, query->dtype, static_cast<hipStream_t>(stream));
    }
  }
  return dispatch_rows(a, query->dtype, k_cache->dtype, static_cast<hipStream_t>(stream), "tsa_paged_tree");
}

extern "C" size_t tsa_paged_rows_workspace_bytes(int64_t num_seqs, int64_t max_nodes, int64_t num_heads,
                                                 int64_t num_kv_heads, int64_t head_dim, int64_t max_blocks_per_seq,
                                                 int64_t block_size, int64_t window, int64_t sinks) {
  if (num_seqs <= 0 || num_heads <= 0 || num_kv_heads <= 0 || num_heads % num_kv_heads || num_seqs >= 65536 ||
      num_heads >= 65536 || head_dim <= 0 || head_dim > 512 || block_size <= 0 || block_size >= (int64_t{1} << 27) ||
      max_blocks_per_seq <= 0 || max_blocks_per_seq >= (int64_t{1} << 27) || max_nodes <= 0 ||
      max_blocks_per_seq * block_size >= (int64_t{1} << 27))
    return 0;  // (calls of such sizes are refused, or have nothing to do)
  const int64_t cap = max_blocks_per_seq * block_size;
  const size_t decode = decode_rows_bytes(num_seqs, num_heads, num_kv_heads, head_dim, cap, window, sinks);
  if (window > 0 || sinks > 0) return decode;
  max_nodes = max_nodes < 65536 ? max_nodes : 65536;  // (the widest mask's)
  const size_t tree = tree_rows_plan(num_seqs, max_nodes, num_heads, num_kv_heads, head_dim, cap).bytes;
  return max_nodes > 1 ? tree : tree > decode ? tree : decode;
}
