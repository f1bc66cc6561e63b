// The 8-bit paged K/V cache (cache8.h): rows quantised as they are stored, and
// read back.
//
// tsa_store_kv_quantized writes what tsa_store_kv_paged writes
// (server/model/kernels/kv_cache.py:6-70 with qwen3.py:296-318's addressing),
// in 8 bits; tsa_load_kv_quantized is its inverse. Both are copies with a row
// maximum or a product between: bound by HBM for prompts, by the chain of
// sequence search, block-table entry and row for a decode step's few tokens.
#include "cache8.h"
#include "kv_store.h"

namespace tsa {

struct Quant8Args {
  const char* k_src; const char* v_src;  // store: (T, H, D) rows; load: not used
  char* k_out; char* v_out;              // load: (T, H, D) rows
  char* kc; char* vc;                    // codes (NB, H, BS, D)
  float* ks; float* vs;                  // scales (NB, H, BS)
  int64_t T, H, D, NB, BS;
  int64_t kr_t, kr_h, kr_d, vr_t, vr_h, vr_d;  // element strides of the packed rows
  int64_t kc_b, kc_h, kc_s, kc_d, vc_b, vc_h, vc_s, vc_d;
  int64_t ks_b, ks_h, ks_s, vs_b, vs_h, vs_s;
};

// Any strides and head_dim: one wave per (token, kv head, K or V) row.
template <typename T, typename C, bool STORE>
__global__ __launch_bounds__(256) void quant8_rows(Quant8Args a, PagedAddr addr) {
  const int lane = threadIdx.x & 63;
  const int64_t rows = 2 * a.T * a.H, waves = static_cast<int64_t>(gridDim.x) * 4;
  for (int64_t r = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6); r < rows; r += waves) {
    const bool is_v = r & 1;
    const int64_t t = (r >> 1) / a.H, h = (r >> 1) - t * a.H;
    int64_t blk, slot;
    const bool ok = addr.locate(t, a.BS, a.NB, blk, slot);
    const int64_t row = is_v ? t * a.vr_t + h * a.vr_h : t * a.kr_t + h * a.kr_h, rd = is_v ? a.vr_d : a.kr_d;
    C* const code = reinterpret_cast<C*>(is_v ? a.vc : a.kc) +
                    (ok ? (is_v ? blk * a.vc_b + h * a.vc_h + slot * a.vc_s : blk * a.kc_b + h * a.kc_h + slot * a.kc_s)
                        : 0);
    const int64_t cd = is_v ? a.vc_d : a.kc_d;
    float* const scale_p = (is_v ? a.vs : a.ks) +
                           (ok ? (is_v ? blk * a.vs_b + h * a.vs_h + slot * a.vs_s
                                       : blk * a.ks_b + h * a.ks_h + slot * a.ks_s)
                               : 0);
    if constexpr (STORE) {
      if (!ok) continue;
      const T* const src = reinterpret_cast<const T*>(is_v ? a.v_src : a.k_src) + row;
      uint32_t top = 0;
      for (int64_t d = lane; d < a.D; d += 64)
        top = max(top, __builtin_bit_cast(uint32_t, to_float(src[d * rd])) & 0x7FFFFFFFu);
#pragma unroll
      for (int off = 32; off >= 1; off >>= 1) top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), off, 64)));
      const float scale = scale8<C>(top);
      for (int64_t d = lane; d < a.D; d += 64)
        code[d * cd] = __builtin_bit_cast(C, static_cast<uint8_t>(codes4<C>(quotient8<C>(to_float(src[d * rd]), scale), 0.f, 0.f, 0.f)));
      if (lane == 0) *scale_p = scale;
    } else {
      T* const dst = reinterpret_cast<T*>(is_v ? a.v_out : a.k_out) + row;
      const float scale = ok ? *scale_p : 0.f;
      for (int64_t d = lane; d < a.D; d += 64)
        dst[d * rd] = from_float<T>(ok ? product8(to_float(code[d * cd]), scale) : 0.f);
    }
  }
}

// 16-bit rows of 64 or 128 dims in 16-byte pieces: D / 8 lanes a row, 8 elements
// a lane, so that a wave's stores of one head's tokens are whole lines. A
// workgroup takes 256 / (D / 8) tokens and `heads` kv heads of each, kBatch at a
// time, K and V together, with all of a batch's loads in flight; a token's
// place is looked up once. The sequences' starts go to LDS first, so the search
// is one round trip to memory and not one for each of its steps.
//
// A quotient is x times the scale's reciprocal, corrected twice by its fma
// residual: with the correctly rounded reciprocal that is the correctly rounded
// x / scale (Markstein's theorem: one step from a quotient within a unit in the
// last place; the first step gives that one). Residuals below the normal range
// would lose bits, so rows of scales under 2^-80 divide. The residual is y scale
// - x, subtracted: that of -0 is +0, and -0 - 0 stays -0 (x - y scale, added,
// would make it +0, another code of e4m3).
constexpr int kQuant8Batch = 2;
constexpr int kQuant8LdsSeqs = 2048;

struct LdsCu {
  const int32_t* cu;  // [nseq + 1] in LDS
  // pos: the token's given position, where there are any.
  __device__ __forceinline__ bool locate(const PagedAddr& a, int64_t t, int64_t pos, int64_t BS, int64_t NB, int64_t& blk,
                                         int64_t& slot) const {
    int lo = 0, hi = static_cast<int>(a.nseq);  // the last s with cu[s] <= t is in [lo, hi)
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (cu[mid] <= t) lo = mid; else hi = mid;
    }
    const int64_t t0 = cu[lo];
    if (t < t0 || t >= cu[lo + 1]) return false;
    const int64_t p = a.pos_kind ? pos : t - t0;
    if (p < 0 || p >= a.max_blocks * BS) return false;
    // (positions within a table fit 32 bits here: checked by the caller)
    const uint32_t lb = static_cast<uint32_t>(p) / static_cast<uint32_t>(BS);
    blk = a.bt[lo * a.bt_s0 + lb * a.bt_s1];
    slot = static_cast<uint32_t>(p) - lb * static_cast<uint32_t>(BS);
    return blk >= 0 && blk < NB;
  }
};

template <typename C> __device__ __forceinline__ void quotients8(const float (&x)[8], float scale, float (&q)[8]) {
  if (scale > 0x1p-80f) {
    const float r = 1.f / scale;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float y = x[i] * r;
      y = fmaf(-fmaf(y, scale, -x[i]), r, y);
      y = fmaf(-fmaf(y, scale, -x[i]), r, y);
      q[i] = fminf(fmaxf(y, -kLargest8<C>), kLargest8<C>);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) q[i] = quotient8<C>(x[i], scale);
  }
}

template <typename T, typename C, int D, bool STORE>
__global__ __launch_bounds__(256) void quant8_vec(Quant8Args a, PagedAddr addr, int heads) {
  constexpr int LG = D / 8, TOK = 256 / LG;
  __shared__ int32_t cu_s[kQuant8LdsSeqs + 1];
  const int tid = threadIdx.x, c = tid % LG;
  const int64_t t = static_cast<int64_t>(blockIdx.x) * TOK + tid / LG, tt = t < a.T ? t : a.T - 1;
  const int h0 = static_cast<int>(blockIdx.y) * heads, h1 = min(h0 + heads, static_cast<int>(a.H));
  // (store) The first batch's rows and the position are asked for before the search.
  u32x4 x[kQuant8Batch][2];
  auto fetch = [&](int h) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < kQuant8Batch; ++i) {
      const int hh = min(h + i, h1 - 1);
      x[i][0] = *reinterpret_cast<const u32x4*>(reinterpret_cast<const T*>(a.k_src) + tt * a.kr_t + hh * a.kr_h + 8 * c);
      x[i][1] = *reinterpret_cast<const u32x4*>(reinterpret_cast<const T*>(a.v_src) + tt * a.vr_t + hh * a.vr_h + 8 * c);
    }
  };
  int64_t pos = 0;
  if (addr.pos_kind == 2) pos = static_cast<const int64_t*>(addr.pos)[tt * addr.pos_stride];
  else if (addr.pos_kind == 1) pos = static_cast<const int32_t*>(addr.pos)[tt * addr.pos_stride];
  for (int i = tid; i <= addr.nseq; i += 256) cu_s[i] = addr.cu[i * addr.cu_stride];
  if constexpr (STORE) fetch(h0);
  lds_barrier();
  int64_t blk = 0, slot = 0;
  const bool found = LdsCu{cu_s}.locate(addr, tt, pos, a.BS, a.NB, blk, slot), ok = found && t < a.T;
  if (!found) blk = slot = 0;
  const int64_t kc = blk * a.kc_b + slot * a.kc_s + 8 * c, vc = blk * a.vc_b + slot * a.vc_s + 8 * c;
  const int64_t ks = blk * a.ks_b + slot * a.ks_s, vs = blk * a.vs_b + slot * a.vs_s;
  for (int h = h0; h < h1; h += kQuant8Batch) {
    if constexpr (STORE) {
      if (h > h0) fetch(h);
#pragma unroll
      for (int i = 0; i < kQuant8Batch; ++i) {
        if (h + i >= h1) break;
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          float f[8], q[8];
          uint32_t top = 0;
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            f[2 * k] = lo_f<T>(x[i][y][k]);
            f[2 * k + 1] = hi_f<T>(x[i][y][k]);
          }
#pragma unroll
          for (int k = 0; k < 8; ++k) top = max(top, __builtin_bit_cast(uint32_t, f[k]) & 0x7FFFFFFFu);
          const int lane = tid & 63;  // (every lane takes part: tokens past the last repeat it)
          top = max(top, xor_lane32<1>(top, lane));
          top = max(top, xor_lane32<2>(top, lane));
          top = max(top, xor_lane32<4>(top, lane));
          if constexpr (LG == 16) top = max(top, xor_lane32<8>(top, lane));
          const float scale = scale8<C>(top);
          quotients8<C>(f, scale, q);
          if (ok) {
            const u32x2 w = {codes4<C>(q[0], q[1], q[2], q[3]), codes4<C>(q[4], q[5], q[6], q[7])};
            *reinterpret_cast<u32x2*>((y ? a.vc + vc + (h + i) * a.vc_h : a.kc + kc + (h + i) * a.kc_h)) = w;
            if (c == 0) (y ? a.vs[vs + (h + i) * a.vs_h] : a.ks[ks + (h + i) * a.ks_h]) = scale;
          }
        }
      }
    } else {
      u32x2 w[kQuant8Batch][2];
      float sc[kQuant8Batch][2];
#pragma unroll
      for (int i = 0; i < kQuant8Batch; ++i) {  // (a token without a page reads page 0's first row, and drops it)
        const int hh = min(h + i, h1 - 1);
        w[i][0] = w[i][1] = u32x2{0, 0};
        sc[i][0] = sc[i][1] = 0.f;
        if (a.NB > 0) {
          w[i][0] = *reinterpret_cast<const u32x2*>(a.kc + kc + hh * a.kc_h);
          w[i][1] = *reinterpret_cast<const u32x2*>(a.vc + vc + hh * a.vc_h);
          sc[i][0] = a.ks[ks + hh * a.ks_h];
          sc[i][1] = a.vs[vs + hh * a.vs_h];
        }
      }
#pragma unroll
      for (int i = 0; i < kQuant8Batch; ++i) {
        if (h + i >= h1 || t >= a.T) break;
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          u32x4 out;
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            float v[4];
            values4<C>(w[i][y][k], v);
#pragma unroll
            for (int e = 0; e < 2; ++e)
              out[2 * k + e] = found ? pack2<T>(product8(v[2 * e], sc[i][y]), product8(v[2 * e + 1], sc[i][y])) : 0u;
          }
          T* const dst = y ? reinterpret_cast<T*>(a.v_out) + t * a.vr_t + (h + i) * a.vr_h
                           : reinterpret_cast<T*>(a.k_out) + t * a.kr_t + (h + i) * a.kr_h;
          *reinterpret_cast<u32x4*>(dst + 8 * c) = out;
        }
      }
    }
  }
}

// Whether the calls' rows are what quant8_vec takes.
static bool quant8_takes_vec(const Quant8Args& a, const PagedAddr& addr, const tsa_view* k, const tsa_view* v,
                             const tsa_view* k_cache, const tsa_view* v_cache) {
  if ((k->dtype != TSA_BF16 && k->dtype != TSA_F16) || (a.D != 64 && a.D != 128)) return false;
  if (!rows_vec16(k) || !rows_vec16(v) || addr.nseq < 1 || addr.nseq > kQuant8LdsSeqs) return false;
  if (addr.max_blocks >= (int64_t{1} << 31) / a.BS || a.T >= (int64_t{1} << 27)) return false;  // (a grid of 2^32 threads)
  for (const tsa_view* x : {k_cache, v_cache}) {
    if (x->stride[3] != 1 || reinterpret_cast<uintptr_t>(x->data) % 8) return false;
    for (int d = 0; d < 3; ++d)
      if (x->size[d] > 1 && x->stride[d] % 8) return false;
  }
  return a.H < 65536;
}

template <typename T, typename C, bool STORE>
static int launch_quant8_vec(const Quant8Args& a, const PagedAddr& addr, hipStream_t stream, const char* what) {
  // Heads a workgroup: one for few tokens, for more workgroups, two for many, which
  // share a token's lookup. Both sides, one / two, us, e4m3, 8 heads of 128 dims: 64
  // tokens store 3.6 / 4.5, load 3.2 / 3.5; 1024 4.5 / 5.3 and 4.3 / 4.4; 2048 6.2 /
  // 6.4 and 5.5 / 5.4; 4096 9.9 / 10.3 and 9.2 / 8.3; 16384 26.9 / 27.3 and 28.9 / 24.7.
  // (Eight: 16 prompts' store 25.3 against 24.7, 8 prefixes' load 26.9 against 25.1.)
  const int tok = 256 / static_cast<int>(a.D / 8), heads = a.T >= 2048 ? 2 : 1;
  const dim3 grid(static_cast<uint32_t>((a.T + tok - 1) / tok), static_cast<uint32_t>((a.H + heads - 1) / heads));
  if (a.D == 128) quant8_vec<T, C, 128, STORE><<<grid, dim3(256), 0, stream>>>(a, addr, heads);
  else quant8_vec<T, C, 64, STORE><<<grid, dim3(256), 0, stream>>>(a, addr, heads);
  return check_launch(what);
}

template <typename T, typename C, bool STORE>
static int launch_quant8(const Quant8Args& a, const PagedAddr& addr, hipStream_t stream, const char* what) {
  const int64_t wgs = (2 * a.T * a.H + 3) / 4;
  quant8_rows<T, C, STORE><<<dim3(static_cast<uint32_t>(wgs < 65536 ? wgs : 65536)), dim3(256), 0, stream>>>(a, addr);
  return check_launch(what);
}

// Rows (T, H, D) (store: the sources, passed as (H, T, D); load: the outputs), codes and scales.
static int check_quant8(const tsa_view* k, const tsa_view* v, bool heads_first, const tsa_view* k_cache,
                        const tsa_view* v_cache, const tsa_view* k_scale, const tsa_view* v_scale, Quant8Args& a) {
  const char* const kn = heads_first ? "k_src" : "k_out";
  const char* const vn = heads_first ? "v_src" : "v_out";
  const int hd = heads_first ? 0 : 1, td = heads_first ? 1 : 0;
  TSA_REQUIRE(view_ok(k, 3) && view_ok(v, 3), "%s and %s must be 3D tensors %s", kn, vn,
              heads_first ? "(num_kv_heads, num_tokens, head_dim)" : "(num_tokens, num_kv_heads, head_dim)");
  TSA_REQUIRE(view_ok(k_cache, 4) && view_ok(v_cache, 4),
              "k_cache and v_cache must be 4D tensors (num_blocks, num_kv_heads, block_size, head_dim)");
  TSA_REQUIRE(view_ok(k_scale, 3) && view_ok(v_scale, 3),
              "k_scale and v_scale must be 3D tensors (num_blocks, num_kv_heads, block_size)");
  for (int d = 0; d < 3; ++d) TSA_REQUIRE(k->size[d] == v->size[d], "%s and %s must have the same shape", kn, vn);
  for (int d = 0; d < 4; ++d)
    TSA_REQUIRE(k_cache->size[d] == v_cache->size[d], "k_cache and v_cache must have the same shape");
  for (int d = 0; d < 3; ++d)
    TSA_REQUIRE(k_scale->size[d] == k_cache->size[d] && v_scale->size[d] == k_cache->size[d],
                "k_scale and v_scale must have the cache's shape but its head_dim");
  TSA_REQUIRE(is_float_dtype(k->dtype) && v->dtype == k->dtype, "%s and %s must share one floating dtype (got %s/%s)",
              kn, vn, dtype_name(k->dtype), dtype_name(v->dtype));
  TSA_REQUIRE(is_cache8_dtype(k_cache->dtype) && v_cache->dtype == k_cache->dtype,
              "k_cache and v_cache must share one 8-bit dtype, e4m3 or int8 (got %s/%s)", dtype_name(k_cache->dtype),
              dtype_name(v_cache->dtype));
  TSA_REQUIRE(k_scale->dtype == TSA_F32 && v_scale->dtype == TSA_F32, "k_scale and v_scale must be float32");
  TSA_REQUIRE(k->size[hd] == k_cache->size[1], "%s has %lld kv heads but the cache has %lld", kn,
              (long long)k->size[hd], (long long)k_cache->size[1]);
  TSA_REQUIRE(k->size[2] == k_cache->size[3], "%s head_dim %lld != cache head_dim %lld", kn, (long long)k->size[2],
              (long long)k_cache->size[3]);
  TSA_REQUIRE(k_cache->size[2] > 0, "block_size must be positive");
  a = Quant8Args{};
  a.T = k->size[td]; a.H = k->size[hd]; a.D = k->size[2];
  a.NB = k_cache->size[0]; a.BS = k_cache->size[2];
  a.kr_t = k->stride[td]; a.kr_h = k->stride[hd]; a.kr_d = k->stride[2];
  a.vr_t = v->stride[td]; a.vr_h = v->stride[hd]; a.vr_d = v->stride[2];
  a.kc = static_cast<char*>(k_cache->data); a.vc = static_cast<char*>(v_cache->data);
  a.ks = static_cast<float*>(k_scale->data); a.vs = static_cast<float*>(v_scale->data);
  a.kc_b = k_cache->stride[0]; a.kc_h = k_cache->stride[1]; a.kc_s = k_cache->stride[2]; a.kc_d = k_cache->stride[3];
  a.vc_b = v_cache->stride[0]; a.vc_h = v_cache->stride[1]; a.vc_s = v_cache->stride[2]; a.vc_d = v_cache->stride[3];
  a.ks_b = k_scale->stride[0]; a.ks_h = k_scale->stride[1]; a.ks_s = k_scale->stride[2];
  a.vs_b = v_scale->stride[0]; a.vs_h = v_scale->stride[1]; a.vs_s = v_scale->stride[2];
  return TSA_OK;
}

template <bool STORE>
static int dispatch_quant8(const Quant8Args& a, const PagedAddr& addr, bool vec, int dt, int cache_dt,
                           hipStream_t stream, const char* what) {
  if (a.T == 0 || a.H == 0 || a.D == 0) return TSA_OK;
  const bool e4m3 = cache_dt == TSA_E4M3;
  if (vec && dt == TSA_BF16)
    return e4m3 ? launch_quant8_vec<bf16_t, e4m3_t, STORE>(a, addr, stream, what)
                : launch_quant8_vec<bf16_t, i8_t, STORE>(a, addr, stream, what);
  if (vec)
    return e4m3 ? launch_quant8_vec<f16_t, e4m3_t, STORE>(a, addr, stream, what)
                : launch_quant8_vec<f16_t, i8_t, STORE>(a, addr, stream, what);
  switch (dt) {
    case TSA_BF16:
      return e4m3 ? launch_quant8<bf16_t, e4m3_t, STORE>(a, addr, stream, what)
                  : launch_quant8<bf16_t, i8_t, STORE>(a, addr, stream, what);
    case TSA_F16:
      return e4m3 ? launch_quant8<f16_t, e4m3_t, STORE>(a, addr, stream, what)
                  : launch_quant8<f16_t, i8_t, STORE>(a, addr, stream, what);
    default:
      return e4m3 ? launch_quant8<float, e4m3_t, STORE>(a, addr, stream, what)
                  : launch_quant8<float, i8_t, STORE>(a, addr, stream, what);
  }
}

}  // namespace tsa

using namespace tsa;

extern "C" int tsa_store_kv_quantized(const tsa_view* k_src, const tsa_view* v_src, const tsa_view* k_cache,
                                      const tsa_view* v_cache, const tsa_view* k_scale, const tsa_view* v_scale,
                                      const tsa_view* block_tables, const tsa_view* cu_seqlens,
                                      const tsa_view* positions, void* stream) {
  Quant8Args a;
  if (int rc = check_quant8(k_src, v_src, true, k_cache, v_cache, k_scale, v_scale, a)) return rc;
  a.k_src = static_cast<const char*>(k_src->data);
  a.v_src = static_cast<const char*>(v_src->data);
  PagedAddr addr;
  if (int rc = make_paged_addr(block_tables, cu_seqlens, positions, a.T, addr)) return rc;
  if (a.NB == 0) return TSA_OK;  // (no page to write)
  return dispatch_quant8<true>(a, addr, quant8_takes_vec(a, addr, k_src, v_src, k_cache, v_cache), k_src->dtype,
                               k_cache->dtype, static_cast<hipStream_t>(stream), "tsa_store_kv_quantized");
}

extern "C" int tsa_load_kv_quantized(const tsa_view* k_out, const tsa_view* v_out, const tsa_view* k_cache,
                                     const tsa_view* v_cache, const tsa_view* k_scale, const tsa_view* v_scale,
                                     const tsa_view* block_tables, const tsa_view* cu_seqlens,
                                     const tsa_view* positions, void* stream) {
  Quant8Args a;
  if (int rc = check_quant8(k_out, v_out, false, k_cache, v_cache, k_scale, v_scale, a)) return rc;
  a.k_out = static_cast<char*>(k_out->data);
  a.v_out = static_cast<char*>(v_out->data);
  PagedAddr addr;
  if (int rc = make_paged_addr(block_tables, cu_seqlens, positions, a.T, addr)) return rc;
  return dispatch_quant8<false>(a, addr, quant8_takes_vec(a, addr, k_out, v_out, k_cache, v_cache), k_out->dtype,
                                k_cache->dtype, static_cast<hipStream_t>(stream), "tsa_load_kv_quantized");
}
