// Varlen prefill attention with a sliding window and first tokens that stay
// visible: query i of a sequence sees the keys j <= i with j > i - window or
// j < sinks (top-left positions, as tsa_varlen_prefill's causal mask).
//
// varlen_window_gqa   bf16/f16, GQA group 2, 4 or 8: the LDS-staged persistent
//                     kernel (prefill_gqa_body), and
// varlen_window_w64   head_dim 128, groups of 12, 16, ...: 64 queries a wave
//                     (prefill_w64_body), both over the blocks of the window and
//                     of the first keys;
// varlen_prefill_mfma other groups (all three round a weight once to the type for the
//                     second product, as the prefill without a window does: at most
//                     2^-8, f16 2^-11, of itself; outputs 0.0021 from 64 bits where
//                     their own rounding is 0.0016, bf16);
// varlen_window_generic  float32, other head_dims, strides and scales: one wave
//                     per (query, q-head), VALU.
#include "varlen_prefill_mfma.h"
#include "varlen_prefill_window.h"

namespace tsa {

template <typename T, int D, int NW, int QS>
__global__ __launch_bounds__(64 * NW) __attribute__((amdgpu_waves_per_eu(2))) void varlen_window_gqa(
    PrefillWindowArgs a, const int32_t* __restrict__ cu_q, const int32_t* __restrict__ cu_k) {
  __shared__ __align__(16) char smem[gqa_window_smem_bytes<D, NW>()];
  prefill_gqa_body<T, D, NW, QS>(a, cu_q, cu_k, smem, 0);
}

// As many workgroups as fit on the device at once.
template <typename T, int D, int NW, int QS = 1>
static int launch_window_gqa(const PrefillWindowArgs& a, hipStream_t stream) {
  int per_cu = 0, dev = 0, cus = 0;
  if (hipOccupancyMaxActiveBlocksPerMultiprocessor(&per_cu, varlen_window_gqa<T, D, NW, QS>, 64 * NW, 0) != hipSuccess ||
      per_cu <= 0)
    per_cu = 1;
  if (hipGetDevice(&dev) != hipSuccess ||
      hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || cus <= 0)
    cus = 256;
  varlen_window_gqa<T, D, NW, QS><<<dim3(per_cu * cus), dim3(64 * NW), 0, stream>>>(a, a.cu_q, a.cu_k);
  return check_launch("tsa_varlen_prefill_window");
}

template <typename T>
static int launch_window_mfma(PrefillWindowArgs& a, int64_t max_seqlen_q, hipStream_t stream) {
  // Groups of 2, 4 and 8: the LDS-staged kernel. Beside it, 64 queries a wave, 16
  // prompts of 128-2048 tokens, window 32 / 512 + 4: 32/8 heads 109 / 257 us
  // against 135 / 273, 64/8 heads 217 / 455 against 253 / 485; four prompts of
  // 100-700, 32/8 heads: 17 / 25 against 17 / 32; one of 16384, 32/8 heads, window
  // 512 / 4096: 231 / 1029 against 229 / 1026. Other multiples of four take 64
  // queries a wave (four of 500-2048, 128/8 heads: 139 / 264 against 236 / 1008 in
  // varlen_prefill_mfma).
  if (prefill_takes_gqa(a)) {
    if (a.D == 128) {
      if (prefill_pairs(a)) return launch_window_gqa<T, 128, 4, 2>(a, stream);
      if (a.G == 2) return launch_window_gqa<T, 128, 2>(a, stream);
      return a.G == 4 ? launch_window_gqa<T, 128, 4>(a, stream) : launch_window_gqa<T, 128, 8>(a, stream);
    }
    if (a.G == 2) return launch_window_gqa<T, 64, 2>(a, stream);
    return a.G == 4 ? launch_window_gqa<T, 64, 4>(a, stream) : launch_window_gqa<T, 64, 8>(a, stream);
  }
  if (prefill_takes_w64(a)) return prefill_w64_window_launch(a, std::is_same<T, bf16_t>::value, stream);
  a.nqb = static_cast<int32_t>((max_seqlen_q + 31) / 32);
  if (a.nqb == 0) return TSA_OK;
  const dim3 grid(a.nqb, a.nseq, (a.Hq + 3) / 4);
  if (a.D == 128) varlen_prefill_mfma<T, 128><<<grid, dim3(256), 0, stream>>>(a);
  else varlen_prefill_mfma<T, 64><<<grid, dim3(256), 0, stream>>>(a);
  return check_launch("tsa_varlen_prefill_window");
}

// Any strides and head_dim up to 512: one wave per (query row, q-head).
template <typename T>
__global__ __launch_bounds__(64) void varlen_window_generic(PrefillWindowArgs a) {
  const int64_t items = a.total_q * a.Hq;
  for (int64_t it = blockIdx.x; it < items; it += gridDim.x) {
    const int64_t qi = it / a.Hq;
    const int h = static_cast<int>(it - qi * a.Hq);
    int lo = 0, hi = a.nseq;  // the sequence of query token qi
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (a.cu_q[mid * a.cuq_s] <= qi) lo = mid; else hi = mid;
    }
    int64_t q_start, q_len, k_start, k_len;
    seq_range(a.cu_q, a.cuq_s, lo, a.total_q, q_start, q_len);
    seq_range(a.cu_k, a.cuk_s, lo, a.total_k, k_start, k_len);
    if (qi < q_start || qi >= q_start + q_len) continue;
    prefill_window_row<T>(a, qi, qi - q_start, h, k_start, k_len);
  }
}

template <typename T>
static int launch_window(const PrefillWindowArgs& a, hipStream_t stream) {
  const int64_t items = a.total_q * a.Hq;
  varlen_window_generic<T><<<dim3(static_cast<uint32_t>(items < (1 << 20) ? items : 1 << 20)), dim3(64), 0, stream>>>(a);
  return check_launch("tsa_varlen_prefill_window");
}

}  // namespace tsa

using namespace tsa;

extern "C" int tsa_varlen_prefill_window(const tsa_view* out, const tsa_view* q, const tsa_view* k, const tsa_view* v,
                                         const tsa_view* cu_seqlens_q, const tsa_view* cu_seqlens_k,
                                         int64_t max_seqlen_q, int64_t max_seqlen_k, int64_t window, int64_t sinks,
                                         double softmax_scale, void* stream) {
  PrefillWindowArgs a;
  bool mfma = false;
  if (int rc = prefill_prepare(out, q, k, v, cu_seqlens_q, cu_seqlens_k, max_seqlen_q, max_seqlen_k, 1, softmax_scale,
                               a, mfma))
    return rc;
  TSA_REQUIRE(window >= 1, "window must be positive (got %lld)", (long long)window);
  TSA_REQUIRE(sinks >= 0, "sinks must be non-negative (got %lld)", (long long)sinks);
  constexpr int64_t kMost = int64_t{1} << 30;
  TSA_UNSUPPORTED(a.total_q <= kMost && a.total_k <= kMost, "more than 2^30 packed tokens are not implemented");
  a.window = static_cast<int32_t>(window < kMost ? window : kMost);
  a.sinks = static_cast<int32_t>(sinks < kMost ? sinks : kMost);
  if (a.nseq == 0 || a.Hq == 0 || a.D == 0 || a.total_q == 0) return TSA_OK;
  const hipStream_t st = static_cast<hipStream_t>(stream);
  if (mfma && a.scale_log2 > 0.f && a.nseq < 65536 && q->dtype != TSA_F32)
    return q->dtype == TSA_BF16 ? launch_window_mfma<bf16_t>(a, max_seqlen_q, st)
                                : launch_window_mfma<f16_t>(a, max_seqlen_q, st);
  switch (q->dtype) {
    case TSA_BF16: return launch_window<bf16_t>(a, st);
    case TSA_F16: return launch_window<f16_t>(a, st);
    default: return launch_window<float>(a, st);
  }
}
