// Varlen prefill attention with a sliding window and first tokens that stay
// visible: query i of a sequence sees the keys j <= i with j > i - window or
// j < sinks (top-left positions, as tsa_varlen_prefill's causal mask).
#include "varlen_prefill_window.h"

namespace tsa {

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
  switch (q->dtype) {
    case TSA_BF16: return launch_window<bf16_t>(a, st);
    case TSA_F16: return launch_window<f16_t>(a, st);
    default: return launch_window<float>(a, st);
  }
}
