// Log probabilities of given tokens, with the entropy of their distribution and the
// most likely alternatives (tsa_token_logprobs).
//
// For a row x of V logits with m = max x, t_i = x_i - m <= 0, S = sum exp(t_i) and
// E = sum exp(t_i) t_i:
//   log p_i = t_i - ln S,   H = -sum p_i ln p_i = ln S - E / S
// (both terms of H are non-negative: nothing cancels). A logit of -inf has p = 0 and
// adds nothing; a NaN, a +inf or a row of nothing but -inf makes S NaN, and with it
// the row's results.
//
// Order of the alternatives: by value, the lowest index first where values tie (0 and
// -0 do), NaN last. One whole number a logit has that order (rank_of), and no two of a
// row are alike.
#include "tsa_common.h"

namespace tsa {

struct LogprobArgs {
  float* logp;
  float* entropy;
  float* top_logp;
  int64_t* top_tok;
  const void* x;
  const void* tokens;
  int64_t lp_s, en_s, tl_s0, tl_s1, tt_s0, tt_s1, x_s0, x_s1, tok_s;
  int64_t N;
  int32_t V, top;
  bool tok64;
};

constexpr int kMaxTop = 64;

__device__ __forceinline__ uint64_t rank_of(float x, uint32_t i) {
  uint32_t b = __float_as_uint(x + 0.f);
  b ^= b & 0x80000000u ? 0xFFFFFFFFu : 0x80000000u;
  if (x != x) b = 0;
  return (static_cast<uint64_t>(b) << 32) | (0xFFFFFFFFu - i);
}
__device__ __forceinline__ uint32_t index_of(uint64_t rank) { return 0xFFFFFFFFu - static_cast<uint32_t>(rank); }

__device__ __forceinline__ int64_t token_of(const LogprobArgs& a, int64_t row) {
  return a.tok64 ? static_cast<const int64_t*>(a.tokens)[row * a.tok_s] : static_cast<const int32_t*>(a.tokens)[row * a.tok_s];
}

// Any strides: a workgroup a row, the row read for the maximum, the sums and each
// alternative.
template <typename T>
__global__ __launch_bounds__(256) void token_logprobs_rows(LogprobArgs a) {
  __shared__ uint64_t best[4];
  __shared__ float sums[2][4];
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  for (int64_t row = blockIdx.x; row < a.N; row += gridDim.x) {
    const T* const x = static_cast<const T*>(a.x) + row * a.x_s0;
    float m = -INFINITY;
    for (int i = tid; i < a.V; i += 256) m = fmaxf(m, to_float(x[i * a.x_s1]));
    for (int off = 32; off >= 1; off >>= 1) m = fmaxf(m, __shfl_xor(m, off, 64));
    if (lane == 0) sums[0][w] = m;
    __syncthreads();
    m = fmaxf(fmaxf(sums[0][0], sums[0][1]), fmaxf(sums[0][2], sums[0][3]));
    __syncthreads();
    float S = 0.f, E = 0.f;
    for (int i = tid; i < a.V; i += 256) {
      const float t = to_float(x[i * a.x_s1]) - m, p = expf(t);
      S += p;
      E += p == 0.f ? 0.f : p * t;
    }
    for (int off = 32; off >= 1; off >>= 1) {
      S += __shfl_xor(S, off, 64);
      E += __shfl_xor(E, off, 64);
    }
    if (lane == 0) {
      sums[0][w] = S;
      sums[1][w] = E;
    }
    __syncthreads();
    S = (sums[0][0] + sums[0][1]) + (sums[0][2] + sums[0][3]);
    E = (sums[1][0] + sums[1][1]) + (sums[1][2] + sums[1][3]);
    const float lse = logf(S);
    if (tid == 0) {
      const int64_t t = token_of(a, row);
      a.logp[row * a.lp_s] = (t >= 0 && t < a.V ? to_float(x[t * a.x_s1]) - m : -INFINITY) - lse;
      a.entropy[row * a.en_s] = lse - E / S;
    }
    uint64_t last = ~uint64_t{0};
    for (int k = 0; k < a.top; ++k) {
      uint64_t b = 0;
      for (int i = tid; i < a.V; i += 256) {
        const uint64_t r = rank_of(to_float(x[i * a.x_s1]), i);
        b = r < last && r > b ? r : b;
      }
      for (int off = 32; off >= 1; off >>= 1) {
        const uint64_t o = __shfl_xor(b, off, 64);
        b = o > b ? o : b;
      }
      if (lane == 0) best[w] = b;
      __syncthreads();
      b = best[0];
      for (int i = 1; i < 4; ++i) b = best[i] > b ? best[i] : b;
      if (tid == 0) {
        const int i = static_cast<int>(index_of(b));
        a.top_tok[row * a.tt_s0 + k * a.tt_s1] = i;
        a.top_logp[row * a.tl_s0 + k * a.tl_s1] = (to_float(x[i * a.x_s1]) - m) - lse;
      }
      last = b;
      __syncthreads();
    }
  }
}

template <typename T>
static int launch_rows(const LogprobArgs& a, hipStream_t stream) {
  const uint32_t grid = static_cast<uint32_t>(a.N < 65536 ? a.N : 65536);
  token_logprobs_rows<T><<<dim3(grid), dim3(256), 0, stream>>>(a);
  return check_launch("tsa_token_logprobs");
}

}  // namespace tsa

using namespace tsa;

extern "C" int tsa_token_logprobs(const tsa_view* logprobs, const tsa_view* entropy, const tsa_view* top_logprobs,
                                  const tsa_view* top_tokens, const tsa_view* logits, const tsa_view* tokens,
                                  void* workspace, size_t workspace_bytes, void* stream) {
  TSA_REQUIRE(view_ok(logits, 2) && is_float_dtype(logits->dtype), "logits must be a 2D floating tensor (num_tokens, vocab_size)");
  const int64_t N = logits->size[0], V = logits->size[1];
  TSA_REQUIRE(V >= 1 || N == 0, "logits must have a vocabulary");
  TSA_REQUIRE(view_ok(tokens, 1) && is_index_dtype(tokens->dtype) && tokens->size[0] == N,
              "tokens must be a 1D int32 or int64 tensor, one for each row of logits");
  TSA_REQUIRE(view_ok(logprobs, 1) && logprobs->dtype == TSA_F32 && logprobs->size[0] == N, "logprobs must be a 1D float32 tensor (num_tokens)");
  TSA_REQUIRE(view_ok(entropy, 1) && entropy->dtype == TSA_F32 && entropy->size[0] == N, "entropy must be a 1D float32 tensor (num_tokens)");
  TSA_REQUIRE(view_ok(top_logprobs, 2) && top_logprobs->dtype == TSA_F32 && top_logprobs->size[0] == N,
              "top_logprobs must be a 2D float32 tensor (num_tokens, num_top)");
  const int64_t top = top_logprobs->size[1];
  TSA_REQUIRE(view_ok(top_tokens, 2) && top_tokens->dtype == TSA_I64 && top_tokens->size[0] == N && top_tokens->size[1] == top,
              "top_tokens must be a 2D int64 tensor shaped like top_logprobs");
  TSA_REQUIRE(top <= V || N == 0, "num_top (%lld) is larger than the vocabulary (%lld)", (long long)top, (long long)V);
  TSA_UNSUPPORTED(top <= kMaxTop, "more than %d alternatives are not implemented (got %lld)", kMaxTop, (long long)top);
  TSA_UNSUPPORTED(V < (int64_t{1} << 30), "a vocabulary of 2^30 and more is not implemented");
  if (N == 0) return TSA_OK;
  LogprobArgs a;
  a.logp = static_cast<float*>(logprobs->data); a.entropy = static_cast<float*>(entropy->data);
  a.top_logp = static_cast<float*>(top_logprobs->data); a.top_tok = static_cast<int64_t*>(top_tokens->data);
  a.x = logits->data; a.tokens = tokens->data;
  a.lp_s = logprobs->stride[0]; a.en_s = entropy->stride[0];
  a.tl_s0 = top_logprobs->stride[0]; a.tl_s1 = top_logprobs->stride[1];
  a.tt_s0 = top_tokens->stride[0]; a.tt_s1 = top_tokens->stride[1];
  a.x_s0 = logits->stride[0]; a.x_s1 = logits->stride[1];
  a.tok_s = tokens->stride[0];
  a.N = N; a.V = static_cast<int32_t>(V); a.top = static_cast<int32_t>(top);
  a.tok64 = tokens->dtype == TSA_I64;
  (void)workspace;
  (void)workspace_bytes;
  const hipStream_t st = static_cast<hipStream_t>(stream);
  switch (logits->dtype) {
    case TSA_BF16: return launch_rows<bf16_t>(a, st);
    case TSA_F16: return launch_rows<f16_t>(a, st);
    default: return launch_rows<float>(a, st);
  }
}

extern "C" size_t tsa_token_logprobs_workspace_bytes(int64_t, int64_t, int64_t) { return 0; }
