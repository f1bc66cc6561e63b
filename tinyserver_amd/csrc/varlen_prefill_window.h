// Windowed prefill (PrefillWindowArgs in varlen_prefill_gqa.h): one row, by one wave.
#pragma once

#include "varlen_prefill_gqa.h"

namespace tsa {

// Row qi of q/out (query qq of its sequence), q-head h, over the sequence's
// keys [k_start, k_start + k_len), by one wave: any strides, head_dim up to
// 512, fp32 on the vector units. Keys the query does not see are not read. A
// query that sees none gives 0.
template <typename T>
__device__ void prefill_window_row(const PrefillWindowArgs& a, int64_t qi, int64_t qq, int h, int64_t k_start,
                                   int64_t k_len) {
  const int lane = threadIdx.x & 63;
  const int kvh = h / a.G, D = a.D;
  const T* const qrow = static_cast<const T*>(a.q) + qi * a.q_st + h * a.q_sh;
  const T* const kb = static_cast<const T*>(a.k) + k_start * a.k_st + kvh * a.k_sh;
  const T* const vb = static_cast<const T*>(a.v) + k_start * a.v_st + kvh * a.v_sh;
  const int64_t kend = k_len < qq + 1 ? k_len : qq + 1;
  const int64_t lo = qq + 1 > a.window ? qq + 1 - a.window : 0;
  const int64_t first_end = a.sinks < lo ? a.sinks : lo;
  constexpr int kMaxPerLane = 8;
  float acc[kMaxPerLane];
#pragma unroll
  for (int i = 0; i < kMaxPerLane; ++i) acc[i] = 0.f;
  float m = kNegInfP, l = 0.f;
  // The first keys' chunks, then the window's (one run where they meet).
  for (int64_t base = first_end > 0 ? 0 : lo & ~int64_t{63}; base < kend;
       base = base + 64 < first_end || base + 64 >= lo ? base + 64 : lo & ~int64_t{63}) {
    const int64_t key = base + lane;
    const bool sees = key < kend && (key >= lo || key < first_end);
    float sc = kNegInfP;
    if (sees) {
      float dot = 0.f;
      for (int d = 0; d < D; ++d) dot += to_float(qrow[d * a.q_sd]) * to_float(kb[key * a.k_st + d * a.k_sd]);
      sc = dot * a.scale_log2;
    }
    float cmax = sc;
    for (int off = 32; off >= 1; off >>= 1) cmax = fmaxf(cmax, __shfl_xor(cmax, off, 64));
    const float m_new = fmaxf(m, cmax), mu = m_new == kNegInfP ? 0.f : m_new;
    const float alpha = fast_exp2(m - mu);
    const float p = fast_exp2(sc - mu);
    float psum = p;
    for (int off = 32; off >= 1; off >>= 1) psum += __shfl_xor(psum, off, 64);
    l = l * alpha + psum;
#pragma unroll
    for (int i = 0; i < kMaxPerLane; ++i) acc[i] *= alpha;
    for (uint64_t left = __ballot(sees); left; left &= left - 1) {
      const int j = __builtin_ctzll(left);
      const float pj = __shfl(p, j, 64);
      const T* const vr = vb + (base + j) * a.v_st;
#pragma unroll
      for (int i = 0; i < kMaxPerLane; ++i) {
        const int d = lane + 64 * i;
        if (d < D) acc[i] += pj * to_float(vr[d * a.v_sd]);
      }
    }
    m = m_new;
  }
  T* const orow = static_cast<T*>(a.out) + qi * a.o_st + h * a.o_sh;
#pragma unroll
  for (int i = 0; i < kMaxPerLane; ++i) {
    const int d = lane + 64 * i;
    if (d < D) orow[d * a.o_sd] = from_float<T>(l == 0.f ? 0.f : acc[i] / l);
  }
}

}  // namespace tsa
