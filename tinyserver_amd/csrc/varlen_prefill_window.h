// Windowed prefill (PrefillWindowArgs in varlen_prefill_gqa.h): one row, by one
// wave on the vector units; and 32 rows again, by one wave on the matrix cores,
// where V values that are not finite may have reached rows that do not see them.
#pragma once

#include "nonfinite.h"
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

// Whether a key of the blocks `win` that some of the queries [q, q + 32) of a
// sequence (those below q_len) do not see has a V that is not finite. Only blocks
// that hold such a key are read: the diagonal's, the window's low end's, that of
// the first tokens' end, and any behind the queries.
template <typename T, int D>
__device__ __forceinline__ bool window_leaks(const PrefillWindowArgs& a, const WindowBlocks& win, int q, int q_len,
                                             int kvh, int64_t k_start, int k_len) {
  constexpr int NU = D / 32;
  typedef typename VPiece<2 * NU>::type VP;
  const int lane = threadIdx.x & 63, h = lane >> 5, c = lane & 31;
  const T* const vb = static_cast<const T*>(a.v) + k_start * a.v_st + kvh * a.v_sh + NU * c;
  bool bad = false;
#pragma unroll 1
  for (int v = 0; v < win.count; ++v) {
    const int k0 = 32 * win.at(v);
    if (window_sees_all(a, q, k0, k_len)) continue;
    uint32_t all = window_bits(a, min(q + c, q_len - 1), k0, k_len);  // keys that every query sees
#pragma unroll
    for (int off = 16; off >= 1; off >>= 1) all &= static_cast<uint32_t>(__shfl_xor(static_cast<int>(all), off, 64));
    const uint32_t unseen = ~all & (k_len - k0 >= 32 ? ~0u : (1u << (k_len - k0)) - 1u);
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const int i = 8 * (e >> 2) + 4 * h + (e & 3);
      if (!((unseen >> i) & 1)) continue;
      const VP w = *reinterpret_cast<const VP*>(vb + (k0 + i) * a.v_st);
#pragma unroll
      for (int x = 0; x < NU / 2; ++x) bad |= nonfinite2<T>(word_of(w, x)) != 0;
    }
  }
  return __any(bad);
}

// The outputs of queries [q0, q0 + 32) of a sequence (those below q_len), q-head
// h, by one wave: S^T = K Q^T and O^T += V^T P^T on v_mfma_f32_32x32x16 as the
// draft trees' register kernel has them (lane (h, c): row c's softmax and
// outputs), K and V straight from memory. Values of V that are not finite reach
// the rows that see them alone (take_nonfinite, in every block).
template <typename T, int D>
__device__ __forceinline__ void prefill_window_tile(const PrefillWindowArgs& a, int64_t q_start, int q0, int q_len,
                                                    int head, int64_t k_start, int k_len) {
  constexpr int KJ = D / 16, NU = D / 32;
  constexpr float kRescale = 8.f;
  typedef typename VPiece<2 * NU>::type VP;
  const int lane = threadIdx.x & 63, h = lane >> 5, c = lane & 31, kvh = head / a.G;
  const int row = q0 + c, live = min(row, q_len - 1);  // (past the last: it again, never stored)
  const T* const kb = static_cast<const T*>(a.k) + k_start * a.k_st + kvh * a.k_sh + 8 * h;
  const T* const vb = static_cast<const T*>(a.v) + k_start * a.v_st + kvh * a.v_sh + NU * c;
  const float cs = a.scale_log2;  // > 0 here
  u32x4 q[KJ];
  {
    const T* const qp = static_cast<const T*>(a.q) + (q_start + live) * a.q_st + head * a.q_sh + 8 * h;
#pragma unroll
    for (int j = 0; j < KJ; ++j) q[j] = *reinterpret_cast<const u32x4*>(qp + 16 * j);
  }
  const WindowBlocks win = window_blocks(a, q0, min(q_len, q0 + 32), k_len);
  float m = kNegInfP, l = 0.f;
  f32x16 acc[NU];
#pragma unroll
  for (int x = 0; x < NU; ++x)
#pragma unroll
    for (int e = 0; e < 16; ++e) acc[x][e] = 0.f;
  u32x4 kr[KJ];
  VP vr[16];
  auto load_k = [&](int v) __attribute__((always_inline)) {  // (keys past the last: it again, never seen)
    const T* const p = kb + min(32 * win.at(v) + c, k_len - 1) * a.k_st;
#pragma unroll
    for (int j = 0; j < KJ; ++j) kr[j] = *reinterpret_cast<const u32x4*>(p + 16 * j);
  };
  auto load_v = [&](int v) __attribute__((always_inline)) {
#pragma unroll
    for (int e = 0; e < 16; ++e)
      vr[e] = *reinterpret_cast<const VP*>(vb + min(32 * win.at(v) + 8 * (e >> 2) + 4 * h + (e & 3), k_len - 1) * a.v_st);
  };
  if (win.count > 0) {
    load_k(0);
    load_v(0);
  }
#pragma unroll 1
  for (int v = 0; v < win.count; ++v) {
    f32x16 sc;
#pragma unroll
    for (int e = 0; e < 16; ++e) sc[e] = 0.f;
#pragma unroll
    for (int j = 0; j < KJ; ++j) sc = mfma_k16x32<T>(kr[j], q[j], sc);
    const int next = min(v + 1, win.count - 1);
    load_k(next);
    const uint32_t seen = window_bits(a, live, 32 * win.at(v), k_len);
#pragma unroll
    for (int e = 0; e < 16; ++e) sc[e] = masked_score(sc[e], seen >> (4 * h), 8 * (e >> 2) + (e & 3));
    float mx = kNegInfP;
#pragma unroll
    for (int e = 0; e < 16; ++e) mx = fmaxf(mx, sc[e]);
    const auto sw = __builtin_amdgcn_permlane32_swap(__float_as_uint(mx), __float_as_uint(mx), false, false);
    const float mt = fmaxf(__uint_as_float(sw[0]), __uint_as_float(sw[1])) * cs;
    if (__any(mt > m + kRescale)) {
      const float mn = fmaxf(m, mt), alpha = mn == kNegInfP ? 1.f : fast_exp2(m - mn);
      l *= alpha;
#pragma unroll
      for (int x = 0; x < NU; ++x)
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[x][e] *= alpha;
      m = mn;
    }
    const float mu = m == kNegInfP ? 0.f : m;
    u32x4 pop[2];
    float p[16];
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      p[e] = fast_exp2(fmaf(sc[e], cs, -mu));
      l += p[e];
    }
#pragma unroll
    for (int e = 0; e < 16; e += 2) pop[e >> 3][(e & 7) >> 1] = pack2<T>(p[e], p[e + 1]);
    bool bad = false;
#pragma unroll
    for (int e = 0; e < 16; ++e)
#pragma unroll
      for (int x = 0; x < NU / 2; ++x) bad |= nonfinite2<T>(word_of(vr[e], x)) != 0;
    if (__any(bad)) take_nonfinite<T>(vr, acc, seen, h);
#pragma unroll
    for (int s2 = 0; s2 < 2; ++s2)
#pragma unroll
      for (int x = 0; x < NU; ++x) {
        u32x4 w;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const uint32_t w0 = word_of(vr[8 * s2 + 2 * k], x >> 1), w1 = word_of(vr[8 * s2 + 2 * k + 1], x >> 1);
          w[k] = x & 1 ? pack_hi(w0, w1) : pack_lo(w0, w1);
        }
        acc[x] = mfma_k16x32<T>(w, pop[s2], acc[x]);
      }
    load_v(next);
  }
  l += __shfl_xor(l, 32, 64);
  if (row >= q_len) return;
  const float inv = l == 0.f ? 0.f : 1.f / l;
  T* const out = static_cast<T*>(a.out) + (q_start + row) * a.o_st + head * a.o_sh;
#pragma unroll
  for (int e = 0; e < 16; ++e) {
    T* const dst = out + NU * (8 * (e >> 2) + 4 * h + (e & 3));
    uint32_t w[NU / 2];
#pragma unroll
    for (int x = 0; x < NU / 2; ++x) w[x] = l == 0.f ? 0u : pack2<T>(acc[2 * x][e] * inv, acc[2 * x + 1][e] * inv);
    if constexpr (NU == 4) *reinterpret_cast<u32x2*>(dst) = u32x2{w[0], w[NU / 2 - 1]};
    else *reinterpret_cast<uint32_t*>(dst) = w[0];
  }
}

// What an item whose sums were not all finite takes after the item loop. Both
// measured at window 512 + 4, 16 prompts of 128-2048 tokens, 32/8 heads (211 us
// without such a value): a NaN in a first token, which every later query sees, 258
// us (each such item is looked at, the first ones computed again), in a middle
// one 298, V of NaN alone (every item computed again, its K/V from memory) 1282;
// the rows one by one on the vector units took 28.6, 11.8 and 97 ms.
template <typename T, int D>
__device__ __forceinline__ void prefill_window_again(const PrefillWindowArgs& a, const WindowBlocks& win,
                                                     int64_t q_start, int q0, int q_len, int head, int64_t k_start,
                                                     int k_len, bool always) {
  if (q0 >= q_len) return;
  if (always || window_leaks<T, D>(a, win, q0, q_len, head / a.G, k_start, k_len))
    prefill_window_tile<T, D>(a, q_start, q0, q_len, head, k_start, k_len);
}

}  // namespace tsa
