// Values of V that are not finite, in blocks of keys that some rows do not see: a
// weight of 0 times an infinity or NaN is NaN, so those values leave the product
// of weights and V and reach the rows that see them through a product of flags.
#pragma once

#include <cmath>
#include <type_traits>

#include "tsa_common.h"

namespace tsa {

// A lane's piece of a V row: N bytes (4, 8 or 16).
template <int N> struct VPiece;
template <> struct VPiece<4> { typedef uint32_t type; };
template <> struct VPiece<8> { typedef u32x2 type; };
template <> struct VPiece<16> { typedef u32x4 type; };
__device__ __forceinline__ uint32_t word_of(uint32_t v, int) { return v; }
__device__ __forceinline__ uint32_t word_of(const u32x2& v, int i) { return v[i]; }
__device__ __forceinline__ uint32_t word_of(const u32x4& v, int i) { return v[i]; }

// Elements of a dword of T that are not finite: which (bit 0: low, 1: high).
template <typename T> __device__ __forceinline__ uint32_t nonfinite2(uint32_t w) {
  constexpr uint32_t kExp = std::is_same<T, bf16_t>::value ? 0x7F80u : 0x7C00u;
  return ((w & kExp) == kExp ? 1u : 0u) | (((w >> 16) & kExp) == kExp ? 2u : 0u);
}
// A 16-bit element as a flag of T: 0 (finite), 1 (+inf), 2^8 (-inf), 2^15 (NaN).
// Sums of up to 32 of each are told apart.
template <typename T> __device__ __forceinline__ uint32_t flag16(uint32_t x) {
  constexpr bool bf = std::is_same<T, bf16_t>::value;
  constexpr uint32_t kExp = bf ? 0x7F80u : 0x7C00u;
  if ((x & kExp) != kExp) return 0;
  if (x & (0x7FFFu ^ kExp)) return bf ? 0x4700u : 0x7800u;
  return x & 0x8000u ? (bf ? 0x4380u : 0x5C00u) : (bf ? 0x3F80u : 0x3C00u);
}
// What a sum of flags adds to an output.
__device__ __forceinline__ float flag_value(float n) {
  const int k = static_cast<int>(n);
  const bool nan = k >= 32768, pos = (k & 255) != 0, neg = ((k >> 8) & 127) != 0;
  return nan || (pos && neg) ? __builtin_nanf("") : pos ? INFINITY : neg ? -INFINITY : 0.f;
}

// A block of 32 keys on v_mfma_f32_32x32x16, O^T(dims x rows) += V^T P^T: lane
// (h, c) holds NU dims of keys 8 (e / 4) + 4 h + e % 4 in vr[e] and accumulates
// row c. Adds to acc, for each row and dim, the infinities and NaN of the keys the
// row sees (bits of vis: P is 1 where it sees a key, V a flag where it is not
// finite) and takes them out of vr.
template <typename T, int NU, typename VP>
__device__ __forceinline__ void take_nonfinite(VP (&vr)[16], f32x16 (&acc)[NU], uint32_t vis, int h) {
  constexpr uint32_t one = std::is_same<T, bf16_t>::value ? 0x3F80u : 0x3C00u;
  u32x4 sees[2];
#pragma unroll
  for (int e = 0; e < 16; e += 2) {
    const uint32_t b = vis >> (8 * (e >> 2) + 4 * h + (e & 3));
    sees[e >> 3][(e & 7) >> 1] = (b & 1 ? one : 0u) | (b & 2 ? one << 16 : 0u);
  }
#pragma unroll
  for (int x = 0; x < NU; ++x) {
    f32x16 n;
#pragma unroll
    for (int e = 0; e < 16; ++e) n[e] = 0.f;
#pragma unroll
    for (int s2 = 0; s2 < 2; ++s2) {
      u32x4 f;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const uint32_t w0 = word_of(vr[8 * s2 + 2 * k], x >> 1), w1 = word_of(vr[8 * s2 + 2 * k + 1], x >> 1);
        f[k] = flag16<T>((x & 1 ? w0 >> 16 : w0) & 0xFFFFu) | flag16<T>((x & 1 ? w1 >> 16 : w1) & 0xFFFFu) << 16;
      }
      n = mfma_k16x32<T>(f, sees[s2], n);
    }
#pragma unroll
    for (int e = 0; e < 16; ++e) acc[x][e] += flag_value(n[e]);
  }
#pragma unroll
  for (int e = 0; e < 16; ++e) {
    uint32_t w[NU / 2];
#pragma unroll
    for (int x = 0; x < NU / 2; ++x) {
      w[x] = word_of(vr[e], x);
      const uint32_t nf = nonfinite2<T>(w[x]);
      w[x] &= (nf & 1 ? 0xFFFF0000u : ~0u) & (nf & 2 ? 0xFFFFu : ~0u);
    }
    if constexpr (NU == 4) vr[e] = u32x2{w[0], w[NU / 2 - 1]};
    else vr[e] = w[0];
  }
}

}  // namespace tsa
