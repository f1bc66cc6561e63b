// The decode step over part of the context or over an 8-bit cache, on the
// matrix cores: one workgroup takes up to NW * KT 16-token tiles of one
// (sequence, kv head) unit, all of them in one shot.
//
// What bounds it: HBM for long contexts (each visible K/V byte is read once,
// for all the q-heads of the kv head), the chain length -> block table -> K/V
// -> merge for short ones. So a unit's visible tiles (those of the first
// tokens, then the window's) are split over workgroups, nothing is computed from other sequences,
// and every K/V row of a workgroup is in flight at once; a wave scores its KT
// tiles together (one row maximum, one exponential pass, no rescaling).
//
// With lane (g, c) = (lane / 16, lane % 16), for up to 16 q-heads of a kv head:
//   S^T(16 tokens x 16 heads) = K Q^T on v_mfma_f32_16x16x32: K's operand is
//     16-byte pieces of token c's row, Q's the same dims of head c; element r
//     of the result is token 4 g + r, head c.
//   O(heads x dims) += P V, a pair of tiles at a time: P's operand is the lane's
//     own weights, V's the lane's D / 16 dims of its 4 tokens of either tile.
// An 8-bit cache is widened in registers, exactly: e4m3 and int8 codes are
// numbers of bf16 and f16. A token's key scale multiplies its scores, its value
// scale its weights, so no element is scaled. K takes 16-byte pieces of 16
// dims, two steps of the product each (Q is read in that order); V's bytes are
// transposed as they are widened. The weights go to the product as two 16-bit
// halves, hi + lo (16 significant bits, 22 in f16): the matrix cores have the
// slack; for an 8-bit cache in bf16 always, whose range holds weight x scale
// whatever the scale.
#pragma once

#include <type_traits>

#include "nonfinite.h"
#include "paged_decode.h"
#include "paged_rows.h"

namespace tsa {

template <typename C> constexpr bool kIs8 = sizeof(C) == 1;
// Tiles of a wave: 64 tokens. (Eight in 8 bits, 512 tokens a workgroup of four
// waves: 4 x 512-1024 tokens, 16/8 heads, 13.2 us against 8.5.)
constexpr int kUnitTiles = 4;
constexpr int kUnitWavesOne = 8;    // a unit that is one workgroup
constexpr int kUnitWavesSplit = 4;  // a split's workgroup
// Floats of one row of a partial: acc[D], m, l, padded to 16 bytes.
__host__ __device__ constexpr int part_floats(int D) { return D + 4; }

// A sequence's visible tiles: first (the first tokens'), then those from w0 on.
struct UnitTiles {
  int L, lo, first, w0, n;
  __device__ __forceinline__ int at(int v) const { return v < first ? v : v - first + w0; }
};
__device__ __forceinline__ UnitTiles unit_tiles(const RowsArgs& a, int len) {
  UnitTiles t{len, 0, 0, 0, (len + 15) >> 4};
  if (a.window > 0 && len > a.window) {
    t.lo = len - a.window;
    t.w0 = t.lo >> 4;
    t.first = min((min(a.sinks, t.lo) + 15) >> 4, t.w0);
    t.n += t.first - t.w0;
  }
  return t;
}
__device__ __forceinline__ int unit_length(const RowsArgs& a, const int32_t* lens, int s) {
  const int cap = a.NB > 0 ? a.max_blocks * a.BS : 0;  // (< 2^27)
  return min(max(lens[s * a.len_s], 0), cap);
}

// Two codes of a dword as a pair of T: the low or the high half-word's.
template <typename C, typename T, bool HI> __device__ __forceinline__ uint32_t widen2(uint32_t w) {
  if constexpr (std::is_same<C, e4m3_t>::value) {
    if constexpr (std::is_same<T, bf16_t>::value)
      return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.f, HI));
    else
      return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.f, HI));
  } else if constexpr (std::is_same<T, f16_t>::value) {
    // 1024 + (code + 128) is the f16 whose low byte is code + 128; less 1152, exactly the code. (Five instructions
    // for four codes; nine by conversions.)
    typedef _Float16 h2 __attribute__((ext_vector_type(2)));
    const h2 x = __builtin_bit_cast(h2, __builtin_amdgcn_perm(0x64646464u, w ^ 0x80808080u, HI ? 0x04030402u : 0x04010400u));
    return __builtin_bit_cast(uint32_t, x - h2{1152, 1152});
  } else {
    constexpr int b = HI ? 16 : 0;
    return pack2<T>(static_cast<float>(static_cast<int8_t>(w >> b)), static_cast<float>(static_cast<int8_t>(w >> (b + 8))));
  }
}

// The K operand of one step: 8 codes of two dwords as 8 T.
template <typename C, typename T> __device__ __forceinline__ u32x4 widen8(uint32_t w0, uint32_t w1) {
  return u32x4{widen2<C, T, false>(w0), widen2<C, T, true>(w0), widen2<C, T, false>(w1), widen2<C, T, true>(w1)};
}

template <bool NT, typename P, typename S> __device__ __forceinline__ P load_piece(const S* p) {
  if constexpr (NT) return __builtin_nontemporal_load(reinterpret_cast<const P*>(p));
  else return *reinterpret_cast<const P*>(p);
}

// Dim u of two tokens' V pieces (a, b) as a pair of the product's type.
template <typename C, typename T, typename P> __device__ __forceinline__ uint32_t v_pair(const P& a, const P& b, int u) {
  if constexpr (!kIs8<C>) {
    return (u & 1) ? pack_hi(word_of(a, u >> 1), word_of(b, u >> 1)) : pack_lo(word_of(a, u >> 1), word_of(b, u >> 1));
  } else {
    // bytes a.x b.x a.x+1 b.x+1 of the dword, x = 0 or 2: the pairs of dims x and x + 1
    const uint32_t w = __builtin_amdgcn_perm(word_of(b, u >> 2), word_of(a, u >> 2), (u & 2) ? 0x07030602u : 0x05010400u);
    return (u & 1) ? widen2<C, T, true>(w) : widen2<C, T, false>(w);
  }
}

// Element r times the value of lane r of the lane's quad (quad_perm
// broadcasts): with lane (g, c) holding the scale of token 4 g + c % 4, the
// four tokens' of its row group.
__device__ __forceinline__ f32x4 scale_tokens(f32x4 x, float s) {
  const uint32_t b = __builtin_bit_cast(uint32_t, s);
  return f32x4{x[0] * __builtin_bit_cast(float, dpp32<0x00, 0xf, false>(b)), x[1] * __builtin_bit_cast(float, dpp32<0x55, 0xf, false>(b)),
               x[2] * __builtin_bit_cast(float, dpp32<0xAA, 0xf, false>(b)), x[3] * __builtin_bit_cast(float, dpp32<0xFF, 0xf, false>(b))};
}

// Wave vw of NW, of unit u, split sp: its partial to slots[vw] ([rows][D + 4]).
template <typename T, typename C, int D, int NW, bool NT>
__device__ __forceinline__ void rows_unit_wave(const RowsArgs& a, const int32_t* __restrict__ bt, int s, int kvh, int g0,
                                               int rows, int t0, const UnitTiles& ut, int vw, float* slots) {
  constexpr int KT = kUnitTiles, kTiles = NW * KT, eb = sizeof(C);
  constexpr int KL = D * eb / 64;   // 16-byte K pieces of a lane
  constexpr int KJ = D / 32;        // steps of the score product
  constexpr int NU = D / 16;        // dims of a lane in the second product
  typedef typename VPiece<NU * eb>::type VP;
  typedef typename std::conditional<kIs8<C>, bf16_t, T>::type PT;
  static_assert(kTiles <= 64, "a lane per tile");
  const int lane = threadIdx.x & 63, g = lane >> 4, c = lane & 15;

  // Lane j: the split's tile j, its page and first slot.
  const int my_v = t0 + (lane & (kTiles - 1));
  // (Without a window a tile's place does not wait for the length: a branch that
  // stays one, so that the page ids load beside it.)
  int my_at = my_v;
  if (a.window > 0) {
    my_at = ut.at(my_v);
    asm volatile("" : "+v"(my_at));
  }
  const uint32_t my_tile = static_cast<uint32_t>(my_at), my_lb = page_of_tile(my_tile, a.page_mul, a.page_shift);
  const int my_slot = static_cast<int>(16u * my_tile - my_lb * static_cast<uint32_t>(a.BS));
  const int my_page = bt[s * a.bt_s0 + min(static_cast<int>(my_lb), a.max_blocks - 1) * a.bt_s1];
  const uint64_t ok64 = __ballot(my_v < ut.n && my_page >= 0 && my_page < a.NB);

  u32x4 q[KJ];
  {
    const T* const qrow = static_cast<const T*>(a.q) + s * a.q_sr + (kvh * a.G + g0 + min(c, rows - 1)) * a.q_sh;
#pragma unroll
    for (int j = 0; j < KJ; ++j) {
      const int d = kIs8<C> ? 16 * (g + 4 * (j >> 1)) + 8 * (j & 1) : 8 * (g + 4 * j);
      q[j] = *reinterpret_cast<const u32x4*>(qrow + d);
    }
  }

  // Rows of pages outside the pool read row 0 of page 0 and are masked; tiles
  // past the unit's end are not read.
  u32x4 ko[KT][KL];
  VP vo[KT][4];
  float ks[KT], vs[KT];  // (8-bit) the scales of token 4 g + c % 4
  uint32_t vis[KT];      // bit i: token i of the tile is seen
  const char* const kbase = static_cast<const char*>(a.kc) + kvh * a.kc_h * eb;
  const char* const vbase = static_cast<const char*>(a.vc) + kvh * a.vc_h * eb;
  const char* const ksbase = reinterpret_cast<const char*>(a.ks + kvh * a.ks_h);
  const char* const vsbase = reinterpret_cast<const char*>(a.vs + kvh * a.vs_h);
  const uint32_t k_lane = static_cast<uint32_t>(c * static_cast<int>(a.kc_s) * eb + 16 * g);
  const uint32_t v_lane = static_cast<uint32_t>((4 * g) * static_cast<int>(a.vc_s) * eb + NU * eb * c);
  const uint32_t ks_lane = static_cast<uint32_t>((4 * g + (c & 3)) * static_cast<int>(a.ks_s) * 4);
  const uint32_t vs_lane = static_cast<uint32_t>((4 * g + (c & 3)) * static_cast<int>(a.vs_s) * 4);
#pragma unroll
  for (int x = 0; x < KT; ++x) {
    const int j = vw + NW * x;
    vis[x] = 0;
    if (t0 + j < ut.n) {  // (uniform)
      const bool ok = (ok64 >> j) & 1;
      const uint32_t page = ok ? __builtin_amdgcn_readlane(my_page, j) : 0;
      const int slot0 = ok ? __builtin_amdgcn_readlane(my_slot, j) : 0;
      const int tok0 = 16 * ut.at(t0 + j), left = ut.L - tok0;
      uint32_t m16 = left >= 16 ? 0xFFFFu : (1u << left) - 1u;
      if (ut.lo > tok0) {
        const uint32_t in_window = ut.lo - tok0 >= 16 ? 0u : 0xFFFFu << (ut.lo - tok0);
        const int first = a.sinks - tok0;
        m16 &= in_window | (first >= 16 ? 0xFFFFu : first > 0 ? (1u << first) - 1u : 0u);
      }
      vis[x] = ok ? m16 : 0u;
      const char* const kp = kbase + static_cast<uint64_t>(page) * a.k_page + slot0 * static_cast<int>(a.kc_s) * eb;
      const char* const vp = vbase + static_cast<uint64_t>(page) * a.v_page + slot0 * static_cast<int>(a.vc_s) * eb;
#pragma unroll
      for (int i = 0; i < KL; ++i) ko[x][i] = load_piece<NT, u32x4>(kp + k_lane + 64 * i);
#pragma unroll
      for (int r = 0; r < 4; ++r) vo[x][r] = load_piece<NT, VP>(vp + r * static_cast<int>(a.vc_s) * eb + v_lane);
      if constexpr (kIs8<C>) {
        ks[x] = *reinterpret_cast<const float*>(ksbase + static_cast<uint64_t>(page) * a.ks_page +
                                                slot0 * static_cast<int>(a.ks_s) * 4 + ks_lane);
        vs[x] = *reinterpret_cast<const float*>(vsbase + static_cast<uint64_t>(page) * a.vs_page +
                                                slot0 * static_cast<int>(a.vs_s) * 4 + vs_lane);
      }
    } else {
#pragma unroll
      for (int i = 0; i < KL; ++i) ko[x][i] = u32x4{0, 0, 0, 0};
#pragma unroll
      for (int r = 0; r < 4; ++r) vo[x][r] = VP{};
      ks[x] = vs[x] = 0.f;
    }
  }

  // ---- Scores and the row maximum.
  float sv[KT][4], m = kNegInfR;
#pragma unroll
  for (int x = 0; x < KT; ++x) {
    f32x4 sc = f32x4{0.f, 0.f, 0.f, 0.f};
    if (t0 + vw + NW * x < ut.n) {  // (uniform)
      if constexpr (kIs8<C>) {
#pragma unroll
        for (int j = 0; j < KJ; ++j)
          sc = mfma_k32<T>(widen8<C, T>(ko[x][j >> 1][2 * (j & 1)], ko[x][j >> 1][2 * (j & 1) + 1]), q[j], sc);
        sc = scale_tokens(sc, ks[x]);
      } else {
#pragma unroll
        for (int j = 0; j < KJ; ++j) sc = mfma_k32<T>(ko[x][j], q[j], sc);
      }
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) sv[x][r] = sc[r] * a.scale_log2;
    if (vis[x] != 0xFFFFu) {  // (uniform) tokens that are not seen: no weight, and no V that 0 would not cancel
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (!((vis[x] >> (4 * g + r)) & 1)) {
          sv[x][r] = kNegInfR;
          vo[x][r] = VP{};
        }
      if constexpr (kIs8<C>)
        if (!((vis[x] >> (4 * g + (c & 3))) & 1)) vs[x] = 0.f;
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) m = fmaxf(m, sv[x][r]);
  }
  m = fmaxf(m, __builtin_bit_cast(float, xor_lane32<16>(__builtin_bit_cast(uint32_t, m), lane)));
  m = fmaxf(m, __builtin_bit_cast(float, xor_lane32<32>(__builtin_bit_cast(uint32_t, m), lane)));
  const float mu = m == kNegInfR ? 0.f : m;  // (-inf: every score is -inf, and weighs 0)

  // ---- O += P V, pairs of tiles. acc[u][r] = O[head 4 g + r][dim NU c + u].
  float l = 0.f;
  f32x4 acc[NU];
#pragma unroll
  for (int u = 0; u < NU; ++u) acc[u] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int x = 0; x < KT; x += 2) {
    if (t0 + vw + NW * x >= ut.n) continue;  // (uniform)
    u32x4 hi, lo;
#pragma unroll
    for (int y = 0; y < 2; ++y) {
      float p[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        p[r] = fast_exp2(sv[x + y][r] - mu);
        l += p[r];
      }
      if constexpr (kIs8<C>) {
        const f32x4 ps = scale_tokens(f32x4{p[0], p[1], p[2], p[3]}, vs[x + y]);
#pragma unroll
        for (int r = 0; r < 4; ++r) p[r] = ps[r];
      }
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        hi[2 * y + k] = pack2<PT>(p[2 * k], p[2 * k + 1]);
        lo[2 * y + k] = pack2<PT>(p[2 * k] - lo_f<PT>(hi[2 * y + k]), p[2 * k + 1] - hi_f<PT>(hi[2 * y + k]));
      }
    }
#pragma unroll
    for (int u = 0; u < NU; ++u) {
      u32x4 b;
#pragma unroll
      for (int y = 0; y < 2; ++y)
#pragma unroll
        for (int k = 0; k < 2; ++k) b[2 * y + k] = v_pair<C, PT>(vo[x + y][2 * k], vo[x + y][2 * k + 1], u);
      acc[u] = mfma_k32<PT>(hi, b, acc[u]);
      acc[u] = mfma_k32<PT>(lo, b, acc[u]);
    }
  }
  l += __builtin_bit_cast(float, xor_lane32<16>(__builtin_bit_cast(uint32_t, l), lane));
  l += __builtin_bit_cast(float, xor_lane32<32>(__builtin_bit_cast(uint32_t, l), lane));
  float* const slot = slots + vw * rows * part_floats(D);
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const int row = 4 * g + r;
    if (row < rows) {
      float* const dst = slot + row * part_floats(D) + NU * c;
#pragma unroll
      for (int u = 0; u < NU; u += 4)
        *reinterpret_cast<f32x4*>(dst + u) = f32x4{acc[u][r], acc[u + 1][r], acc[u + 2][r], acc[u + 3][r]};
    }
  }
  if (g == 0 && c < rows) {
    slot[c * part_floats(D) + D] = m;
    slot[c * part_floats(D) + D + 1] = l;
  }
}

// Grid: splits x (units x groups of 16 heads), the latter fastest.
template <typename T, typename C, int D, int NW, bool NT>
__global__ __launch_bounds__(64 * NW) __attribute__((amdgpu_waves_per_eu(2))) void paged_rows_unit(
    RowsArgs a, const int32_t* __restrict__ bt, const int32_t* __restrict__ lens, float* __restrict__ part) {
  extern __shared__ __align__(16) float slots[];  // [NW][rows][D + 4]
  constexpr int kTiles = NW * kUnitTiles, PF = part_floats(D);
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int groups = (a.G + 15) / 16, items = a.B * a.Hkv * groups;
  const int sp = static_cast<int>(blockIdx.x) / items, it = static_cast<int>(blockIdx.x) - sp * items;
  const int u = it / groups, g0 = 16 * (it - u * groups), rows = min(16, a.G - g0);
  const int s = u / a.Hkv, kvh = u - s * a.Hkv;
  const UnitTiles ut = unit_tiles(a, __builtin_amdgcn_readfirstlane(unit_length(a, lens, s)));
  const int t0 = kTiles * sp, nt = min(max(ut.n - t0, 0), kTiles);
  if (nt == 0 && a.S > 1) return;  // (the merge takes the splits that have tiles)
  if (wave < nt) rows_unit_wave<T, C, D, NW, NT>(a, bt, s, kvh, g0, rows, t0, ut, wave, slots);
  lds_barrier();
  const int nw = min(nt, NW);
  for (int idx = tid; idx < rows * D; idx += 64 * NW) {
    const int row = idx / D, d = idx - row * D;
    float M = kNegInfR, den = 0.f, o = 0.f;
    for (int w = 0; w < nw; ++w) {
      const float* const x = slots + (w * rows + row) * PF;
      combine_partial(M, den, o, x[D], x[D + 1], x[d]);
    }
    if (a.S == 1) {
      static_cast<T*>(a.out)[s * a.o_sr + (kvh * a.G + g0 + row) * a.o_sh + d * a.o_sd] =
          from_float<T>(den == 0.f ? 0.f : o / den);
    } else {
      float* const out = part + ((static_cast<int64_t>(u) * a.S + sp) * a.G + g0 + row) * PF;
      out[d] = o;
      if (d == 0) {
        out[D] = M;
        out[D + 1] = den;
      }
    }
  }
}

// Outputs from the partials of a unit's splits, 4 dims a lane, 64 / (D / 4) rows
// a wave. Few rows with many splits (SHARE): the four waves of a workgroup take
// the same rows, a quarter of the splits each, then the quarters in order; else
// each wave takes rows of its own and all their splits. Splits go in batches
// whose loads are issued together (past the last: repeated and dropped). Grid:
// units x row groups. tiles_per_split: decode's (trees: tree_per_split).
template <typename T, int D, bool SHARE>
__global__ __launch_bounds__(256) void paged_rows_merge(RowsArgs a, const int32_t* __restrict__ lens,
                                                        const float* __restrict__ part, int tiles_per_split) {
  constexpr int LR = D / 4, RW = 64 / LR, PF = part_floats(D), kBatch = SHARE ? 8 : 4;
  __shared__ __align__(16) float red[SHARE ? 4 : 1][RW][PF];
  const int u = blockIdx.x, s = u / a.Hkv, kvh = u - s * a.Hkv;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int n;  // splits with tiles
  int64_t row0;
  int nrows;
  if (a.cu) {
    const SeqRange r = seq_of(a, s);
    const int nblk = (r.end + 31) >> 5, per = tree_per_split(a, nblk);
    n = (nblk + per - 1) / per;
    row0 = r.row0;
    nrows = r.nodes * a.G;
  } else {
    n = (unit_tiles(a, unit_length(a, lens, s)).n + tiles_per_split - 1) / tiles_per_split;
    row0 = s;
    nrows = a.G;
  }
  const int all_rows = a.T * a.G;
  const int group = SHARE ? static_cast<int>(blockIdx.y) : 4 * static_cast<int>(blockIdx.y) + wave;
  const int row = group * RW + lane / LR, d = 4 * (lane % LR);
  if (group * RW >= nrows) return;
  const int rr = min(row, nrows - 1);
  const int per = SHARE ? (n + 3) / 4 : n;
  const int first = SHARE ? min(n, wave * per) : 0, last = SHARE ? min(n, first + per) : n;
  const float* const base = part + (static_cast<int64_t>(u) * a.S * all_rows + rr) * PF;
  const int64_t step = static_cast<int64_t>(all_rows) * PF;
  float M = kNegInfR, den = 0.f;
  f32x4 o = f32x4{0.f, 0.f, 0.f, 0.f};
  auto take = [&](float m, float l, f32x4 x) {
    const float mn = fmaxf(M, m), mu = mn == kNegInfR ? 0.f : mn;
    const float c_old = fast_exp2(M - mu), c_new = fast_exp2(m - mu);
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = fmaf(x[i], c_new, o[i] * c_old);
    den = fmaf(l, c_new, den * c_old);
    M = mn;
  };
  for (int sp = first; sp < last; sp += kBatch) {
    f32x4 po[kBatch];
    f32x2 ml[kBatch];
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      const float* const x = base + min(sp + k, last - 1) * step;
      po[k] = *reinterpret_cast<const f32x4*>(x + d);
      ml[k] = *reinterpret_cast<const f32x2*>(x + D);
    }
#pragma unroll
    for (int k = 0; k < kBatch; ++k)
      if (sp + k < last) take(ml[k][0], ml[k][1], po[k]);
  }
  if constexpr (SHARE) {
    float* const mine = red[wave][lane / LR];
    *reinterpret_cast<f32x4*>(mine + d) = o;
    if (d == 0) {
      mine[D] = M;
      mine[D + 1] = den;
    }
    __syncthreads();
    if (wave > 0) return;
#pragma unroll
    for (int w = 1; w < 4; ++w) {
      const float* const x = red[w][lane / LR];
      take(x[D], x[D + 1], *reinterpret_cast<const f32x4*>(x + d));
    }
  }
  if (row >= nrows) return;
  const int node = row / a.G;
  T* const out = static_cast<T*>(a.out) + (row0 + node) * a.o_sr + (kvh * a.G + row - node * a.G) * a.o_sh;
  const float inv = den == 0.f ? 0.f : 1.f / den;
  if (a.out8) {
    u32x2 w;
#pragma unroll
    for (int i = 0; i < 2; ++i) w[i] = den == 0.f ? 0u : pack2<T>(o[2 * i] * inv, o[2 * i + 1] * inv);
    *reinterpret_cast<u32x2*>(out + d) = w;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) out[(d + i) * a.o_sd] = from_float<T>(den == 0.f ? 0.f : o[i] * inv);
  }
}

// Splits from which the waves of the merge share rows. Both sides, rows of their
// own / shared, us, the call with its merge: decode, e4m3, 8 sequences, 32/8 heads, 3
// splits 11.3 / 11.4, 4 11.5 / 11.7 (128/8 heads: 13.2 / 13.9), 5 13.8 / 13.8, 6 14.3 /
// 14.2, 8 15.1 / 15.0, 4 sequences of 16 16.9 / 15.2, one of 128 (64/8 heads) 27.6 /
// 20.9; trees of 4-8 nodes, 32/8 heads, 4 splits 43.9 / 46.1, 6 38.1 / 38.8, 8 30.3 /
// 30.8, 16 21.9 / 19.7; of 40-64 nodes, 64/8 heads, 2 splits 145 / 161, 8 39.1 / 42.2.
constexpr int kMergeShare = 6;
template <typename T, int D>
inline void launch_rows_merge(const RowsArgs& a, int rows, int tiles_per_split, hipStream_t stream) {
  constexpr int RW = 64 / (D / 4);
  const int groups = (rows + RW - 1) / RW;
  if (a.S >= kMergeShare)
    paged_rows_merge<T, D, true><<<dim3(a.B * a.Hkv, groups), dim3(256), 0, stream>>>(a, a.lens, a.part, tiles_per_split);
  else
    paged_rows_merge<T, D, false><<<dim3(a.B * a.Hkv, (groups + 3) / 4), dim3(256), 0, stream>>>(a, a.lens, a.part, tiles_per_split);
}

}  // namespace tsa
