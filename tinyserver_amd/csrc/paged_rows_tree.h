// Attention of drafted tokens' trees on the matrix cores: the rows of a unit
// (sequence, kv head) are its nodes' q-heads of that kv head, so every K/V byte
// read serves nodes x heads rows. This kernel takes up to 32 rows a unit
// (paged_rows_tree_lds.h the others).
//
// What bounds it: HBM (each K/V byte once; 64 sequences of 512-4096 tokens, 4
// nodes, 32/8 heads: 114 us, 5.3 TB/s). A workgroup of four waves takes a unit's
// rows, wave kg every fourth 32-key block. A unit's keys are split over
// workgroups, whose partials a second launch merges.
//
// With lane (h, c) = (lane / 32, lane % 32), v_mfma_f32_32x32x16:
//   S^T(32 keys x 32 rows) = K Q^T over D / 16 steps: lane (h, c) reads key c,
//     dims 16 j + 8 h..+8, and holds row c's Q; element e of the result is the
//     score of key 8 (e / 4) + 4 h + e % 4 for row c.
//   O^T(dims x rows) += V^T P^T over two 16-key steps s: the P^T operand is the
//     lane's own weights 8 s .. 8 s + 7, and V's operand is dim (D / 32) c + u of
//     those same eight keys, from rows read 8 (4) bytes a lane. Lane (h, c)
//     accumulates row c, so the softmax's scales are the lane's own.
// K of the next block is asked for as soon as the scores have taken this
// block's, V after the second product.
// A weight goes to the second product rounded once to T, off by at most 2^-8 (f16:
// 2^-11) of itself, as in the prefill kernels; the decode kernels' two halves would
// double that product, which bounds wide trees. So a tree's outputs are a little
// further from 64 bits (2-norm, relative: 0.0023, f16 0.00029) than a decode
// step's (0.0017, 0.00021, their own rounding), a tree of one node's too.
//
// A block of keys that every row sees (all of the context's but the last) takes
// no mask. In the others each row has 32 bits: the context's tokens and its own
// mask words' nodes. A weight of 0 times an infinity or NaN in V would be NaN, so
// there V is tested, and elements that are not finite leave the product and
// reach the rows that see them by a product of their own (take_nonfinite).
#pragma once

#include "paged_rows_unit.h"

namespace tsa {

constexpr float kTreeRescale = 8.f;  // log2 units a maximum grows before it moves

// Which unit (sequence s, kv head), split and row block a workgroup takes; false:
// none. Ids go round the XCDs, so those of one XCD and the row blocks of a unit
// and split follow each other. With a.order the sequences go by falling length,
// and every other run of 32 workgroups of an XCD (its CUs) backwards: a CU that
// gets two has a long and a short one. (In the sequences' own order, 8 sequences
// of 2000-8192 tokens, 40-64 nodes, 64/8 heads: 133 us against 122; 64 of
// 512-4096, 4-16 nodes, 32/8 heads: 137 against 123.) keys: LDS, 128
// words; all threads call.
struct TreeWork {
  int s, kvh, sp, rb, u;
};
__device__ __forceinline__ bool tree_work(const RowsArgs& a, int32_t* keys, TreeWork& w) {
  const int U = a.B * a.Hkv, total = (U * a.S + 7) / 8 * a.RB;  // workgroups of an XCD
  int k = static_cast<int>(blockIdx.x) >> 3;
  if (a.order) {
    const int lo = k & ~31;
    if (lo & 32) k = lo + min(lo + 32, total) - 1 - k;
  }
  w.rb = k % a.RB;
  const int us = k / a.RB * 8 + (static_cast<int>(blockIdx.x) & 7);
  if (us >= U * a.S) return false;
  w.sp = us / U;
  const int u = us - w.sp * U;
  w.s = u / a.Hkv;
  w.kvh = u - w.s * a.Hkv;
  if (a.order) {
    const int t = threadIdx.x;
    if (t < kTreeOrderSeqs) keys[t] = t < a.B ? max(a.lens[t * a.len_s], 0) : -1;
    __syncthreads();
    int rank = 0, mine = t < a.B ? keys[t] : -1;
    for (int j = 0; j < a.B; ++j) rank += keys[j] > mine || (keys[j] == mine && j < t);
    __syncthreads();
    if (t < a.B && rank == w.s) keys[0] = t;
    __syncthreads();
    w.s = __builtin_amdgcn_readfirstlane(keys[0]);
    __syncthreads();
  }
  w.u = w.s * a.Hkv + w.kvh;
  return true;
}

template <typename T, int D>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2))) void paged_rows_tree(
    RowsArgs a, const int32_t* __restrict__ bt, const uint32_t* __restrict__ mask, float* __restrict__ part) {
  constexpr int KJ = D / 16, NU = D / 32, PF = part_floats(D);
  typedef typename VPiece<2 * NU>::type VP;
  __shared__ __align__(16) float slots[4 * 32 * PF];
  // ---- Which unit and split.
  TreeWork w;
  if (!tree_work(a, reinterpret_cast<int32_t*>(slots), w)) return;
  const int sp = w.sp, u = w.u, s = w.s, kvh = w.kvh;
  const SeqRange r = seq_of(a, s);
  const int rows = r.nodes * a.G;  // up to 32
  if (rows <= 0) return;
  const int nblk = (r.end + 31) >> 5, per = tree_per_split(a, nblk), b0 = sp * per, b1 = min(nblk, b0 + per);
  if (b0 >= b1 && a.S > 1) return;  // (the merge takes the splits that have blocks)
  const int tid = threadIdx.x, lane = tid & 63, h = lane >> 5, c = lane & 31;
  constexpr int KG = 4;
  const int kg = __builtin_amdgcn_readfirstlane(tid >> 6);

  const int row = min(c, rows - 1);  // (past the last: it again, never stored)
  const int node = row / a.G, head = kvh * a.G + row - node * a.G;
  const int64_t prow = r.row0 + node;
  const uint32_t* const my_mask = mask + prow * a.mask_s;
  u32x4 q[KJ];
  {
    const T* const qp = static_cast<const T*>(a.q) + prow * a.q_sr + head * a.q_sh + 8 * h;
#pragma unroll
    for (int j = 0; j < KJ; ++j) q[j] = *reinterpret_cast<const u32x4*>(qp + 16 * j);
  }
  const float cs = a.scale_log2;  // > 0 here
  float m = kNegInfR, l = 0.f;
  f32x16 acc[NU];
#pragma unroll
  for (int x = 0; x < NU; ++x)
#pragma unroll
    for (int e = 0; e < 16; ++e) acc[x][e] = 0.f;

  const int mine = b0 + kg < b1 ? (b1 - b0 - kg + KG - 1) / KG : 0;  // this wave's blocks
  if (mine > 0) {
    // Lane 2 i + half: the page and first slot of that half of the wave's
    // block i0 + i, for 32 blocks at a time.
    int my_page = 0, my_slot = 0;
    uint64_t ok64 = 0;
    auto lookup = [&](int i0) __attribute__((always_inline)) {
      const int blk = b0 + kg + KG * (i0 + (lane >> 1));
      const uint32_t tile = static_cast<uint32_t>(2 * blk + (lane & 1)), lb = page_of_tile(tile, a.page_mul, a.page_shift);
      my_slot = static_cast<int>(16u * tile - lb * static_cast<uint32_t>(a.BS));
      const bool in = static_cast<int>(16u * tile) < r.end;
      my_page = bt[s * a.bt_s0 + min(static_cast<int>(lb), a.max_blocks - 1) * a.bt_s1];
      ok64 = __ballot(in && my_page >= 0 && my_page < a.NB);
    };
    const char* const kb = static_cast<const char*>(a.kc) + kvh * a.kc_h * 2;
    const char* const vb = static_cast<const char*>(a.vc) + kvh * a.vc_h * 2;
    const uint32_t k_slot = static_cast<uint32_t>(a.kc_s) * 2, v_slot = static_cast<uint32_t>(a.vc_s) * 2;
    const uint32_t k_lane = static_cast<uint32_t>(c & 15) * k_slot + 16u * h;
    const uint32_t v_lane = 4u * h * v_slot + 2u * NU * c;
    u32x4 kr[KJ];
    VP vr[16];
    // Rows of pages outside the pool, and of halves past the end, are row 0 of
    // page 0 (and masked).
    auto load_k = [&](int i) __attribute__((always_inline)) {
      const int x = 2 * (i & 31);
      const char* p[2];
#pragma unroll
      for (int y = 0; y < 2; ++y) {
        const bool ok = (ok64 >> (x + y)) & 1;
        const uint32_t page = ok ? __builtin_amdgcn_readlane(my_page, x + y) : 0;
        const uint32_t slot = ok ? __builtin_amdgcn_readlane(my_slot, x + y) : 0;
        p[y] = kb + static_cast<uint64_t>(page) * a.k_page + slot * k_slot;
      }
      const char* const kp = (c < 16 ? p[0] : p[1]) + k_lane;
#pragma unroll
      for (int j = 0; j < KJ; ++j) kr[j] = *reinterpret_cast<const u32x4*>(kp + 32 * j);
    };
    auto load_v = [&](int i) __attribute__((always_inline)) {
      const int x = 2 * (i & 31);
#pragma unroll
      for (int y = 0; y < 2; ++y) {
        const bool ok = (ok64 >> (x + y)) & 1;
        const uint32_t page = ok ? __builtin_amdgcn_readlane(my_page, x + y) : 0;
        const uint32_t slot = ok ? __builtin_amdgcn_readlane(my_slot, x + y) : 0;
        const char* const p = vb + static_cast<uint64_t>(page) * a.v_page + slot * v_slot;
#pragma unroll
        for (int t = 0; t < 8; ++t)
          vr[8 * y + t] = *reinterpret_cast<const VP*>(p + ((t & 3) + 8 * (t >> 2)) * v_slot + v_lane);
      }
    };
    lookup(0);
    load_k(0);
    load_v(0);
    for (int i = 0; i < mine; ++i) {
      const int blk = b0 + kg + KG * i;
      const uint32_t okb = static_cast<uint32_t>(ok64 >> (2 * (i & 31))) & 3u;
      f32x16 sc;
#pragma unroll
      for (int e = 0; e < 16; ++e) sc[e] = 0.f;
#pragma unroll
      for (int j = 0; j < KJ; ++j) sc = mfma_k16x32<T>(kr[j], q[j], sc);
      const bool more = i + 1 < mine;
      if (((i + 1) & 31) == 0 && more) lookup(i + 1);
      load_k(more ? i + 1 : i);  // (the last block's again: unconditional, so that the waits count it)
      uint32_t vis = ~0u;
      if (okb != 3u || 32 * blk + 32 > r.ctx) {  // (uniform) some key that some row does not see
        auto below = [](int n) { return n >= 32 ? ~0u : n > 0 ? (1u << n) - 1u : 0u; };
        const uint32_t there = below(r.end - 32 * blk) & ((okb & 1 ? 0xFFFFu : 0u) | (okb & 2 ? 0xFFFF0000u : 0u));
        const int j0 = 32 * blk - r.ctx, w = j0 >> 5, sh = j0 & 31;
        const uint32_t lo = w >= 0 && w < a.words ? my_mask[w] : 0u;
        const uint32_t hi = w + 1 >= 0 && w + 1 < a.words ? my_mask[w + 1] : 0u;
        const uint32_t nodes = sh ? (lo >> sh) | (hi << (32 - sh)) : lo;
        vis = (below(r.ctx - 32 * blk) | nodes) & there;
#pragma unroll
        for (int e = 0; e < 16; ++e)
          if (!((vis >> (8 * (e >> 2) + 4 * h + (e & 3))) & 1)) sc[e] = kNegInfR;
        bool bad = false;
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          if (!((there >> (8 * (e >> 2) + 4 * h + (e & 3))) & 1)) vr[e] = VP{};  // unread rows
#pragma unroll
          for (int x = 0; x < NU / 2; ++x) bad |= nonfinite2<T>(word_of(vr[e], x)) != 0;
        }
        if (__any(bad)) take_nonfinite<T>(vr, acc, vis, h);
      }
      float mx = kNegInfR;
#pragma unroll
      for (int e = 0; e < 16; ++e) mx = fmaxf(mx, sc[e]);
      const auto sw = __builtin_amdgcn_permlane32_swap(__float_as_uint(mx), __float_as_uint(mx), false, false);
      const float mt = fmaxf(__uint_as_float(sw[0]), __uint_as_float(sw[1])) * cs;
      if (__any(mt > m + kTreeRescale)) {
        const float mn = fmaxf(m, mt), alpha = mn == kNegInfR ? 1.f : fast_exp2(m - mn);
        l *= alpha;
#pragma unroll
        for (int x = 0; x < NU; ++x)
#pragma unroll
          for (int e = 0; e < 16; ++e) acc[x][e] *= alpha;
        m = mn;
      }
      const float mu = m == kNegInfR ? 0.f : m;
      u32x4 pop[2];
      {
        float p[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          p[e] = fast_exp2(fmaf(sc[e], cs, -mu));
          l += p[e];
        }
#pragma unroll
        for (int e = 0; e < 16; e += 2) pop[e >> 3][(e & 7) >> 1] = pack2<T>(p[e], p[e + 1]);
      }
#pragma unroll
      for (int s2 = 0; s2 < 2; ++s2)
#pragma unroll
        for (int x = 0; x < NU; ++x) {
          u32x4 w;
#pragma unroll
          for (int k = 0; k < 4; ++k) w[k] = v_pair<T, T>(vr[8 * s2 + 2 * k], vr[8 * s2 + 2 * k + 1], x);
          acc[x] = mfma_k16x32<T>(w, pop[s2], acc[x]);
        }
      load_v(more ? i + 1 : i);
    }
    l += __builtin_bit_cast(float, xor_lane32<32>(__builtin_bit_cast(uint32_t, l), lane));
  }
  // ---- The waves' partials to LDS, then the runs of keys together.
  float* const slot = slots + (kg * 32 + c) * PF;
#pragma unroll
  for (int e = 0; e < 16; ++e) {
    const int i = 8 * (e >> 2) + 4 * h + (e & 3);
    if constexpr (NU == 4) *reinterpret_cast<f32x4*>(slot + 4 * i) = f32x4{acc[0][e], acc[1][e], acc[2][e], acc[NU - 1][e]};
    else *reinterpret_cast<f32x2*>(slot + 2 * i) = f32x2{acc[0][e], acc[1][e]};
  }
  if (h == 0) {
    slot[D] = m;
    slot[D + 1] = l;
  }
  __syncthreads();
  for (int idx = tid; idx < rows * (D / 2); idx += 256) {
    const int rr = idx / (D / 2), d = 2 * (idx - rr * (D / 2));
    float M = kNegInfR, den = 0.f, o0 = 0.f, o1 = 0.f;
    for (int g = 0; g < KG; ++g) {
      const float* const x = slots + (32 * g + rr) * PF;
      const f32x2 v = *reinterpret_cast<const f32x2*>(x + d), ml = *reinterpret_cast<const f32x2*>(x + D);
      const float mn = fmaxf(M, ml[0]), mu = mn == kNegInfR ? 0.f : mn;
      const float c_old = fast_exp2(M - mu), c_new = fast_exp2(ml[0] - mu);
      o0 = fmaf(v[0], c_new, o0 * c_old);
      o1 = fmaf(v[1], c_new, o1 * c_old);
      den = fmaf(ml[1], c_new, den * c_old);
      M = mn;
    }
    if (a.S == 1) {
      const int nd = rr / a.G;
      T* const out = static_cast<T*>(a.out) + (r.row0 + nd) * a.o_sr + (kvh * a.G + rr - nd * a.G) * a.o_sh;
      out[d * a.o_sd] = from_float<T>(den == 0.f ? 0.f : o0 / den);
      out[(d + 1) * a.o_sd] = from_float<T>(den == 0.f ? 0.f : o1 / den);
    } else {
      float* const out = part + ((static_cast<int64_t>(u) * a.S + sp) * (a.T * a.G) + rr) * PF;
      *reinterpret_cast<f32x2*>(out + d) = f32x2{o0, o1};
      if (d == 0) *reinterpret_cast<f32x2*>(out + D) = f32x2{M, den};
    }
  }
}

}  // namespace tsa
