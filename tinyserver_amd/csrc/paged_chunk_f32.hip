// Attention of a chunk over the paged cache in float32, on the f32 matrix
// instructions.
//
// What bounds it: v_mfma_f32_16x16x4_f32, 32 cycles for 2,048 FLOP a SIMD, and for few
// tokens the segments' serial parts (lengths, pages, the first loads, the waves' join).
//
// Work is dealt as paged_chunk_stream.h does it: runs of 32-key blocks over all items,
// an item being QB queries times the G q-heads of a kv head, here up to 32 rows. A
// workgroup of four waves takes a segment, whose 16-key tiles go to the waves in turn,
// K and V from their pages straight into registers: V is in flight under the score
// products, the next tile's K under the softmax and P V. The waves' sums meet in LDS.
//
// With lane (g, c) = (lane / 16, lane % 16) and row tiles t = 0, 1:
//   S^T(16 keys x 16 rows) = K Q^T: step 4 j + i takes dims 16 j + 4 g + i, so a lane's
//     K and Q operands are 16-byte pieces of key c's and row c's vectors; element r of
//     the result is the score of key 4 g + r.
//   O^T(dims x 16 rows) += V^T P^T: step r takes keys 4 g + r, whose weights are element
//     r of the lane's own scores. Dim tile (y, i) has dim 64 y + 4 c + i in its row c, so
//     a lane's V operands are 16-byte pieces of a key's row. A lane holds row c's
//     outputs, so the softmax's scales are the lane's own.
// A tile that some row does not see whole takes masks; there elements of V that are
// not finite leave the product and reach the rows that see them by one of flags.
// Measured (16 q-heads, 8 kv heads, head_dim 128, 4 sequences of 16-128 new tokens over
// 100-1,024): 26 us and 6 for the items that were cut; one wave a row on the vector
// units 810.
#include "paged_chunk_stream.h"

namespace tsa {

constexpr int kF32Rows = 32, kF32Threads = 256;
template <int D> constexpr int chunk_f32_pitch() { return D + 4; }  // LDS rows: 16-byte aligned, 4 banks apart
// LDS: the four waves' sums (Q's rows sit in the first until then), their m and l, and
// the work.
template <int D> constexpr int chunk_f32_floats() { return 4 * kF32Rows * chunk_f32_pitch<D>() + 2 * 4 * kF32Rows; }

template <int D>
__global__ __launch_bounds__(kF32Threads) __attribute__((amdgpu_waves_per_eu(2, 2))) void paged_chunk_f32(ChunkArgs a) {
  constexpr int NJ = D / 16;  // 16-byte pieces of a lane's K or Q operand
  constexpr int NH = D / 64;  // 16-byte pieces of a lane's V operand of one key
  constexpr int RP = chunk_f32_pitch<D>();
  __shared__ __align__(16) float smem[chunk_f32_floats<D>()];
  __shared__ ChunkWork work_s;
  ChunkWork* const work = &work_s;
  float* const ml = smem + 4 * kF32Rows * RP;  // m[4][32], l[4][32]

  int64_t total;
  int per, run;
  ChunkStart st;
  ChunkFound* const found = reinterpret_cast<ChunkFound*>(smem + 16);
  const bool has = chunk_start<kF32Threads>(a, reinterpret_cast<uint64_t*>(smem), found, static_cast<int>(gridDim.x), total,
                                            per, run, st);
  const int tid = threadIdx.x, lane = tid & 63, g = lane >> 4, c = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  if (blockIdx.x == 0 && tid == 0) *a.runs = static_cast<int32_t>((total + per - 1) / per);
  if (!has) return;
  if (tid == 0) work->start(a, found->r, st, total, run, per);
  __syncthreads();

  auto of = [](const int32_t& x) { return __builtin_amdgcn_readfirstlane(x); };
#pragma unroll 1
  for (int turn = 0; work->seg[turn].blk1 > 0; turn ^= 1) {
    const ChunkSegment& seg = work->seg[turn];
    const int blk0 = of(seg.blk0), blk1 = of(seg.blk1), pos = of(seg.pos), end = of(seg.end), nq = of(seg.nq);
    const int kvh = of(seg.kvh), G = a.G, rows = nq * G;
    const int64_t seg_row = seg.row;
    auto q_of = [&](int r) { return (r * a.g_mul) >> 16; };
    // ---- This wave's tiles: the first + 4 i, i < count; pages of 64 at a time, a lane each.
    const int first = 2 * blk0 + wave, last_tile = (end - 1) >> 4, tiles = min(2 * blk1, last_tile + 1);
    const int count = first < tiles ? (tiles - first + 3) / 4 : 0;
    int my_page = 0;
    uint64_t ok64 = 0;
    auto look_up = [&](int i0) {
      const int tile = min(first + 4 * (i0 + lane), last_tile);
      const uint32_t lb = page_of_tile(static_cast<uint32_t>(tile), a.page_mul, a.page_shift);
      my_page = a.bt[of(seg.s) * a.bt_s0 + min(static_cast<int>(lb), a.max_blocks - 1) * a.bt_s1];
      const bool ok = my_page >= 0 && my_page < a.NB;
      ok64 = __ballot(ok);
      if (!ok) my_page = 0;  // (its rows are read, and masked)
    };
    if (count > 0) look_up(0);
    // ---- Q's rows (those past the last repeat it).
    constexpr int kQ = kF32Rows * (D / 4) / kF32Threads;  // 16-byte pieces a thread
    f32x4 qv[kQ];
#pragma unroll
    for (int x = 0; x < kQ; ++x) {
      const int i = tid + x * kF32Threads, r = min(i / (D / 4), rows - 1), ch = i % (D / 4), qq = q_of(r);
      qv[x] = *reinterpret_cast<const f32x4*>(static_cast<const float*>(a.q) + (seg_row + qq) * a.q_sr +
                                              (kvh * G + r - qq * G) * a.q_sh + 4 * ch);
    }
    const float* const kb = static_cast<const float*>(a.kc) + kvh * a.kc_h + 4 * g;
    const float* const vb = static_cast<const float*>(a.vc) + kvh * a.vc_h + 4 * c;
    auto slot_of = [&](int tile) {  // of its first row in its page
      return 16 * tile - static_cast<int>(page_of_tile(static_cast<uint32_t>(tile), a.page_mul, a.page_shift)) * a.BS;
    };
    f32x4 kop[NJ];
    // (keys past the sequence's last re-read it; their scores are masked)
    auto load_k = [&](int i) __attribute__((always_inline)) {
      const int tile = first + 4 * i, row = slot_of(tile) + min(c, end - 1 - 16 * tile);
      const float* const p = kb + static_cast<int64_t>(__builtin_amdgcn_readlane(my_page, i & 63)) * a.kc_b + row * a.kc_s;
#pragma unroll
      for (int j = 0; j < NJ; ++j) kop[j] = *reinterpret_cast<const f32x4*>(p + 16 * j);
    };
    if (count > 0) load_k(0);
#pragma unroll
    for (int x = 0; x < kQ; ++x) {
      const int i = tid + x * kF32Threads;
      *reinterpret_cast<f32x4*>(smem + i / (D / 4) * RP + 4 * (i % (D / 4))) = qv[x];
    }
    int my_end[2];  // keys that rows c and 16 + c see
#pragma unroll
    for (int t = 0; t < 2; ++t) my_end[t] = min(pos + q_of(min(16 * t + c, rows - 1)) + 1, end);
    const int full = min(pos + 1, end);  // keys below it are seen by every row
    __syncthreads();
    if (tid == 0) work->next(a, seg, work->seg[turn ^ 1]);

    float m[2] = {kChunkNone, kChunkNone}, l[2] = {0.f, 0.f};
    f32x4 acc[2][NH][4];
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int y = 0; y < NH; ++y)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[t][y][i] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
    for (int it = 0; it < count; ++it) {
      const int tile = first + 4 * it, k0 = 16 * tile;
      const bool there = (ok64 >> (it & 63)) & 1;
      f32x4 vop[4][NH];
      {
        const float* const p = vb + static_cast<int64_t>(__builtin_amdgcn_readlane(my_page, it & 63)) * a.vc_b;
        const int slot = slot_of(tile);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float* const q = p + (slot + min(4 * g + r, end - 1 - k0)) * a.vc_s;
#pragma unroll
          for (int y = 0; y < NH; ++y) vop[r][y] = *reinterpret_cast<const f32x4*>(q + 64 * y);
        }
      }
      __builtin_amdgcn_sched_barrier(0);  // in flight under the score products
      f32x4 sc[2] = {f32x4{0.f, 0.f, 0.f, 0.f}, f32x4{0.f, 0.f, 0.f, 0.f}};
      const float* const qrow = smem + c * RP + 4 * g;
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        const f32x4 q0 = *reinterpret_cast<const f32x4*>(qrow + 16 * j);
        const f32x4 q1 = *reinterpret_cast<const f32x4*>(qrow + 16 * RP + 16 * j);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          sc[0] = __builtin_amdgcn_mfma_f32_16x16x4f32(kop[j][i], q0[i], sc[0], 0, 0, 0);
          sc[1] = __builtin_amdgcn_mfma_f32_16x16x4f32(kop[j][i], q1[i], sc[1], 0, 0, 0);
        }
      }
      if (((it + 1) & 63) == 0 && it + 1 < count) look_up(it + 1);
      load_k(min(it + 1, count - 1));     // the wave's next tile (its last: a repeat)
      __builtin_amdgcn_sched_barrier(0);  // in flight under the softmax and P V

      const bool edge = k0 + 16 > full || !there;  // some row does not see some key of the tile
      float p[2][4];
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        float s[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) s[r] = sc[t][r] * a.scale_log2;
        if (edge) {
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (k0 + 4 * g + r >= my_end[t] || !there) s[r] = kNegInfC;
        }
        float mx = fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3]));
        mx = fmaxf(mx, __builtin_bit_cast(float, xor_lane32<16>(__builtin_bit_cast(uint32_t, mx), lane)));
        mx = fmaxf(mx, __builtin_bit_cast(float, xor_lane32<32>(__builtin_bit_cast(uint32_t, mx), lane)));
        const float m_new = fmaxf(m[t], mx);
        if (__any(m_new > m[t])) {
          const float alpha = fast_exp2(m[t] - m_new);
          l[t] *= alpha;
#pragma unroll
          for (int y = 0; y < NH; ++y)
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
              for (int e = 0; e < 4; ++e) acc[t][y][i][e] *= alpha;
          m[t] = m_new;
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          p[t][r] = fast_exp2(s[r] - m[t]);
          l[t] += p[t][r];
        }
      }
      if (edge) {
        float z = 0.f;
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
          for (int y = 0; y < NH; ++y)
#pragma unroll
            for (int i = 0; i < 4; ++i) z = fmaf(vop[r][y][i], 0.f, z);
        if (__any(z != 0.f)) {  // (NaN)
          float sees[2][4];
#pragma unroll
          for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int r = 0; r < 4; ++r) sees[t][r] = there && k0 + 4 * g + r < my_end[t] ? 1.f : 0.f;
#pragma unroll
          for (int y = 0; y < NH; ++y)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              f32x4 n[2] = {f32x4{0.f, 0.f, 0.f, 0.f}, f32x4{0.f, 0.f, 0.f, 0.f}};
#pragma unroll
              for (int r = 0; r < 4; ++r) {
                const bool bad = !(fabsf(vop[r][y][i]) < INFINITY);
                const float flag = bad ? 1.f : 0.f;
                if (bad) vop[r][y][i] = 0.f;
                n[0] = __builtin_amdgcn_mfma_f32_16x16x4f32(flag, sees[0][r], n[0], 0, 0, 0);
                n[1] = __builtin_amdgcn_mfma_f32_16x16x4f32(flag, sees[1][r], n[1], 0, 0, 0);
              }
#pragma unroll
              for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                  if (n[t][e] > 0.f) acc[t][y][i][e] = __builtin_nanf("");
            }
        }
      }
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int y = 0; y < NH; ++y)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            acc[0][y][i] = __builtin_amdgcn_mfma_f32_16x16x4f32(vop[r][y][i], p[0][r], acc[0][y][i], 0, 0, 0);
            acc[1][y][i] = __builtin_amdgcn_mfma_f32_16x16x4f32(vop[r][y][i], p[1][r], acc[1][y][i], 0, 0, 0);
          }
    }
    // ---- The waves' sums to LDS, then together. Element e of acc[t][y][i] is row 16 t
    // + c, dim 64 y + 4 (4 g + e) + i.
    __syncthreads();  // (Q is no longer read)
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      l[t] += __builtin_bit_cast(float, xor_lane32<16>(__builtin_bit_cast(uint32_t, l[t]), lane));
      l[t] += __builtin_bit_cast(float, xor_lane32<32>(__builtin_bit_cast(uint32_t, l[t]), lane));
      if (g == 0) {
        ml[wave * kF32Rows + 16 * t + c] = m[t];
        ml[(4 + wave) * kF32Rows + 16 * t + c] = l[t];
      }
      float* const mine = smem + (wave * kF32Rows + 16 * t + c) * RP + 16 * g;
#pragma unroll
      for (int y = 0; y < NH; ++y)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          *reinterpret_cast<f32x4*>(mine + 64 * y + 4 * e) =
              f32x4{acc[t][y][0][e], acc[t][y][1][e], acc[t][y][2][e], acc[t][y][3][e]};
    }
    __syncthreads();
    const int r = tid >> 3;  // eight threads a row
    float f[4], M = kChunkNone, den = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) M = fmaxf(M, ml[w * kF32Rows + r]);
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      f[w] = fast_exp2(ml[w * kF32Rows + r] - M);
      den = fmaf(f[w], ml[(4 + w) * kF32Rows + r], den);
    }
    const bool whole = blk0 == 0 && blk1 == of(seg.nblk);
    const int qq = q_of(r);
    float* const out = static_cast<float*>(a.out) + (seg_row + qq) * a.o_sr + (kvh * G + r - qq * G) * a.o_sh;
    // Slot 0: of the item that the run starts inside of; 1: of the one it starts.
    float* const slot = a.part + (2 * static_cast<int64_t>(work->run) + (blk0 == 0 ? 1 : 0)) * chunk_part_floats(D, 1);
    if (r < rows) {
#pragma unroll
      for (int x = 0; x < D / 32; ++x) {
        const int d = 4 * ((tid & 7) + 8 * x);
        f32x4 o = *reinterpret_cast<const f32x4*>(smem + r * RP + d) * f[0];
#pragma unroll
        for (int w = 1; w < 4; ++w) o += *reinterpret_cast<const f32x4*>(smem + (w * kF32Rows + r) * RP + d) * f[w];
        if (whole) {
          o = den == 0.f ? f32x4{0.f, 0.f, 0.f, 0.f} : o / den;
          if (a.out8) {
            *reinterpret_cast<f32x4*>(out + d) = o;
          } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) out[(d + e) * a.o_sd] = o[e];
          }
        } else {
          *reinterpret_cast<f32x4*>(slot + r * D + d) = o;
        }
      }
      if (!whole && (tid & 7) == 0) *reinterpret_cast<f32x2*>(slot + kF32Rows * D + 2 * r) = f32x2{M, den};
    }
    if (!whole && blk0 > 0 && tid == 0) a.splits[work->run] = work->split(seg);
    __syncthreads();
  }
}

// Items that a cut goes through (paged_chunk_merge).
template <int D>
__global__ __launch_bounds__(256) void paged_chunk_f32_merge(ChunkArgs a) {
  const int run = static_cast<int>(blockIdx.x) + 1, tid = threadIdx.x, r = tid >> 3;
  if (run >= *a.runs) return;
  const ChunkSplit sp = a.splits[run];
  if (sp.runs == 0 || r >= sp.queries * a.G) return;
  f32x4 o[D / 32];
  const float den = chunk_join<D / 32>(
      sp.runs + 1, kF32Rows * D, r,
      [&](int k) { return a.part + (2 * static_cast<int64_t>(run + k - 1) + (k == 0 ? 1 : 0)) * chunk_part_floats(D, 1); },
      [&](int x) { return r * D + 4 * ((tid & 7) + 8 * x); }, o);
  const int qq = (r * a.g_mul) >> 16;
  float* const out = static_cast<float*>(a.out) + (sp.row0 + qq) * a.o_sr + (sp.kvh * a.G + r - qq * a.G) * a.o_sh;
#pragma unroll
  for (int x = 0; x < D / 32; ++x) {
    const f32x4 v = den == 0.f ? f32x4{0.f, 0.f, 0.f, 0.f} : o[x] / den;
    const int d = 4 * ((tid & 7) + 8 * x);
#pragma unroll
    for (int e = 0; e < 4; ++e) out[(d + e) * a.o_sd] = v[e];
  }
}

template <int D>
static int launch_f32(const ChunkArgs& a, const ChunkPlan& p, hipStream_t stream) {
  paged_chunk_f32<D><<<dim3(p.runs), dim3(kF32Threads), 0, stream>>>(a);
  if (int rc = check_launch("tsa_paged_chunk")) return rc;
  if (p.whole || p.runs < 2) return TSA_OK;
  paged_chunk_f32_merge<D><<<dim3(p.runs - 1), dim3(256), 0, stream>>>(a);
  return check_launch("tsa_paged_chunk");
}

int chunk_f32_launch(const ChunkArgs& a, const ChunkPlan& p, hipStream_t stream) {
  return a.D == 128 ? launch_f32<128>(a, p, stream) : launch_f32<64>(a, p, stream);
}

}  // namespace tsa
