// The decode step over part of the context or over an 8-bit cache, for batches
// with many tiles: a fixed grid whose waves each stream an equal, contiguous
// run of the batch's pairs of 16-token tiles.
//
// What bounds it: HBM. In the unit form (paged_rows_unit.h) a workgroup waits
// for its length, its pages and its rows before it computes, and no more of
// them fit a CU than hide that in part: 4.2 to 4.4 TB/s. Here the list of
// visible tile pairs of every unit (sequence, kv head, group of 16 q-heads),
// unit-major, is dealt evenly to the waves of a grid that is resident at once,
// whatever the lengths; a wave's ring keeps RING - 1 pairs of rows in flight
// and runs on across units, with the page ids of the next pair already in
// scalar registers when its loads are issued. A wave's partial of a unit goes
// to workspace slot unit + wave (a wave's units start where the previous
// wave's ended, so no slot is written twice); a second launch merges.
// The arithmetic is the unit form's, with a running maximum: rescaling only
// where a head's maximum grows by more than 2^8 (the weights and l share it, so
// the result is unchanged).
#pragma once

#include "paged_rows_unit.h"

namespace tsa {

constexpr int kStreamWaves = 4;

struct StreamCur {
  int s, k, n, t;  // sequence, unit of the sequence (kv head x group), its pairs, the pair
  UnitTiles ut;
};
// Pairs of a wave, and x / y for run positions: in 32 bits where the list's
// length allows (a 64-bit division is some hundred instructions).
__device__ __forceinline__ int64_t div_pos(int64_t x, int64_t y) {
  return ((x | y) >> 32) == 0 ? static_cast<int64_t>(static_cast<uint32_t>(x) / static_cast<uint32_t>(y)) : x / y;
}
__device__ __forceinline__ int64_t stream_share(int64_t total, int waves) { return div_pos(total + waves - 1, waves); }

// What the loads of a unit start from.
struct StreamBase {
  const char *k, *v, *ks, *vs;
  int64_t bt;  // (an offset: the block table's entries are read through the __restrict__ parameter, by scalar loads)
};

template <typename T, typename C, int D, int RING>
__global__ __launch_bounds__(64 * kStreamWaves) __attribute__((amdgpu_waves_per_eu(2))) void paged_rows_stream(
    RowsArgs a, const int32_t* __restrict__ bt, const int32_t* __restrict__ lens, float* __restrict__ part,
    int32_t* __restrict__ pref_out) {
  constexpr int eb = sizeof(C), KL = D * eb / 64, KJ = D / 32, NU = D / 16, PF = part_floats(D);
  typedef typename VPiece<NU * eb>::type VP;
  typedef typename std::conditional<kIs8<C>, bf16_t, T>::type PT;
  extern __shared__ int32_t pref[];  // [B + 1] pairs before each sequence, per unit of it, then [B] lengths
  int32_t* const len_s = pref + a.B + 1;
  __shared__ int32_t wave_tot[kStreamWaves];
  const int tid = threadIdx.x, lane = tid & 63, g = lane >> 4, c = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int groups = (a.G + 15) / 16, units = a.Hkv * groups;  // units of a sequence

  // ---- The prefix: thread t sums a run of sequences, a scan of the threads.
  {
    const int per = (a.B + 64 * kStreamWaves - 1) / (64 * kStreamWaves);
    int sum = 0;
    for (int i = 0; i < per; ++i) {
      const int s = tid * per + i;
      if (s < a.B) {
        const int len = unit_length(a, lens, s);
        len_s[s] = len;
        sum += (unit_tiles(a, len).n + 1) >> 1;
      }
    }
    const int incl = static_cast<int>(wave_scan_u32(static_cast<uint32_t>(sum)));
    if (lane == 63) wave_tot[wave] = incl;
    __syncthreads();
    int run = incl - sum;
    for (int w = 0; w < wave; ++w) run += wave_tot[w];
    for (int i = 0; i < per; ++i) {
      const int s = tid * per + i;
      if (s < a.B) {
        pref[s] = run;
        run += (unit_tiles(a, len_s[s]).n + 1) >> 1;
      }
    }
    if (tid == 64 * kStreamWaves - 1) pref[a.B] = run;
    __syncthreads();
    if (blockIdx.x == 0)
      for (int i = tid; i <= a.B; i += 64 * kStreamWaves) pref_out[i] = pref[i];
  }
  const int v = blockIdx.x * kStreamWaves + wave;
  const int64_t total = static_cast<int64_t>(units) * pref[a.B];
  const int64_t share = stream_share(total, a.NW);
  const int64_t lo = v * share, hi = min(total, lo + share);
  if (lo >= hi) return;  // (no barrier follows)
  const int n_pairs = static_cast<int>(hi - lo);

  auto set_seq = [&](StreamCur& x, int s) __attribute__((always_inline)) {
    x.s = s;
    x.n = __builtin_amdgcn_readfirstlane(pref[s + 1] - pref[s]);
    x.ut = unit_tiles(a, __builtin_amdgcn_readfirstlane(len_s[s]));
  };
  auto advance = [&](StreamCur& x) __attribute__((always_inline)) {
    if (++x.t < x.n) return;
    x.t = 0;
    if (++x.k < units) return;
    x.k = 0;
    int s = x.s + 1;
    while (s < a.B && pref[s + 1] == pref[s]) ++s;
    s = __builtin_amdgcn_readfirstlane(s);
    if (s < a.B) set_seq(x, s);
  };
  StreamCur cur;
  {
    int l0 = 0, h0 = a.B;  // units pref[l0] <= lo < units pref[h0]
    while (h0 - l0 > 1) {
      const int mid = (l0 + h0) >> 1;
      if (static_cast<int64_t>(units) * pref[mid] <= lo) l0 = mid; else h0 = mid;
    }
    set_seq(cur, __builtin_amdgcn_readfirstlane(l0));
    const int64_t off = lo - static_cast<int64_t>(units) * __builtin_amdgcn_readfirstlane(pref[cur.s]);
    cur.k = __builtin_amdgcn_readfirstlane(static_cast<int>(div_pos(off, cur.n)));
    cur.t = __builtin_amdgcn_readfirstlane(static_cast<int>(off - static_cast<int64_t>(cur.k) * cur.n));
  }

  auto base_of = [&](const StreamCur& x) __attribute__((always_inline)) {
    const int kvh = groups == 1 ? x.k : x.k / groups;
    StreamBase b;
    b.k = static_cast<const char*>(a.kc) + kvh * a.kc_h * eb;
    b.v = static_cast<const char*>(a.vc) + kvh * a.vc_h * eb;
    b.ks = reinterpret_cast<const char*>(a.ks + kvh * a.ks_h);
    b.vs = reinterpret_cast<const char*>(a.vs + kvh * a.vs_h);
    b.bt = x.s * a.bt_s0;
    return b;
  };
  // The page id and first slot of a pair's two tiles. The ids are asked for one
  // pair ahead of the loads that need them, and nothing here looks at them: a
  // test of an id would wait for it.
  struct Ids {
    int page[2], slot[2];
  };
  auto ask = [&](const StreamCur& x, const StreamBase& b) __attribute__((always_inline)) {
    Ids r;
#pragma unroll
    for (int y = 0; y < 2; ++y) {
      const uint32_t tile = static_cast<uint32_t>(x.ut.at(min(2 * x.t + y, x.ut.n - 1)));
      const uint32_t lb = page_of_tile(tile, a.page_mul, a.page_shift);
      r.slot[y] = static_cast<int>(16u * tile - lb * static_cast<uint32_t>(a.BS));
      r.page[y] = bt[b.bt + lb * a.bt_s1];
    }
    return r;
  };
  struct Buf {
    u32x4 k[2][KL];
    VP v[2][4];
    float ks[2], vs[2];
    uint32_t vis;  // bits of the 32 tokens (uniform)
  };
  const uint32_t k_lane = static_cast<uint32_t>(c * static_cast<int>(a.kc_s) * eb + 16 * g);
  const uint32_t v_lane = static_cast<uint32_t>((4 * g) * static_cast<int>(a.vc_s) * eb + NU * eb * c);
  const uint32_t ks_lane = static_cast<uint32_t>((4 * g + (c & 3)) * static_cast<int>(a.ks_s) * 4);
  const uint32_t vs_lane = static_cast<uint32_t>((4 * g + (c & 3)) * static_cast<int>(a.vs_s) * 4);
  const uint32_t k_slot = static_cast<uint32_t>(a.kc_s) * eb, v_slot = static_cast<uint32_t>(a.vc_s) * eb;
  const uint32_t ks_slot = static_cast<uint32_t>(a.ks_s) * 4, vs_slot = static_cast<uint32_t>(a.vs_s) * 4;
  const uint32_t nb = static_cast<uint32_t>(min(a.NB, int64_t{0x7FFFFFFF}));
  auto load = [&](Buf& b, const StreamCur& x, const StreamBase& base, const Ids& id) __attribute__((always_inline)) {
    uint32_t vis = ~0u;
#pragma unroll
    for (int y = 0; y < 2; ++y) {
      const bool ok = static_cast<uint32_t>(id.page[y]) < nb;
      const uint32_t page = ok ? id.page[y] : 0, slot0 = ok ? id.slot[y] : 0;
      const char* const kp = base.k + static_cast<uint64_t>(page) * a.k_page + slot0 * k_slot;
      const char* const vp = base.v + static_cast<uint64_t>(page) * a.v_page + slot0 * v_slot;
#pragma unroll
      for (int i = 0; i < KL; ++i) b.k[y][i] = load_piece<true, u32x4>(kp + k_lane + 64 * i);
#pragma unroll
      for (int r = 0; r < 4; ++r) b.v[y][r] = load_piece<true, VP>(vp + r * v_slot + v_lane);
      if constexpr (kIs8<C>) {
        b.ks[y] = *reinterpret_cast<const float*>(base.ks + static_cast<uint64_t>(page) * a.ks_page + slot0 * ks_slot + ks_lane);
        b.vs[y] = *reinterpret_cast<const float*>(base.vs + static_cast<uint64_t>(page) * a.vs_page + slot0 * vs_slot + vs_lane);
      }
      if (!ok) vis &= y ? 0xFFFFu : 0xFFFF0000u;
    }
    // Pairs inside the visible range are seen whole; the others' bits are made out here.
    const int tok0 = 16 * x.ut.at(2 * x.t), tok1 = 16 * x.ut.at(2 * x.t + 1);
    if (tok0 < x.ut.lo || tok1 + 16 > x.ut.L) {
      auto bits = [&](int tok) {
        const int left = x.ut.L - tok;
        uint32_t m16 = left >= 16 ? 0xFFFFu : left > 0 ? (1u << left) - 1u : 0u;
        if (x.ut.lo > tok) {
          const uint32_t in_window = x.ut.lo - tok >= 16 ? 0u : 0xFFFFu << (x.ut.lo - tok);
          const int first = a.sinks - tok;
          m16 &= in_window | (first >= 16 ? 0xFFFFu : first > 0 ? (1u << first) - 1u : 0u);
        }
        return m16 & 0xFFFFu;
      };
      vis &= bits(tok0) | (2 * x.t + 1 < x.ut.n ? bits(tok1) << 16 : 0u);
    }
    b.vis = __builtin_amdgcn_readfirstlane(vis);
  };
  u32x4 q[KJ];
  auto load_q = [&](const StreamCur& x, u32x4 (&to)[KJ]) __attribute__((always_inline)) {
    const int kvh = groups == 1 ? x.k : x.k / groups, g0 = 16 * (x.k - kvh * groups), rows = min(16, a.G - g0);
    const T* const qrow = static_cast<const T*>(a.q) + x.s * a.q_sr + (kvh * a.G + g0 + min(c, rows - 1)) * a.q_sh;
#pragma unroll
    for (int j = 0; j < KJ; ++j) {
      const int d = kIs8<C> ? 16 * (g + 4 * (j >> 1)) + 8 * (j & 1) : 8 * (g + 4 * j);
      to[j] = *reinterpret_cast<const u32x4*>(qrow + d);
    }
  };

  float m = kNegInfR, l = 0.f;
  f32x4 acc[NU];
#pragma unroll
  for (int u = 0; u < NU; ++u) acc[u] = f32x4{0.f, 0.f, 0.f, 0.f};
  constexpr float kRescale = 8.f;
  auto compute = [&](Buf& b) __attribute__((always_inline)) {
    float sv[2][4];
#pragma unroll
    for (int y = 0; y < 2; ++y) {
      f32x4 sc = f32x4{0.f, 0.f, 0.f, 0.f};
      if constexpr (kIs8<C>) {
#pragma unroll
        for (int j = 0; j < KJ; ++j)
          sc = mfma_k32<T>(widen8<C, T>(b.k[y][j >> 1][2 * (j & 1)], b.k[y][j >> 1][2 * (j & 1) + 1]), q[j], sc);
        sc = scale_tokens(sc, b.ks[y]);
      } else {
#pragma unroll
        for (int j = 0; j < KJ; ++j) sc = mfma_k32<T>(b.k[y][j], q[j], sc);
      }
#pragma unroll
      for (int r = 0; r < 4; ++r) sv[y][r] = sc[r] * a.scale_log2;
    }
    if (b.vis != ~0u) {  // (uniform) tokens that are not seen: no weight, and no V that 0 would not cancel
#pragma unroll
      for (int y = 0; y < 2; ++y) {
        const uint32_t vis = b.vis >> (16 * y);
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (!((vis >> (4 * g + r)) & 1)) {
            sv[y][r] = kNegInfR;
            b.v[y][r] = VP{};
          }
        if constexpr (kIs8<C>)
          if (!((vis >> (4 * g + (c & 3))) & 1)) b.vs[y] = 0.f;
      }
    }
    float mx = kNegInfR;
#pragma unroll
    for (int y = 0; y < 2; ++y)
#pragma unroll
      for (int r = 0; r < 4; ++r) mx = fmaxf(mx, sv[y][r]);
    mx = fmaxf(mx, __builtin_bit_cast(float, xor_lane32<16>(__builtin_bit_cast(uint32_t, mx), lane)));
    mx = fmaxf(mx, __builtin_bit_cast(float, xor_lane32<32>(__builtin_bit_cast(uint32_t, mx), lane)));
    if (__any(mx > m + kRescale)) {
      const float mn = fmaxf(m, mx);
      const float alpha = mn == kNegInfR ? 1.f : fast_exp2(m - mn);
      l *= alpha;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float ar = __shfl(alpha, 4 * g + r, 64);  // head 4 g + r's
#pragma unroll
        for (int u = 0; u < NU; ++u) acc[u][r] *= ar;
      }
      m = mn;
    }
    const float mu = m == kNegInfR ? 0.f : m;
    u32x4 ph, pl;
#pragma unroll
    for (int y = 0; y < 2; ++y) {
      f32x4 p;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        p[r] = fast_exp2(sv[y][r] - mu);
        l += p[r];
      }
      if constexpr (kIs8<C>) p = scale_tokens(p, b.vs[y]);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        ph[2 * y + i] = pack2<PT>(p[2 * i], p[2 * i + 1]);
        pl[2 * y + i] = pack2<PT>(p[2 * i] - lo_f<PT>(ph[2 * y + i]), p[2 * i + 1] - hi_f<PT>(ph[2 * y + i]));
      }
    }
#pragma unroll
    for (int u = 0; u < NU; ++u) {
      u32x4 w;
#pragma unroll
      for (int y = 0; y < 2; ++y)
#pragma unroll
        for (int i = 0; i < 2; ++i) w[2 * y + i] = v_pair<C, PT>(b.v[y][2 * i], b.v[y][2 * i + 1], u);
      acc[u] = mfma_k32<PT>(ph, w, acc[u]);
      acc[u] = mfma_k32<PT>(pl, w, acc[u]);
    }
  };
  // The wave's partial of the unit, and a fresh state.
  auto flush = [&](const StreamCur& x) __attribute__((always_inline)) {
    float lt = l;
    lt += __builtin_bit_cast(float, xor_lane32<16>(__builtin_bit_cast(uint32_t, lt), lane));
    lt += __builtin_bit_cast(float, xor_lane32<32>(__builtin_bit_cast(uint32_t, lt), lane));
    const int rows = min(16, a.G - 16 * (x.k % groups)), cap = min(16, a.G);
    float* const slot = part + (static_cast<int64_t>(x.s) * units + x.k + v) * (cap * PF);
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int row = 4 * g + r;
      if (row < rows) {
        float* const dst = slot + row * PF + NU * c;
#pragma unroll
        for (int u = 0; u < NU; u += 4)
          *reinterpret_cast<f32x4*>(dst + u) = f32x4{acc[u][r], acc[u + 1][r], acc[u + 2][r], acc[u + 3][r]};
      }
    }
    if (g == 0 && c < rows) {
      slot[c * PF + D] = m;
      slot[c * PF + D + 1] = lt;
    }
    m = kNegInfR;
    l = 0.f;
#pragma unroll
    for (int u = 0; u < NU; ++u) acc[u] = f32x4{0.f, 0.f, 0.f, 0.f};
  };

  // The load cursor runs RING pairs ahead of the compute cursor, the ids one
  // pair ahead of it. Past the wave's last pair the loads go on (so that the
  // compiler's counts of what is in flight hold), all of page 0's first rows of the
  // kv head, which stay in L2: the last pair again would be read from memory again (8-bit,
  // 64 x 512-4096 tokens: 10% of the bytes). qn: the Q operand of the unit that
  // the load cursor entered last.
  Buf buf[RING];
  u32x4 qn[KJ];
  StreamCur ld = cur;
  StreamBase lbase = base_of(ld);
  int left = n_pairs - 1;  // advances the load cursor may still make
  load_q(cur, q);
  int qn_unit = -1;  // s * units + k of qn
  Ids ids = ask(ld, lbase);
  auto next = [&]() __attribute__((always_inline)) {
    if (left > 0) {
      --left;
      advance(ld);
      if (ld.t == 0) {
        lbase = base_of(ld);
        load_q(ld, qn);
        qn_unit = ld.s * units + ld.k;
      }
      ids = ask(ld, lbase);
    } else {
      ids = Ids{{0, 0}, {0, 0}};
    }
  };
#pragma unroll
  for (int d = 0; d < RING; ++d) {
    load(buf[d], ld, lbase, ids);
    next();
    __builtin_amdgcn_sched_barrier(0);
  }
  for (int i = 0; i < n_pairs; i += RING) {
#pragma unroll
    for (int d = 0; d < RING; ++d) {
      if (i + d < n_pairs) {
        if (cur.t == 0 && i + d > 0) {  // a unit starts
          if (cur.s * units + cur.k == qn_unit) {
#pragma unroll
            for (int j = 0; j < KJ; ++j) q[j] = qn[j];
          } else {  // (the load cursor has entered a later unit since)
            load_q(cur, q);
          }
          // Q has landed here: after this branch the compiler would otherwise
          // wait for it (and for every load since) before each pair's product.
#pragma unroll
          for (int j = 0; j < KJ; ++j) asm volatile("" : "+v"(q[j]));
        }
        compute(buf[d]);
        if (cur.t + 1 == cur.n || i + d + 1 == n_pairs) flush(cur);
        if (i + d + 1 < n_pairs) advance(cur);
      }
      __builtin_amdgcn_sched_barrier(0);
      load(buf[d], ld, lbase, ids);
      next();
      __builtin_amdgcn_sched_barrier(0);
    }
  }
}

// Outputs from the partials of the waves whose runs cover a unit: wave w of a
// workgroup takes every fourth of them from the w-th, batches of 4 whose loads
// are issued together, 4 dims a lane and 64 / (D / 4) rows; then the four in
// order. (Four to sixteen partials are the usual, so one or two round trips.)
// Grid: units x row groups.
template <typename T, int D>
__global__ __launch_bounds__(256) void paged_rows_stream_merge(RowsArgs a, const float* __restrict__ part,
                                                               const int32_t* __restrict__ pref) {
  constexpr int LR = D / 4, RW = 64 / LR, PF = part_floats(D);
  __shared__ __align__(16) float red[4][RW][PF];
  const int groups = (a.G + 15) / 16, units = a.Hkv * groups, cap = min(16, a.G);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int s = static_cast<int>(blockIdx.x) / units, k = static_cast<int>(blockIdx.x) - s * units;
  const int kvh = k / groups, g0 = 16 * (k - kvh * groups), rows = min(16, a.G - g0);
  const int row0 = static_cast<int>(blockIdx.y) * RW;
  if (row0 >= rows) return;
  const int row = row0 + lane / LR, rr = min(row, rows - 1), d = 4 * (lane % LR);
  const int p0 = pref[s], n = pref[s + 1] - p0;
  const int64_t total = static_cast<int64_t>(units) * pref[a.B];
  float M = kNegInfR, den = 0.f;
  f32x4 o = f32x4{0.f, 0.f, 0.f, 0.f};
  auto take = [&](float m, float l, f32x4 x) {
    const float mn = fmaxf(M, m), mu = mn == kNegInfR ? 0.f : mn;
    const float c_old = fast_exp2(M - mu), c_new = fast_exp2(m - mu);
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = fmaf(x[e], c_new, o[e] * c_old);
    den = fmaf(l, c_new, den * c_old);
    M = mn;
  };
  if (n > 0) {
    const int64_t share = stream_share(total, a.NW);
    const int64_t P = static_cast<int64_t>(units) * p0 + static_cast<int64_t>(k) * n;
    const int v0 = static_cast<int>(div_pos(P, share)), v1 = static_cast<int>(div_pos(P + n - 1, share));
    const float* const base = part + (static_cast<int64_t>(s) * units + k) * (cap * PF) + rr * PF;
    for (int v = v0 + wave; v <= v1; v += 16) {
      f32x4 po[4];
      f32x2 ml[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float* const x = base + static_cast<int64_t>(min(v + 4 * i, v1)) * (cap * PF);
        po[i] = *reinterpret_cast<const f32x4*>(x + d);
        ml[i] = *reinterpret_cast<const f32x2*>(x + D);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (v + 4 * i <= v1) take(ml[i][0], ml[i][1], po[i]);
    }
  }
  float* const mine = red[wave][lane / LR];
  *reinterpret_cast<f32x4*>(mine + d) = o;
  if (d == 0) {
    mine[D] = M;
    mine[D + 1] = den;
  }
  __syncthreads();
  if (wave > 0 || row >= rows) return;
#pragma unroll
  for (int w = 1; w < 4; ++w) {
    const float* const x = red[w][lane / LR];
    take(x[D], x[D + 1], *reinterpret_cast<const f32x4*>(x + d));
  }
  T* const out = static_cast<T*>(a.out) + s * a.o_sr + (kvh * a.G + g0 + row) * a.o_sh;
  const float inv = den == 0.f ? 0.f : 1.f / den;
  if (a.out8) {
    u32x2 w;
#pragma unroll
    for (int i = 0; i < 2; ++i) w[i] = den == 0.f ? 0u : pack2<T>(o[2 * i] * inv, o[2 * i + 1] * inv);
    *reinterpret_cast<u32x2*>(out + d) = w;
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) out[(d + e) * a.o_sd] = from_float<T>(den == 0.f ? 0.f : o[e] * inv);
  }
}

}  // namespace tsa
