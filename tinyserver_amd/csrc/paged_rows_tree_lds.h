// Draft trees of more than 32 rows a unit: the keys go through LDS, once for all
// of a workgroup's rows.
//
// A workgroup of NW = 2 or 4 waves takes 32 NW rows (nodes x q-heads of a kv
// head) over one split of the unit's keys, wave w the w-th 32 rows. 32-key
// blocks of K and V go from their pages straight into LDS
// (global_load_lds_dwordx4, no registers), NB slots of each, A = NB - 1 blocks
// ahead, the page ids from a table of the split's that the prologue puts in
// LDS. The products, the LDS layout (16-byte chunk ch of row r at position ch ^
// swz(r)), the transposed reads of V and the two-stage pipeline (S(j + 1) under
// the exponentials of block j, P V of block j - 1 under its maximum) are
// prefill_gqa_body's; the rows, the pages, the masks and what is written differ.
// The pipeline takes the blocks that every row sees whole; those from the
// context's end on (or from a page outside the pool) follow one at a time.
// Of four waves, two workgroups give a SIMD two waves of up to 256 registers, and
// one's exponentials run under the other's products.
#pragma once

#include "paged_rows_tree.h"

namespace tsa {

constexpr int kTreeMaxSplit = 256;  // 32-key blocks of a split: its page table in LDS
// K/V slots: two workgroups fit a CU, which is what the plan's 512 give it, with
// three blocks each in flight (64 sequences of 512-4096 tokens, 16 nodes, 32/8
// heads, in the sequences' own order: four 138 us, two, with four workgroups to a
// CU, 155).
constexpr int kTreeSlots = 4;
template <int D> constexpr int tree_lds_bytes() { return 2 * kTreeSlots * 32 * 2 * D + kTreeMaxSplit * 8 + 16; }

template <typename T, int D, int NW>
__global__ __launch_bounds__(64 * NW) __attribute__((amdgpu_waves_per_eu(NW == 2 ? 1 : 2))) void paged_rows_tree_lds(
    RowsArgs a, const int32_t* __restrict__ bt, const uint32_t* __restrict__ mask, float* __restrict__ part) {
  constexpr int KJ = D / 16, NU = D / 32, CPR = D / 8, RB = 2 * D, BLKB = 32 * RB, PF = part_floats(D);
  constexpr int NB = kTreeSlots, A = NB - 1;
  constexpr int RPI = 1024 / RB;            // rows of a 1 KB load instruction
  constexpr int IPW = 2 * (32 / RPI) / NW;  // load instructions of a wave and block
  constexpr int IPH = 16 / RPI;             // load instructions of a 16-row half
  constexpr int VOFF = NB * BLKB, TOFF = 2 * NB * BLKB;
  constexpr int kInFlight = (A - 1) * IPW;
  __shared__ __align__(16) char smem[tree_lds_bytes<D>()];
  int32_t* const tab = reinterpret_cast<int32_t*>(smem + TOFF);  // page id of each half of the split's blocks, -1: none
  int32_t* const first_bad = tab + 2 * kTreeMaxSplit;            // the first block with such a half

  // ---- Which unit, split and row block.
  TreeWork w;
  if (!tree_work(a, tab, w)) return;
  const int rb = w.rb, sp = w.sp, u = w.u, s = w.s, kvh = w.kvh;
  const SeqRange r = seq_of(a, s);
  const int all = r.nodes * a.G, row_first = rb * 32 * NW;
  if (row_first >= all) return;
  const int nblk = (r.end + 31) >> 5, per = tree_per_split(a, nblk), b0 = sp * per, n = min(nblk, b0 + per) - b0;  // blocks
  if (n <= 0 && a.S > 1) return;  // (the merge takes the splits that have blocks)
  const int tid = threadIdx.x, lane = tid & 63, h = lane >> 5, c = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int row_w = row_first + 32 * wave;
  const bool active = row_w < all;

  const int row = min(row_w + c, all - 1);  // (past the last: it again, never stored)
  const int node = row / a.G, head = kvh * a.G + row - node * a.G;
  const int64_t prow = r.row0 + node;
  const uint32_t* const my_mask = mask + prow * a.mask_s;
  u32x4 qop[KJ];
  {
    const T* const qp = static_cast<const T*>(a.q) + prow * a.q_sr + head * a.q_sh + 8 * h;
#pragma unroll
    for (int j = 0; j < KJ; ++j) qop[j] = *reinterpret_cast<const u32x4*>(qp + 16 * j);
  }
  // ---- The split's page table.
  if (tid == 0) *first_bad = n;
  __syncthreads();
  for (int i = tid; i < 2 * n; i += 64 * NW) {
    const uint32_t tile = static_cast<uint32_t>(2 * b0 + i), lb = page_of_tile(tile, a.page_mul, a.page_shift);
    const bool in = static_cast<int>(16u * tile) < r.end;
    const int page = bt[s * a.bt_s0 + min(static_cast<int>(lb), a.max_blocks - 1) * a.bt_s1];
    const bool ok = in && page >= 0 && page < a.NB;
    tab[i] = ok ? page : -1;
    if (!ok) atomicMin(first_bad, i >> 1);
  }
  __syncthreads();
  const int jm = min(__builtin_amdgcn_readfirstlane(*first_bad), max((r.ctx >> 5) - b0, 0));  // first masked block
  const float cs = a.scale_log2;  // > 0 here

  // ---- Loads: waves 0 .. NW / 2 - 1 the K rows, the others the V rows, IPW
  // instructions of RPI rows; lane l of one whose first row is R0 fetches the
  // chunk that belongs at row R0 + l / CPR, position l % CPR. Halves without a
  // page read page 0's first rows (masked); blocks past the last repeat it.
  auto swz = [](int x) {
    return D == 128 ? ((x & 3) << 2) | ((x >> 2) & 3) : (((x >> 1) & 1) << 2) | ((x >> 2) & 3);
  };
  typedef __attribute__((address_space(3))) void lds_void;
  const uint32_t smem_lds = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((lds_void*)smem));
  const bool k_wave = wave < NW / 2;
  const int row0w = (wave % (NW / 2)) * IPW * RPI;
  const uint32_t slot_b = static_cast<uint32_t>(k_wave ? a.kc_s : a.vc_s) * 2, page_b = k_wave ? a.k_page : a.v_page;
  const char* const pool = k_wave ? static_cast<const char*>(a.kc) + kvh * a.kc_h * 2
                                  : static_cast<const char*>(a.vc) + kvh * a.vc_h * 2;
  const int lrow = lane / CPR;
  uint32_t doff[IPW];  // of the lane within instruction i: rows from the half's first
#pragma unroll
  for (int i = 0; i < IPW; ++i)
    doff[i] = static_cast<uint32_t>((row0w + i * RPI) % 16 + lrow) * slot_b +
              16u * static_cast<uint32_t>((lane % CPR) ^ swz(row0w + i * RPI + lrow));
  constexpr int NH = IPW > IPH ? 2 : 1;  // halves a wave loads
  auto load_block = [&](int blk, int slot) __attribute__((always_inline)) {
    const int j = min(blk, n - 1);
    const int lds0 = (k_wave ? 0 : VOFF) + slot * BLKB + row0w * RB;
    const char* base[NH];
#pragma unroll
    for (int y = 0; y < NH; ++y) {
      const int half = row0w / 16 + y;
      const int ent = __builtin_amdgcn_readfirstlane(tab[2 * j + half]);
      const uint32_t tile = static_cast<uint32_t>(2 * (b0 + j) + half), lb = page_of_tile(tile, a.page_mul, a.page_shift);
      const uint32_t page = ent < 0 ? 0u : static_cast<uint32_t>(ent);
      const uint32_t slot0 = ent < 0 ? 0u : 16u * tile - lb * static_cast<uint32_t>(a.BS);
      base[y] = pool + static_cast<uint64_t>(page) * page_b + slot0 * slot_b;
    }
#pragma unroll
    for (int i = 0; i < IPW; ++i) dma16_sv(base[NH == 1 ? 0 : i / IPH], doff[i], smem_lds + lds0 + i * 1024);
  };

  int kaj[KJ];
#pragma unroll
  for (int j = 0; j < KJ; ++j) kaj[j] = (c * RB + 16 * (h ^ swz(c))) ^ (32 * j);
  u32x4 kop[KJ];
  auto kread = [&](int ks) __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < KJ; ++j) kop[j] = *reinterpret_cast<const u32x4*>(smem + ks * BLKB + kaj[j]);
  };
  auto qk = [&](f32x16& sc) __attribute__((always_inline)) {
#pragma unroll
    for (int e = 0; e < 16; ++e) sc[e] = 0.f;
#pragma unroll
    for (int j = 0; j < KJ; ++j) sc = mfma_k16x32<T>(kop[j], qop[j], sc);
  };
  float m = kNegInfR, l = 0.f;
  f32x16 acc[NU];
#pragma unroll
  for (int x = 0; x < NU; ++x)
#pragma unroll
    for (int e = 0; e < 16; ++e) acc[x][e] = 0.f;
  // Blocks from jm on: the keys the lane's row sees, and those that are there
  // at all.
  uint32_t vis = ~0u, there = ~0u;
  auto mask_block = [&](f32x16& sc, int j) __attribute__((always_inline)) {
    auto below = [](int x) { return x >= 32 ? ~0u : x > 0 ? (1u << x) - 1u : 0u; };
    const int blk = b0 + j, j0 = 32 * blk - r.ctx, w = j0 >> 5, sh = j0 & 31;
    const int e0 = __builtin_amdgcn_readfirstlane(tab[2 * j]), e1 = __builtin_amdgcn_readfirstlane(tab[2 * j + 1]);
    there = below(r.end - 32 * blk) & ((e0 < 0 ? 0u : 0xFFFFu) | (e1 < 0 ? 0u : 0xFFFF0000u));
    const uint32_t lo = w >= 0 && w < a.words ? my_mask[w] : 0u;
    const uint32_t hi = w + 1 >= 0 && w + 1 < a.words ? my_mask[w + 1] : 0u;
    vis = (below(r.ctx - 32 * blk) | (sh ? (lo >> sh) | (hi << (32 - sh)) : lo)) & there;
#pragma unroll
    for (int e = 0; e < 16; ++e)
      if (!((vis >> (8 * (e >> 2) + 4 * h + (e & 3))) & 1)) sc[e] = kNegInfR;
  };
  auto block_max = [&](const f32x16& sc) __attribute__((always_inline)) {
    float mx = kNegInfR;
#pragma unroll
    for (int e = 0; e < 16; ++e) mx = fmaxf(mx, sc[e]);
    const auto sw = __builtin_amdgcn_permlane32_swap(__float_as_uint(mx), __float_as_uint(mx), false, false);
    return fmaxf(__uint_as_float(sw[0]), __uint_as_float(sw[1])) * cs;
  };
  auto rescale = [&](float mt) __attribute__((always_inline)) {
    if (__any(mt > m + kTreeRescale)) {
      const float mn = fmaxf(m, mt), alpha = mn == kNegInfR ? 1.f : fast_exp2(m - mn);
      l *= alpha;
#pragma unroll
      for (int x = 0; x < NU; ++x)
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[x][e] *= alpha;
      m = mn;
    }
  };
  u32x4 pop[2];
  auto softmax_exp = [&](const f32x16& sc) __attribute__((always_inline)) {
    const float mu = m == kNegInfR ? 0.f : m;
    float p[16];
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      p[e] = fast_exp2(fmaf(sc[e], cs, -mu));
      l += p[e];
    }
#pragma unroll
    for (int e = 0; e < 16; e += 2) pop[e >> 3][(e & 7) >> 1] = pack2<T>(p[e], p[e + 1]);
  };
  typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
  int vofs[NU];
#pragma unroll
  for (int x = 0; x < NU; ++x) {
    const int jl = c & 15, rr = 4 * h + (jl >> 2), ch = 4 * x + 2 * (c >> 4) + ((jl & 3) >> 1);
    vofs[x] = rr * RB + 16 * (ch ^ swz(rr)) + 8 * (jl & 1);
  }
  u32x4 vop[2][NU];  // V[keys of P's slots][dim 32 x + c]
  auto vread = [&](int vs) __attribute__((always_inline)) {
#pragma unroll
    for (int s2 = 0; s2 < 2; ++s2)
#pragma unroll
      for (int x = 0; x < NU; ++x) {
        const int base = VOFF + vs * BLKB + 16 * s2 * RB;
        const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(smem + base + vofs[x]));
        const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(smem + base + 8 * RB + (vofs[x] ^ 32)));
        const u32x2 lo2 = __builtin_bit_cast(u32x2, lo), hi2 = __builtin_bit_cast(u32x2, hi);
        vop[s2][x] = u32x4{lo2[0], lo2[1], hi2[0], hi2[1]};
      }
  };
  // Masked blocks, after their V is in registers: rows that are not there
  // become 0; elements that are not finite reach the rows that see them through
  // a product of flags, and leave V.
  auto fix_v = [&]() __attribute__((always_inline)) {
    bool bad = false;
#pragma unroll
    for (int s2 = 0; s2 < 2; ++s2)
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int e = 8 * s2 + 2 * k;
        const uint32_t b = there >> (8 * (e >> 2) + 4 * h + (e & 3));
        const uint32_t keep = (b & 1 ? 0xFFFFu : 0u) | (b & 2 ? 0xFFFF0000u : 0u);
#pragma unroll
        for (int x = 0; x < NU; ++x) {
          vop[s2][x][k] &= keep;
          bad |= nonfinite2<T>(vop[s2][x][k]) != 0;
        }
      }
    if (!__any(bad)) return;
    constexpr uint32_t one = std::is_same<T, bf16_t>::value ? 0x3F80u : 0x3C00u;
    u32x4 sees[2];
#pragma unroll
    for (int e = 0; e < 16; e += 2) {
      const uint32_t b = vis >> (8 * (e >> 2) + 4 * h + (e & 3));
      sees[e >> 3][(e & 7) >> 1] = (b & 1 ? one : 0u) | (b & 2 ? one << 16 : 0u);
    }
#pragma unroll
    for (int x = 0; x < NU; ++x) {
      f32x16 f;
#pragma unroll
      for (int e = 0; e < 16; ++e) f[e] = 0.f;
#pragma unroll
      for (int s2 = 0; s2 < 2; ++s2) {
        u32x4 w;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const uint32_t v = vop[s2][x][k], nf = nonfinite2<T>(v);
          w[k] = flag16<T>(v & 0xFFFFu) | flag16<T>(v >> 16) << 16;
          vop[s2][x][k] = v & (nf & 1 ? 0xFFFF0000u : ~0u) & (nf & 2 ? 0xFFFFu : ~0u);
        }
        f = mfma_k16x32<T>(w, sees[s2], f);
      }
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[x][e] += flag_value(f[e]);
    }
  };
  auto pv = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int s2 = 0; s2 < 2; ++s2)
#pragma unroll
      for (int x = 0; x < NU; ++x) acc[x] = mfma_k16x32<T>(vop[s2][x], pop[s2], acc[x]);
  };

  f32x16 sca, scb;  // S of the even / odd blocks
  // One block that every row sees whole (prefill_gqa_body's full()): on entry
  // S(j) is in registers, K block j + 1 and V block j in their slots, and (PREV)
  // block j - 1's P and V operands in registers.
  auto full = [&](int j, auto S, auto prev) __attribute__((always_inline)) {
    constexpr int s0 = decltype(S)::value;
    f32x16& cur = (s0 & 1) ? scb : sca;
    f32x16& nxt = (s0 & 1) ? sca : scb;
    const bool issue = j < n - A;
    if (issue) load_block(j + A + (k_wave ? 1 : 0), k_wave ? s0 : (s0 + NB - 1) % NB);
    if (active) {
      kread((s0 + 1) % NB);
      if constexpr (decltype(prev)::value) pv();
      const float mt = block_max(cur);
      if constexpr (decltype(prev)::value) {
#pragma unroll
        for (int i = 0; i < 2 * NU; ++i) {
          __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
          __builtin_amdgcn_sched_group_barrier(0x002, 2, 0);
        }
      }
      rescale(mt);
      qk(nxt);
      softmax_exp(cur);
      vread(s0);
#pragma unroll
      for (int jj = 0; jj < KJ; ++jj) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x002, 56 / KJ, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, 4 * NU / KJ, 0);
      }
      asm volatile("" : "+v"(pop[0]), "+v"(pop[1]), "+v"(l));
    }
    if (issue) wait_vmcnt<kInFlight>();
    else wait_vmcnt<0>();
    lds_barrier();
  };

  using std::integral_constant;
  if (n > 0) {
    if (k_wave) {
      load_block(0, 0);
#pragma unroll
      for (int x = 0; x < A; ++x)
        if (x < n) load_block(x + 1, x + 1);
    } else {
#pragma unroll
      for (int x = 0; x < A; ++x)
        if (x < n) load_block(x, x);
    }
    // K(0) and step 0. (Also the Q loads, which the compiler's own waits would
    // otherwise put into the loop.)
    if (n >= A) wait_vmcnt<kInFlight>();
    else wait_vmcnt<0>();
    lds_barrier();
    // ---- The blocks before jm, in the pipeline.
    const int n1 = min(n, jm);
    if (n1 > 0) {
      kread(0);
      qk(sca);
      lds_barrier();  // iteration 0's loads overwrite K(0)'s slot
      full(0, integral_constant<int, 0>{}, std::false_type{});
      for (int j = 1; j < n1;) {
        full(j, integral_constant<int, 1>{}, std::true_type{});
        if (++j == n1) break;
        full(j, integral_constant<int, 2>{}, std::true_type{});
        if (++j == n1) break;
        full(j, integral_constant<int, 3>{}, std::true_type{});
        if (++j == n1) break;
        full(j, integral_constant<int, 0>{}, std::true_type{});
        ++j;
      }
      if (active) pv();
    }
    // ---- The others (a few: those of the nodes and the context's last), one
    // at a time: masks and what they need stay out of the pipeline's registers.
#pragma unroll 1
    for (int j = n1; j < n; ++j) {
      if (active) kread(j % NB);
      lds_barrier();  // step j + A overwrites K(j)'s slot and V(j - 1)'s
      const bool issue = j < n - A;
      if (issue) load_block(j + A + (k_wave ? 1 : 0), k_wave ? j % NB : (j + NB - 1) % NB);
      if (active) {
        qk(sca);
        mask_block(sca, j);
        rescale(block_max(sca));
        softmax_exp(sca);
        vread(j % NB);
        fix_v();
        pv();
      }
      if (issue) wait_vmcnt<kInFlight>();
      else wait_vmcnt<0>();
      lds_barrier();
    }
  }
  if (!active) return;  // (no barrier follows)
  l += __builtin_bit_cast(float, xor_lane32<32>(__builtin_bit_cast(uint32_t, l), lane));
  if (row_w + c >= all) return;
  if (a.S == 1) {
    T* const out = static_cast<T*>(a.out) + prow * a.o_sr + head * a.o_sh;
    const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
    for (int x = 0; x < NU; ++x)
#pragma unroll
      for (int e = 0; e < 16; e += 4) {
        const int d = 32 * x + 8 * (e >> 2) + 4 * h;
        u32x2 w = {pack2<T>(acc[x][e] * inv, acc[x][e + 1] * inv), pack2<T>(acc[x][e + 2] * inv, acc[x][e + 3] * inv)};
        if (l == 0.f) w = u32x2{0, 0};
        if (a.out8) {
          *reinterpret_cast<u32x2*>(out + d) = w;
        } else {
          uint16_t* const o16 = reinterpret_cast<uint16_t*>(out);
#pragma unroll
          for (int i = 0; i < 4; ++i) o16[(d + i) * a.o_sd] = static_cast<uint16_t>(w[i >> 1] >> (16 * (i & 1)));
        }
      }
  } else {
    float* const out = part + ((static_cast<int64_t>(u) * a.S + sp) * (a.T * a.G) + row) * PF;
#pragma unroll
    for (int x = 0; x < NU; ++x)
#pragma unroll
      for (int e = 0; e < 16; e += 4)
        *reinterpret_cast<f32x4*>(out + 32 * x + 8 * (e >> 2) + 4 * h) =
            f32x4{acc[x][e], acc[x][e + 1], acc[x][e + 2], acc[x][e + 3]};
    if (h == 0) *reinterpret_cast<f32x2*>(out + D) = f32x2{m, l};
  }
}

}  // namespace tsa
