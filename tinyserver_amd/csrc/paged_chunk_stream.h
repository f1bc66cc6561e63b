// Attention of a chunk over the paged cache on the matrix cores: a run of 32-key
// blocks a workgroup, whatever sequences they belong to.
//
// An item is (sequence, kv head, row block): QB queries times the G q-heads of the kv
// head, up to 32 NW rows (row = query G + head), so that one K/V byte serves all of
// them and a wave takes 32 rows. Item i has as many 32-key blocks as its last query
// sees. A step may hold one sequence with 2048 new tokens beside sixty with one, over
// a few or 30,000 cached ones, so work is not dealt by sequence: all items' blocks in
// a row (sequence, kv head, row block), total W, are cut into runs of ceil(W / P)
// blocks, one a workgroup, and an item that a cut goes through is put together by a
// second launch from its runs' partial results. The lengths are on the device only:
// each workgroup sums them itself and looks its start up (chunk_start).
// Runs that follow each other share K and V and go to one XCD.
//
// In a workgroup K and V go from their pages straight into LDS
// (global_load_lds_dwordx4, no registers), NB slots of each, A = NB - 1 blocks ahead;
// page ids come from a table in LDS that a segment's prologue fills. With lane (h, c)
// = (lane / 32, lane % 32), v_mfma_f32_32x32x16:
//   S^T(32 keys x 32 rows) = K Q^T: lane (h, c) reads key c, dims 16 j + 8 h..+8, and
//     holds row c's Q; element e of the result is the score of key 8 (e / 4) + 4 h +
//     e % 4 for row c;
//   O^T(dims x 32 rows) += V^T P^T over two 16-key steps: the P^T operand is the lane's
//     own weights, V's comes from transposed LDS reads. Lane (h, c) accumulates row c,
//     so the softmax's scales are the lane's own.
// The 16-byte chunk ch of LDS row r sits at position ch ^ swz(r), free of bank
// conflicts in both reads. S(j + 1) runs under the exponentials of block j, P V of
// block j - 1 under its maximum; two workgroups a CU give a SIMD two waves, of which
// one's exponentials run under the other's products.
//
// The chunk's own last blocks take their masks in the pipeline; blocks before them
// need none. From the first block with a page that is not there on, the blocks of a
// table's 480 go one at a time, behind the pipeline. Rows of V that no row sees repeat the last key's there. Where an item's sums are not
// finite, V of a key that some row does not see may be why (a weight of 0 times NaN):
// the item goes again with every masked block one at a time, where V rows that are not
// there become 0 and elements of V that are not finite reach the rows that see them
// through a product of flags.
// A weight goes to the second product rounded once to T, off by at most 2^-8 (f16:
// 2^-11) of itself, as in the prefill kernels.
//
// At head_dim 128 the kernel holds 256 registers and spills 17; 190 and none at 64.
#pragma once

#include "nonfinite.h"
#include "varlen_prefill_gqa.h"
#include "paged_chunk.h"

namespace tsa {

constexpr int kChunkSlots = 4;       // K/V blocks in LDS
constexpr int kChunkTab = 480;       // 32-key blocks whose places the table in LDS holds
// What an item costs beside its blocks, in blocks (its table, Q, first loads and
// results: 5 us where a block takes 0.9), which the deal counts at its start.
constexpr int kItemCost = 6;
constexpr float kChunkRescale = 8.f; // log2 units a maximum grows before it moves
constexpr float kChunkNone = -3.402823466e38f;  // the maximum of no score: below every one but -inf, and its weights 0

// ---- The plan on the device.
// 32-key blocks of a sequence's row blocks 0 .. i - 1: sum of ceil(min(ctx + (k + 1)
// QB, end) / 32), and kItemCost for each. With QB = 32 qh + ql the remainders of ql repeat after 32 terms.
__device__ __forceinline__ int64_t chunk_blocks(int ctx, int end, int QB, int i) {
  const int full = min(i, (end - ctx) / QB), ql = QB & 31, y = ctx + QB + 31;
  int64_t sum = static_cast<int64_t>(i) * kItemCost + static_cast<int64_t>(i - full) * ((end + 31) >> 5) + static_cast<int64_t>(y >> 5) * full +
                static_cast<int64_t>(QB >> 5) * full * (full - 1) / 2;
  if (ql) {
    const int K = full >> 5, J = full & 31;
    int all = 0, part = 0, v = y & 31;
    for (int j = 0; j < 32; ++j, v += ql) {
      all += v >> 5;
      part += j < J ? v >> 5 : 0;
    }
    sum += static_cast<int64_t>(K) * all + static_cast<int64_t>(ql) * (16 * static_cast<int64_t>(K) * (K - 1) + static_cast<int64_t>(K) * J) + part;
  }
  return sum;
}
__device__ __forceinline__ int chunk_row_blocks(const ChunkSeq& r, int QB) { return (r.n + QB - 1) / QB; }
__device__ __forceinline__ int64_t uniform64(int64_t x) {
  const uint32_t lo = static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(x)));
  const uint32_t hi = static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(x >> 32)));
  return static_cast<int64_t>((static_cast<uint64_t>(hi) << 32) | lo);
}
// Where a run starts: block `blk` of row block rb of (sequence s, kv head kvh), or -blk
// of its cost before the first.
struct ChunkStart {
  int s, kvh, rb, blk;
};
// A segment: blocks blk0 .. blk1 - 1 of an item's nblk. In LDS, with what its next
// one follows from.
struct ChunkSegment {
  int32_t s, kvh, nq, pos, end;  // pos: position of the item's first query
  int32_t blk0, blk1, nblk;      // blk1 0: no more
  int64_t row;                   // packed row of that query
};
struct ChunkWork {
  ChunkSegment seg[2];  // in turn: the one in hand, and the next
  ChunkSeq r;
  int32_t rb, left, run, per;  // left: blocks (whole items: items) of the run
  int32_t redo;         // what a segment gave is not finite
  int32_t bad[2];       // of each segment: its first block (from its table's first) with a page that is not there
  // One thread: the segment from block blk of row block rb on, `cost` before it.
  __device__ __forceinline__ void set(const ChunkArgs& a, ChunkSegment& x, int s, int kvh, int blk, int cost) {
    const int q0 = rb * a.QB;
    x.s = s;
    x.kvh = kvh;
    x.nq = min(a.QB, r.n - q0);
    x.pos = r.ctx + q0;
    x.end = r.end;
    x.row = r.row0 + q0;
    x.nblk = (min(x.pos + x.nq, r.end) + 31) >> 5;  // keys that its last query sees
    x.blk0 = blk;
    left -= cost;
    x.blk1 = left <= 0 ? 0 : a.whole ? x.nblk : min(x.nblk, blk + left);
    left -= a.whole ? 1 : x.blk1 - blk;
  }
  // One thread: run `run`, from st on.
  __device__ __forceinline__ void start(const ChunkArgs& a, const ChunkSeq& first, const ChunkStart& st, int64_t total,
                                        int run_, int per_) {
    a.splits[run_].runs = 0;
    run = run_;
    per = per_;
    bad[0] = INT32_MAX;
    redo = 0;
    r = first;
    rb = st.rb;
    const int64_t rest = total - static_cast<int64_t>(run) * per;
    left = static_cast<int>(rest < per ? rest : per);
    set(a, seg[0], st.s, st.kvh, max(st.blk, 0), max(-st.blk, 0));
  }
  // What the second launch needs of segment x, which the run starts inside of.
  __device__ __forceinline__ ChunkSplit split(const ChunkSegment& x) const {
    const int64_t item = static_cast<int64_t>(run) * per - x.blk0;  // its first block
    ChunkSplit sp;
    sp.row0 = x.row;
    sp.kvh = x.kvh;
    sp.queries = x.nq;
    sp.runs = item >= static_cast<int64_t>(run - 1) * per ? static_cast<int>((item + x.nblk - 1) / per) - run + 1 : 0;
    return sp;
  }
  // One thread: the segment behind `from`.
  __device__ __forceinline__ void next(const ChunkArgs& a, const ChunkSegment& from, ChunkSegment& x) {
    x = from;  // (without a next, its Q and first page are read again)
    x.blk1 = 0;
    if (left <= 0) return;
    int s = from.s, kvh = from.kvh;
    if (++rb * a.QB >= r.n) {
      rb = 0;
      if (++kvh == a.Hkv) {
        kvh = 0;
        do r = chunk_seq(a, ++s);
        while (r.n == 0 && s < a.B - 1);
      }
    }
    set(a, x, s, kvh, 0, a.whole ? 0 : kItemCost);
  }
};
constexpr size_t kChunkHead = 64;  // bytes before the splits: the number of runs
// A partial result: 32 NW rows, in the order of the lanes' accumulators, then each
// row's maximum and sum.
__host__ __device__ constexpr int chunk_part_floats(int D, int NW) { return 32 * NW * (D + 2); }

template <int NT>
__device__ __forceinline__ uint64_t chunk_scan(uint64_t x, uint64_t* waves, uint64_t& total) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const uint64_t incl = wave_scan_u64(x);
  if (lane == 63) waves[w] = incl;
  __syncthreads();
  uint64_t before = 0;
  total = 0;
#pragma unroll
  for (int i = 0; i < NT / 64; ++i) {
    before += i < w ? waves[i] : 0;
    total += waves[i];
  }
  __syncthreads();
  return before + incl - x;
}

// The blocks of all items, and the place of block run * per of them, per = the blocks
// of a run. (Whole items: their number, and item run * per.) Up to NT sequences are
// read once. found: in LDS, where the thread that has the run's sequence leaves it;
// waves: 64 bytes of LDS. All threads call.
struct ChunkFound {
  ChunkSeq r;
  int64_t off, head;  // blocks of the sequence before the start; of one kv head
  int32_t s;
};
template <int NT>
__device__ __forceinline__ bool chunk_start(const ChunkArgs& a, uint64_t* waves, ChunkFound* found, int P, int64_t& total,
                                            int& per, int& run, ChunkStart& st) {
  const int tid = threadIdx.x, lane = tid & 63;
  ChunkSeq r{};
  int64_t head = 0;
  auto weight = [&](int s) -> uint64_t {
    if (s >= a.B) return 0;
    r = chunk_seq(a, s);
    head = chunk_row_blocks(r, a.QB);
    if (!a.whole) head = chunk_blocks(r.ctx, r.end, a.QB, static_cast<int>(head));
    return static_cast<uint64_t>(head) * a.Hkv;
  };
  uint64_t mine = weight(tid), sum;
  const uint64_t first = mine;
  for (int s = tid + NT; s < a.B; s += NT) mine += weight(s);
  uint64_t b = chunk_scan<NT>(mine, waves, sum);
  total = uniform64(static_cast<int64_t>(sum));
  // (32-bit divisions where they do: a 64-bit one is a hundred instructions)
  const int64_t even = total < (int64_t{1} << 31) ? (static_cast<uint32_t>(total) + P - 1) / static_cast<uint32_t>(P)
                                                  : (total + P - 1) / P;
  per = __builtin_amdgcn_readfirstlane(static_cast<int>(even > a.min_run ? even : a.min_run));
  const int runs = total < (int64_t{1} << 31) ? static_cast<int>((static_cast<uint32_t>(total) + per - 1) / static_cast<uint32_t>(per))
                                              : static_cast<int>((total + per - 1) / per);
  // Runs of an XCD (workgroups go round the XCDs) follow each other.
  const int of_xcd = (runs + 7) >> 3, i = static_cast<int>(blockIdx.x) >> 3;
  run = (static_cast<int>(blockIdx.x) & 7) * of_xcd + i;
  if (i >= of_xcd || run >= runs) return false;
  const uint64_t x0 = static_cast<uint64_t>(run) * per;
  uint64_t before = 0;
  for (int base = 0; base < a.B; base += NT) {
    uint64_t w = first;
    if (a.B > NT) {  // (uniform)
      w = weight(base + tid);
      b = before + chunk_scan<NT>(w, waves, sum);
      before += sum;
    }
    if (b <= x0 && x0 < b + w) {
      found->r = r;
      found->head = head;
      found->off = static_cast<int64_t>(x0 - b);
      found->s = base + tid;
    }
    if (a.B > NT && x0 < before) break;  // (uniform)
  }
  __syncthreads();
  st.s = __builtin_amdgcn_readfirstlane(found->s);
  int64_t off = uniform64(found->off);
  const int64_t of_head = uniform64(found->head);
  const int ctx = __builtin_amdgcn_readfirstlane(found->r.ctx), end = __builtin_amdgcn_readfirstlane(found->r.end);
  st.kvh = __builtin_amdgcn_readfirstlane(
      (off | of_head) < (int64_t{1} << 31) ? static_cast<int>(static_cast<uint32_t>(off) / static_cast<uint32_t>(of_head))
                                           : static_cast<int>(off / of_head));
  off -= of_head * st.kvh;
  st.rb = static_cast<int>(off);
  st.blk = 0;
  if (a.whole) return true;
  int lo = 0, n = chunk_row_blocks(found->r, a.QB);  // the row block is one of lo .. lo + n - 1
  n = __builtin_amdgcn_readfirstlane(n);
  int64_t at_lo = 0;  // blocks before it
  while (n > 1) {
    const int step = (n + 63) >> 6;
    const int64_t mine_at = lane * step < n ? chunk_blocks(ctx, end, a.QB, lo + lane * step) : INT64_MAX;
    const int at = __builtin_popcountll(__ballot(mine_at <= off)) - 1;
    at_lo = static_cast<int64_t>(static_cast<uint64_t>(static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(mine_at >> 32), at))) << 32 |
                                 static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(mine_at), at)));
    n = min(step, n - at * step);
    lo += at * step;
  }
  st.rb = lo;
  st.blk = __builtin_amdgcn_readfirstlane(static_cast<int>(off - at_lo)) - kItemCost;  // (below 0: in what it costs)
  return true;
}

// The arguments, read where they are used: held in registers from the start, those
// that only a segment's ends need would spill others' out of the loop over blocks.
// (The kernel's first parameter is its ChunkArgs.)
__device__ __forceinline__ const ChunkArgs& chunk_args() {
  typedef const __attribute__((address_space(4))) ChunkArgs* Ptr;
  Ptr p = (Ptr)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(p));
  return *(const ChunkArgs*)p;
}

template <int D> constexpr int chunk_lds_bytes() { return 2 * kChunkSlots * 32 * 2 * D + kChunkTab * 32 + sizeof(ChunkWork); }

template <typename T, int D, int NW>
__global__ __launch_bounds__(64 * NW) __attribute__((amdgpu_waves_per_eu(2))) void paged_chunk_stream(
    ChunkArgs a) {
  constexpr int KJ = D / 16, NU = D / 32, CPR = D / 8, RB = 2 * D, BLKB = 32 * RB;
  constexpr int NB = kChunkSlots, A = NB - 1;
  constexpr int RPI = 1024 / RB;            // rows of a 1 KB load instruction
  constexpr int IPW = 2 * (32 / RPI) / NW;  // load instructions of a wave and block
  constexpr int IPH = 16 / RPI;             // load instructions of a 16-row half
  constexpr int VOFF = NB * BLKB, TOFF = 2 * NB * BLKB;
  constexpr int kInFlight = (A - 1) * IPW;
  __shared__ __align__(16) char smem[chunk_lds_bytes<D>()];
  // For the halves (16 keys) of a segment's blocks, the byte offset of the first row
  // in the K pool, then (kChunkTab blocks on) in the V pool; bit 63: no such page.
  uint64_t* const tab = reinterpret_cast<uint64_t*>(smem + TOFF);
  ChunkWork* const work = reinterpret_cast<ChunkWork*>(tab + 4 * kChunkTab);

  int64_t total;
  int per, run;
  ChunkStart st;
  const int P = static_cast<int>(gridDim.x);
  ChunkFound* const found = reinterpret_cast<ChunkFound*>(smem + 64);
  const bool has = chunk_start<64 * NW>(a, reinterpret_cast<uint64_t*>(smem), found, P, total, per, run, st);
  if (blockIdx.x == 0 && threadIdx.x == 0) *a.runs = static_cast<int32_t>((total + per - 1) / per);
  if (!has) return;

  const int tid = threadIdx.x, lane = tid & 63, h = lane >> 5, c = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const float cs = a.scale_log2;  // > 0 here
  // Of two workgroups on a CU the one that came first has its waves served first, and
  // the other ran 20 us alone at the end of 80: three blocks of four it goes first now
  // (2 x 12-40 tokens over 24000-32768: 89 -> 85.5 us; all four: 87).
  const bool second = NW == 4 && (blockIdx.x >> 3) * 16 >= gridDim.x;
  if (NW == 4 && !second) __builtin_amdgcn_s_setprio(1);

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
  const uint32_t slot_b = static_cast<uint32_t>(k_wave ? a.kc_s : a.vc_s) * 2;
  const uint32_t lds_w = smem_lds + (k_wave ? 0 : VOFF) + row0w * RB;  // this wave's rows of slot 0
  const int lrow = lane / CPR;
  // The lane's place in instruction i: row r0w % 16 + i RPI + lrow of the half, chunk
  // (lane % CPR) ^ swz(that row), where i changes two bits of swz (one at D = 64).
  const uint32_t rpart = static_cast<uint32_t>(row0w % 16 + lrow) * slot_b;
  const uint32_t cpart = 16u * static_cast<uint32_t>((lane % CPR) ^ swz(row0w + lrow));
  static_assert(IPW <= IPH, "a wave loads rows of one half");
  const int ka0 = c * RB + 16 * (h ^ swz(c));  // K operand j at ka0 ^ 32 j of a slot
  typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
  int vofs[NU];
#pragma unroll
  for (int x = 0; x < NU; ++x) {
    const int jl = c & 15, rr = 4 * h + (jl >> 2), ch = 4 * x + 2 * (c >> 4) + ((jl & 3) >> 1);
    vofs[x] = rr * RB + 16 * (ch ^ swz(rr)) + 8 * (jl & 1);
  }

  // The run's segments, one after the other: thread 0 keeps them in LDS (held in
  // registers they cost the loop over blocks 160 spilled ones).
  if (tid == 0) work->start(a, found->r, st, total, run, per);
  lds_barrier();
  auto of = [&](const int32_t& x) { return __builtin_amdgcn_readfirstlane(x); };
  // The lane's row of a segment, looked up where it is used: query and q-head, and the
  // packed row of q/out. (Rows past the item's last: its query again, never stored.)
  struct Row {
    int q, head;
    int64_t at;
    bool ok;
  };
  auto my_row = [&](const ChunkArgs& x, const ChunkSegment& seg) __attribute__((always_inline)) {
    int t = threadIdx.x;
    asm volatile("" : "+v"(t));
    const int rw = (t >> 6) * 32 + (t & 31), rq = (rw * x.g_mul) >> 16;
    Row row;
    row.q = min(rq, of(seg.nq) - 1);
    row.head = of(seg.kvh) * x.G + rw - rq * x.G;
    row.at = seg.row + row.q;
    row.ok = rq < of(seg.nq);
    return row;
  };
  auto page_at = [&](const ChunkArgs& x, const ChunkSegment& seg, int tile) __attribute__((always_inline)) {
    // (halves behind the last key: the last one's place again)
    const uint32_t lb = page_of_tile(static_cast<uint32_t>(min(tile, (of(seg.end) - 1) >> 4)), x.page_mul, x.page_shift);
    return x.bt[of(seg.s) * x.bt_s0 + min(static_cast<int>(lb), x.max_blocks - 1) * x.bt_s1];
  };
  // A segment's Q, and the page of the thread's first half block: asked for while the
  // one before stores its results.
  u32x4 qop[KJ];
  int page0;
  auto ask = [&](const ChunkSegment& seg) __attribute__((always_inline)) {
    const ChunkArgs& g = chunk_args();
    page0 = page_at(g, seg, 2 * of(seg.blk0) + tid);
    const Row row = my_row(g, seg);
    const T* const qp = static_cast<const T*>(g.q) + row.at * g.q_sr + row.head * g.q_sh + 8 * h;
#pragma unroll
    for (int j = 0; j < KJ; ++j) qop[j] = *reinterpret_cast<const u32x4*>(qp + 16 * j);
  };
  ask(work->seg[0]);
#pragma unroll 1
  for (int turn = 0; work->seg[turn].blk1 > 0; turn ^= 1) {
    const ChunkSegment& seg = work->seg[turn];
    const ChunkArgs& g = chunk_args();
    const int blk0 = of(seg.blk0), blk1 = of(seg.blk1), pos = of(seg.pos), end = of(seg.end);
    const bool active = 32 * wave < of(seg.nq) * g.G;
    {
      const char* const pool = k_wave ? static_cast<const char*>(g.kc) + of(seg.kvh) * g.kc_h * 2
                                      : static_cast<const char*>(g.vc) + of(seg.kvh) * g.vc_h * 2;
      float m, l;
      f32x16 acc[NU];
      u32x4 kop[KJ];
      // (`it`, the loop's counter, keeps the operands' places from being computed once
      // and held: they would spill.)
      auto kread = [&](int ks, int it) __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < KJ; ++j) {
          int ka = ka0;
          if (j > 0) asm("v_xor_b32 %0, %1, %2" : "=v"(ka) : "n"(32 * j), "v"(ka0), "s"(it));
          kop[j] = *reinterpret_cast<const u32x4*>(smem + ks * BLKB + ka);
        }
      };
      auto qk = [&](f32x16& sc) __attribute__((always_inline)) {
#pragma unroll
        for (int e = 0; e < 16; ++e) sc[e] = 0.f;
#pragma unroll
        for (int j = 0; j < KJ; ++j) sc = mfma_k16x32<T>(kop[j], qop[j], sc);
      };
      auto block_max = [&](const f32x16& sc) __attribute__((always_inline)) {
        float mx = kNegInfC;
#pragma unroll
        for (int e = 0; e < 16; ++e) mx = fmaxf(mx, sc[e]);
        const auto sw = __builtin_amdgcn_permlane32_swap(__float_as_uint(mx), __float_as_uint(mx), false, false);
        return fmaxf(__uint_as_float(sw[0]), __uint_as_float(sw[1])) * cs;
      };
      auto rescale = [&](float mt) __attribute__((always_inline)) {
        // (A row's own scores alone move its maximum, so that what other rows of the
        // wave see does not change its rounding.)
        const bool up = mt > m + kChunkRescale;
        if (__any(up)) {
          const float mn = up ? mt : m, alpha = up ? fast_exp2(m - mn) : 1.f;
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
        float p[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          p[e] = fast_exp2(fmaf(sc[e], cs, -m));
          l += p[e];
        }
#pragma unroll
        for (int e = 0; e < 16; e += 2) pop[e >> 3][(e & 7) >> 1] = pack2<T>(p[e], p[e + 1]);
      };
      u32x4 vop[2][NU];  // V[keys of P's slots][dim 32 x + c]
      auto vread = [&](int vs, int it) __attribute__((always_inline)) {
#pragma unroll
        for (int x = 0; x < NU; ++x) {
          int vofx;  // (8 rows on)
          asm("v_xor_b32 %0, 32, %1" : "=v"(vofx) : "v"(vofs[x]), "s"(it));
#pragma unroll
          for (int s2 = 0; s2 < 2; ++s2) {
            const int base = VOFF + vs * BLKB + 16 * s2 * RB;
            const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(smem + base + vofs[x]));
            const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(smem + base + 8 * RB + vofx));
            const u32x2 lo2 = __builtin_bit_cast(u32x2, lo), hi2 = __builtin_bit_cast(u32x2, hi);
            vop[s2][x] = u32x4{lo2[0], lo2[1], hi2[0], hi2[1]};
          }
        }
      };
      auto pv = [&]() __attribute__((always_inline)) {
#pragma unroll
        for (int s2 = 0; s2 < 2; ++s2)
#pragma unroll
          for (int x = 0; x < NU; ++x) acc[x] = mfma_k16x32<T>(vop[s2][x], pop[s2], acc[x]);
      };

      // ---- The segment's blocks, kChunkTab at a time. A first time with every block
      // whose pages are there in the pipeline; if what that gives is not finite, V of a
      // key that some row does not see may be why, and those go one at a time.
#pragma unroll 1
      for (bool safe = false;; safe = true) {
      m = kChunkNone;
      l = 0.f;
#pragma unroll
      for (int x = 0; x < NU; ++x)
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[x][e] = 0.f;
#pragma unroll 1
      for (int b0 = blk0; b0 < blk1; b0 += kChunkTab) {
        const int n = min(blk1 - b0, kChunkTab);
        int32_t* const first_bad = &work->bad[turn];
        if (safe || b0 != blk0) {  // (else the one before left it so)
          lds_barrier();
          if (tid == 0) {
            *first_bad = INT32_MAX;
            work->redo = 0;
          }
          lds_barrier();
        }
        const ChunkArgs& f = chunk_args();
        auto put = [&](int i, int page) __attribute__((always_inline)) {
          const int tile = min(2 * b0 + i, (end - 1) >> 4);
          const uint32_t lb = page_of_tile(static_cast<uint32_t>(tile), f.page_mul, f.page_shift);
          const bool ok = page >= 0 && page < f.NB;
          const uint32_t slot0 = 16u * tile - lb * static_cast<uint32_t>(f.BS);
          const uint64_t none = uint64_t{1} << 63;
          tab[i] = ok ? static_cast<uint64_t>(page) * f.k_page + slot0 * static_cast<uint64_t>(2 * f.kc_s) : none;
          tab[2 * kChunkTab + i] = ok ? static_cast<uint64_t>(page) * f.v_page + slot0 * static_cast<uint64_t>(2 * f.vc_s) : none;
          if (!ok) atomicMin(first_bad, i >> 1);
        };
        int from = tid;
        if (b0 == blk0 && !safe) {
          if (tid < 2 * n) put(tid, page0);
          from += 64 * NW;
        }
        for (int i = from; i < 2 * n; i += 64 * NW) put(i, page_at(f, seg, 2 * b0 + i));
        lds_barrier();
        // The first block that some row does not see whole, and the first outside the
        // pipeline.
        const int jc = max((min(pos + 1, end) >> 5) - b0, 0);
        const int jm = min(min(__builtin_amdgcn_readfirstlane(*first_bad), n), safe ? jc : n);
        // The wave's places of a block; the loads of one, and of the places of the one
        // after it.
        const int whole = 32 * (b0 + n) > end ? n - 1 : n + A + 2;  // blocks below it have all their keys
        uint64_t at;
        const uint64_t* const my_tab = tab + (k_wave ? 0 : 2 * kChunkTab) + row0w / 16;
        auto look_up = [&](int blk) __attribute__((always_inline)) { at = my_tab[2 * min(blk, n - 1)]; };
        auto load_block = [&](int blk, int slot) __attribute__((always_inline)) {
          uint32_t lds0 = lds_w;
          asm("" : "+s"(lds0) : "s"(blk));  // (each load's place is added to it here: sixteen of them held would spill)
          const uint32_t lo = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(at));
          const uint32_t hi = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(at >> 32)) & 0x7FFFFFFFu;
          const char* const base = pool + ((static_cast<uint64_t>(hi) << 32) | lo);
          constexpr uint32_t kBits = D == 128 ? 16u : 32u;
          if (blk < whole) {
#pragma unroll
            for (int i = 0; i < IPW; ++i) {
              // (rpart + (cpart ^ bits of i), made here)
              uint32_t off;
              const uint32_t x = kBits * (D == 128 ? i & 3 : i & 1);
              asm("v_xad_u32 %0, %1, %2, %3" : "=v"(off) : "v"(cpart), "n"(x), "v"(rpart), "s"(blk));
              dma16_sv(base + static_cast<uint32_t>(i * RPI) * slot_b, off, lds0 + slot * BLKB + i * 1024);
            }
          } else {  // The last block: rows behind the last key repeat its row (no row sees them, but 0 times NaN is NaN).
            const int there = end - 16 * (2 * (b0 + n - 1) + row0w / 16), most = there >= 16 ? 15 : (end - 1) & 15;
#pragma unroll
            for (int i = 0; i < IPW; ++i) {
              int t = threadIdx.x;
              asm("" : "+v"(t) : "s"(blk));
              const uint32_t row = static_cast<uint32_t>(min(row0w % 16 + i * RPI + (t & 63) / CPR, most));
              dma16_sv(base, row * slot_b + (cpart ^ (kBits * (D == 128 ? i & 3 : i & 1))), lds0 + slot * BLKB + i * 1024);
            }
          }
          look_up(blk + 1);
        };
        // Masked blocks: the keys that the lane's row sees, and those that are there
        // at all.
        uint32_t vis = ~0u, there = ~0u;
        int sees = 0;  // (of masked blocks) keys that the lane's row sees
        int hm = h;  // (h again: what is computed from it here stays here)
        auto mask_block = [&](f32x16& sc, int j) __attribute__((always_inline)) {
          auto below = [](int x) { return x >= 32 ? ~0u : x > 0 ? (1u << x) - 1u : 0u; };
          const int k0 = 32 * (b0 + j);
          const int e0 = __builtin_amdgcn_readfirstlane(static_cast<int>(tab[2 * j] >> 32));
          const int e1 = __builtin_amdgcn_readfirstlane(static_cast<int>(tab[2 * j + 1] >> 32));
          there = below(end - k0) & ((e0 < 0 ? 0u : 0xFFFFu) | (e1 < 0 ? 0u : 0xFFFF0000u));
          vis = below(sees - k0) & there;
#pragma unroll
          for (int e = 0; e < 16; ++e) sc[e] = masked_score(sc[e], vis >> (4 * hm), 8 * (e >> 2) + (e & 3));
        };
        auto fix_v = [&]() __attribute__((always_inline)) {
          bool bad = false;
#pragma unroll
          for (int s2 = 0; s2 < 2; ++s2)
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const int e = 8 * s2 + 2 * k;
              const uint32_t b = there >> (8 * (e >> 2) + 4 * hm + (e & 3));
              const uint32_t keep = (b & 1 ? 0xFFFFu : 0u) | (b & 2 ? 0xFFFF0000u : 0u);
#pragma unroll
              for (int x = 0; x < NU; ++x) {
                vop[s2][x][k] &= keep;
                bad |= nonfinite2<T>(vop[s2][x][k]) != 0;
              }
            }
          if (!__any(bad)) return;
          constexpr uint32_t one = std::is_same<T, bf16_t>::value ? 0x3F80u : 0x3C00u;
          u32x4 see[2];
#pragma unroll
          for (int e = 0; e < 16; e += 2) {
            const uint32_t b = vis >> (8 * (e >> 2) + 4 * hm + (e & 3));
            see[e >> 3][(e & 7) >> 1] = (b & 1 ? one : 0u) | (b & 2 ? one << 16 : 0u);
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
              f = mfma_k16x32<T>(w, see[s2], f);
            }
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[x][e] += flag_value(f[e]);
          }
        };
        f32x16 sca, scb;  // S of the even / odd blocks
        // One block in the pipeline: on entry S(j) is in registers, K block j + 1 and V
        // block j in their slots, and (PREV) block j - 1's P and V operands in registers.
        auto full = [&](int j, auto S, auto prev) __attribute__((always_inline)) {
          constexpr int s0 = decltype(S)::value;
          f32x16& cur = (s0 & 1) ? scb : sca;
          f32x16& nxt = (s0 & 1) ? sca : scb;
          if (second) __builtin_amdgcn_s_setprio(s0 ? 2 : 0);
          const bool issue = j < n - A;
          if (issue) load_block(j + A + (k_wave ? 1 : 0), k_wave ? s0 : (s0 + NB - 1) % NB);
          if (active) {
            if (j >= jc) {  // (uniform) the chunk's own last blocks
              int hm = h;
              asm("" : "+v"(hm) : "s"(j));
              const int upto = min(pos + my_row(chunk_args(), seg).q + 1, end) - 32 * (b0 + j) - 4 * hm;
              const uint32_t keep = upto >= 32 ? ~0u : upto > 0 ? (1u << upto) - 1u : 0u;  // (of the lane's keys, from its first)
#pragma unroll
              for (int e = 0; e < 16; ++e) cur[e] = masked_score(cur[e], keep, 8 * (e >> 2) + (e & 3));
            }
            kread((s0 + 1) % NB, j);
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
            vread(s0, j);
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
        look_up(0);
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
        if (tid == 0 && b0 == blk0 && !safe) {  // (while they are on their way)
          work->next(chunk_args(), seg, work->seg[turn ^ 1]);
          work->bad[turn ^ 1] = INT32_MAX;
        }
        // K(0) and step 0. (Also the Q loads, which the compiler's own waits would
        // otherwise put into the loop.)
        if (n >= A) wait_vmcnt<kInFlight>();
        else wait_vmcnt<0>();
        lds_barrier();
        // ---- The blocks before jm, in the pipeline.
        const int n1 = min(n, jm);
        if (n1 > 0) {
          kread(0, b0);
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
        // ---- The others, one at a time: masks and what they need stay out of the
        // pipeline's registers.
        if (n1 < n) sees = min(pos + my_row(chunk_args(), seg).q + 1, end);
#pragma unroll 1
        for (int j = n1; j < n; ++j) {
          if (active) kread(j % NB, j);
          lds_barrier();  // step j + A overwrites K(j)'s slot and V(j - 1)'s
          const bool issue = j < n - A;
          if (issue) load_block(j + A + (k_wave ? 1 : 0), k_wave ? j % NB : (j + NB - 1) % NB);
          if (active) {
            asm volatile("" : "+v"(hm));
            qk(sca);
            mask_block(sca, j);
            rescale(block_max(sca));
            softmax_exp(sca);
            vread(j % NB, j);
            fix_v();
            pv();
          }
          if (issue) wait_vmcnt<kInFlight>();
          else wait_vmcnt<0>();
          lds_barrier();
        }
      }
      // (P's sum is 0 times NaN where an unseen key's V is; l tells of NaN scores)
      float finite[4] = {l * 0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int x = 0; x < NU; ++x)
#pragma unroll
        for (int e = 0; e < 16; ++e) finite[e & 3] = fmaf(acc[x][e], 0.f, finite[e & 3]);
      if (safe) break;
      if (active && (finite[0] + finite[1]) + (finite[2] + finite[3]) != 0.f) work->redo = 1;
      lds_barrier();
      if (of(work->redo) == 0) break;
      }
      ask(work->seg[turn ^ 1]);
      // ---- What the segment gives: the item's rows, or a partial result.
      l += __builtin_bit_cast(float, xor_lane32<32>(__builtin_bit_cast(uint32_t, l), lane));
      const ChunkArgs& o = chunk_args();
      int he = h;
      asm volatile("" : "+v"(he));
      if (blk0 == 0 && blk1 == of(seg.nblk)) {
        const Row row = my_row(o, seg);
        if (active && row.ok) {
          T* const out = static_cast<T*>(o.out) + row.at * o.o_sr + row.head * o.o_sh;
          const int64_t o_sd = o.o_sd;
          const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
          for (int x = 0; x < NU; ++x)
#pragma unroll
            for (int e = 0; e < 16; e += 4) {
              const int d = 32 * x + 8 * (e >> 2) + 4 * he;
              u32x2 w = {pack2<T>(acc[x][e] * inv, acc[x][e + 1] * inv), pack2<T>(acc[x][e + 2] * inv, acc[x][e + 3] * inv)};
              if (l == 0.f) w = u32x2{0, 0};
              if (o.out8) {
                *reinterpret_cast<u32x2*>(out + d) = w;
              } else {
                uint16_t* const o16 = reinterpret_cast<uint16_t*>(out);
#pragma unroll
                for (int i = 0; i < 4; ++i) o16[(d + i) * o_sd] = static_cast<uint16_t>(w[i >> 1] >> (16 * (i & 1)));
              }
            }
        }
      } else {
        // Slot 0: of the item that the run starts inside of; 1: of the one it starts.
        float* const slot = o.part + (2 * static_cast<int64_t>(of(work->run)) + (blk0 == 0 ? 1 : 0)) * chunk_part_floats(D, NW);
        if (active && my_row(o, seg).ok) {
#pragma unroll
          for (int x = 0; x < NU; ++x)
#pragma unroll
            for (int e = 0; e < 16; e += 4)
              *reinterpret_cast<f32x4*>(slot + 4 * ((wave * (4 * NU) + 4 * x + (e >> 2)) * 64 + lane)) =
                  f32x4{acc[x][e], acc[x][e + 1], acc[x][e + 2], acc[x][e + 3]};
          if (h == 0) *reinterpret_cast<f32x2*>(slot + 32 * NW * D + 2 * (32 * wave + c)) = f32x2{m, l};
        }
        if (blk0 > 0 && tid == 0) o.splits[work->run] = work->split(seg);
      }
    }
  }
}

// The partial results of an item that a cut goes through, put together, the reads of
// four runs' in flight at once (32 runs an item 21 -> 11.5 us, two 13 -> 11; eight at once
// by four times the threads: 12.3 and 12 to 14). slot(k): the k-th of n; row: the
// thread's, whose maximum and sum are behind the slot's first `sums` floats; at(i): its
// i-th four floats.
template <int NU, typename S, typename F>
__device__ __forceinline__ float chunk_join(int n, int sums, int row, S slot, F at, f32x4 (&o)[NU]) {
  float M = kChunkNone, den = 0.f;
#pragma unroll
  for (int i = 0; i < NU; ++i) o[i] = f32x4{0.f, 0.f, 0.f, 0.f};
  auto some = [&](int k0, auto K) __attribute__((always_inline)) {
    f32x4 v[K][NU];
    f32x2 ml[K];
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const float* const p = slot(k0 + k);
      ml[k] = *reinterpret_cast<const f32x2*>(p + sums + 2 * row);
#pragma unroll
      for (int i = 0; i < NU; ++i) v[k][i] = *reinterpret_cast<const f32x4*>(p + at(i));
    }
    __builtin_amdgcn_sched_barrier(0);
    float mn = M;
#pragma unroll
    for (int k = 0; k < K; ++k) mn = fmaxf(mn, ml[k][0]);
    const float c_old = fast_exp2(M - mn);
    den *= c_old;
#pragma unroll
    for (int i = 0; i < NU; ++i)
#pragma unroll
      for (int x = 0; x < 4; ++x) o[i][x] *= c_old;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const float f = fast_exp2(ml[k][0] - mn);
      den = fmaf(ml[k][1], f, den);
#pragma unroll
      for (int i = 0; i < NU; ++i)
#pragma unroll
        for (int x = 0; x < 4; ++x) o[i][x] = fmaf(v[k][i][x], f, o[i][x]);
    }
    M = mn;
  };
  int k = 0;
  for (; k + 4 <= n; k += 4) some(k, std::integral_constant<int, 4>{});
  if (n - k == 3) some(k, std::integral_constant<int, 3>{});
  if (n - k == 2) some(k, std::integral_constant<int, 2>{});
  if (n - k == 1) some(k, std::integral_constant<int, 1>{});
  return den;
}

// Items that a cut goes through: the first run that starts inside of one, a wave's rows
// a workgroup.
template <typename T, int D, int NW>
__global__ __launch_bounds__(256) void paged_chunk_merge(ChunkArgs a) {
  constexpr int NU = D / 32;
  const int run = static_cast<int>(blockIdx.x) + 1, wave = blockIdx.y;
  if (run >= *a.runs) return;
  const ChunkSplit sp = a.splits[run];
  const float* __restrict__ const part = a.part;
  if (sp.runs == 0 || 32 * wave >= sp.queries * a.G) return;
  const int lane = threadIdx.x & 63, h = lane >> 5, c = lane & 31, rw = 32 * wave + c, rq = (rw * a.g_mul) >> 16;
  if (rq >= sp.queries) return;
  f32x4 o[NU];
  const float den = chunk_join<NU>(
      sp.runs + 1, 32 * NW * D, rw,
      [&](int k) { return part + (2 * static_cast<int64_t>(run + k - 1) + (k == 0 ? 1 : 0)) * chunk_part_floats(D, NW); },
      [&](int i) { return 4 * ((wave * (4 * NU) + (threadIdx.x >> 6) + 4 * i) * 64 + lane); }, o);
  T* const out = static_cast<T*>(a.out) + (sp.row0 + rq) * a.o_sr + (sp.kvh * a.G + rw - rq * a.G) * a.o_sh;
  const float inv = den == 0.f ? 0.f : 1.f / den;
#pragma unroll
  for (int i = 0; i < NU; ++i) {
    const int d = 32 * i + 8 * (threadIdx.x >> 6) + 4 * h;
    u32x2 w = {pack2<T>(o[i][0] * inv, o[i][1] * inv), pack2<T>(o[i][2] * inv, o[i][3] * inv)};
    if (den == 0.f) w = u32x2{0, 0};
    if (a.out8) {
      *reinterpret_cast<u32x2*>(out + d) = w;
    } else {
      uint16_t* const o16 = reinterpret_cast<uint16_t*>(out);
#pragma unroll
      for (int x = 0; x < 4; ++x) o16[(d + x) * a.o_sd] = static_cast<uint16_t>(w[x >> 1] >> (16 * (x & 1)));
    }
  }
}

}  // namespace tsa
