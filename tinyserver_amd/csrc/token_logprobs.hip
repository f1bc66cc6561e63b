// Log probabilities of given tokens, with the entropy of their distribution and the
// most likely alternatives (tsa_token_logprobs).
//
// For a row x of V logits with m = max x, t_i = x_i - m <= 0, S = sum exp(t_i) and
// E = sum exp(t_i) t_i:
//   log p_i = t_i - ln S,   H = -sum p_i ln p_i = ln S - E / S
// (both terms of H are non-negative: nothing cancels). The sums are taken relative to the
// largest logit that the wave has met, and end relative to m itself: S is at least 1 and
// E at most 0 however they round, so no log p is above 0 and no H below. A logit of -inf
// has p = 0 and adds nothing; a NaN, a +inf or a row of nothing but -inf makes S NaN,
// and with it the row's results.
//
// One read of the logits; what bounds it: for many rows the vector units, with 7.5
// operations and an exponential a logit (89% busy in 16 bits, 4,096 rows of 151,936 at
// 5.0 to 6.0 TB/s; 40% in float32, where it is HBM), and for a few the chain load -> sums
// -> threshold -> candidates -> rank.
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
  int32_t per_group, parts;  // tiles of a group; parts that rows are cut into
  bool tok64;
};

constexpr int kMaxTop = 64;
constexpr int kThreads = 256;
constexpr int64_t kWholeRows = 512;  // rows of a call from which on none is cut

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

// What sorts in the other order than its bits: rank_of's value.
__device__ __forceinline__ float value_of(uint64_t rank) {
  uint32_t b = static_cast<uint32_t>(rank >> 32);
  if (b == 0) return __builtin_nanf("");
  return __uint_as_float(b & 0x80000000u ? b ^ 0x80000000u : ~b);
}

// The k-th largest (k from 1) of the wave's 64 numbers: a bitonic sort over the
// lanes, the largest in lane 0.
template <int J>
__device__ __forceinline__ void sort_step(uint64_t& x, int lane, bool down) {
  const uint64_t o = xor_lane64<J>(x, lane);
  x = ((lane & J) == 0) == down ? (o > x ? o : x) : (o < x ? o : x);
}
__device__ __forceinline__ uint64_t wave_kth(uint64_t x, int k, int lane) {
  sort_step<1>(x, lane, !(lane & 2));
  sort_step<2>(x, lane, !(lane & 4)); sort_step<1>(x, lane, !(lane & 4));
  sort_step<4>(x, lane, !(lane & 8)); sort_step<2>(x, lane, !(lane & 8)); sort_step<1>(x, lane, !(lane & 8));
  sort_step<8>(x, lane, !(lane & 16)); sort_step<4>(x, lane, !(lane & 16)); sort_step<2>(x, lane, !(lane & 16));
  sort_step<1>(x, lane, !(lane & 16));
  sort_step<16>(x, lane, !(lane & 32)); sort_step<8>(x, lane, !(lane & 32)); sort_step<4>(x, lane, !(lane & 32));
  sort_step<2>(x, lane, !(lane & 32)); sort_step<1>(x, lane, !(lane & 32));
  sort_step<32>(x, lane, true); sort_step<16>(x, lane, true); sort_step<8>(x, lane, true);
  sort_step<4>(x, lane, true); sort_step<2>(x, lane, true); sort_step<1>(x, lane, true);
  const uint32_t lo = __builtin_amdgcn_readlane(static_cast<int>(x), k - 1);
  const uint32_t hi = __builtin_amdgcn_readlane(static_cast<int>(x >> 32), k - 1);
  return (static_cast<uint64_t>(hi) << 32) | lo;
}

// The candidates of a row, in LDS.
constexpr int kCand = 1024, kWork = 8 * kMaxTop + 64;
struct Candidates {
  uint64_t list[kCand];
  uint64_t fours[64];  // the largest of four lanes
  int count, reach;
  int work[kWork];     // groups of tiles to read again: group << 8 | thread
};
// The k-th largest of the 64 groups' largest, where each thread gives the largest of
// its part: at least k of all the numbers reach it. All threads call.
__device__ __forceinline__ uint64_t group_kth(Candidates& c, uint64_t mine, int k) {
  const int lane = threadIdx.x & 63;
  uint64_t o = xor_lane64<1>(mine, lane);
  mine = o > mine ? o : mine;
  o = xor_lane64<2>(mine, lane);
  mine = o > mine ? o : mine;
  __syncthreads();
  if ((lane & 3) == 0) c.fours[threadIdx.x >> 2] = mine;
  __syncthreads();
  return wave_kth(c.fours[lane], k, lane);
}
// Leaves out candidates that k others are larger than, while more than `most` are left
// (no two are alike, so each round leaves out one at least). All threads call.
__device__ __forceinline__ uint64_t prune(Candidates& c, int k, int most, uint64_t floor) {
  constexpr int kPer = kCand / kThreads;
  while (true) {
    __syncthreads();
    const int n = c.count;
    if (n <= most) return floor;
    uint64_t x[kPer], top = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int at = static_cast<int>(threadIdx.x) + i * kThreads;
      x[i] = at < n ? c.list[at] : 0;
      top = x[i] > top ? x[i] : top;
    }
    const uint64_t t = group_kth(c, top, k);
    floor = t > floor ? t : floor;
    __syncthreads();
    if (threadIdx.x == 0) c.count = 0;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kPer; ++i)
      if (x[i] != 0 && x[i] >= floor) c.list[atomicAdd(&c.count, 1)] = x[i];
  }
}
// The k largest candidates in order, write(place, number); places past the last
// candidate get 0.
template <typename F>
__device__ __forceinline__ void write_top(Candidates& c, int k, F write) {
  prune(c, k, kThreads, 0);
  __syncthreads();
  const int n = c.count, tid = threadIdx.x;
  if (tid < n) {
    const uint64_t x = c.list[tid];
    int place = 0;
#pragma unroll 8
    for (int i = 0; i < n; ++i) place += c.list[i] > x;
    if (place < k) write(place, x);
  }
  if (tid >= n && tid < k) write(tid, uint64_t{0});
}

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr float kNoMax = -3.402823466e38f;  // the reference of no logit

// Sums over logits x, relative to the largest of them, m: s = sum 2^y, e = sum 2^y y, y
// = (x - m) log2 e.
struct Sums {
  float m, s, e;
  __device__ __forceinline__ void move(float to) {
    const float d = fmaxf((m - to) * kLog2e, -1e30f), f = fast_exp2(d);
    e = f * fmaf(d, s, e);
    s *= f;
    m = to;
  }
  // (a logit of -inf adds 0; a NaN, or an infinity's inf - inf, makes s NaN)
  __device__ __forceinline__ void add(float x) {
    const float y = (x - m) * kLog2e, p = fast_exp2(y);
    s += p;
    e = fmaf(p, fmaxf(y, -1e30f), e);
  }
  __device__ __forceinline__ void join(const Sums& o) {
    Sums b = o;
    const float to = fmaxf(m, o.m);
    move(to);
    b.move(to);
    s += b.s;
    e += b.e;
  }
};
__device__ __forceinline__ Sums wave_sums(Sums v) {
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) {
    Sums o;
    o.m = __shfl_xor(v.m, off, 64);
    o.s = __shfl_xor(v.s, off, 64);
    o.e = __shfl_xor(v.e, off, 64);
    v.join(o);
  }
  // (Lanes round their joins in different orders; a row's results are written by threads
  // that the order of an atomic chooses.)
  auto first = [](float x) { return __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(x))); };
  return Sums{first(v.m), first(v.s), first(v.e)};
}
__device__ __forceinline__ Sums block_sums(Sums v, Sums* waves) {
  v = wave_sums(v);
  if ((threadIdx.x & 63) == 0) waves[threadIdx.x >> 6] = v;
  __syncthreads();
  v = waves[0];
#pragma unroll
  for (int w = 1; w < kThreads / 64; ++w) v.join(waves[w]);
  return v;
}

// The largest of the wave's numbers.
__device__ __forceinline__ float wave_max(float x) {
  const int lane = threadIdx.x & 63;
  auto step = [&](auto J) { x = fmaxf(x, __uint_as_float(xor_lane32<decltype(J)::value>(__float_as_uint(x), lane))); };
  step(std::integral_constant<int, 1>{});
  step(std::integral_constant<int, 2>{});
  step(std::integral_constant<int, 4>{});
  step(std::integral_constant<int, 8>{});
  step(std::integral_constant<int, 16>{});
  step(std::integral_constant<int, 32>{});
  return __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(x)));
}

// 16 bytes of logits.
template <typename T> struct Piece;
template <> struct Piece<float> {
  static constexpr int n = 4;
  static constexpr uint32_t none = 0xFF800000u;
  static __device__ __forceinline__ float at(const u32x4& v, int i) { return __uint_as_float(v[i]); }
};
template <> struct Piece<bf16_t> {
  static constexpr int n = 8;
  static constexpr uint32_t none = 0xFF80FF80u;
  static __device__ __forceinline__ float at(const u32x4& v, int i) { return i & 1 ? hi_f<bf16_t>(v[i >> 1]) : lo_f<bf16_t>(v[i >> 1]); }
};
template <> struct Piece<f16_t> {
  static constexpr int n = 8;
  static constexpr uint32_t none = 0xFC00FC00u;
  static __device__ __forceinline__ float at(const u32x4& v, int i) { return i & 1 ? hi_f<f16_t>(v[i >> 1]) : lo_f<f16_t>(v[i >> 1]); }
};

constexpr int kUnroll = 8;   // pieces of a thread in flight: a tile is 256 x 8 pieces
constexpr int kGroups = 12;  // runs of tiles of a row, of which each thread keeps its largest logit
constexpr int kTilePieces = kThreads * kUnroll;

// A row: `head` logits before the first 16-byte boundary, whole pieces, `tail` behind
// them. Thread i has the i-th of the head, thread 32 + i that of the tail (the edges).
template <typename T>
struct Row {
  typedef Piece<T> PT;
  static constexpr int VE = PT::n;
  const T* x;
  const T* body;
  int V, head, pieces, tail, tiles;
  __device__ __forceinline__ Row(const LogprobArgs& a, int64_t row) {
    x = static_cast<const T*>(a.x) + row * a.x_s0;
    V = a.V;
    head = min(V, static_cast<int>((16 - reinterpret_cast<uintptr_t>(x) % 16) % 16 / sizeof(T)));
    body = x + head;
    pieces = (V - head) / VE;
    tail = V - head - pieces * VE;
    tiles = (pieces + kTilePieces - 1) / kTilePieces;
  }
  __device__ __forceinline__ int edge() const {  // the thread's, -1: none
    const int t = threadIdx.x;
    return t < head ? t : t >= 32 && t - 32 < tail ? V - tail + t - 32 : -1;
  }
  // A tile's pieces of this thread; those past the row's are of -inf.
  __device__ __forceinline__ void load(int t, u32x4 (&w)[kUnroll]) const {
    const u32x4* const p = reinterpret_cast<const u32x4*>(body);
    const int p0 = t * kTilePieces + static_cast<int>(threadIdx.x);
    if ((t + 1) * kTilePieces <= pieces) {
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) w[u] = __builtin_nontemporal_load(p + p0 + u * kThreads);
    } else {
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        w[u] = u32x4{PT::none, PT::none, PT::none, PT::none};
        if (p0 + u * kThreads < pieces) w[u] = p[p0 + u * kThreads];
      }
    }
  }
  // Sums over tiles t .. end - 1; the thread's largest of them. A piece is summed by
  // itself, then a tile, then all. All lanes of a wave have one reference, which moves
  // at a new largest logit, a few times a row. (4,096 rows of 151,936: log probabilities
  // and entropies off by at most 1.2e-6 and 1.5e-6; with one float32 sum over a thread's
  // 600 logits 6.2e-6 and 5.8e-6; with references of the lanes' own that a logit may pass
  // by 16, whose offsets then cancel, 2.5e-6 and 7.9e-6, and 231 us, not 217.)
  __device__ __forceinline__ float sum(Sums& v, int t, int end) const {
    float gm = -INFINITY;
    for (; t < end; ++t) {
      u32x4 w[kUnroll];
      load(t, w);
      Sums tile{v.m, 0.f, 0.f};
      // (a piece at a time: its logits as floats, a few registers, serve both loops)
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        float mx = -INFINITY;
#pragma unroll
        for (int i = 0; i < VE; i += 2) mx = fmaxf(fmaxf(mx, PT::at(w[u], i)), PT::at(w[u], i + 1));
        if (__any(mx > tile.m)) tile.move(wave_max(mx));
        gm = fmaxf(gm, mx);
        Sums piece{tile.m, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < VE; ++i) piece.add(PT::at(w[u], i));
        tile.s += piece.s;
        tile.e += piece.e;
      }
      if (tile.m > v.m) v.move(tile.m);
      v.s += tile.s;
      v.e += tile.e;
    }
    return gm;
  }
  __device__ __forceinline__ void sum_edge(Sums& v) const {
    const int e = edge();
    if (e < 0) return;
    const float xe = to_float(x[e]);
    if (xe > v.m) v.move(xe);
    v.add(xe);
  }
};

// The candidates of a row's `top` largest logits. The top-th largest of 64 groups'
// largest is a threshold that at least `top` logits reach and few others (about 24 for
// 20 where their places are random), and threads with a group of tiles (group_max[g],
// tiles per g) that reaches it read that again. More than kCand of them: those above
// the threshold and the lowest of those that tie with it, or else all of them a wave's
// piece at a time, under a floor that rises. All threads call.
template <typename T>
__device__ __forceinline__ void candidates(const Row<T>& r, int top, int per, const float (&group_max)[kGroups][kThreads],
                                           Candidates& c) {
  typedef Piece<T> PT;
  constexpr int VE = PT::n;
  const int tid = threadIdx.x, groups = (r.tiles + per - 1) / per, edge = r.edge();
  const float at_edge = edge >= 0 ? to_float(r.x[edge]) : -INFINITY;
  float largest = at_edge;
  for (int g = 0; g < groups; ++g) largest = fmaxf(largest, group_max[g][tid]);
  const float threshold = value_of(group_kth(c, rank_of(fmaxf(largest, -INFINITY), 0xFFFFFFFFu), top));
  auto append = [&](uint64_t rank) __attribute__((always_inline)) {
    const int at = atomicAdd(&c.count, 1);
    if (at < kCand) c.list[at] = rank;
  };
  // The logits that reach the threshold, from the groups that do (whole pieces at
  // once); `above`: those past it. False: there are too many. (Of 64 groups, about
  // -64 ln(1 - top / 64) threads' groups reach it; all do where it is a mask's value.)
  const int most = r.V <= kCand ? kThreads : min(min(8 * top + 64, kWork), groups * kThreads - 1);
  auto gather = [&](bool above) {
    auto in = [&](float x) { return above ? x > threshold : !(x < threshold); };  // (a NaN reaches any, and passes none)
    __syncthreads();
    if (tid == 0) c.count = c.reach = 0;
    __syncthreads();
    for (int g = 0; g < groups; ++g) {
      if (!in(group_max[g][tid])) continue;
      const int at = atomicAdd(&c.reach, 1);
      if (at < kWork) c.work[at] = g << 8 | tid;
    }
    __syncthreads();
    if (c.reach > most) return false;
    if (edge >= 0 && in(at_edge)) append(rank_of(at_edge, edge));
    // (a piece a thread: they are all in flight at once)
    const int reads = c.reach * per * kUnroll;
    for (int i = tid; i < reads; i += kThreads) {
      const int w = c.work[i / (per * kUnroll)], u = i % (per * kUnroll);
      const int p = (w >> 8) * per * kTilePieces + u * kThreads + (w & 255);
      if (p >= r.pieces) continue;
      const u32x4 v = reinterpret_cast<const u32x4*>(r.body)[p];
#pragma unroll
      for (int e = 0; e < VE; ++e)
        if (in(PT::at(v, e))) append(rank_of(PT::at(v, e), r.head + p * VE + e));
    }
    __syncthreads();
    return c.count <= kCand;
  };
  if (gather(false)) return;
  if (gather(true)) {
    // Many tie at the threshold (a mask's value, with fewer tokens allowed than asked
    // for): those of them among the row's first logits are the lowest.
    __syncthreads();  // (every wave has read the count)
    if (tid < min(r.V, 2 * top + 16) && to_float(r.x[tid]) == threshold) append(rank_of(threshold, tid));
    __syncthreads();
    if (c.count >= top && c.count <= kCand) return;
  }
  uint64_t floor = 0;
  __syncthreads();
  if (tid == 0) c.count = 0;
  __syncthreads();
  if (edge >= 0) append(rank_of(at_edge, edge));
#pragma unroll 1
  for (int y = 0; y < r.tiles; ++y) {
    // (the largest that this thread's logits of the tile can be)
    const bool may = floor == 0 || rank_of(group_max[y / per][tid], r.head + y * kTilePieces * VE) > floor;
    if (!__syncthreads_or(may)) continue;
#pragma unroll 1
    for (int i = 0; i < kUnroll * (kThreads / 64); ++i) {
      const int p = y * kTilePieces + (i >> 2) * kThreads + tid;
      floor = prune(c, top, kCand - 64 * VE, floor);
      __syncthreads();  // (every wave has read the count that prune left)
      if (may && tid >> 6 == (i & 3) && p < r.pieces) {
#pragma unroll 1
        for (int e = 0; e < VE; ++e) {
          const uint64_t rank = rank_of(to_float(r.body[p * VE + e]), r.head + p * VE + e);
          if (rank > floor) append(rank);
        }
      }
    }
  }
  __syncthreads();
}

// A row's results from its sums and the candidates of its largest logits.
template <typename T>
__device__ __forceinline__ void write_row(const LogprobArgs& a, int64_t row, const T* x, Sums v, Candidates& c) {
  const float s = v.s == 0.f ? __builtin_nanf("") : v.s, lse = logf(s);  // (nothing but -inf: no distribution)
  if (threadIdx.x == 0) {
    const int64_t t = token_of(a, row);
    a.logp[row * a.lp_s] = ((t >= 0 && t < a.V ? to_float(x[t]) : -INFINITY) - v.m) - lse;
    a.entropy[row * a.en_s] = lse - kLn2 * (v.e / s);
  }
  if (a.top > 0)
    write_top(c, a.top, [&](int place, uint64_t rank) {
      a.top_tok[row * a.tt_s0 + place * a.tt_s1] = index_of(rank);
      a.top_logp[row * a.tl_s0 + place * a.tl_s1] = (value_of(rank) - v.m) - lse;
    });
}

// A workgroup a row.
template <typename T>
__global__ __launch_bounds__(kThreads) __attribute__((amdgpu_waves_per_eu(6))) void token_logprobs_stream(LogprobArgs a) {
  __shared__ Candidates c;
  __shared__ float group_max[kGroups][kThreads];
  __shared__ Sums waves[kThreads / 64];
  for (int64_t row = blockIdx.x; row < a.N; row += gridDim.x) {
    const Row<T> r(a, row);
    Sums v{kNoMax, 0.f, 0.f};
    for (int g = 0; g * a.per_group < r.tiles; ++g)
      group_max[g][threadIdx.x] = r.sum(v, g * a.per_group, min((g + 1) * a.per_group, r.tiles));
    r.sum_edge(v);
    if (a.top > 0) candidates<T>(r, a.top, a.per_group, group_max, c);
    v = block_sums(v, waves);
    write_row<T>(a, row, r.x, v, c);
    __syncthreads();
  }
}

// Few rows: a workgroup a group of a row's tiles, whose sums and threads' largest go
// to the workspace, then one a row for the rest. The choice of the alternatives once a
// row, and not once a part of it, is what keeps the second launch short (64 rows of
// 151936, 20 alternatives: 17.2 + 6.6 us with each part's own 20).
__host__ __device__ constexpr int part_words(int top) { return 4 + (top > 0 ? kThreads : 0); }

template <typename T>
__global__ __launch_bounds__(kThreads) __attribute__((amdgpu_waves_per_eu(6))) void token_logprobs_parts(
    LogprobArgs a, float* __restrict__ part) {
  __shared__ Sums waves[kThreads / 64];
  const int64_t items = a.N * a.parts;
  for (int64_t item = blockIdx.x; item < items; item += gridDim.x) {
    const int64_t row = item / a.parts;
    const int g = static_cast<int>(item - row * a.parts);
    const Row<T> r(a, row);
    Sums v{kNoMax, 0.f, 0.f};
    const float gm = r.sum(v, g * a.per_group, min((g + 1) * a.per_group, r.tiles));
    if (g == 0) r.sum_edge(v);
    float* const out = part + item * part_words(a.top);
    if (a.top > 0) out[4 + threadIdx.x] = gm;
    v = block_sums(v, waves);
    if (threadIdx.x == 0) *reinterpret_cast<f32x4*>(out) = f32x4{v.m, v.s, v.e, 0.f};
    __syncthreads();
  }
}

template <typename T>
__global__ __launch_bounds__(kThreads) void token_logprobs_join(LogprobArgs a, const float* __restrict__ part) {
  __shared__ Candidates c;
  __shared__ float group_max[kGroups][kThreads];
  for (int64_t row = blockIdx.x; row < a.N; row += gridDim.x) {
    const Row<T> r(a, row);
    const float* const mine = part + row * a.parts * part_words(a.top);
    Sums v{kNoMax, 0.f, 0.f};  // (a part a lane, the same in every wave)
    const int lane = threadIdx.x & 63;
    if (lane < a.parts) {
      const f32x4 p = *reinterpret_cast<const f32x4*>(mine + lane * part_words(a.top));
      v = Sums{p[0], p[1], p[2]};
    }
    if (a.top > 0) {
      float gm[kGroups];
#pragma unroll
      for (int g = 0; g < kGroups; ++g)
        gm[g] = g < a.parts ? mine[g * part_words(a.top) + 4 + threadIdx.x] : -INFINITY;
#pragma unroll
      for (int g = 0; g < kGroups; ++g) group_max[g][threadIdx.x] = gm[g];
    }
    v = wave_sums(v);
    if (a.top > 0) candidates<T>(r, a.top, a.per_group, group_max, c);
    write_row<T>(a, row, r.x, v, c);
    __syncthreads();
  }
}

// Tiles of a group, and the parts that rows are cut into (1: none).
struct RowCut {
  int per_group, parts;
};
static RowCut cut_rows(int64_t N, int64_t V, int elem_bytes) {
  const int64_t tiles = (V * elem_bytes / 16 + kTilePieces - 1) / kTilePieces;
  const int64_t per = tiles > kGroups ? (tiles + kGroups - 1) / kGroups : 1, groups = (tiles + per - 1) / per;
  return RowCut{static_cast<int>(per), static_cast<int>(N < kWholeRows && groups > 1 ? groups : 1)};
}
static size_t cut_bytes(int64_t N, const RowCut& r, int64_t top) {
  return r.parts > 1 ? sizeof(float) * static_cast<size_t>(N) * r.parts * part_words(static_cast<int>(top)) : 0;
}

template <typename T>
static int launch_stream(LogprobArgs& a, const RowCut& r, void* workspace, hipStream_t stream) {
  a.per_group = r.per_group;
  a.parts = r.parts;
  auto grid = [](int64_t n) { return dim3(static_cast<uint32_t>(n < (1 << 22) ? n : 1 << 22)); };
  if (r.parts == 1) {
    token_logprobs_stream<T><<<grid(a.N), dim3(kThreads), 0, stream>>>(a);
    return check_launch("tsa_token_logprobs");
  }
  float* const part = static_cast<float*>(workspace);
  token_logprobs_parts<T><<<grid(a.N * r.parts), dim3(kThreads), 0, stream>>>(a, part);
  if (int rc = check_launch("tsa_token_logprobs")) return rc;
  token_logprobs_join<T><<<grid(a.N), dim3(kThreads), 0, stream>>>(a, part);
  return check_launch("tsa_token_logprobs");
}

// Logits that do not lie side by side: a workgroup a row, the row read for the maximum,
// the sums and each alternative.
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
  const hipStream_t st = static_cast<hipStream_t>(stream);
  if (a.x_s1 == 1 || V == 1) {
    a.x_s1 = 1;
    const RowCut r = cut_rows(N, V, dtype_bytes(logits->dtype));
    const size_t need = cut_bytes(N, r, top);
    TSA_REQUIRE(need == 0 || (workspace != nullptr && workspace_bytes >= need),
                "workspace of %zu bytes is too small: %zu needed", workspace_bytes, need);
    TSA_REQUIRE(need == 0 || reinterpret_cast<uintptr_t>(workspace) % 256 == 0, "workspace must be 256-byte aligned");
    switch (logits->dtype) {
      case TSA_BF16: return launch_stream<bf16_t>(a, r, workspace, st);
      case TSA_F16: return launch_stream<f16_t>(a, r, workspace, st);
      default: return launch_stream<float>(a, r, workspace, st);
    }
  }
  switch (logits->dtype) {
    case TSA_BF16: return launch_rows<bf16_t>(a, st);
    case TSA_F16: return launch_rows<f16_t>(a, st);
    default: return launch_rows<float>(a, st);
  }
}

extern "C" size_t tsa_token_logprobs_workspace_bytes(int64_t num_tokens, int64_t vocab_size, int64_t num_top) {
  if (num_tokens <= 0 || vocab_size <= 0 || vocab_size >= (int64_t{1} << 30) || num_top < 0 || num_top > kMaxTop)
    return 0;  // (calls of such sizes are refused, or have nothing to do)
  size_t most = 0;
  for (const int bytes : {2, 4}) {
    const size_t n = cut_bytes(num_tokens, cut_rows(num_tokens, vocab_size, bytes), num_top);
    most = n > most ? n : most;
  }
  return most;
}
