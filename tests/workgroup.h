// A kernel's workgroups on the CPU, one after the other: a fibre a thread, waves of
// 64. Barriers and cross-lane operations are where fibres stop; between two barriers
// each wave runs as far as it can before the next one starts, the one named by
// wg_order first, so a value that a wave reads behind a barrier and another one
// changes before the next barrier differs from wave to wave. Waves that wait at
// different barriers are an error (wg_error), not a hang.
#pragma once

#include <sys/mman.h>
#include <ucontext.h>

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <functional>
#include <vector>

#define __device__
#define __host__
#define __global__
#define __shared__ static
#define __forceinline__ inline
#define __launch_bounds__(...)
#define amdgpu_waves_per_eu(...) unused
#define __syncthreads() wg::block_wait(__LINE__, false)
#define __syncthreads_or(x) wg::block_wait(__LINE__, (x) != 0)
#define __builtin_amdgcn_readlane(v, l) wg::from_lane(static_cast<int>(v), l)
#define __builtin_amdgcn_readfirstlane(v) wg::from_lane(static_cast<int>(v), 0)
#define __any(x) wg::any_lane(x)
#define __shfl_xor(v, off, n) wg::from_lane(v, (threadIdx.x & 63) ^ (off))

struct dim3 {
  uint32_t x, y, z;
  dim3(uint32_t x_ = 1, uint32_t y_ = 1, uint32_t z_ = 1) : x(x_), y(y_), z(z_) {}
};
typedef void* hipStream_t;
typedef int hipError_t;
constexpr hipError_t hipSuccess = 0;
inline hipError_t hipGetLastError() { return hipSuccess; }
inline const char* hipGetErrorString(hipError_t) { return ""; }

static dim3 threadIdx, blockIdx, gridDim, blockDim;
using std::max;
using std::min;
inline uint32_t __float_as_uint(float x) { return __builtin_bit_cast(uint32_t, x); }
inline float __uint_as_float(uint32_t x) { return __builtin_bit_cast(float, x); }
inline int atomicAdd(int* p, int v) {
  const int old = *p;
  *p += v;
  return old;
}

namespace wg {
enum State { kReady, kAtWave, kAtBlock, kDone };
struct Fibre {
  ucontext_t ctx;
  State state;
  int site;
  bool flag;
};
constexpr int kMost = 1024;
constexpr size_t kStack = 256 << 10;
static Fibre fibres[kMost];
static char* stacks;
static ucontext_t home;
static int current, threads, order;
static bool any;
static char error[256];
static std::function<void()> body;
static uint64_t slots[2][kMost];
static int turn[kMost];

inline void stop(State s, int site) {
  Fibre& f = fibres[current];
  f.state = s;
  f.site = site;
  const int me = current;
  swapcontext(&f.ctx, &home);
  current = me;
  threadIdx.x = me;
}
inline bool block_wait(int site, bool flag) {
  fibres[current].flag = flag;
  stop(kAtBlock, site);
  return any;
}
template <typename T>
inline T from_lane(T v, int lane) {
  const int me = current, t = turn[me] ^= 1;
  std::memcpy(&slots[t][me], &v, sizeof(T));
  stop(kAtWave, 0);
  T r;
  std::memcpy(&r, &slots[t][(me & ~63) + lane], sizeof(T));
  return r;
}
inline bool any_lane(bool x) {
  const int me = current, t = turn[me] ^= 1;
  slots[t][me] = x;
  stop(kAtWave, 0);
  bool r = false;
  for (int l = 0; l < 64; ++l) r |= slots[t][(me & ~63) + l] != 0;
  return r;
}
inline void enter() {
  body();
  fibres[current].state = kDone;
  swapcontext(&fibres[current].ctx, &home);
}
// The wave's fibres, until all are at a block's barrier or done.
inline bool run_wave(int w) {
  const int t0 = 64 * w, t1 = std::min(t0 + 64, threads);
  while (true) {
    for (int t = t0; t < t1; ++t)
      if (fibres[t].state == kReady) {
        current = t;
        threadIdx.x = t;
        swapcontext(&home, &fibres[t].ctx);
      }
    int waiting = 0;
    for (int t = t0; t < t1; ++t) waiting += fibres[t].state == kAtWave;
    if (waiting == 0) return true;
    if (waiting != t1 - t0) {
      std::snprintf(error, sizeof(error), "wave %d: %d of its lanes at a cross-lane operation", w, waiting);
      return false;
    }
    for (int t = t0; t < t1; ++t) fibres[t].state = kReady;
  }
}
inline bool run_block() {
  for (int t = 0; t < threads; ++t) {
    Fibre& f = fibres[t];
    getcontext(&f.ctx);
    f.ctx.uc_stack.ss_sp = stacks + t * kStack;
    f.ctx.uc_stack.ss_size = kStack;
    f.ctx.uc_link = nullptr;
    makecontext(&f.ctx, reinterpret_cast<void (*)()>(enter), 0);
    f.state = kReady;
    turn[t] = 0;
  }
  const int waves = (threads + 63) / 64;
  while (true) {
    for (int i = 0; i < waves; ++i)
      if (!run_wave((i + order) % waves)) return false;
    int at = 0;
    any = false;
    for (int t = 0; t < threads; ++t) {
      at += fibres[t].state == kAtBlock;
      any |= fibres[t].state == kAtBlock && fibres[t].flag;
    }
    if (at == 0) return true;
    for (int t = 0; t < threads; ++t)
      if (fibres[t].state != kAtBlock || fibres[t].site != fibres[0].site) {
        std::snprintf(error, sizeof(error), "threads 0 and %d wait at different barriers (lines %d and %d)", t,
                      fibres[0].site, fibres[t].state == kAtBlock ? fibres[t].site : -1);
        return false;
      }
    for (int t = 0; t < threads; ++t) fibres[t].state = kReady;
  }
}
inline void launch(dim3 grid, dim3 block, std::function<void()> f) {
  if (!stacks)
    stacks = static_cast<char*>(mmap(nullptr, kMost * kStack, PROT_READ | PROT_WRITE, MAP_PRIVATE | MAP_ANONYMOUS | MAP_NORESERVE, -1, 0));
  threads = static_cast<int>(block.x);
  if (error[0]) return;
  gridDim = grid;
  blockDim = block;
  body = f;
  for (uint32_t b = 0; b < grid.x; ++b) {
    blockIdx = dim3(b, 0, 0);
    if (!run_block()) return;
  }
}
}  // namespace wg

extern "C" {
// The wave that runs first, and no error.
void wg_order(int first) {
  wg::order = first;
  wg::error[0] = 0;
}
const char* wg_error() { return wg::error; }
}
