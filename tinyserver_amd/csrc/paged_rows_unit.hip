// Instances and launch of the unit form (paged_rows_unit.h).
#include "paged_rows_stream.h"

namespace tsa {

// Split calls of up to this many workgroups take the unit form. Both sides, 32/8
// heads, e4m3 / bf16, us, unit form against stream: 16 x 256-1024 tokens (512
// workgroups) 10.9 / 14.4 against 14.5 / 17.2; 16 x 512-2048 (1024) 17.2 / 20.6
// against 18.4 / 22.3; 64 x 256-1024 (2048) 23.6 / 31.2 against 26.2 / 33.5; 16 x
// 1024-4096 (2048) 26.3 / 37.4 against 26.7 / 36.1; 4 x 8192-32768 (4096) 47.5 /
// 72 against 40 / 60.
constexpr int64_t kUnitMaxWorkgroups = 2048;
// The stream's grid: a four-wave workgroup a CU (two a CU, e4m3, 64 x 512-4096
// tokens: 68.5 us against 64.0; 32 x 32768: 361 against 348).
static int stream_workgroups() {
  int dev = 0, cus = 0;
  if (hipGetDevice(&dev) != hipSuccess ||
      hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || cus <= 0)
    cus = 256;
  return cus;
}

// A unit that is one workgroup reads K/V with ordinary loads, a split's workgroup
// with non-temporal ones. Both sides, ordinary / non-temporal, us, caches of several
// calls in turn (past what the chip keeps, but for the first): one workgroup, e4m3 /
// bf16, 4 x 16-512 tokens, 16/8 heads 8.2 / 8.6 and 9.4 / 10.9, 64 x 100-512, 32/8
// heads 16.4 / 15.5 and 25.0 / 23.9, 256 of them 45.2 / 44.3 and 79.1 / 79.9; splits,
// 32/8 heads, 16 x 512-1024 14.7 / 13.8 and 18.8 / 16.2, 16 x 1024-2048 21.1 / 19.8
// and 29.7 / 26.4, 4 x 2048-4096 15.7 / 15.2 and 18.8 / 17.3, 1 x 16384-32768 21.3 /
// 19.6 and 27.5 / 24.4.
template <typename T, typename C, int D>
static int launch_unit(const RowsArgs& a, hipStream_t stream, const char* what) {
  const int groups = (a.G + 15) / 16, items = a.B * a.Hkv * groups, rows = a.G < 16 ? a.G : 16;
  const size_t row_bytes = static_cast<size_t>(rows) * part_floats(D) * sizeof(float);
  if (a.S == 1) {
    paged_rows_unit<T, C, D, kUnitWavesOne, false>
        <<<dim3(items), dim3(64 * kUnitWavesOne), kUnitWavesOne * row_bytes, stream>>>(a, a.bt, a.lens, a.part);
    return check_launch(what);
  }
  const dim3 grid(static_cast<uint32_t>(items) * a.S), threads(64 * kUnitWavesSplit);
  paged_rows_unit<T, C, D, kUnitWavesSplit, true><<<grid, threads, kUnitWavesSplit * row_bytes, stream>>>(a, a.bt, a.lens, a.part);
  if (int rc = check_launch(what)) return rc;
  launch_rows_merge<T, D>(a, a.G, kUnitWavesSplit * kUnitTiles, stream);
  return check_launch(what);
}

template <typename T, typename C>
static int launch_unit_d(const RowsArgs& a, hipStream_t stream, const char* what) {
  return a.D == 128 ? launch_unit<T, C, 128>(a, stream, what) : launch_unit<T, C, 64>(a, stream, what);
}

int rows_unit_launch(const RowsArgs& a, int dt, int cache_dt, hipStream_t stream, const char* what) {
  if (dt == TSA_BF16)
    return cache_dt == TSA_E4M3 ? launch_unit_d<bf16_t, e4m3_t>(a, stream, what)
           : cache_dt == TSA_I8 ? launch_unit_d<bf16_t, i8_t>(a, stream, what)
                                : launch_unit_d<bf16_t, bf16_t>(a, stream, what);
  return cache_dt == TSA_E4M3 ? launch_unit_d<f16_t, e4m3_t>(a, stream, what)
         : cache_dt == TSA_I8 ? launch_unit_d<f16_t, i8_t>(a, stream, what)
                              : launch_unit_d<f16_t, f16_t>(a, stream, what);
}

// One workgroup of eight waves a unit where its visible tiles fit it, else
// splits of four waves each, else the stream.
DecodeRowsPlan decode_rows_plan(int64_t B, int64_t Hq, int64_t Hkv, int64_t D, int64_t cap, int64_t window,
                                int64_t sinks) {
  int64_t tiles = (cap + 15) / 16;
  if (window > 0 && window < cap) {
    const int64_t seen = ((sinks < cap ? sinks : cap) + 15) / 16 + (window + 15) / 16 + 1;
    tiles = seen < tiles ? seen : tiles;
  }
  const int64_t G = Hq / Hkv, items = B * Hkv * ((G + 15) / 16), rows = G < 16 ? G : 16;
  const size_t slot = static_cast<size_t>(rows) * (D + 4) * sizeof(float);
  auto align = [](size_t n) { return (n + 255) & ~size_t{255}; };
  DecodeRowsPlan p{};
  const int64_t S = tiles <= kUnitWavesOne * kUnitTiles ? 1 : (tiles + kUnitWavesSplit * kUnitTiles - 1) / (kUnitWavesSplit * kUnitTiles);
  if (S == 1 || items * S <= kUnitMaxWorkgroups) {
    p.S = static_cast<int>(S);
    p.total = p.part_bytes = S == 1 ? 0 : align(static_cast<size_t>(B * Hkv * S * G) * (D + 4) * sizeof(float));
    return p;
  }
  p.waves = kStreamWaves * stream_workgroups();
  p.part_bytes = align((static_cast<size_t>(items) + p.waves) * slot);
  p.total = p.part_bytes + align((static_cast<size_t>(B) + 1) * sizeof(int32_t));
  return p;
}

}  // namespace tsa
