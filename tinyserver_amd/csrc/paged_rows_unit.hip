// Instances and launch of the unit form (paged_rows_unit.h).
#include "paged_rows_unit.h"

namespace tsa {

// Units of this many splits or more read K/V with non-temporal loads.
constexpr int kRowsNtSplits = 16;

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
  if (a.S >= kRowsNtSplits)
    paged_rows_unit<T, C, D, kUnitWavesSplit, true><<<grid, threads, kUnitWavesSplit * row_bytes, stream>>>(a, a.bt, a.lens, a.part);
  else
    paged_rows_unit<T, C, D, kUnitWavesSplit, false><<<grid, threads, kUnitWavesSplit * row_bytes, stream>>>(a, a.bt, a.lens, a.part);
  if (int rc = check_launch(what)) return rc;
  constexpr int RW = 64 / (D / 4);
  paged_rows_merge<T, D><<<dim3(a.B * a.Hkv, (a.G + RW - 1) / RW), dim3(256), 0, stream>>>(
      a, a.lens, a.part, kUnitWavesSplit * kUnitTiles<C>);
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

// Splits: one workgroup of eight waves where a unit's visible tiles fit it, else
// workgroups of four.
int rows_unit_splits(int64_t max_tiles, bool cache8) {
  const int kt = cache8 ? kUnitTiles<i8_t> : kUnitTiles<bf16_t>;
  if (max_tiles <= kUnitWavesOne * kt) return 1;
  return static_cast<int>((max_tiles + kUnitWavesSplit * kt - 1) / (kUnitWavesSplit * kt));
}

}  // namespace tsa
