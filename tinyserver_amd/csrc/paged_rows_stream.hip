// Instances and launch of the stream (paged_rows_stream.h).
#include "paged_rows_stream.h"

namespace tsa {

// Tile pairs a wave keeps in registers. e4m3, 64 x 512-4096 / 32 x 32768 tokens:
// three 64.0 / 348 us, four 66.4 / 351, six 69.4 / 353; bf16, window 1024 + 4 of
// 64: two 51.8, three 55.0, four 54.5, five 59.1 (more have to land before the
// first is computed).
constexpr int kRing8 = 3, kRing16 = 2;

template <typename T, typename C, int D>
static int launch_stream(const RowsArgs& a, hipStream_t stream, const char* what) {
  constexpr int RING = kIs8<C> ? kRing8 : kRing16;
  const int groups = (a.G + 15) / 16, units = a.Hkv * groups, rows = a.G < 16 ? a.G : 16;
  paged_rows_stream<T, C, D, RING><<<dim3(a.NW / kStreamWaves), dim3(64 * kStreamWaves), (2 * a.B + 1) * sizeof(int32_t), stream>>>(
      a, a.bt, a.lens, a.part, a.pref);
  if (int rc = check_launch(what)) return rc;
  constexpr int RW = 64 / (D / 4);
  paged_rows_stream_merge<T, D><<<dim3(a.B * units, (rows + RW - 1) / RW), dim3(256), 0, stream>>>(a, a.part, a.pref);
  return check_launch(what);
}

template <typename T, typename C>
static int launch_stream_d(const RowsArgs& a, hipStream_t stream, const char* what) {
  return a.D == 128 ? launch_stream<T, C, 128>(a, stream, what) : launch_stream<T, C, 64>(a, stream, what);
}

int rows_stream_launch(const RowsArgs& a, int dt, int cache_dt, hipStream_t stream, const char* what) {
  if (dt == TSA_BF16)
    return cache_dt == TSA_E4M3 ? launch_stream_d<bf16_t, e4m3_t>(a, stream, what)
           : cache_dt == TSA_I8 ? launch_stream_d<bf16_t, i8_t>(a, stream, what)
                                : launch_stream_d<bf16_t, bf16_t>(a, stream, what);
  return cache_dt == TSA_E4M3 ? launch_stream_d<f16_t, e4m3_t>(a, stream, what)
         : cache_dt == TSA_I8 ? launch_stream_d<f16_t, i8_t>(a, stream, what)
                              : launch_stream_d<f16_t, f16_t>(a, stream, what);
}

}  // namespace tsa
