// Instances and launch of the stream (paged_rows_stream.h).
#include "paged_rows_stream.h"

namespace tsa {

#ifndef TSA_ROWS_RING8
#define TSA_ROWS_RING8 3
#endif
#ifndef TSA_ROWS_RING16
#define TSA_ROWS_RING16 2
#endif

template <typename T, typename C, int D>
static int launch_stream(const RowsArgs& a, hipStream_t stream, const char* what) {
  constexpr int RING = kIs8<C> ? TSA_ROWS_RING8 : TSA_ROWS_RING16;
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
