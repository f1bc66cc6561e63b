// Plan and launch of the matrix-core form of attention of a chunk
// (paged_chunk_stream.h).
#include "paged_chunk_stream.h"

namespace tsa {

constexpr int kChunkWaves = 4;

static int chunk_runs() {
  int dev = 0, cus = 0;
  if (hipGetDevice(&dev) != hipSuccess ||
      hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || cus <= 0)
    cus = 256;
  return (2 * cus + 7) / 8 * 8;  // two workgroups a CU
}

ChunkPlan chunk_plan(int64_t B, int64_t N, int64_t T, int64_t Hq, int64_t Hkv, int64_t D, int64_t cap) {
  ChunkPlan p{};
  const int64_t G = Hq / Hkv, R = 32 * kChunkWaves;
  if (G > R) return p;
  p.QB = static_cast<int>(R / G);
  p.min_run = 8;
  // Items of this call at most: row blocks of its tokens, one more a sequence.
  T = T < N ? T : N;
  const int64_t rows = N < B * T ? N : B * T;
  const int64_t items = Hkv * (rows / p.QB + B), blocks = (cap + 31) / 32;
  if (items >= (int64_t{1} << 38) / (blocks + 1)) return p;  // (a run's blocks stay in 31 bits)
  // Items of a few blocks are not cut: there is nothing to gain from a second launch.
  p.whole = blocks <= 16;
  const int64_t most = p.whole ? items : (items * blocks + p.min_run - 1) / p.min_run;
  const int64_t P = chunk_runs();
  p.runs = static_cast<int>(P < (most + 7) / 8 * 8 ? P : (most + 7) / 8 * 8);
  const size_t part = sizeof(float) * (D == 128 ? chunk_part_floats<128, kChunkWaves>() : chunk_part_floats<64, kChunkWaves>());
  const size_t head = (kChunkHead + p.runs * sizeof(ChunkSplit) + 255) / 256 * 256;
  p.bytes = head + (p.whole ? 0 : 2 * p.runs * part);
  return p;
}

template <typename T, int D>
static int launch_stream(const ChunkArgs& a, const ChunkPlan& p, void* workspace, hipStream_t stream) {
  int32_t* const head = static_cast<int32_t*>(workspace);
  ChunkSplit* const splits = reinterpret_cast<ChunkSplit*>(static_cast<char*>(workspace) + kChunkHead);
  float* const part = reinterpret_cast<float*>(static_cast<char*>(workspace) +
                                               (kChunkHead + p.runs * sizeof(ChunkSplit) + 255) / 256 * 256);
  paged_chunk_stream<T, D, kChunkWaves><<<dim3(p.runs), dim3(64 * kChunkWaves), 0, stream>>>(a, a.bt, head, splits, part);
  if (int rc = check_launch("tsa_paged_chunk")) return rc;
  if (p.whole || p.runs < 2) return TSA_OK;
  paged_chunk_merge<T, D, kChunkWaves><<<dim3(p.runs - 1, kChunkWaves), dim3(256), 0, stream>>>(a, head, splits, part);
  return check_launch("tsa_paged_chunk");
}

int chunk_stream_launch(const ChunkArgs& a, const ChunkPlan& p, int dt, void* workspace, hipStream_t stream) {
  if (dt == TSA_BF16)
    return a.D == 128 ? launch_stream<bf16_t, 128>(a, p, workspace, stream) : launch_stream<bf16_t, 64>(a, p, workspace, stream);
  return a.D == 128 ? launch_stream<f16_t, 128>(a, p, workspace, stream) : launch_stream<f16_t, 64>(a, p, workspace, stream);
}

}  // namespace tsa
