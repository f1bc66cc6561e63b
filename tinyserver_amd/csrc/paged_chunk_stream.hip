// Plan and launch of the matrix-core form of attention of a chunk
// (paged_chunk_stream.h).
#include "paged_chunk_stream.h"

namespace tsa {

// Waves of a workgroup: eight (256 rows, one workgroup a CU) where sequences have rows
// for it on average, four (128 rows, two a CU) else: half the K/V reads against twice
// the items in flight. (28 sequences with one token beside four with 128-512, 32/8
// heads: 100 us in fours, 127 in eights; 16 with 64-512: 214 in eights, 217 in fours;
// 2048 over 30720, 64/8 heads: 1.96 ms and 2.2.) Eight also from 128 rows on where no
// sequence has more than 256: K/V are read once then. (20 tokens each over 2 x
// 24000-32768, 64/8 heads: 81 us, 94 in fours; 12 and 40 each: 108 and 98.)
static int chunk_waves(int64_t B, int64_t rows, int64_t G, int64_t T) {
  return rows * G > (T * G <= 256 ? 128 : 192) * B ? 8 : 4;
}

static int chunk_runs(int waves) {
  int dev = 0, cus = 0;
  if (hipGetDevice(&dev) != hipSuccess ||
      hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || cus <= 0)
    cus = 256;
  return ((waves == 8 ? cus : 2 * cus) + 7) / 8 * 8;  // as many as fit at once
}

ChunkPlan chunk_plan(int64_t B, int64_t N, int64_t T, int64_t Hq, int64_t Hkv, int64_t D, int64_t cap,
                     bool f32) {
  ChunkPlan p{};
  T = T < N ? T : N;
  const int64_t G = Hq / Hkv;
  const int64_t rows = N < B * T ? N : B * T;
  p.waves = f32 ? 1 : G > 128 ? 8 : chunk_waves(B, rows, G, T);  // (float32: 32 rows a workgroup)
  const int64_t R = 32 * p.waves;
  if (G > R) return p;
  p.QB = static_cast<int>(R / G);
  // Items of this call at most: row blocks of its tokens, one more a sequence.
  const int64_t items = Hkv * (rows / p.QB + B), blocks = (cap + 31) / 32;
  if (items >= (int64_t{1} << 38) / (blocks + kItemCost)) return p;  // (a run's blocks stay in 31 bits)
  // Items of a few blocks are not cut, which saves the second launch and the partial
  // results; few items of more blocks are, as there are workgroups left for their runs.
  // (16/8 heads. f16: 4 sequences of one token under tables of 256 tokens 11.2 us whole
  // and 13.9 cut, of 8 under 512 16.1 and 14.4; 16 of 8 under 512 17.1 and 19.8, under 768
  // 21.3 and 22.4, under 1024 25.5 and 24.3. float32: 4 of one token under 256 17.0 and
  // 16.3, under 512 24.6 and 17.0; 16 under 512 27.6 and 27.8, 4 of 64 28.3 and 32. Over
  // 87 bf16 calls of each table of 12, 14 and 16 blocks, 1 to 192 items, these bounds lie 0.6,
  // 0.9 and 0.6% above the better side on average; float32, 58 calls, 0.5, 0.1 and 0.5%.)
  // Longer tables are always cut: their sequences may be of very different lengths. Runs
  // are as short as four blocks (4 sequences of 1-8 tokens over up to 1000: 17.6 us with
  // eight, 15.6).
  p.whole = blocks <= (f32 ? 8 : 12) || (blocks <= 16 && items >= (f32 ? 112 : 64));
  p.min_run = p.whole ? 1 : 4;
  const int64_t most = p.whole ? items : (items * (blocks + kItemCost) + p.min_run - 1) / p.min_run;
  const int64_t P = chunk_runs(p.waves);
  p.runs = static_cast<int>(P < (most + 7) / 8 * 8 ? P : (most + 7) / 8 * 8);
  const size_t part = sizeof(float) * (chunk_part_floats(static_cast<int>(D), p.waves));
  const size_t head = (kChunkHead + p.runs * sizeof(ChunkSplit) + 255) / 256 * 256;
  p.bytes = head + (p.whole ? 0 : 2 * p.runs * part);
  return p;
}

template <typename T, int D, int NW>
static int launch_stream(const ChunkArgs& a, const ChunkPlan& p, hipStream_t stream) {
  paged_chunk_stream<T, D, NW><<<dim3(p.runs), dim3(64 * NW), 0, stream>>>(a);
  if (int rc = check_launch("tsa_paged_chunk")) return rc;
  if (p.whole || p.runs < 2) return TSA_OK;
  paged_chunk_merge<T, D, NW><<<dim3(p.runs - 1, NW), dim3(256), 0, stream>>>(a);
  return check_launch("tsa_paged_chunk");
}

template <typename T>
static int launch_stream(const ChunkArgs& a, const ChunkPlan& p, hipStream_t stream) {
  if (p.waves == 8) return a.D == 128 ? launch_stream<T, 128, 8>(a, p, stream) : launch_stream<T, 64, 8>(a, p, stream);
  return a.D == 128 ? launch_stream<T, 128, 4>(a, p, stream) : launch_stream<T, 64, 4>(a, p, stream);
}

int chunk_stream_launch(ChunkArgs& a, const ChunkPlan& p, int dt, void* workspace, hipStream_t stream) {
  char* const ws = static_cast<char*>(workspace);
  a.QB = p.QB;
  a.min_run = p.min_run;
  a.whole = p.whole;
  a.g_mul = (65536 + a.G - 1) / a.G;
  a.runs = reinterpret_cast<int32_t*>(ws);
  a.splits = reinterpret_cast<ChunkSplit*>(ws + kChunkHead);
  a.part = reinterpret_cast<float*>(ws + (kChunkHead + p.runs * sizeof(ChunkSplit) + 255) / 256 * 256);
  if (dt == TSA_F32) return chunk_f32_launch(a, p, stream);
  return dt == TSA_BF16 ? launch_stream<bf16_t>(a, p, stream) : launch_stream<f16_t>(a, p, stream);
}

}  // namespace tsa
