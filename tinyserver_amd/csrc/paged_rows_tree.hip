// Instances, plan and launch of the tree kernels (paged_rows_tree.h,
// paged_rows_tree_lds.h).
#include "paged_rows_tree_lds.h"

namespace tsa {

// Workgroups a call's units are split into, at least, where there are tokens for
// it (64 sequences of 512-4096 tokens, 16 nodes, 32/8 heads: 512 126 us, 1024 158;
// 32 nodes: 144, 187; 8 of 8192 with 64 nodes, 64/8 heads: 177, 188), and the least
// blocks of a split. (16 was the faster before tree_per_split dealt the blocks evenly;
// with it 4 is: 8 nodes, 32/8 heads, one sequence of 300 / 1000 / 2000 tokens: 13.8 /
// 17.7 / 17.7 us against 12.7 / 14.3 / 13.7. Larger plans have not been measured so.)
constexpr int64_t kTreeWorkgroups = 512, kTreeMinSplit = 16;

TreeRowsPlan tree_rows_plan(int64_t B, int64_t T, int64_t Hq, int64_t Hkv, int64_t D, int64_t cap) {
  TreeRowsPlan p{};
  const int64_t rows = T * (Hq / Hkv), blocks = (cap + 31) / 32;
  p.RT = rows <= 32 ? 1 : rows <= 64 ? 2 : 4;
  p.RB = static_cast<int>((rows + 32 * p.RT - 1) / (32 * p.RT));
  const int64_t wgs = B * Hkv * p.RB;
  int64_t S = (kTreeWorkgroups + wgs - 1) / wgs;
  const int64_t most = (blocks + kTreeMinSplit - 1) / kTreeMinSplit;
  S = S < most ? S : most;
  const int64_t least = (blocks + kTreeMaxSplit - 1) / kTreeMaxSplit;
  S = S < least ? least : S;
  S = S < 1 ? 1 : S;
  const int64_t per = ((blocks + S - 1) / S + 3) / 4 * 4;
  p.per_split = static_cast<int>(per < 4 ? 4 : per);
  p.S = static_cast<int>((blocks + p.per_split - 1) / p.per_split);
  if (p.S < 1) p.S = 1;
  if (wgs * p.S >= (int64_t{1} << 22) || rows > 65536) return TreeRowsPlan{};  // (grids' limits)
  p.bytes = p.S == 1 ? 0 : static_cast<size_t>(B * Hkv * p.S) * static_cast<size_t>(rows) * (D + 4) * sizeof(float);
  return p;
}
static_assert(kTreeMaxSplit % 4 == 0, "a split rounded up to four blocks still fits its table");

template <typename T, int D>
static int launch_tree(const RowsArgs& a, hipStream_t stream) {
  const int64_t us = int64_t{a.B} * a.Hkv * a.S;
  const dim3 grid(static_cast<uint32_t>((us + 7) / 8 * 8 * a.RB));
  if (a.RT == 1) paged_rows_tree<T, D><<<grid, dim3(256), 0, stream>>>(a, a.bt, a.mask, a.part);
  else if (a.RT == 2) paged_rows_tree_lds<T, D, 2><<<grid, dim3(128), 0, stream>>>(a, a.bt, a.mask, a.part);
  else paged_rows_tree_lds<T, D, 4><<<grid, dim3(256), 0, stream>>>(a, a.bt, a.mask, a.part);
  if (int rc = check_launch("tsa_paged_tree")) return rc;
  if (a.S == 1) return TSA_OK;
  launch_rows_merge<T, D>(a, a.T * a.G, 0, stream);
  return check_launch("tsa_paged_tree");
}

int rows_tree_launch(const RowsArgs& a, int dt, hipStream_t stream) {
  if (dt == TSA_BF16) return a.D == 128 ? launch_tree<bf16_t, 128>(a, stream) : launch_tree<bf16_t, 64>(a, stream);
  return a.D == 128 ? launch_tree<f16_t, 128>(a, stream) : launch_tree<f16_t, 64>(a, stream);
}

}  // namespace tsa
