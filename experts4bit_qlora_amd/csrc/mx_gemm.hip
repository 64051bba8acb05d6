// Launchers of the microscaled products.
#include "mx_gemm.h"

#include "mx_launch.h"

#include <algorithm>

namespace e4b {

namespace {

template <int DT>
void launch_rows(const MxGemmArgs& a, hipStream_t s) {
  const int64_t row_chunks = mx_chunks(a.w.k), chunks = a.M * row_chunks;
  constexpr int kPer = kMxRowThreads / (kMxChunk / 8);
  hipLaunchKernelGGL(mx_rows_kernel<DT>, dim3(static_cast<unsigned>((chunks + kPer - 1) / kPer)), dim3(kMxRowThreads), 0, s,
                     a.x, static_cast<int>(a.w.k), static_cast<uint32_t>(row_chunks), static_cast<uint32_t>(chunks),
                     reinterpret_cast<uint32_t*>(a.a), a.as);
}

int group_tiles(const MxTiling& tl, int size) { return size > tl.lo && size <= tl.hi ? (size + tl.tm - 1) / tl.tm : 0; }

template <class K>
void launch_tiles(K kernel, int threads, MxGemmArgs a, MxGroups& g, MxTiling tl, int columns, hipStream_t s,
                  unsigned most = 0x7fffffff, int lds = 0) {
  a.tl = tl;
  a.tl.one = 1;
  int tiles = 0;
  for (int i = 0; i < a.groups; ++i) {
    g.tile[i] = static_cast<uint16_t>(tiles);
    const int n = group_tiles(tl, g.off[i + 1] - g.off[i]);
    tiles += n;
    a.tl.one &= n == 1;
  }
  for (int i = a.groups; i <= kMxGroupsMax; ++i) g.tile[i] = static_cast<uint16_t>(tiles);
  if (!tiles) return;
  a.tiles = tiles;
  a.n_blocks = static_cast<int>((a.w.n + columns - 1) / columns);
  const unsigned total = static_cast<unsigned>(tiles) * static_cast<unsigned>(a.n_blocks);
  hipLaunchKernelGGL(kernel, dim3(std::min((total + 7) / 8 * 8, most)), dim3(threads), lds, s, a, g);
}

// Groups of more than 32 rows take 256-row tiles; smaller ones 32-row tiles, unless there are only a few beside
// larger groups: a tile of either kind costs about its weights' bytes (5,760 x 2,880: 3.1 us of the card in
// the 256-row launch, 2 in the other), a launch 5 us. K of at most one chunk has no 256-row kernel.
// Where no group has more than kDirect rows, and their codes fit 16 KB (four workgroups per CU with the 17 KB of
// partial sums), the 32-row tiles quantize their rows themselves: four experts of 5,760 x 2,880 take 11.4 us so at
// four rows each, 11.3 and a launch more in two kernels; at eight 14.7 and 11.6.
template <int ODT>
void launch_groups(const MxGemmArgs& a, MxGroups& g, hipStream_t s) {
  constexpr int kAll = 0x7fffffff, kFew = 5, kDirect = 4;
  int small = 0, large = 0, most = 0;
  for (int i = 0; i < a.groups; ++i) {
    const int size = g.off[i + 1] - g.off[i];
    small += size > 0 && size <= kMxTileM;
    large += size > kMxTileM;
    most = std::max(most, size);
  }
  const int threads = kMxNarrowWaves * kWave;
  const MxTiling tiles32 = {kMxTileM, 0, kAll, 0};
  const bool bf16 = a.act_dtype == E4B_BF16;
  const int64_t lds = most * mx_chunks(a.w.k) * (kMxChunk / 2 + kMxChunk / kMxBlock);
  if (most <= kDirect && lds <= 16384) {
    const unsigned all = 0x7fffffff;
    if (bf16) launch_tiles(mx_narrow_kernel<ODT, E4B_BF16>, threads, a, g, tiles32, 32, s, all, static_cast<int>(lds));
    else launch_tiles(mx_narrow_kernel<ODT, E4B_FP16>, threads, a, g, tiles32, 32, s, all, static_cast<int>(lds));
    return;
  }
  if (bf16) launch_rows<E4B_BF16>(a, s);
  else launch_rows<E4B_FP16>(a, s);
  const bool wide = large && a.w.k > kMxChunk;
  const int narrow_to = !wide ? kAll : small > kFew ? kMxTileM : 0;
  if (wide) launch_tiles(mx_wide_kernel<ODT>, kMxWideThreads, a, g, {kMxWideM, narrow_to, kAll, 0}, kMxWideN, s, 256);
  if (narrow_to) launch_tiles(mx_narrow_kernel<ODT, -1>, threads, a, g, {kMxTileM, 0, narrow_to, 0}, 32, s);
}

}  // namespace

void launch_mx_gemm_groups(const MxGemmArgs& a, MxGroups& g, int out_dtype, hipStream_t s) {
  switch (out_dtype) {
    case E4B_BF16: return launch_groups<E4B_BF16>(a, g, s);
    case E4B_FP16: return launch_groups<E4B_FP16>(a, g, s);
    default: return launch_groups<E4B_FP32>(a, g, s);
  }
}

}  // namespace e4b
