// Launchers of the microscaled products.
#include "mx_gemm.h"

#include "mx_launch.h"

#include <algorithm>

namespace e4b {

namespace {

// A launch holds fewer than 2^32 work items: 2^26 chunks of the rows' kernel (32 threads each) and 2^24 workgroups of
// 256 threads are taken per launch at most.
constexpr int64_t kRowChunks = int64_t(1) << 26, kWorkgroups = (int64_t(1) << 24) - 8;

template <int DT>
void launch_rows(const MxGemmArgs& a, hipStream_t s) {
  const int64_t row_chunks = mx_chunks(a.w.k), most = kRowChunks / row_chunks;  // (k below 2^24: at least 2^10 rows)
  constexpr int kPer = kMxRowThreads / (kMxChunk / 8);
  for (int64_t row = 0; row < a.M; row += most) {
    const int64_t chunks = std::min(most, a.M - row) * row_chunks, first = row * row_chunks;
    hipLaunchKernelGGL(mx_rows_kernel<DT>, dim3(static_cast<unsigned>((chunks + kPer - 1) / kPer)), dim3(kMxRowThreads), 0, s,
                       static_cast<const uint16_t*>(a.x) + row * a.w.k, static_cast<int>(a.w.k),
                       static_cast<uint32_t>(row_chunks), static_cast<uint32_t>(chunks),
                       reinterpret_cast<uint32_t*>(a.a) + first * (kMxChunk / 8), a.as + first * (kMxChunk / kMxBlock));
  }
}

int group_tiles(const MxTiling& tl, int size) { return size > tl.lo && size <= tl.hi ? (size + tl.tm - 1) / tl.tm : 0; }

// most: the workgroups of a launch, which stay and take all tiles; 0: one workgroup for every tile and column block,
// in launches of as many groups as one holds. (No group alone passes that: one of more than 32 rows takes 256-row
// tiles, unless its call has few tiles or its stack fewer than eight scale bytes, which are one column block.)
template <class K>
void launch_tiles(K kernel, int threads, MxGemmArgs a, MxGroups& g, MxTiling tl, int columns, hipStream_t s, unsigned most = 0,
                  int lds = 0) {
  a.tl = tl;
  a.n_blocks = static_cast<int>((a.w.n + columns - 1) / columns);
  const int64_t fit = most ? int64_t(1) << 31 : kWorkgroups / a.n_blocks;
  for (int from = 0; from < a.groups;) {
    a.tl.one = from == 0;
    a.tiles = 0;
    int i = 0;
    for (; i < a.groups; ++i) {
      const int n = i < from ? 0 : group_tiles(tl, g.off[i + 1] - g.off[i]);
      if (a.tiles && a.tiles + n > fit) break;
      g.tile[i] = static_cast<uint16_t>(a.tiles);
      a.tiles += n;
      a.tl.one &= n == 1;
    }
    a.tl.one &= i == a.groups;
    from = i;
    for (; i <= kMxGroupsMax; ++i) g.tile[i] = static_cast<uint16_t>(a.tiles);
    if (!a.tiles) return;
    const unsigned total = (static_cast<unsigned>(a.tiles) * static_cast<unsigned>(a.n_blocks) + 7) / 8 * 8;
    hipLaunchKernelGGL(kernel, dim3(most ? std::min(total, most) : total), dim3(threads), lds, s, a, g);
  }
}

// Calls of at most kNarrowTiles tiles of 32 x 32 (2.5 for each workgroup that the card holds) take those alone: they
// spread over the CUs and start at once, where a 256-row tile keeps one CU for ~10 us and longer. Both grow alike
// with K, so the bound holds for any: in us, 32-row tiles / 256-row tiles,
//   2,880 tiles: K 128 11.3 / 11.6, 256 12.8 / 10.4, 1,024 19.9 / 13.6, 2,880 29.9 / 24.8
//   1,664 to 1,792: K 128 8.3 / 12.4, 512 9.6 / 11.2, 1,024 13.0 / 15.4, 2,880 20.2 / 27.0
//   832: K 512 6.0 / 11.9, 2,880 12.8 / 25.4;  23,040: K 128 64.9 / 23.4, 2,880 206.9 / 60.2
// In larger calls the groups of more than 32 rows take 256-row tiles, and smaller ones ride along unless there are
// many: a launch of 32-row tiles for them gains only where it is mostly their weights (us a call, own launch /
// along: 24 groups of 30 rows + 8 of 300, 2,880 x 2,880 79.6 / 67.7, 1,408 x 1,216 31.4 / 25.2; 8 of 8 + 24 of 200 84.2
// / 74.1, 29.7 / 25.6; 26 of 2 + 6 of 500 68.5 / 72.5, 30.2 / 25.5).
//
// Small groups all round quantize their rows inside the 32-row tiles, without a launch for that: up to eight rows
// each, up to sixteen where there are tiles enough for runs of column blocks (more than twice 1,024), which share
// the quantized rows (one row or four are cheaper quantized again for every block than runs are). Per call in us,
// against the rows' kernel and the product's (and a gap between them):
//   experts x rows of 5,760 x 2,880: 4 x 1 8.6 (4.4 + 9.7); 4 x 8 12.1 (4.4 + 9.4); 4 x 16 16.9 (4.4 + 10.4);
//   32 x 1 56.8 (4.4 + 61.7); 32 x 4 63.5 (4.3 + 66.9), in runs 66.3; 32 x 12 72.3 (4.4 + 76.7), without runs 84.0;
//   32 x 16 75.6 (4.5 + 80.7); 32 x 24 87.8 (4.5 + 88.5); of 2,880 x 2,880: 32 x 16 38.9 (4.5 + 37.5)
template <int ODT>
void launch_groups(const MxGemmArgs& a, MxGroups& g, hipStream_t s) {
  constexpr int kAll = 0x7fffffff, kFew = 32, kNarrowThreads = kMxNarrowWaves * kWave;
  constexpr int kDirect = 8, kDirectInRuns = 16, kDirectLds = 32768, kOnce = 4, kRunItems = 1024, kRunMost = 4, kNarrowTiles = 2560;
  int small = 0, large = 0, most = 0;
  int64_t tiles = 0;
  for (int i = 0; i < a.groups; ++i) {
    const int size = g.off[i + 1] - g.off[i];
    small += size > 0 && size <= kMxTileM;
    large += size > kMxTileM;
    most = std::max(most, size);
    tiles += (size + kMxTileM - 1) / kMxTileM;
  }
  const bool bf16 = a.act_dtype == E4B_BF16;
  const int64_t blocks = (a.w.n + 31) / 32;
  const int64_t lds = most * mx_chunks(a.w.k) * (kMxChunk / 2 + kMxChunk / kMxBlock);
  const int64_t run = std::clamp<int64_t>(tiles * blocks / kRunItems, 1, kRunMost);
  if (most <= (run > 1 ? kDirectInRuns : kDirect) && lds <= kDirectLds) {
    MxGemmArgs d = a;
    d.run = most > kOnce ? static_cast<int>(run) : 1;
    const auto kernel = bf16 ? mx_narrow_kernel<ODT, E4B_BF16> : mx_narrow_kernel<ODT, E4B_FP16>;
    launch_tiles(kernel, kNarrowThreads, d, g, {kMxTileM, 0, kAll, 0}, 32 * d.run, s, 0, static_cast<int>(lds));
    return;
  }
  if (bf16) launch_rows<E4B_BF16>(a, s);
  else launch_rows<E4B_FP16>(a, s);
  const bool wide = large && tiles * blocks > kNarrowTiles && mx_wide(a.w);
  const int narrow_to = !wide ? kAll : small > kFew ? kMxTileM : 0;
  if (wide) launch_tiles(mx_wide_kernel<ODT>, kMxWideThreads, a, g, {kMxWideM, narrow_to, kAll, 0}, kMxWideN, s, 256);
  if (narrow_to) launch_tiles(mx_narrow_kernel<ODT, -1>, kNarrowThreads, a, g, {kMxTileM, 0, narrow_to, 0}, 32, s);
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
