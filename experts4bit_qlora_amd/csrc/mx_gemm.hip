// Launchers of the microscaled products.
#include "mx_gemm.h"

#include "mx_launch.h"

#include <algorithm>
#include <cstdlib>

namespace e4b {

namespace {

template <int DT>
void launch_rows(const void* x, int64_t rows, int64_t k, uint8_t* codes, uint8_t* scales, hipStream_t s) {
  const int64_t row_pieces = mx_chunks(k) * (kMxChunk / 8), pieces = rows * row_pieces;
  const dim3 grid(static_cast<unsigned>((pieces + kMxRowThreads - 1) / kMxRowThreads));
  hipLaunchKernelGGL(mx_rows_kernel<DT>, grid, dim3(kMxRowThreads), 0, s, x, k, static_cast<int>(row_pieces), pieces,
                     reinterpret_cast<uint32_t*>(codes), scales);
}

}  // namespace

void launch_mx_rows(const void* x, int dtype, int64_t rows, int64_t k, uint8_t* codes, uint8_t* scales, hipStream_t s) {
  if (dtype == E4B_BF16) launch_rows<E4B_BF16>(x, rows, k, codes, scales, s);
  else launch_rows<E4B_FP16>(x, rows, k, codes, scales, s);
}

namespace {

int group_tiles(const MxTiling& tl, int size) {
  if (tl.rest_only) {
    const int rest = size % tl.big;
    return rest > 0 && rest <= tl.tm ? 1 : 0;
  }
  return size / tl.tm + (size % tl.tm > tl.rest_above ? 1 : 0);
}

template <class K>
void launch_tiles(K kernel, int threads, MxGemmArgs a, MxGroups& g, MxTiling tl, int columns, hipStream_t s,
                  unsigned most = 0x7fffffff) {
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
  hipLaunchKernelGGL(kernel, dim3(std::min((total + 7) / 8 * 8, most)), dim3(threads), 0, s, a, g);
}

template <int ODT>
void launch_groups(const MxGemmArgs& a, MxGroups& g, hipStream_t s) {
  int largest = 0;
  for (int i = 0; i < a.groups; ++i) largest = std::max(largest, g.off[i + 1] - g.off[i]);
  const int threads = kMxNarrowWaves * kWave;
  if (largest <= kMxTileM) {
    launch_tiles(mx_narrow_kernel<ODT>, threads, a, g, {kMxTileM, 0, 0, 1, 0}, 32, s);
    return;
  }
  if (largest <= kMxTileM || a.w.k <= kMxChunk) {
    launch_tiles(mx_narrow_kernel<ODT>, threads, a, g, {kMxTileM, 0, 0, 1, 0}, 32, s);
    return;
  }
  const char* env = getenv("MXT");
  const int rest = env ? atoi(env) : 32;
  launch_tiles(mx_wide_kernel<ODT>, kMxWideThreads, a, g, {kMxWideM, rest, 0, 1, 0}, kMxWideN, s, 256);
  if (rest) launch_tiles(mx_narrow_kernel<ODT>, threads, a, g, {kMxTileM, 0, 1, kMxWideM, 0}, 32, s);
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
