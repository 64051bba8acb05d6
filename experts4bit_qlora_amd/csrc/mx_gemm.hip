// Launchers of the microscaled products.
#include "mx_gemm.h"

#include "mx_launch.h"

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

void launch_mx_gemm_groups(MxGemmArgs a, const MxGroups& g, int out_dtype, hipStream_t s) {
  a.tiles = 0;
  a.one = 1;
  for (int i = 0; i < a.groups; ++i) {
    const int tiles = (g.off[i + 1] - g.off[i] + kMxTileM - 1) / kMxTileM;
    a.tiles += tiles;
    a.one &= tiles == 1;
  }
  a.n_blocks = static_cast<int>((a.w.n + 31) / 32);
  const dim3 grid(static_cast<unsigned>(a.tiles) * static_cast<unsigned>(a.n_blocks)), b(kMxNarrowWaves * kWave);
  switch (out_dtype) {
    case E4B_BF16: hipLaunchKernelGGL(mx_narrow_kernel<E4B_BF16>, grid, b, 0, s, a, g); break;
    case E4B_FP16: hipLaunchKernelGGL(mx_narrow_kernel<E4B_FP16>, grid, b, 0, s, a, g); break;
    default: hipLaunchKernelGGL(mx_narrow_kernel<E4B_FP32>, grid, b, 0, s, a, g); break;
  }
}

}  // namespace e4b
