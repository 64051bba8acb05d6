// Launch-side view of the products of microscaled operands (mx_gemm.h), instantiated in mx_gemm.hip.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "e4b_amd.h"

namespace e4b {

// Activation rows are quantized into the workspace with K padded to whole chunks of 256, two at least (zero codes,
// scale bytes 0): a chunk is 128 bytes of codes and 8 scale bytes.
constexpr int kMxChunk = 256;
__host__ __device__ inline int64_t mx_chunks(int64_t k) { return k > kMxChunk ? (k + kMxChunk - 1) / kMxChunk : 2; }

// Row groups given by the host: group g holds rows off[g] .. off[g + 1] - 1 for the expert ids[g].
constexpr int kMxGroupsMax = 512;
// tile: a launch's first row tile of each group.
struct MxGroups {
  int32_t off[kMxGroupsMax + 1];
  uint16_t tile[kMxGroupsMax + 1];
};
// The 256-row tiles read scale bytes eight at a time.
inline bool mx_wide(const e4b_qweight& w) { return w.num_experts * w.n * (w.k / 32) >= 8; }
// Fewer than 2^16 row tiles, one more than the rows fill per group: of 256 rows, or of 32 for stacks so small.
inline int64_t mx_rows_max(const e4b_qweight& w) { return int64_t(1) << (mx_wide(w) ? 23 : 20); }

// A launch's row tiles: tiles of tm rows over the groups of above lo and at most hi rows.
struct MxTiling {
  int tm, lo, hi;
  int one;  // every group is one tile
};

struct MxGemmArgs {
  const void* x;      // the rows [rows, k] as given, of type act_dtype
  int act_dtype;
  uint8_t* a;         // workspace: codes [rows, 128 * chunks]
  uint8_t* as;        // workspace: scale bytes [rows, 8 * chunks]
  e4b_qweight w;
  const int64_t* ids;  // group form: the groups' experts (device); a group outside [0, E) gets zero rows
  int groups;
  int64_t M;
  void* out;  // [M, n] in the kernel's output type
  MxTiling tl;
  int tiles;     // row tiles of the launch
  int n_blocks;  // columns of the launch's tiles
  int run;       // 32-row tiles: column blocks of 32 that a workgroup takes one after the other
};

// The whole product of the group form, the rows' quantization included (g.tile is filled for each launch).
void launch_mx_gemm_groups(const MxGemmArgs& a, MxGroups& g, int out_dtype, hipStream_t s);

}  // namespace e4b
