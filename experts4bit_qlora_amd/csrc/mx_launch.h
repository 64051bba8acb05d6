// Launch-side view of the products of microscaled operands (mx_gemm.h), instantiated in mx_gemm.hip.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "e4b_amd.h"

namespace e4b {

// Activation rows are quantized into the workspace with K padded to whole chunks of 256 (zero codes):
// a chunk is 128 bytes of codes and 8 scale bytes.
constexpr int kMxChunk = 256;
inline int64_t mx_chunks(int64_t k) { return (k + kMxChunk - 1) / kMxChunk; }

// Row groups given by the host: group g holds rows off[g] .. off[g + 1] - 1 for the expert ids[g].
constexpr int kMxGroupsMax = 512;
// tile: a launch's first row tile of each group.
struct MxGroups {
  int32_t off[kMxGroupsMax + 1];
  uint16_t tile[kMxGroupsMax + 1];
};
constexpr int64_t kMxRowsMax = int64_t(1) << 23;  // below 2^16 tiles of 256 rows, one more per group

// A launch's row tiles: tiles of tm rows over the groups of above lo and at most hi rows.
struct MxTiling {
  int tm, lo, hi;
  int one;  // every group is one tile
};

struct MxGemmArgs {
  const uint8_t* a;   // codes [rows, 128 * chunks]
  const uint8_t* as;  // scale bytes [rows, 8 * chunks]
  e4b_qweight w;
  const int64_t* ids;  // group form: the groups' experts (device); a group outside [0, E) gets zero rows
  int groups;
  int64_t M;
  void* out;  // [M, n] in the kernel's output type
  MxTiling tl;
  int tiles;     // row tiles of the launch
  int n_blocks;  // column blocks of the launch
};

// Rows [rows, k] of dtype to padded codes and scale bytes; a block with an infinity or a NaN takes the
// scale byte 255, which makes its products NaN.
void launch_mx_rows(const void* x, int dtype, int64_t rows, int64_t k, uint8_t* codes, uint8_t* scales, hipStream_t s);

// The whole product of the group form (g.tile is filled for each launch).
void launch_mx_gemm_groups(const MxGemmArgs& a, MxGroups& g, int out_dtype, hipStream_t s);

}  // namespace e4b
