// Grouped product of microscaled operands: rows of MXFP4 activations times the MXFP4 weights of their
// expert, y[m, n] = sum over blocks b of 2^(sa[m, b] + sw[n, b] - 254) * sum_{i < 32} a[m, b, i] w[n, b, i],
// on the block-scaled matrix instructions (v_mfma_scale_f32_32x32x64_f8f6f4, both operands e2m1): the
// products and the scaling are exact, the sums fp32. A scale byte of 255 makes its block NaN.
//
// Operand layout: lane l of an MFMA holds row l % 32 and the 32 values of one block (16 bytes, one
// scale byte), half h = l / 32 the second block of the 64. The order of K is free as long as both
// operands agree, so in a chunk of 256 values (eight blocks) step j takes block 4 h + j of lane half
// h: a lane's four steps are 64 contiguous bytes of its row and the four bytes of one scale word, from
// which the instruction selects byte j. The weights are the first operand: lane l then holds the sums
// of row (token) l % 32 and weight rows 8 (i / 4) + 4 (l / 32) + i % 4, i = 0..15.
#pragma once

#include "common.h"
#include "mx.h"
#include "mx_launch.h"

namespace e4b {

typedef int i32x8_t __attribute__((ext_vector_type(8)));
typedef float mx_acc_t __attribute__((ext_vector_type(16)));

template <int J>
E4B_DEV mx_acc_t mx_mfma(const uint4& w, const uint4& a, uint32_t ws, uint32_t as, const mx_acc_t& c) {
  const i32x8_t wv = {static_cast<int>(w.x), static_cast<int>(w.y), static_cast<int>(w.z), static_cast<int>(w.w)};
  const i32x8_t av = {static_cast<int>(a.x), static_cast<int>(a.y), static_cast<int>(a.z), static_cast<int>(a.w)};
  constexpr int kE2M1 = 4;
  return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(wv, av, c, kE2M1, kE2M1, J, static_cast<int>(ws), J,
                                                         static_cast<int>(as));
}

// Four scale bytes of a weight row from block b on (rows of scale bytes start at any address); blocks
// past the row's end, whose activation codes are zero, get the byte of 1.
E4B_DEV uint32_t mx_scales4(const uint8_t* row, int b, int blocks) {
  uint32_t v;
  if (b + 4 <= blocks) {
    __builtin_memcpy(&v, row + b, 4);
  } else {
    v = 0x7f7f7f7fu;
    for (int j = 0; b + j < blocks; ++j) v = (v & ~(0xffu << (8 * j))) | (static_cast<uint32_t>(row[b + j]) << (8 * j));
  }
  return v;
}

constexpr int kMxRowThreads = 256;

// Activation rows to padded codes and scale bytes (a block with an infinity or a NaN: 255). Thread =
// piece of eight values; pieces past k are zero.
template <int DT>
__global__ void __launch_bounds__(kMxRowThreads) mx_rows_kernel(const void* __restrict__ x, int64_t k, int row_pieces,
                                                                int64_t pieces, uint32_t* __restrict__ codes,
                                                                uint8_t* __restrict__ scales) {
  const int64_t p = int64_t(blockIdx.x) * kMxRowThreads + threadIdx.x;
  if (p >= pieces) return;  // whole quads: a row's pieces are a multiple of 32
  const int64_t row = p / row_pieces;
  const int q = static_cast<int>(p - row * row_pieces);
  const bool in = q < k / 8;
  MxPiece<DT> v = mx_load<DT>(x, row * (k / 8) + (in ? q : 0));
  const uint32_t m = quad_max(mx_amax<DT>(v));
  const uint32_t e = mx_scale_byte<DT>(m, true);
  const uint32_t c = mx_codes<DT>(v, e);
  codes[p] = in ? c : 0u;
  if ((p & 3) == 0) scales[p >> 2] = in ? static_cast<uint8_t>(e) : 0;
}

// A row tile of the group form: its expert (-1: outside [0, E)) and rows row0 .. end - 1. The tiles of
// group g are ceil(size / TM) consecutive ones, in group order; every wave finds its tile by itself
// (eight groups per lane, a prefix sum over the lanes).
template <int TM>
E4B_DEV void mx_group_tile(const MxGemmArgs& p, const MxGroups& go, int t, int& e, int& row0, int& end) {
  int g = t, first = t;
  if (!p.one) {
    const int lane = threadIdx.x & (kWave - 1);
    constexpr int kPer = kMxGroupsMax / kWave;
    int mine = 0;
    for (int i = 0; i < kPer; ++i) {
      const int gi = kPer * lane + i;
      if (gi < p.groups) mine += (go.off[gi + 1] - go.off[gi] + TM - 1) / TM;
    }
    int upto = mine;
#pragma unroll
    for (int o = 1; o < kWave; o <<= 1) {
      const int v = __shfl_up(upto, o);
      upto += lane >= o ? v : 0;
    }
    const int owner = __builtin_ctzll(__ballot(upto > t));
    first = __builtin_amdgcn_readlane(upto - mine, owner);
    g = kPer * owner;
    for (;; ++g) {
      const int n = (go.off[g + 1] - go.off[g] + TM - 1) / TM;
      if (first + n > t) break;
      first += n;
    }
  }
  const int64_t id = p.ids[g];
  e = id >= 0 && id < p.w.num_experts ? static_cast<int>(id) : -1;
  row0 = go.off[g] + (t - first) * TM;
  end = min(row0 + TM, go.off[g + 1]);
}

// Four sums of a row to the output's columns n .. n + 3.
template <int ODT>
E4B_DEV void mx_store4(void* out, int64_t at, int left, bool vec, const float (&v)[4]) {
  if constexpr (ODT == E4B_FP32) {
    float* o = static_cast<float*>(out) + at;
    if (vec && left >= 4) {
      *reinterpret_cast<float4*>(o) = make_float4(v[0], v[1], v[2], v[3]);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (j < left) o[j] = v[j];
    }
  } else {
    uint16_t* o = static_cast<uint16_t*>(out) + at;
    const uint16_t h[4] = {from_f<ODT>(v[0]), from_f<ODT>(v[1]), from_f<ODT>(v[2]), from_f<ODT>(v[3])};
    if (vec && left >= 4) {
      *reinterpret_cast<uint2*>(o) = make_uint2(pack2(h[0], h[1]), pack2(h[2], h[3]));
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (j < left) o[j] = h[j];
    }
  }
}

// A tile of at most 32 rows times 32 weight rows per workgroup: each of the four waves takes every
// fourth chunk of K straight into the operand registers, their sums join in LDS. Bound by the weights'
// bytes: each is read once per tile.
constexpr int kMxTileM = 32;
constexpr int kMxNarrowWaves = 4;

template <int ODT>
__global__ void __launch_bounds__(kMxNarrowWaves* kWave) mx_narrow_kernel(MxGemmArgs p, MxGroups go) {
  __shared__ float red[kMxNarrowWaves][32][33];
  const int tid = threadIdx.x;
  const int lane = tid & (kWave - 1);
  const int wid = __builtin_amdgcn_readfirstlane(tid) / kWave;
  const int half = lane >> 5, r32 = lane & 31;
  const int t = blockIdx.x / p.n_blocks, nb = blockIdx.x % p.n_blocks;
  int e, row0, end;
  mx_group_tile<kMxTileM>(p, go, t, e, row0, end);
  const int64_t n = p.w.n, n0 = int64_t(nb) * 32;
  const int chunks = static_cast<int>((p.w.k + kMxChunk - 1) / kMxChunk);
  mx_acc_t acc = {};
  if (e >= 0) {
    const int blocks = static_cast<int>(p.w.k / kMxBlock);
    const int64_t wrow = int64_t(e) * n + min(n0 + r32, n - 1);  // rows past n are not stored
    const uint8_t* wc = p.w.packed + wrow * (p.w.k / 2);
    const uint8_t* ws = static_cast<const uint8_t*>(p.w.absmax) + wrow * blocks;
    const int64_t arow = min(row0 + r32, end - 1);  // columns past the tile's rows are not stored
    const uint8_t* ac = p.a + arow * (chunks * 128);
    const uint8_t* as = p.as + arow * (chunks * 8);
    for (int c = wid; c < chunks; c += kMxNarrowWaves) {
      uint4 wv[4], av[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int b = 8 * c + 4 * half + j;
        wv[j] = *reinterpret_cast<const uint4*>(wc + 16 * (b < blocks ? b : 0));
        av[j] = *reinterpret_cast<const uint4*>(ac + 16 * b);
      }
      const uint32_t wsc = mx_scales4(ws, 8 * c + 4 * half, blocks);
      const uint32_t asc = *reinterpret_cast<const uint32_t*>(as + 8 * c + 4 * half);
      acc = mx_mfma<0>(wv[0], av[0], wsc, asc, acc);
      acc = mx_mfma<1>(wv[1], av[1], wsc, asc, acc);
      acc = mx_mfma<2>(wv[2], av[2], wsc, asc, acc);
      acc = mx_mfma<3>(wv[3], av[3], wsc, asc, acc);
    }
  }
#pragma unroll
  for (int i = 0; i < 16; ++i) red[wid][8 * (i / 4) + 4 * half + i % 4][r32] = acc[i];
  __syncthreads();
  const int row = row0 + (tid >> 3), c0 = 4 * (tid & 7);
  if (row >= end) return;
  float v[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    float s = 0.0f;
#pragma unroll
    for (int w = 0; w < kMxNarrowWaves; ++w) s += red[w][c0 + j][tid >> 3];
    v[j] = s;
  }
  const int64_t left = n - (n0 + c0);
  if (left > 0) mx_store4<ODT>(p.out, int64_t(row) * n + n0 + c0, static_cast<int>(min<int64_t>(left, 4)), n % 4 == 0, v);
}

}  // namespace e4b
