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

#include <utility>

#include "common.h"
#include "mx.h"
#include "mx_launch.h"

namespace e4b {

typedef int i32x8_t __attribute__((ext_vector_type(8)));
typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));
typedef float mx_acc_t __attribute__((ext_vector_type(16)));

template <int J>
E4B_DEV mx_acc_t mx_mfma(const u32x4_t& w, const u32x4_t& a, uint32_t ws, uint32_t as, const mx_acc_t& c) {
  const i32x8_t wv = {static_cast<int>(w.x), static_cast<int>(w.y), static_cast<int>(w.z), static_cast<int>(w.w)};
  const i32x8_t av = {static_cast<int>(a.x), static_cast<int>(a.y), static_cast<int>(a.z), static_cast<int>(a.w)};
  constexpr int kE2M1 = 4;
  return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(wv, av, c, kE2M1, kE2M1, J, static_cast<int>(ws), J,
                                                         static_cast<int>(as));
}

// Four scale bytes of a weight row from block b on. Rows of scale bytes start at any address and are read in
// whole words: one that would pass the row's end is read back from it and shifted where it is used (`past` bytes;
// blocks past the end, whose activation codes are zero, get byte 0). Rows of fewer than four: by bytes.
struct MxScales {
  uint32_t word;
  int past;
};
E4B_DEV MxScales mx_scales4(const uint8_t* row, int b, int blocks) {
  MxScales s = {0, 0};
  if (blocks >= 4) {
    s.past = min(max(b + 4 - blocks, 0), 4);
    __builtin_memcpy(&s.word, row + min(b, blocks - 4), 4);
  } else {
    for (int j = 0; b + j < blocks; ++j) s.word |= static_cast<uint32_t>(row[b + j]) << (8 * j);
  }
  return s;
}
E4B_DEV uint32_t mx_scale_word(const MxScales& s) { return s.past < 4 ? s.word >> (8 * s.past) : 0u; }

constexpr int kMxRowThreads = 256;

// Activation rows to padded codes and scale bytes (a block with an infinity or a NaN: 255). Thread =
// piece of eight values; 32 threads take a chunk of a row, pieces past k are zero. Bound by HBM: 16,384 rows of
// 2,880 bf16 values (120 MB with the codes) take 24 us, 5.0 TB/s.
template <int DT>
__global__ void __launch_bounds__(kMxRowThreads) mx_rows_kernel(const void* __restrict__ x, int row_values, uint32_t row_chunks,
                                                                uint32_t chunks, uint32_t* __restrict__ codes,
                                                                uint8_t* __restrict__ scales) {
  constexpr int kPieces = kMxChunk / 8;
  const uint32_t chunk = blockIdx.x * (kMxRowThreads / kPieces) + threadIdx.x / kPieces;
  if (chunk >= chunks) return;
  const uint32_t row = chunk / row_chunks;
  const int q = static_cast<int>(chunk - row * row_chunks) * kPieces + threadIdx.x % kPieces;
  const int64_t p = int64_t(blockIdx.x) * kMxRowThreads + threadIdx.x;
  const bool in = q < row_values / 8;
  MxPiece<DT> v = mx_load<DT>(x, int64_t(row) * (row_values / 8) + (in ? q : 0));
  const uint32_t m = quad_max(mx_amax<DT>(v));
  const uint32_t e = mx_scale_byte(m, true);
  const uint32_t c = mx_codes<DT>(v, e);
  codes[p] = in ? c : 0u;
  if ((p & 3) == 0) scales[p >> 2] = in ? static_cast<uint8_t>(e) : 0;
}

// The group of row tile t, its first tile and its number of tiles: every wave finds them by itself in the
// launch's table of first tiles, by two reads of 64 and of eight entries.
E4B_DEV void mx_find_group(const MxGemmArgs& p, const MxGroups& go, int t, int& g, int& first, int& count) {
  if (p.tl.one) {  // every group is one tile
    g = first = t;
    count = 1;
    return;
  }
  static_assert(kMxGroupsMax == 8 * kWave, "eight groups per lane");
  const int lane = threadIdx.x & (kWave - 1);
  const int owner = __builtin_ctzll(__ballot(go.tile[8 * lane + 8] > t));
  g = 8 * owner + __builtin_ctzll(__ballot(go.tile[8 * owner + (lane & 7) + 1] > t));
  g = __builtin_amdgcn_readfirstlane(g);
  first = go.tile[g];
  count = go.tile[g + 1] - first;
}

// A workgroup's tile: expert (-1: the group's id is outside [0, E)), rows row0 .. end - 1, column block nb.
struct MxTile {
  int e, row0, end, nb;
};

// Items (row tile, column block) in group order, within a group the row tiles of one column block
// next to each other; the launch's items are cut into eight equal runs, one per XCD (workgroups go
// round-robin over the XCDs), so the tiles that share weights share an L2.
constexpr int kXcds = 8;
E4B_DEV bool mx_tile(const MxGemmArgs& p, const MxGroups& go, MxTile& o) {
  const int total = p.tiles * p.n_blocks;
  const int per = (total + kXcds - 1) / kXcds;
  const int w = static_cast<int>(blockIdx.x % kXcds) * per + static_cast<int>(blockIdx.x / kXcds);
  if (static_cast<int>(blockIdx.x / kXcds) >= per || w >= total) return false;
  int g, first, count;
  mx_find_group(p, go, w / p.n_blocks, g, first, count);
  const int i = w - first * p.n_blocks;
  o.nb = i / count;
  const int64_t id = p.ids[g];
  o.e = id >= 0 && id < p.w.num_experts ? static_cast<int>(id) : -1;
  const int lo = go.off[g], hi = go.off[g + 1];
  o.row0 = lo + (i % count) * p.tl.tm;
  o.end = min(o.row0 + p.tl.tm, hi);
  return true;
}

// Four sums of a row to the output's columns n .. n + 3, at any address.
template <int ODT>
E4B_DEV void mx_store4(void* out, int64_t at, int left, const float (&v)[4]) {
  if constexpr (ODT == E4B_FP32) {
    float* o = static_cast<float*>(out) + at;
    if (left >= 4) {
      __builtin_memcpy(o, v, 16);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (j < left) o[j] = v[j];
    }
  } else {
    uint16_t* o = static_cast<uint16_t*>(out) + at;
    const uint16_t h[4] = {from_f<ODT>(v[0]), from_f<ODT>(v[1]), from_f<ODT>(v[2]), from_f<ODT>(v[3])};
    if (left >= 4) {
      __builtin_memcpy(o, h, 8);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (j < left) o[j] = h[j];
    }
  }
}

// Four pieces of 16 bytes per lane, piece 4 (i / 2) + l / 16 of row 16 (i % 2) + l % 16 in v[i] as loaded (64
// contiguous bytes of a row by four lanes), to the operands' order: v[j] piece 4 (l / 32) + j of row l % 32. A
// 4 x 4 transposition of registers and groups of 16 lanes, in two steps of 2 x 2.
E4B_DEV void mx_to_rows(u32x4_t (&v)[4]) {
#pragma unroll
  for (int d = 0; d < 4; ++d) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const auto s = __builtin_amdgcn_permlane32_swap(v[i][d], v[2 + i][d], false, false);
      v[i][d] = s[0];
      v[2 + i][d] = s[1];
    }
#pragma unroll
    for (int i = 0; i < 4; i += 2) {
      const auto s = __builtin_amdgcn_permlane16_swap(v[i][d], v[i + 1][d], false, false);
      v[i][d] = s[0];
      v[i + 1][d] = s[1];
    }
  }
}

// A tile of at most 32 rows times 32 weight rows per workgroup: each of the four waves takes every
// fourth chunk of K straight into the operand registers, the next one's loads in flight while it computes; their
// sums join in LDS. Bound by the weights' bytes: each is read once per tile. Loads take 64 contiguous bytes of a
// row by four lanes and are turned in registers (mx_to_rows).
// 148 rows over 32 experts of 2,880 x 2,880 (141 MB of weights and scales): 30.4 us, 4.6 TB/s; with each lane
// loading its own row's 64 bytes 31.0, at three waves per SIMD instead of four 32.0, without the next chunk's
// loads in flight 33.6.
// DT >= 0: the workgroup quantizes its rows itself into LDS, from values of type DT, and takes p.run column blocks one
// after the other with them, each block's first loads in flight while the one before is joined (the 148 rows: 30.4
// us for everything, against 4.4 + 30.4 in two kernels).
constexpr int kMxTileM = 32;
constexpr int kMxNarrowWaves = 4;

template <int ODT, int DT>
__global__ void __launch_bounds__(kMxNarrowWaves* kWave, 4) mx_narrow_kernel(MxGemmArgs p, MxGroups go) {
  __shared__ float red[kMxNarrowWaves][32][33];
  extern __shared__ u32x4_t own[];  // DT >= 0: the rows' codes, 8 * chunks pieces each, then their scale bytes
  const int tid = threadIdx.x;
  const int lane = tid & (kWave - 1);
  const int wid = __builtin_amdgcn_readfirstlane(tid) / kWave;
  const int half = lane >> 5, r32 = lane & 31;
  MxTile t;
  if (!mx_tile(p, go, t)) return;
  const int e = t.e, row0 = t.row0, end = t.end, rows = end - row0;
  const int n = static_cast<int>(p.w.n);
  const int blocks = static_cast<int>(p.w.k / kMxBlock);
  const int chunks = static_cast<int>(mx_chunks(p.w.k));
  const int run = DT < 0 ? 1 : p.run;  // the workgroup's column blocks
  const int first = t.nb * run, last = min(first + run, (n + 31) / 32);
  const int r16 = lane & 15, quarter = lane >> 4;
  const int arow = min(r32, rows - 1);  // columns past the tile's rows are not stored
  const uint8_t *wc[2], *ac[2];         // the rows of which the lane loads pieces
  const uint8_t *ws, *as = p.as + int64_t(row0 + arow) * (chunks * 8);
  auto aim = [&](int nb) {  // at a column block's weights; rows past n are not stored
#pragma unroll
    for (int i = 0; i < 2; ++i)
      wc[i] = p.w.packed + (int64_t(e) * n + min(32 * nb + 16 * i + r16, n - 1)) * (16 * blocks);
    ws = static_cast<const uint8_t*>(p.w.absmax) + (int64_t(e) * n + min(32 * nb + r32, n - 1)) * blocks;
  };
#pragma unroll
  for (int i = 0; i < 2; ++i) ac[i] = p.a + int64_t(row0 + min(16 * i + r16, rows - 1)) * (chunks * 128);
  struct Part {
    u32x4_t w[4], a[4];
    MxScales ws;
    uint32_t as;
  } even, odd;
  auto load = [&](Part& f, int c) {
    const int b0 = 8 * c + 4 * half;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int b = 8 * c + 4 * (j / 2) + quarter;
      f.w[j] = *reinterpret_cast<const u32x4_t*>(wc[j % 2] + 16 * (b < blocks ? b : 0));
      if constexpr (DT < 0) f.a[j] = *reinterpret_cast<const u32x4_t*>(ac[j % 2] + 16 * b);
    }
    f.ws = mx_scales4(ws, b0, blocks);
    if constexpr (DT < 0) f.as = *reinterpret_cast<const uint32_t*>(as + b0);
  };
  uint8_t* const own_scales = reinterpret_cast<uint8_t*>(own + rows * 8 * chunks);
  mx_acc_t acc;
  auto add = [&](Part& f, int c) {
    if constexpr (DT >= 0) {
      const int b0 = 8 * (arow * chunks + c) + 4 * half;
#pragma unroll
      for (int j = 0; j < 4; ++j) f.a[j] = own[b0 + j];
      f.as = *reinterpret_cast<const uint32_t*>(own_scales + b0);
    } else {
      mx_to_rows(f.a);
    }
    mx_to_rows(f.w);
    const uint32_t wsc = mx_scale_word(f.ws);
    acc = mx_mfma<0>(f.w[0], f.a[0], wsc, f.as, acc);
    acc = mx_mfma<1>(f.w[1], f.a[1], wsc, f.as, acc);
    acc = mx_mfma<2>(f.w[2], f.a[2], wsc, f.as, acc);
    acc = mx_mfma<3>(f.w[3], f.a[3], wsc, f.as, acc);
  };
  const bool busy = e >= 0 && wid < chunks;
  if (busy) {
    aim(first);
    load(even, wid);
  }
  if constexpr (DT >= 0) {
    constexpr int kThreads = kMxNarrowWaves * kWave, kAhead = 4;
    const int pieces = 32 * chunks, in = 4 * blocks;  // of a row, eight values each: padded and given
    for (int q0 = tid; q0 < rows * pieces; q0 += kAhead * kThreads) {  // whole quads: a block's four pieces
      MxPiece<DT> v[kAhead];
      bool some[kAhead];
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        const int q = min(q0 + u * kThreads, rows * pieces - 1), r = q / pieces;
        some[u] = q - r * pieces < in;
        v[u] = mx_load<DT>(p.x, int64_t(row0 + r) * in + (some[u] ? q - r * pieces : 0));
      }
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        const int q = q0 + u * kThreads;
        const uint32_t s = mx_scale_byte(quad_max(mx_amax<DT>(v[u])), true);
        const uint32_t code = mx_codes<DT>(v[u], s);
        if (q < rows * pieces) {
          reinterpret_cast<uint32_t*>(own)[q] = some[u] ? code : 0u;
          if ((q & 3) == 0) own_scales[q >> 2] = some[u] ? static_cast<uint8_t>(s) : 0;
        }
      }
    }
    __syncthreads();
  }
  for (int nb = first; nb < (DT < 0 ? first + 1 : last); ++nb) {
    acc = mx_acc_t{};
    if (busy) {
      for (int c = wid; c < chunks; c += 2 * kMxNarrowWaves) {
        const int d = c + kMxNarrowWaves;
        if (d < chunks) load(odd, d);
        add(even, c);
        if (d >= chunks) break;
        if (d + kMxNarrowWaves < chunks) load(even, d + kMxNarrowWaves);
        add(odd, d);
      }
      if (DT >= 0 && nb + 1 < last) {  // the next block's first chunk, in flight while this one is joined
        aim(nb + 1);
        load(even, wid);
      }
    }
    if (DT >= 0 && nb > first) __syncthreads();  // the previous block's sums have been read
#pragma unroll
    for (int i = 0; i < 16; ++i) red[wid][8 * (i / 4) + 4 * half + i % 4][r32] = acc[i];
    __syncthreads();
    const int row = tid >> 3, c0 = 4 * (tid & 7), left = n - 32 * nb - c0;
    if (row < rows && left > 0) {
      float v[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float s = 0.0f;
#pragma unroll
        for (int w = 0; w < kMxNarrowWaves; ++w) s += red[w][c0 + j][row];
        v[j] = s;
      }
      mx_store4<ODT>(p.out, int64_t(row0 + row) * n + 32 * nb + c0, left, v);
    }
  }
}

// ---- large groups

// f(integral_constant<int, 0>) ... : indices known at compile time, so that the accumulators never need
// an address.
template <class F, int... I>
E4B_DEV void mx_for_impl(F&& f, std::integer_sequence<int, I...>) {
  (f(std::integral_constant<int, I>{}), ...);
}
template <int N, class F>
E4B_DEV void mx_for(F&& f) {
  mx_for_impl(f, std::make_integer_sequence<int, N>{});
}

constexpr int kMxWideThreads = 256;

// `size` bytes from base on; 16 of them at offset + uniform, zeros at and past the end.
E4B_DEV __amdgpu_buffer_rsrc_t mx_rows_of(const uint8_t* base, int64_t size) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(base), 0, static_cast<int>(static_cast<uint32_t>(size)), 0x00027000);
}
E4B_DEV u32x4_t mx_piece(__amdgpu_buffer_rsrc_t rows, uint32_t offset, uint32_t uniform) {
  return __builtin_amdgcn_raw_buffer_load_b128(rows, static_cast<int>(offset), static_cast<int>(uniform), 0);
}

// Two sums as a pair of 16-bit outputs.
template <int ODT>
E4B_DEV uint32_t mx_pair(float a, float b) {
  typedef float f32x2_t __attribute__((ext_vector_type(2)));
  const f32x2_t v = {a, b};
  if constexpr (ODT == E4B_BF16) return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, bf16x2_t));
  else return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, f16x2_t));
}

// An MFMA block's sums of a lane, columns 8 (i / 4) + 4 half + i % 4 of row l % 32, to a tile's output rows, the
// block's first output at byte `uniform` of the buffer (rows past the tile's last lie past its end).
// All 32 columns of 16-bit outputs: v_permlane32_swap joins the halves' runs of four into eight neighbouring
// columns, v_permlane16_swap hands a lane's second eight to the lane sixteen rows on for that lane's first
// eight: four lanes then write a row's whole 64 bytes, sixteen rows per store. `offset`: of row l % 16,
// columns 16 (l / 16 % 2) + 8 half.
template <int ODT>
E4B_DEV void mx_store_whole(__amdgpu_buffer_rsrc_t out, uint32_t offset, uint32_t uniform, uint32_t row_bytes,
                            const mx_acc_t& v) {
  uint32_t o[2][4];
#pragma unroll
  for (int g = 0; g < 2; ++g) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const auto s = __builtin_amdgcn_permlane32_swap(mx_pair<ODT>(v[8 * g + 2 * j], v[8 * g + 2 * j + 1]),
                                                      mx_pair<ODT>(v[8 * g + 4 + 2 * j], v[8 * g + 5 + 2 * j]), false, false);
      o[g][j] = s[0];
      o[g][2 + j] = s[1];
    }
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const auto s = __builtin_amdgcn_permlane16_swap(o[0][j], o[1][j], false, false);
    o[0][j] = s[0];
    o[1][j] = s[1];
  }
#pragma unroll
  for (int g = 0; g < 2; ++g)
    __builtin_amdgcn_raw_buffer_store_b128(u32x4_t{o[g][0], o[g][1], o[g][2], o[g][3]}, out, static_cast<int>(offset),
                                           static_cast<int>(uniform + 16 * g * row_bytes), 0);
}
// The first `left` of the 32 columns, or fp32 outputs. `offset`: of row l % 32, column 4 half.
template <int ODT>
E4B_DEV void mx_store_part(__amdgpu_buffer_rsrc_t out, uint32_t offset, uint32_t uniform, int left, int half,
                           const mx_acc_t& v) {
  constexpr int kOut = ODT == E4B_FP32 ? 4 : 2;
#pragma unroll
  for (int g = 0; g < 4; ++g) {
    u32x4_t o;  // the next output lowest
    if constexpr (ODT == E4B_FP32)
      o = u32x4_t{__float_as_uint(v[4 * g]), __float_as_uint(v[4 * g + 1]), __float_as_uint(v[4 * g + 2]),
                  __float_as_uint(v[4 * g + 3])};
    else
      o = u32x4_t{mx_pair<ODT>(v[4 * g], v[4 * g + 1]), mx_pair<ODT>(v[4 * g + 2], v[4 * g + 3]), 0, 0};
    const int c = 8 * g + 4 * half, at = static_cast<int>(uniform + 8 * g * kOut);
    if (ODT == E4B_FP32 && c + 4 <= left) {
      __builtin_amdgcn_raw_buffer_store_b128(o, out, static_cast<int>(offset), at, 0);
      continue;
    }
#pragma unroll 1
    for (int j = 0; j < 4 && c + j < left; ++j) {
      const int to = static_cast<int>(offset + kOut * j);
      if constexpr (ODT == E4B_FP32) {
        __builtin_amdgcn_raw_buffer_store_b32(o[0], out, to, at, 0);
        o = u32x4_t{o[1], o[2], o[3], 0};
      } else {
        __builtin_amdgcn_raw_buffer_store_b16(static_cast<uint16_t>(o[0]), out, to, at, 0);
        o = u32x4_t{__builtin_amdgcn_alignbit(o[1], o[0], 16), o[1] >> 16, 0, 0};
      }
    }
  }
}

// A tile of 256 rows times 256 weight rows, four waves (one per SIMD) of 128 x 128. Both operands pass through LDS
// a chunk of 256 values at a time: 128-byte rows whose eight 16-byte pieces are stored in the order piece ^ (row
// / 2 & 7): a row is half of the 64 banks, and sixteen rows' reads of one piece fall in distinct ones, as do the
// stores (eight lanes a row). Chunk g is computed from one buffer while chunk g + 1 goes from registers into the other, and a register
// that is stored takes its piece of chunk g + 2: every load has a whole chunk's time. Fragments are read a
// step ahead (two sets); the one barrier per chunk stands before its last step, which then reads the next
// chunk's first fragments. The order is pinned: left to the compiler, the fragments are read right before
// their use.
// The workgroups (one per CU) stay, and the chunks of a workgroup's tiles are one stream: the first chunks of its
// next tile are loaded while the last ones of this tile are computed, and a tile's stores drain while the next one
// is computed.
// 16,384 rows over 32 experts of 5,760 x 2,880: 242 to 250 us on most cards, medians of 270 to 290 on some (1.9 to 2.2
// PFLOP/s). On one of the former the products alone take 117 us (the card's power limit: 105 for a loop of these
// instructions on random operands), 139 with the LDS reads; the loads and LDS stores of the chunks bring it to 200, the
// output's 189 MB to 246. Tried against it: 128 x 256 tiles, two
// workgroups per CU, 270 us; the same tiles without persistent workgroups 258; fewer row blocks for the last,
// mostly empty row tile of a group 250 (such a tile waits for its weights all the same).
constexpr int kMxWideM = 256, kMxWideN = 256;

template <int ODT>
__global__ void __launch_bounds__(kMxWideThreads, 1) mx_wide_kernel(MxGemmArgs p, MxGroups go) {
  constexpr int NA = 4, NB = 4, TN = kMxWideN, TM = kMxWideM;
  constexpr int PW = TN / 32, PA = TM / 32;  // 16-byte pieces per thread and chunk
  __shared__ u32x4_t wl[2][TN * 8];
  __shared__ u32x4_t al[2][TM * 8];
  __shared__ u32x2_t wsl[2][TN], asl[2][TM];
  __shared__ int tab[3][kMxGroupsMax + 1];  // first row, first tile and expert (-1: none) of each group
  constexpr int kItems = 128;
  __shared__ int4 items[kItems];
  const int tid = threadIdx.x;
  for (int i = tid; i <= p.groups; i += kMxWideThreads) {
    tab[0][i] = go.off[i];
    tab[1][i] = go.tile[i];
    const int64_t id = i < p.groups ? p.ids[i] : -1;
    tab[2][i] = id >= 0 && id < p.w.num_experts ? static_cast<int>(id) : -1;
  }
  __syncthreads();
  // the workgroup's items: of its XCD's run, every 32nd or as many as workgroups there are
  const int total = p.tiles * p.n_blocks, per = (total + kXcds - 1) / kXcds;
  const int xcd = static_cast<int>(blockIdx.x) % kXcds;
  const int stride = static_cast<int>(gridDim.x) / kXcds;
  const int last = min((xcd + 1) * per, total);
  int item = xcd * per + static_cast<int>(blockIdx.x) / kXcds;
  if (item >= last) return;

  const int lane = tid & (kWave - 1);
  const int wid = __builtin_amdgcn_readfirstlane(tid) / kWave;
  const int wn = wid & 1, wm = wid >> 1;  // the wave's columns and rows of the tile
  const int half = lane >> 5, r32 = lane & 31;
  const int64_t n = p.w.n;
  const int blocks = static_cast<int>(p.w.k / kMxBlock);
  const int chunks = static_cast<int>(mx_chunks(p.w.k));  // two at least: the loads are two ahead, at most one tile
  const uint32_t wstride = 16 * blocks, astride = 128 * chunks;

  // the workgroup's next kItems tiles, one per thread, from the tables: a tile is then one broadcast read
  auto fill = [&](int first_item) {
    const int w = first_item + tid * stride;
    if (tid < kItems && w < last) {
      const int t = w / p.n_blocks;
      int lo = 0, hi = p.groups;  // the group whose tiles hold t
      while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (tab[1][mid] <= t) lo = mid;
        else hi = mid;
      }
      const int first = tab[1][lo], count = tab[1][lo + 1] - first, i = w - first * p.n_blocks;
      const int nb = i / count, row0 = tab[0][lo] + (i - nb * count) * TM;
      items[tid] = make_int4(tab[2][lo], nb, row0, min(row0 + TM, tab[0][lo + 1]));
    }
  };
  int filled = item;  // the first item of the table
  fill(filled);
  __syncthreads();
  auto tile_of = [&](int w) {
    const int4 v = items[(w - filled) / stride];
    return MxTile{__builtin_amdgcn_readfirstlane(v.x), __builtin_amdgcn_readfirstlane(v.z),
                  __builtin_amdgcn_readfirstlane(v.w), __builtin_amdgcn_readfirstlane(v.y)};
  };
  // a tile's operands. Rows past the ends and pieces past the last row's end are zeros; a piece past another
  // row's end is the next row's first, against zero codes. A group without an expert computes on expert 0 and
  // stores zeros.
  struct Source {
    __amdgpu_buffer_rsrc_t w, a;
    const uint8_t *ws, *as;  // ws: `before` bytes (8, fewer at the stack's start) before the tile's first
    int wrows, arows, before;
  };
  auto source_of = [&](const MxTile& t) {
    Source o;
    const int64_t n0 = int64_t(t.nb) * TN, first = int64_t(max(t.e, 0)) * n + n0;
    o.wrows = min(static_cast<int>(n) - t.nb * TN, TN);
    o.arows = t.end - t.row0;
    o.w = mx_rows_of(p.w.packed + first * wstride, int64_t(o.wrows) * wstride);
    o.a = mx_rows_of(p.a + int64_t(t.row0) * astride, int64_t(o.arows) * astride);
    o.before = first * blocks < 8 ? static_cast<int>(first * blocks) : 8;
    o.ws = static_cast<const uint8_t*>(p.w.absmax) + (first * blocks - o.before);
    o.as = p.as + int64_t(t.row0) * (chunks * 8);
    return o;
  };

  const int part = tid & 7, prow = tid >> 3;
  const uint32_t woff = prow * wstride + 16 * part, aoff = prow * astride + 16 * part;
  u32x4_t wr[PW], ar[PA];
  u32x2_t wsr, asr;
  int wshift = 0;
  uint64_t wmask = 0;
  const int slot = prow * 8 + (part ^ ((prow >> 1) & 7));  // of rows 32 i + prow: 32 rows apart, the same order
  // eight scale bytes of a weight row, those that would pass the row's end read back from it (in a row of fewer, at the
  // stack's start, from there); shifted and cut to the row's where they are stored: the load is not waited for here
  auto load_s = [&](const Source& f, int c) {
    const int left = blocks - 8 * c, past = max(8 - left, 0);
    const int at = min(tid, f.wrows - 1) * blocks + (8 * c - past + f.before);
    __builtin_memcpy(&wsr, f.ws + static_cast<uint32_t>(max(at, 0)), 8);
    wshift = 8 * (past + min(at, 0)) & 63;
    wmask = left >= 8 ? ~0ull : (1ull << (8 * max(left, 0))) - 1;
    asr = *reinterpret_cast<const u32x2_t*>(f.as + (static_cast<uint32_t>(min(tid, f.arows - 1)) * (chunks * 8) + 8 * c));
  };
  auto store_s = [&](int buf) {
    wsl[buf][tid] = __builtin_bit_cast(u32x2_t, (__builtin_bit_cast(uint64_t, wsr) >> wshift) & wmask);
    asl[buf][tid] = asr;
  };
  auto load = [&](auto i, const Source& f, int c) {  // piece i of the thread: the weights' first
    if constexpr (i() < PW) wr[i()] = mx_piece(f.w, woff, 32 * i() * wstride + 128 * c);
    else ar[i() - PW] = mx_piece(f.a, aoff, 32 * (i() - PW) * astride + 128 * c);
  };
  auto store = [&](auto i, int buf) {
    if constexpr (i() < PW) wl[buf][256 * i() + slot] = wr[i()];
    else al[buf][256 * (i() - PW) + slot] = ar[i() - PW];
  };

  mx_acc_t acc[NA][NB];
  mx_for<NA>([&](auto a) { mx_for<NB>([&](auto b) { acc[a()][b()] = mx_acc_t{}; }); });
  u32x4_t wf[2][NA], af[2][NB];
  uint32_t ws[NA], as[NB], wsn[NA], asn[NB];
  const int wrow = 32 * NA * wn + r32, arow = 32 * NB * wm + r32;
  auto frags = [&](auto set, int buf, int q) {
    const int x = q ^ ((r32 >> 1) & 7);
    mx_for<NA>([&](auto a) { wf[set()][a()] = wl[buf][(wrow + 32 * a()) * 8 + x]; });
    mx_for<NB>([&](auto b) { af[set()][b()] = al[buf][(arow + 32 * b()) * 8 + x]; });
  };
  auto scales = [&](int buf) {
    mx_for<NA>([&](auto a) { wsn[a()] = reinterpret_cast<const uint32_t*>(wsl[buf])[2 * (wrow + 32 * a()) + half]; });
    mx_for<NB>([&](auto b) { asn[b()] = reinterpret_cast<const uint32_t*>(asl[buf])[2 * (arow + 32 * b()) + half]; });
  };
  auto pin = [] { __builtin_amdgcn_sched_barrier(0); };

  MxTile now = tile_of(item), then = now;
  Source from = source_of(now);
  int lc = 0;  // the next chunk to load, of the tile that `from` describes
  auto advance = [&] {
    if (++lc < chunks) return;
    lc = 0;
    item += stride;
    if (item < last) {
      if (item - filled == kItems * stride) {  // (uniform; every wave has read the table's last tile)
        __syncthreads();
        filled = item;
        fill(filled);
        __syncthreads();
      }
      then = tile_of(item);
      from = source_of(then);
    } else {
      then.nb = -1;  // no tile: `from` is loaded once more, and not computed
    }
  };
  mx_for<PW + PA>([&](auto i) { load(i, from, 0); });
  load_s(from, 0);
  advance();
  mx_for<PW + PA>([&](auto i) {
    store(i, 0);
    load(i, from, lc);
  });
  store_s(0);
  load_s(from, lc);
  __syncthreads();
  frags(std::integral_constant<int, 0>{}, 0, 4 * half);
  scales(0);
  int buf = 0;
  auto chunk = [&] {  // one chunk, from LDS buffer `buf`
    const int other = 1 - buf;
    advance();
    mx_for<NA>([&](auto a) { ws[a()] = wsn[a()]; });
    mx_for<NB>([&](auto b) { as[b()] = asn[b()]; });
    mx_for<4>([&](auto j) {
      constexpr std::integral_constant<int, j() & 1> set;
      constexpr std::integral_constant<int, 1 - (j() & 1)> next;
      if constexpr (j() < 3) {
        frags(next, buf, 4 * half + j() + 1);
      } else {
        __syncthreads();
        scales(other);
        frags(next, other, 4 * half);
      }
      pin();
      mx_for<NA>([&](auto a) {
        mx_for<NB>([&](auto b) {
          acc[a()][b()] = mx_mfma<j()>(wf[set()][a()], af[set()][b()], ws[a()], as[b()], acc[a()][b()]);
        });
        pin();
        if constexpr (j() < 3) {  // the pieces of twelve slots
          constexpr int at = NA * j() + a(), lo = at * (PW + PA) / 12, hi = (at + 1) * (PW + PA) / 12;
          mx_for<hi - lo>([&](auto i) {
            constexpr std::integral_constant<int, lo + i()> piece;
            store(piece, other);
            load(piece, from, lc);
          });
          if constexpr (at == 11) {
            store_s(other);
            load_s(from, lc);
          }
          pin();
        }
      });
    });
    buf = other;
  };
  for (;;) {
    for (int c = 0; c < chunks; ++c) chunk();
    constexpr uint32_t kOut = ODT == E4B_FP32 ? 4 : 2;
    const uint32_t ostride = static_cast<uint32_t>(n) * kOut;
    const auto out = mx_rows_of(static_cast<uint8_t*>(p.out) + (int64_t(now.row0) * n + now.nb * TN) * kOut,
                                int64_t(now.end - now.row0) * ostride - now.nb * TN * kOut);
    if (now.e < 0) mx_for<NA>([&](auto a) { mx_for<NB>([&](auto b) { acc[a()][b()] = mx_acc_t{}; }); });
    const int left = static_cast<int>(n) - now.nb * TN - 32 * NA * wn;
    auto write = [&](auto&& block) {
      mx_for<NA>([&](auto a) {
        mx_for<NB>([&](auto b) {
          block(acc[a()][b()], (32 * (NB * wm + b())) * ostride + 32 * (NA * wn + a()) * kOut, left - 32 * a());
          pin();  // (else all of the tile's sums are read ahead)
        });
      });
    };
    if (ODT != E4B_FP32) {
      const uint32_t o = (lane & 15) * ostride + 2 * (lane & 16) + 16 * half;
      write([&](const mx_acc_t& v, uint32_t at, int l) {
        if (l >= 32) mx_store_whole<ODT == E4B_FP32 ? E4B_BF16 : ODT>(out, o, at, ostride, v);
      });
    }
    if (ODT == E4B_FP32 || (left < 32 * NA && left % 32)) {  // (a whole block's stores must not be repeated by parts)
      const uint32_t o = r32 * ostride + 4 * kOut * half;
      write([&](const mx_acc_t& v, uint32_t at, int l) {
        if (ODT == E4B_FP32 || l < 32) mx_store_part<ODT>(out, o, at, l, half, v);
      });
    }
    mx_for<NA>([&](auto a) { mx_for<NB>([&](auto b) { acc[a()][b()] = mx_acc_t{}; }); });
    if (then.nb < 0) return;
    now = then;
  }
}

}  // namespace e4b
