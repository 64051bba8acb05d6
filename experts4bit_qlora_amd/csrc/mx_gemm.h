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

// Four (eight) scale bytes of a weight row from block b on. Rows of scale bytes start at any address and are
// read in whole words: one that would pass the row's end is read back from it and shifted. Blocks past
// the end, whose activation codes are zero, get byte 0.
E4B_DEV uint32_t mx_scales4(const uint8_t* row, int b, int blocks) {
  uint32_t v = 0;
  if (blocks >= 4) {
    const int past = b + 4 - blocks;
    if (past >= 4) return 0;
    __builtin_memcpy(&v, row + (past > 0 ? blocks - 4 : b), 4);
    return v >> (past > 0 ? 8 * past : 0);
  }
  for (int j = 0; b + j < blocks; ++j) v |= static_cast<uint32_t>(row[b + j]) << (8 * j);
  return v;
}
E4B_DEV u32x2_t mx_scales8(const uint8_t* row, int b, int blocks) {
  uint64_t v = 0;
  if (blocks >= 8) {
    const int past = max(b + 8 - blocks, 0);  // at most 7: a chunk has a block
    __builtin_memcpy(&v, row + (b - past), 8);
    v >>= 8 * past;
  } else {
    for (int j = 0; b + j < blocks; ++j) v |= static_cast<uint64_t>(row[b + j]) << (8 * j);
  }
  return __builtin_bit_cast(u32x2_t, v);
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
E4B_DEV bool mx_tile(const MxGemmArgs& p, const MxGroups& go, MxTile& o) {
  constexpr int kXcds = 8;
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
  o.row0 = p.tl.rest_only ? hi - (hi - lo) % p.tl.big : lo + (i % count) * p.tl.tm;
  o.end = min(o.row0 + p.tl.tm, hi);
  return true;
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
  MxTile t;
  if (!mx_tile(p, go, t)) return;
  const int e = t.e, row0 = t.row0, end = t.end;
  const int64_t n = p.w.n, n0 = int64_t(t.nb) * 32;
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
      u32x4_t wv[4], av[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int b = 8 * c + 4 * half + j;
        wv[j] = *reinterpret_cast<const u32x4_t*>(wc + 16 * (b < blocks ? b : 0));
        av[j] = *reinterpret_cast<const u32x4_t*>(ac + 16 * b);
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

constexpr int kMxWideThreads = 512;
constexpr int kMxWideTile = 256;

// Sixteen 16-bit outputs of one row, columns c0 + 8 (i / 4) + 4 half + i % 4 (an MFMA block's sums of a lane):
// v_permlane32_swap joins the halves' runs of four into eight neighbouring columns, one 16-byte store.
template <int ODT>
E4B_DEV void mx_store_block(void* out, int64_t at, int64_t left, bool vec, bool live, int half, const mx_acc_t& v) {
  if (ODT != E4B_FP32 && vec && left >= 32) {
#pragma unroll
    for (int g = 0; g < 4; g += 2) {
      uint32_t lo[2], hi[2];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        lo[j] = pack2(from_f<ODT == E4B_FP32 ? E4B_BF16 : ODT>(v[4 * g + 2 * j]),
                      from_f<ODT == E4B_FP32 ? E4B_BF16 : ODT>(v[4 * g + 2 * j + 1]));
        hi[j] = pack2(from_f<ODT == E4B_FP32 ? E4B_BF16 : ODT>(v[4 * g + 4 + 2 * j]),
                      from_f<ODT == E4B_FP32 ? E4B_BF16 : ODT>(v[4 * g + 4 + 2 * j + 1]));
      }
      const auto a = __builtin_amdgcn_permlane32_swap(lo[0], hi[0], false, false);
      const auto b = __builtin_amdgcn_permlane32_swap(lo[1], hi[1], false, false);
      const u32x4_t o = {a[0], b[0], a[1], b[1]};
      if (live) *reinterpret_cast<u32x4_t*>(static_cast<uint16_t*>(out) + at + 8 * g + 8 * half) = o;
    }
    return;
  }
  if (!live) return;
#pragma unroll
  for (int g = 0; g < 4; ++g) {
    const int c = 8 * g + 4 * half;
    const float f[4] = {v[4 * g], v[4 * g + 1], v[4 * g + 2], v[4 * g + 3]};
    if (c < left) mx_store4<ODT>(out, at + c, static_cast<int>(min<int64_t>(left - c, 4)), vec, f);
  }
}

// A tile of 256 rows times 256 weight rows per workgroup, eight waves of 64 rows x 128 weight rows (two per
// SIMD). Both operands pass through LDS a chunk of 256 values at a time: 128-byte rows whose eight 16-byte
// pieces are stored in the order piece ^ (row & 7), so that the stores (eight lanes a row) and the fragment
// reads (one piece of 32 rows) fall in distinct banks. Chunk c is computed from one buffer while chunk c + 1
// goes from registers into the other, and a register that is stored takes its piece of chunk c + 2: every
// load has a whole chunk's time. Fragments are read a step ahead (two sets); the one barrier per chunk
// stands before its last step, which then reads the next chunk's first fragments.
// A wave whose 64 rows lie past the tile's end only moves data: a tile of at most 128 rows leaves one
// computing wave per SIMD.
template <int ODT>
__global__ void __launch_bounds__(kMxWideThreads, 2) mx_wide_kernel(MxGemmArgs p, MxGroups go) {
  constexpr int TN = kMxWideTile, TM = kMxWideTile, NA = 4, NB = 2, P = 4;
  __shared__ u32x4_t wl[2][TN * 8];
  __shared__ u32x4_t al[2][TM * 8];
  __shared__ u32x2_t scl[2][TN + TM];  // the weight rows' scale bytes, then the activation rows'
  MxTile t;
  if (!mx_tile(p, go, t)) return;
  const int tid = threadIdx.x;
  const int lane = tid & (kWave - 1);
  const int wid = __builtin_amdgcn_readfirstlane(tid) / kWave;
  const int wn = wid & 1, wm = wid >> 1;  // the wave's columns and rows of the tile
  const int half = lane >> 5, r32 = lane & 31;
  const int64_t n = p.w.n, n0 = int64_t(t.nb) * TN;
  const int blocks = static_cast<int>(p.w.k / kMxBlock);
  const int chunks = (blocks + 7) / 8;
  const int e = max(t.e, 0);  // a group without an expert computes on expert 0 and stores zeros
  const uint8_t* wbase = p.w.packed + (int64_t(e) * n + n0) * (16 * int64_t(blocks));
  const uint8_t* wsbase = static_cast<const uint8_t*>(p.w.absmax) + (int64_t(e) * n + n0) * blocks;
  const uint8_t* abase = p.a + int64_t(t.row0) * (chunks * 128);
  const uint8_t* asbase = p.as + int64_t(t.row0) * (chunks * 8);
  // rows past the ends repeat the last one; their sums are not stored
  const int wlast = static_cast<int>(min<int64_t>(n - n0, TN)) - 1, alast = t.end - t.row0 - 1;
  const int part = tid & 7, prow = tid >> 3;
  uint32_t woff[P], aoff[P];
  mx_for<P>([&](auto i) {
    woff[i()] = static_cast<uint32_t>(min(64 * i() + prow, wlast)) * static_cast<uint32_t>(16 * blocks);
    aoff[i()] = static_cast<uint32_t>(min(64 * i() + prow, alast)) * static_cast<uint32_t>(chunks * 128) + 16 * part;
  });
  // waves 0..3 carry the weights' scale bytes, 4..7 the activations', eight bytes per thread and chunk
  const bool ws_wave = wid < 4;
  const uint32_t srow = static_cast<uint32_t>(min(tid & (TN - 1), ws_wave ? wlast : alast));
  const uint8_t* sbase = ws_wave ? wsbase + srow * static_cast<uint32_t>(blocks) : asbase + srow * static_cast<uint32_t>(chunks * 8);
  const int sblocks = ws_wave ? blocks : 8 * chunks;

  u32x4_t wr[P], ar[P];
  u32x2_t sr;
  auto load_w = [&](auto i, int c) {
    const int b = 8 * c + part;  // past the row's end: its first block, against zero codes
    wr[i()] = *reinterpret_cast<const u32x4_t*>(wbase + (woff[i()] + 16 * (b < blocks ? b : 0)));
  };
  auto load_a = [&](auto i, int c) { ar[i()] = *reinterpret_cast<const u32x4_t*>(abase + 128 * c + aoff[i()]); };
  auto load_s = [&](int c) { sr = mx_scales8(sbase, 8 * c, sblocks); };
  const int slot = prow * 8 + (part ^ (prow & 7));  // of rows 64 i + prow: 64 rows apart, the same order
  auto store_w = [&](auto i, int buf) { wl[buf][512 * i() + slot] = wr[i()]; };
  auto store_a = [&](auto i, int buf) { al[buf][512 * i() + slot] = ar[i()]; };
  auto store_s = [&](int buf) { scl[buf][tid] = sr; };

  mx_acc_t acc[NA][NB];
  mx_for<NA>([&](auto a) { mx_for<NB>([&](auto b) { acc[a()][b()] = mx_acc_t{}; }); });
  u32x4_t wf[2][NA], af[2][NB];
  uint32_t ws[2][NA], as[2][NB];
  const int wrow = 32 * NA * wn + r32, arow = 32 * NB * wm + r32;
  const bool live = 32 * NB * wm <= alast;  // the wave has rows
  auto frags = [&](auto set, int buf, int q) {
    const int x = (q ^ (r32 & 7));
    mx_for<NA>([&](auto a) { wf[set()][a()] = wl[buf][(wrow + 32 * a()) * 8 + x]; });
    mx_for<NB>([&](auto b) { af[set()][b()] = al[buf][(arow + 32 * b()) * 8 + x]; });
  };
  auto scales = [&](auto set, int buf) {
    const uint32_t* s = reinterpret_cast<const uint32_t*>(scl[buf]) + half;
    mx_for<NA>([&](auto a) { ws[set()][a()] = s[2 * (wrow + 32 * a())]; });
    mx_for<NB>([&](auto b) { as[set()][b()] = s[2 * (TN + arow + 32 * b())]; });
  };
  auto products = [&](auto set, auto sset, auto j, auto from, auto to) {
    mx_for<to() - from()>([&](auto i) {
      constexpr int a = (from() + i()) / NB, b = (from() + i()) % NB;
      acc[a][b] = mx_mfma<j()>(wf[set()][a], af[set()][b], ws[sset()][a], as[sset()][b], acc[a][b]);
    });
  };
  constexpr std::integral_constant<int, 0> c0;
  constexpr std::integral_constant<int, 1> c1;
  constexpr std::integral_constant<int, 2> c2;
  constexpr std::integral_constant<int, 3> c3;
  constexpr std::integral_constant<int, 4> c4;
  constexpr std::integral_constant<int, 8> c8;
  // one piece moved on: into the other buffer, its register to the chunk after
  auto move_w = [&](auto i, int buf, int c) { store_w(i, buf ^ 1); load_w(i, c); };
  auto move_a = [&](auto i, int buf, int c) { store_a(i, buf ^ 1); load_a(i, c); };

  mx_for<P>([&](auto i) { load_w(i, 0); load_a(i, 0); });
  load_s(0);
  {
    const int c = min(1, chunks - 1);
    mx_for<P>([&](auto i) {
      store_w(i, 0);
      load_w(i, c);
      store_a(i, 0);
      load_a(i, c);
    });
    store_s(0);
    load_s(c);
  }
  __syncthreads();
  frags(c0, 0, 4 * half);
  scales(c0, 0);
  // a chunk whose scales are in set s; the next chunk's go to set 1 - s
  auto chunk = [&](auto s, auto s1, int c) {
    const int buf = c & 1, cn = min(c + 2, chunks - 1);  // past the last chunk: again the last one, never stored
    frags(c1, buf, 4 * half + 1);
    if (live) products(c0, s, c0, c0, c4);
    move_w(c0, buf, cn);
    move_w(c1, buf, cn);
    if (live) products(c0, s, c0, c4, c8);
    move_w(c2, buf, cn);
    frags(c0, buf, 4 * half + 2);
    if (live) products(c1, s, c1, c0, c4);
    move_w(c3, buf, cn);
    move_a(c0, buf, cn);
    if (live) products(c1, s, c1, c4, c8);
    move_a(c1, buf, cn);
    frags(c1, buf, 4 * half + 3);
    if (live) products(c0, s, c2, c0, c4);
    move_a(c2, buf, cn);
    move_a(c3, buf, cn);
    store_s(buf ^ 1);
    load_s(cn);
    if (live) products(c0, s, c2, c4, c8);
    __syncthreads();
    frags(c0, buf ^ 1, 4 * half);
    scales(s1, buf ^ 1);
    if (live) products(c1, s, c3, c0, c8);
  };
  int c = 0;
  for (; c + 2 < chunks; c += 2) {
    chunk(c0, c1, c);
    chunk(c1, c0, c + 1);
  }
  if (c + 1 < chunks) chunk(c0, c1, c++);
  // the last chunk's blocks in (left + 1) / 2 steps: step j takes blocks j and steps + j
  if (live) {
    const int buf = c & 1, left = blocks - 8 * c, steps = (left + 1) / 2;
    uint32_t wz[NA], az[NB];
    auto bytes = [&](int row) {  // the scale bytes of the half's blocks, the first lowest
      return static_cast<uint32_t>(__builtin_bit_cast(uint64_t, scl[buf][row]) >> (half ? 8 * steps : 0));
    };
    mx_for<NA>([&](auto a) { wz[a()] = bytes(wrow + 32 * a()); });
    mx_for<NB>([&](auto b) { az[b()] = bytes(TN + arow + 32 * b()); });
    for (int j = 0; j < steps; ++j) {
      frags(c0, buf, steps * half + j);
      mx_for<NA>([&](auto a) {
        mx_for<NB>([&](auto b) { acc[a()][b()] = mx_mfma<0>(wf[0][a()], af[0][b()], wz[a()], az[b()], acc[a()][b()]); });
      });
      mx_for<NA>([&](auto a) { wz[a()] >>= 8; });
      mx_for<NB>([&](auto b) { az[b()] >>= 8; });
    }
  }
  const bool vec = n % 8 == 0;
  mx_for<NB>([&](auto b) {
    const int row = t.row0 + arow + 32 * b();
    mx_for<NA>([&](auto a) {
      const int64_t col = n0 + 32 * (NA * wn + a());
      mx_acc_t v = acc[a()][b()];
      if (t.e < 0) v = mx_acc_t{};
      if (col < n) mx_store_block<ODT>(p.out, int64_t(row) * n + col, n - col, vec, row < t.end, half, v);
    });
  });
}

}  // namespace e4b
