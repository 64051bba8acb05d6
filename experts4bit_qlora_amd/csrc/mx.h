// Microscaled 4-bit floating point (OCP MX, e2m1 values with one e8m0 scale per 32): quantization of
// dense rows. Per block of 32 the exponent X = floor(log2(amax)) - 2 gives the scale byte
// e = clamp(X + 127, 0, 254), and every value becomes the e2m1 code nearest to v / 2^(e - 127), ties
// to the even code, saturating at 6; a zero has no sign. Low nibble first. The values divide by a
// power of two and are rounded once, so nothing depends on the order of the arithmetic.
//
// gfx950 converts a pair of values per instruction (v_cvt_scalef32_pk_fp4_{f32,bf16,f16}: the scale's
// exponent divided out, round to nearest even, saturating, checked here against the definition over
// every code, midpoint and scale byte); it keeps the sign of a value that rounds to zero, which three
// bit operations per eight codes take off.
#pragma once

#include "common.h"

namespace e4b {

typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));
typedef uint16_t u16x2_t __attribute__((ext_vector_type(2)));

constexpr int kMxBlock = 32;

// Eight values as loaded: four words of pairs (bf16, fp16) or eight floats.
template <int DT>
struct MxPiece {
  uint32_t w[DT == E4B_FP32 ? 8 : 4];
};

template <int DT>
E4B_DEV MxPiece<DT> mx_load(const void* src, int64_t piece) {
  MxPiece<DT> p;
  const uint4* s = static_cast<const uint4*>(src) + piece * (DT == E4B_FP32 ? 2 : 1);
#pragma unroll
  for (int i = 0; i < (DT == E4B_FP32 ? 2 : 1); ++i) {
    const uint4 v = s[i];
    p.w[4 * i] = v.x; p.w[4 * i + 1] = v.y; p.w[4 * i + 2] = v.z; p.w[4 * i + 3] = v.w;
  }
  return p;
}

// The largest magnitude of a piece as fp32 bits. Magnitudes order like their bit patterns and a NaN
// lies above infinity, so it stays the maximum.
template <int DT>
E4B_DEV uint32_t mx_amax(const MxPiece<DT>& p) {
  if constexpr (DT == E4B_FP32) {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max(m, p.w[i] & 0x7fffffffu);
    return m;
  } else {
    u16x2_t m = {0, 0};
#pragma unroll
    for (int i = 0; i < 4; ++i) m = __builtin_elementwise_max(m, __builtin_bit_cast(u16x2_t, p.w[i] & 0x7fff7fffu));
    return __float_as_uint(to_f<DT>(max(m.x, m.y)));
  }
}

// The scale byte of a block whose largest magnitude has the fp32 bits m: floor(log2) is its exponent field. A block
// with an infinity or a NaN: 255, which makes the whole block NaN in a product (nan_scale), or the torch
// formulation's 254 and 0.
E4B_DEV uint32_t mx_scale_byte(uint32_t m, bool nan_scale) {
  const uint32_t f = m >> 23;
  if (f == 255) return nan_scale ? 255u : (m == 0x7f800000u ? 254u : 0u);
  return f > 2 ? f - 2 : 0;
}

// The eight codes of a piece under scale byte e (255 converts as 254; its codes are not read as values).
template <int DT>
E4B_DEV uint32_t mx_codes(const MxPiece<DT>& p, uint32_t e) {
  const float scale = e8m0_to_f32(e < 254 ? e : 254u);
  uint32_t c = 0;
  if constexpr (DT == E4B_FP32) {
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, __uint_as_float(p.w[0]), __uint_as_float(p.w[1]), scale, 0);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, __uint_as_float(p.w[2]), __uint_as_float(p.w[3]), scale, 1);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, __uint_as_float(p.w[4]), __uint_as_float(p.w[5]), scale, 2);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, __uint_as_float(p.w[6]), __uint_as_float(p.w[7]), scale, 3);
  } else if constexpr (DT == E4B_BF16) {
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, __builtin_bit_cast(bf16x2_t, p.w[0]), scale, 0);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, __builtin_bit_cast(bf16x2_t, p.w[1]), scale, 1);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, __builtin_bit_cast(bf16x2_t, p.w[2]), scale, 2);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, __builtin_bit_cast(bf16x2_t, p.w[3]), scale, 3);
  } else {
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(c, __builtin_bit_cast(f16x2_t, p.w[0]), scale, 0);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(c, __builtin_bit_cast(f16x2_t, p.w[1]), scale, 1);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(c, __builtin_bit_cast(f16x2_t, p.w[2]), scale, 2);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(c, __builtin_bit_cast(f16x2_t, p.w[3]), scale, 3);
  }
  const uint32_t some = (c | (c >> 1) | (c >> 2)) & 0x11111111u;  // codes that are not zero
  return c & (0x77777777u | (some << 3));
}

// A NaN's code is +6 (the torch formulation's search ends there), whatever its sign bit.
template <int DT>
E4B_DEV uint32_t mx_nan_codes(const MxPiece<DT>& p, uint32_t c) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    float v;
    if constexpr (DT == E4B_FP32) v = __uint_as_float(p.w[i]);
    else v = (i & 1) ? hi_f<DT>(p.w[i / 2]) : lo_f<DT>(p.w[i / 2]);
    if (v != v) c = (c & ~(15u << (4 * i))) | (7u << (4 * i));
  }
  return c;
}

constexpr int kMxThreads = 256;
constexpr int kMxUnroll = 4;  // pieces per thread, their loads in flight together

// Dense values in blocks of 32 to codes [values / 2] and scale bytes [values / 32].
//
// Bound by HBM: 2 bytes of a bf16 value read, 17 / 32 written. A quad of lanes holds one block, so a
// wave's loads and its code stores are contiguous. 32 experts of 5,760 x 2,880 in bf16 (1.34 GB): at the rate of a
// large copy, 4.9 TB/s; in fp32 (2.4 GB) 453 us, 5.3 TB/s.
template <int DT>
__global__ void __launch_bounds__(kMxThreads) mx_quantize_kernel(const void* __restrict__ x, int64_t pieces,
                                                                 uint32_t* __restrict__ codes,
                                                                 uint8_t* __restrict__ scales) {
  const int64_t first = int64_t(blockIdx.x) * (kMxThreads * kMxUnroll) + threadIdx.x;
  MxPiece<DT> raw[kMxUnroll];
#pragma unroll
  for (int u = 0; u < kMxUnroll; ++u) {
    const int64_t p = first + u * kMxThreads;
    raw[u] = mx_load<DT>(x, p < pieces ? p : 0);  // past the end: piece 0, never stored
  }
#pragma unroll
  for (int u = 0; u < kMxUnroll; ++u) {
    const int64_t p = first + u * kMxThreads;
    const uint32_t m = quad_max(mx_amax<DT>(raw[u]));
    const uint32_t e = mx_scale_byte(m, false);
    uint32_t c = mx_codes<DT>(raw[u], e);
    if (m > 0x7f800000u) c = mx_nan_codes<DT>(raw[u], c);
    if (p < pieces) {
      codes[p] = c;
      if ((p & 3) == 0) scales[p >> 2] = static_cast<uint8_t>(e);
    }
  }
}

}  // namespace e4b
