// mxfp4.hpp -- the microscaled 4-bit format: blocks of 32 elements e2m1 on one
// power-of-two scale (OCP Microscaling Formats 1.0, MXFP4), and the layout of a packed
// matrix.
//
//   scale byte e of a block: 2^(e - 127), 255 NaN.  From the largest magnitude, whose
//   floor(log2) is E: 2^(E - 2), the largest power of two that takes it to at most
//   twice 4, the largest one of e2m1; at least 2^-127; NaN if the block holds one or an
//   infinity.
//   code of x: the nearest of 0, 0.5, 1, 1.5, 2, 3, 4, 6 to |x| / scale, ties to the
//   even code, 6 at most, and x's sign in bit 3.
//
// gfx950's conversions compute both directions, and the tests go through what decides a
// code: all bf16 values under each largest exponent, so on every scale, 2^-127 among them;
// of f32 the three values on either side of each border on every scale; and back, every
// code on every scale byte, of which 255 in a float's exponent field gives NaN.  They read
// a float's exponent field alone, so a scale byte takes one shift.
#pragma once

#include <stdint.h>

#if defined(__HIPCC__)
#include "common.hpp"
#endif

namespace mxfp4 {

constexpr uint32_t kBlock = 32;    // elements on one scale
constexpr uint32_t kPanel = 256;   // columns of a panel: eight scales of a row beside each other
constexpr uint32_t kRowBytes = kPanel / 2;  // a row's codes of one panel
constexpr uint32_t kMaxPanels = 65535;      // 256 rows of codes stay below 2^31 bytes

// Sizes of a packed [rows, cols] matrix: codes [rows][panels * 128], scales
// [panels][scale_rows][8], so that the rows of a tile have their scales of a panel in
// one piece.  0 <= rows, cols < 2^32.
struct Packed {
  uint32_t panels;
  uint64_t scale_rows;  // rows rounded up to 16
  uint64_t codes, scales;  // bytes
  static inline Packed of(uint32_t rows, uint32_t cols) {
    Packed p;
    p.panels = (uint32_t)(((uint64_t)cols + kPanel - 1u) / kPanel);
    p.scale_rows = ((uint64_t)rows + 15u) / 16u * 16u;
    p.codes = (uint64_t)rows * p.panels * kRowBytes;      // below 2^63
    p.scales = p.scale_rows * p.panels * (kPanel / kBlock);
    return p;
  }
};

#if defined(__HIPCC__)
typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));

// The scale byte of a block whose largest magnitude has these bits (sign bit 0; a NaN or
// an infinity is larger than every finite one).
FE2O3_DEVICE uint32_t scale_byte(uint32_t top) {
  const uint32_t e = top >> 23;
  return e == 255u ? 255u : max(e, 2u) - 2u;
}
// What the conversions take for it.
FE2O3_DEVICE float scale_float(uint32_t byte) { return __uint_as_float(byte << 23); }

// Eight codes of f32 values, the first in the low bits.
FE2O3_DEVICE uint32_t encode8(const float (&x)[8], float scale) {
  uint32_t q = 0;
  q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, x[0], x[1], scale, 0);
  q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, x[2], x[3], scale, 1);
  q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, x[4], x[5], scale, 2);
  return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, x[6], x[7], scale, 3);
}
// Of packed bf16 values.
FE2O3_DEVICE uint32_t encode8(u32x4_t x, float scale) {
  // a bit cast of a vector's element takes the vector's first: scalars
  const uint32_t w[4] = {x[0], x[1], x[2], x[3]};
  uint32_t q = 0;
  q = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(q, __builtin_bit_cast(bf16x2_t, w[0]), scale, 0);
  q = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(q, __builtin_bit_cast(bf16x2_t, w[1]), scale, 1);
  q = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(q, __builtin_bit_cast(bf16x2_t, w[2]), scale, 2);
  return __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(q, __builtin_bit_cast(bf16x2_t, w[3]), scale, 3);
}
// The values of eight codes as packed bf16: exact, since a value has two significant
// bits and no scale leaves bf16's range at the small end; at the large one 2 and more
// times 2^127 and 4 and 6 times 2^126 are infinities, in f32 as well.
FE2O3_DEVICE u32x4_t decode8_bf16(uint32_t q, float scale) {
  u32x4_t x;
  x[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(q, scale, 0));
  x[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(q, scale, 1));
  x[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(q, scale, 2));
  x[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(q, scale, 3));
  return x;
}
// Of four codes, in f32.
FE2O3_DEVICE void decode4_f32(uint32_t q, float scale, float (&x)[4]) {
  const fe2o3::f32x2_t a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, scale, 0);
  const fe2o3::f32x2_t b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, scale, 1);
  x[0] = a[0];
  x[1] = a[1];
  x[2] = b[0];
  x[3] = b[1];
}

// The largest magnitude's bits of eight values.
FE2O3_DEVICE uint32_t top8(const float (&x)[8]) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(x[i]) & 0x7fffffffu);
  return m;
}
FE2O3_DEVICE uint32_t top8(u32x4_t x) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    m = max(m, (x[i] << 16) & 0x7fffffffu);
    m = max(m, x[i] & 0x7fff0000u);
  }
  return m;
}
// The largest of the four lanes l & ~3 .. + 3, which hold a block, by lane exchanges
// within quads.
FE2O3_DEVICE uint32_t quad_max(uint32_t v) {
  v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0xb1, 0xf, 0xf, true));  // 1 0 3 2
  return max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x4e, 0xf, 0xf, true));  // 2 3 0 1
}
#endif

}  // namespace mxfp4
