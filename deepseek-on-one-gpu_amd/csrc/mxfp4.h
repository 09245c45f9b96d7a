// MXFP4 device helpers and the launches shared by the MXFP4 translation units.
//
// A row of K values is K/2 bytes of e2m1 codes (value 2i in the low half of byte
// i) and K/32 bytes of e8m0 exponents: value = e2m1(code) * 2^(byte - 127), byte
// 255 a NaN block.  Quantising a block: byte = max(E - 2, 0) with E the biased
// fp32 exponent of its largest magnitude (floor(log2) - 2, the largest e2m1
// exponent being 2; the clamp is e8m0's lower end), codes rounded to nearest
// even by the hardware convert, which saturates at 6.  A block that holds an
// infinity or a NaN is a NaN block with zero codes.
#pragma once

#include "amla_common.h"
#include "amla_internal.h"

namespace amla {

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x4_a4 __attribute__((ext_vector_type(4), aligned(4)));
typedef __bf16 bf16x2_v __attribute__((ext_vector_type(2)));

// amax: bits of the largest |value| of a block as fp32 (sign cleared)
AMLA_DEV uint32_t mx_byte(uint32_t amax) {
  const uint32_t e = amax >> 23;
  return e == 255 ? 255u : (e > 2 ? e - 2 : 0u);
}
// 2^(byte - 127) for byte <= 254
AMLA_DEV float mx_scale(uint32_t byte) { return __uint_as_float(byte ? byte << 23 : 1u << 22); }

// Eight fp32 values -> eight codes (the callers clear those of a NaN block)
AMLA_DEV uint32_t mx_codes8(const float *v, float scale) {
  uint32_t c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0u, v[0], v[1], scale, 0);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[2], v[3], scale, 1);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[4], v[5], scale, 2);
  return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[6], v[7], scale, 3);
}
// Eight bf16 values (packed pairs) -> eight codes
AMLA_DEV uint32_t mx_codes8(u32x4 v, float scale) {
  uint32_t c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(0u, __builtin_bit_cast(bf16x2_v, (uint32_t)v.x), scale, 0);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, __builtin_bit_cast(bf16x2_v, (uint32_t)v.y), scale, 1);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, __builtin_bit_cast(bf16x2_v, (uint32_t)v.z), scale, 2);
  return __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, __builtin_bit_cast(bf16x2_v, (uint32_t)v.w), scale, 3);
}
typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
// largest magnitudes of the even and of the odd bf16 values of four packed pairs
AMLA_DEV u16x2 mx_absmax(u16x2 a, u32x4 v) {
#pragma unroll
  for (int i = 0; i < 4; ++i)
    a = __builtin_elementwise_max(a, __builtin_bit_cast(u16x2, (uint32_t)(v[i] & 0x7fff7fffu)));
  return a;
}
AMLA_DEV uint32_t mx_amax_bits(u16x2 a) { return (uint32_t)(a.x > a.y ? a.x : a.y) << 16; }

// acc += A (16 x 128) B (128 x 16), both MXFP4: lane l holds 32 codes of row
// (column) l % 16 at K = 32 (l / 16) .. +31 and, in byte SEL of its scale dword,
// that block's exponent.  The products are exact; fp32 sums, magnitudes below
// 2^-126 flushed.  D: column l % 16, rows 4 (l / 16) .. +3.
template <int SEL>
AMLA_DEV f32x4 mfma_mx(u32x4 a, uint32_t as, u32x4 b, uint32_t bs, f32x4 c) {
  const i32x8 av = {(int)a.x, (int)a.y, (int)a.z, (int)a.w, 0, 0, 0, 0};
  const i32x8 bv = {(int)b.x, (int)b.y, (int)b.z, (int)b.w, 0, 0, 0, 0};
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(av, bv, c, 4, 4, SEL, as, SEL, bs);
}

// Quantises rows of bf16 (row stride ldx) for a product that follows on the stream.
int launch_mx_quantize_bf16(const uint16_t *x, int64_t rows, int64_t k, int64_t ldx, uint8_t *codes, uint8_t *scales,
                            hipStream_t st);

}  // namespace amla
