// MXFP4 quantisation and its inverse (format and rounding: mxfp4.h).
//
// Both are streams bound by HBM: four lanes share a block of 32 values, eight
// each, so every load and store of a wave is contiguous (codes 4 bytes per lane);
// the block's maximum takes two lane swaps inside the vector unit.  1999 x 7168 bf16 in
// 8.2 us (4.4 TB/s), a block-FP8 weight of 7168 x 16384 in 45 us (4.0 TB/s, of which two
// thirds are reads), back to bf16 in 43 us (6.9 TB/s).
#include <algorithm>

#include "mxfp4.h"

namespace amla {

enum { MX_BF16 = AMLA_BF16, MX_FP16 = AMLA_FP16, MX_FP32 = AMLA_FP32, MX_FP8 = 3 };

// fp8: the value is f32(weight) * scale_inv, one fp32 rounding
template <int TYPE>
__global__ __launch_bounds__(256) void mx_quantize_kernel(const void *__restrict__ x, int64_t chunks, int row_chunks,
                                                          int64_t ldx, const float *__restrict__ scale_inv, int sk,
                                                          uint32_t *__restrict__ codes, uint8_t *__restrict__ scales) {
  typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
  const int64_t stride = (int64_t)gridDim.x * 256;
  // chunks is a multiple of 4: the four lanes of a block leave the loop together
  for (int64_t c = (int64_t)blockIdx.x * 256 + threadIdx.x; c < chunks; c += stride) {
    const int64_t row = c / row_chunks;
    const int64_t at = row * ldx + (c - row * row_chunks) * 8;
    uint32_t amax;
    float v[8];
    u32x4 raw;
    if constexpr (TYPE == MX_BF16) {
      raw = ldg16(static_cast<const uint16_t *>(x) + at);
      amax = mx_amax_bits(mx_absmax(u16x2{0, 0}, raw));
    } else {
      if constexpr (TYPE == MX_FP16) {
        raw = ldg16(static_cast<const uint16_t *>(x) + at);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const f16x2 h = __builtin_bit_cast(f16x2, (uint32_t)raw[i]);
          v[2 * i] = (float)h.x;
          v[2 * i + 1] = (float)h.y;
        }
      } else if constexpr (TYPE == MX_FP32) {
        const f32x4 *src = reinterpret_cast<const f32x4 *>(static_cast<const float *>(x) + at);
        const f32x4 a = src[0], b = src[1];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          v[i] = a[i];
          v[4 + i] = b[i];
        }
      } else {
        const u32x2 w = ldg8(static_cast<const uint8_t *>(x) + at);
        const float s = scale_inv[(row >> 7) * sk + ((c - row * row_chunks) >> 4)];
        const f32x2 a = fp8x2_to_f32<false>(w.x), b = fp8x2_to_f32<true>(w.x);
        const f32x2 d = fp8x2_to_f32<false>(w.y), e = fp8x2_to_f32<true>(w.y);
        const float t[8] = {a.x, a.y, b.x, b.y, d.x, d.y, e.x, e.y};
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = __fmul_rn(t[i], s);
      }
      amax = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) amax = max(amax, __float_as_uint(v[i]) & 0x7fffffffu);
    }
    amax = max(amax, dpp_u32<0xB1>(amax));  // quad_perm [1,0,3,2]
    amax = max(amax, dpp_u32<0x4E>(amax));  // quad_perm [2,3,0,1]
    const uint32_t byte = mx_byte(amax);
    const float s = mx_scale(byte);
    uint32_t q;
    if constexpr (TYPE == MX_BF16) q = mx_codes8(raw, s);
    else q = mx_codes8(v, s);
    codes[c] = byte == 255 ? 0u : q;
    if ((c & 3) == 0) scales[c >> 2] = (uint8_t)byte;
  }
}

template <bool F32>
__global__ __launch_bounds__(256) void mx_dequantize_kernel(const uint32_t *__restrict__ codes,
                                                            const uint8_t *__restrict__ scales, int64_t chunks,
                                                            void *__restrict__ out) {
  const int64_t stride = (int64_t)gridDim.x * 256;
  for (int64_t c = (int64_t)blockIdx.x * 256 + threadIdx.x; c < chunks; c += stride) {
    const uint32_t q = codes[c], byte = scales[c >> 2];
    const float s = byte == 255 ? __uint_as_float(0x7fc00000u) : mx_scale(byte);
    float v[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      // (unit scale: the product with s is exact but for an overflow to infinity)
      const f32x2 p = i == 0   ? __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, 1.f, 0)
                      : i == 1 ? __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, 1.f, 1)
                      : i == 2 ? __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, 1.f, 2)
                               : __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, 1.f, 3);
      v[2 * i] = p.x * s;
      v[2 * i + 1] = p.y * s;
    }
    if constexpr (F32) {
      f32x4 *dst = static_cast<f32x4 *>(out) + 2 * c;
      dst[0] = f32x4{v[0], v[1], v[2], v[3]};
      dst[1] = f32x4{v[4], v[5], v[6], v[7]};
    } else {
      static_cast<u32x4 *>(out)[c] =
          u32x4{pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]), pack_bf16(v[4], v[5]), pack_bf16(v[6], v[7])};
    }
  }
}

static unsigned mx_blocks(int64_t chunks) { return (unsigned)std::min<int64_t>((chunks + 255) / 256, 256 * 64); }

template <int TYPE>
static int launch_mx_quantize(const void *x, int64_t rows, int64_t k, int64_t ldx, const float *scale_inv,
                              uint8_t *codes, uint8_t *scales, hipStream_t st) {
  const int64_t chunks = rows * (k / 8);
  mx_quantize_kernel<TYPE><<<dim3(mx_blocks(chunks)), 256, 0, st>>>(x, chunks, (int)(k / 8), ldx, scale_inv,
                                                                    (int)((k + 127) / 128),
                                                                    reinterpret_cast<uint32_t *>(codes), scales);
  return check_launch("mxfp4_quantize");
}

int launch_mx_quantize_bf16(const uint16_t *x, int64_t rows, int64_t k, int64_t ldx, uint8_t *codes, uint8_t *scales,
                            hipStream_t st) {
  return launch_mx_quantize<MX_BF16>(x, rows, k, ldx, nullptr, codes, scales, st);
}

}  // namespace amla

using namespace amla;

extern "C" {

int amla_mxfp4_quantize(const void *x, int dtype, int64_t rows, int64_t k, int64_t ldx, void *codes, void *scales,
                        void *stream) {
  if (!x || !codes || !scales) return fail(AMLA_EINVAL, "mxfp4_quantize: null pointer");
  if (rows < 0 || k < 0 || ldx < k) return fail(AMLA_EINVAL, "mxfp4_quantize: bad shape");
  if (dtype != AMLA_BF16 && dtype != AMLA_FP16 && dtype != AMLA_FP32)
    return fail(AMLA_EINVAL, "mxfp4_quantize: unknown dtype %d", dtype);
  if (rows == 0 || k == 0) return AMLA_OK;
  if (k % 32 || k > INT32_MAX || ldx % (dtype == AMLA_FP32 ? 4 : 8) || !aligned16(x) || !aligned16(codes))
    return fail(AMLA_EUNSUPPORTED, "mxfp4_quantize: needs k %% 32 == 0 and 16-byte aligned rows and codes (k=%lld)",
                (long long)k);
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  uint8_t *c = static_cast<uint8_t *>(codes), *s = static_cast<uint8_t *>(scales);
  if (dtype == AMLA_BF16) return launch_mx_quantize<MX_BF16>(x, rows, k, ldx, nullptr, c, s, st);
  if (dtype == AMLA_FP16) return launch_mx_quantize<MX_FP16>(x, rows, k, ldx, nullptr, c, s, st);
  return launch_mx_quantize<MX_FP32>(x, rows, k, ldx, nullptr, c, s, st);
}

int amla_mxfp4_quantize_fp8(const void *weight, const float *scale_inv, int64_t n, int64_t k, void *codes,
                            void *scales, void *stream) {
  if (!weight || !scale_inv || !codes || !scales) return fail(AMLA_EINVAL, "mxfp4_quantize_fp8: null pointer");
  if (n < 0 || k < 0) return fail(AMLA_EINVAL, "mxfp4_quantize_fp8: negative shape");
  if (n == 0 || k == 0) return AMLA_OK;
  if (k % 32 || k > INT32_MAX || !aligned16(weight) || !aligned16(codes))
    return fail(AMLA_EUNSUPPORTED,
                "mxfp4_quantize_fp8: needs k %% 32 == 0 and 16-byte aligned weight and codes (k=%lld)", (long long)k);
  return launch_mx_quantize<MX_FP8>(weight, n, k, k, scale_inv, static_cast<uint8_t *>(codes),
                                    static_cast<uint8_t *>(scales), reinterpret_cast<hipStream_t>(stream));
}

int amla_mxfp4_dequantize(const void *codes, const void *scales, int64_t rows, int64_t k, int dtype, void *out,
                          void *stream) {
  if (!codes || !scales || !out) return fail(AMLA_EINVAL, "mxfp4_dequantize: null pointer");
  if (rows < 0 || k < 0) return fail(AMLA_EINVAL, "mxfp4_dequantize: negative shape");
  if (dtype != AMLA_BF16 && dtype != AMLA_FP32)
    return fail(AMLA_EINVAL, "mxfp4_dequantize: dtype %d (bf16 and fp32 hold every value)", dtype);
  if (rows == 0 || k == 0) return AMLA_OK;
  if (k % 32 || !aligned16(codes) || !aligned16(out))
    return fail(AMLA_EUNSUPPORTED, "mxfp4_dequantize: needs k %% 32 == 0 and 16-byte aligned codes and out (k=%lld)",
                (long long)k);
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  const int64_t chunks = rows * (k / 8);
  const uint32_t *c = static_cast<const uint32_t *>(codes);
  const uint8_t *s = static_cast<const uint8_t *>(scales);
  if (dtype == AMLA_FP32) mx_dequantize_kernel<true><<<dim3(mx_blocks(chunks)), 256, 0, st>>>(c, s, chunks, out);
  else mx_dequantize_kernel<false><<<dim3(mx_blocks(chunks)), 256, 0, st>>>(c, s, chunks, out);
  return check_launch("mxfp4_dequantize");
}

}  // extern "C"
