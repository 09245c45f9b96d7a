// Rows into and out of the paged latent cache (latent.h).
//
// The reference keeps the raw outputs of kv_a_proj and norms and rotates every cached row
// on every step (inference/ops.py:136-159); here a row is normed, rotated and rounded once,
// as it is written:
//   n = x rsqrt(mean(x^2) + eps) gamma      (fp32, one rounding: to bf16, or to the codes)
//   e = min { e : max |n| <= 448 2^e } in [-32, 32],  code = e4m3(n 2^-e)
//   (r0, r1) = (x0 cos - x1 sin, x0 sin + x1 cos) at the row's position
// 448 is the largest code, so no value of the row saturates (the choice of
// floor(log2 max) - 8 would cut maxima above 448 / 512 of a binade); a row with an
// infinity or a NaN among its normed values is a row of NaN (byte 255, codes 0x7f).
#include <algorithm>

#include "latent.h"

namespace amla {

int latent_pages(const amla_latent_cache *c, const char *what, LatentPages *p) {
  if (!c || !c->latent || !c->k_pe || (!c->block_table && c->cols)) return fail(AMLA_EINVAL, "%s: null pointer", what);
  if (c->page_size <= 0 || c->page_size > 65536 || (c->page_size & (c->page_size - 1)))
    return fail(AMLA_EUNSUPPORTED, "%s: page_size %d is no power of two up to 65536", what, c->page_size);
  if (c->pages <= 0 || c->cols < 0 || c->ld_table < c->cols) return fail(AMLA_EINVAL, "%s: bad shape", what);
  if (c->pages > INT32_MAX / c->page_size || c->cols > INT32_MAX / c->page_size)
    return fail(AMLA_EUNSUPPORTED, "%s: pool and sequences hold at most 2^31 - 1 rows", what);
  if (!aligned16(c->latent) || !aligned16(c->k_pe))
    return fail(AMLA_EUNSUPPORTED, "%s: latents and rope keys must be 16-byte aligned", what);
  *p = LatentPages{static_cast<uint8_t *>(c->latent),
                   static_cast<uint16_t *>(c->k_pe),
                   static_cast<uint8_t *>(c->scales),
                   c->block_table,
                   c->ld_table,
                   (int32_t)c->pages,
                   (int32_t)c->cols,
                   __builtin_ctz((unsigned)c->page_size)};
  return AMLA_OK;
}

constexpr int LC_WAVES = 4;

// One wave per row: lane l holds latents 8l .. 8l+7 and, for l < 32, the rope pair l.  Bound by latency (offsets, table,
// row, table of angles): 4.0 us for 32 rows, 7.1 for 8111 (14.5 MB; 3.1 at a copy's rate).
template <bool F8>
__global__ __launch_bounds__(64 * LC_WAVES) void latent_write_kernel(LatentPages pg, PackedRows map,
                                                                     const uint16_t *__restrict__ kv, int rows,
                                                                     int64_t ldkv, const uint16_t *__restrict__ gamma,
                                                                     float eps, const f32x2 *__restrict__ rope,
                                                                     int rope_rows) {
  const int i = __builtin_amdgcn_readfirstlane(blockIdx.x * LC_WAVES + (threadIdx.x >> 6));
  const int lane = threadIdx.x & 63;
  if (i >= rows) return;
  const uint16_t *x = kv + i * ldkv;
  const u32x4 v = ldg16(x + 8 * lane);
  const u32x4 g = ldg16(gamma + 8 * lane);
  const uint32_t pe = *reinterpret_cast<const uint32_t *>(x + LC_LORA + 2 * (lane & 31));
  const int2 at = map.at(i);
  if (at.x < 0 || at.y >= rope_rows) return;
  const int slot = pg.slot(at.x, at.y);
  if (slot < 0) return;
  const f32x2 cs = rope[(size_t)at.y * (LC_ROPE / 2) + (lane & 31)];
  float n[8], sum = 0.f;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    n[2 * e] = lo_bf(v[e]);
    n[2 * e + 1] = hi_bf(v[e]);
    sum += n[2 * e] * n[2 * e] + n[2 * e + 1] * n[2 * e + 1];
  }
  const float r = rsqrtf(wave_sum(sum) * (1.f / LC_LORA) + eps);
  uint32_t amax = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    n[e] *= r * (e & 1 ? hi_bf(g[e >> 1]) : lo_bf(g[e >> 1]));
    amax = max(amax, __float_as_uint(n[e]) & 0x7fffffffu);
  }
  if (lane < LC_ROPE / 2) {
    const float a = lo_bf(pe), b = hi_bf(pe);
    reinterpret_cast<uint32_t *>(pg.k_pe)[(size_t)slot * (LC_ROPE / 2) + lane] =
        pack_bf16(a * cs.x - b * cs.y, a * cs.y + b * cs.x);
  }
  if constexpr (!F8) {
    reinterpret_cast<u32x4 *>(pg.latent)[(size_t)slot * (LC_LORA / 8) + lane] =
        u32x4{pack_bf16(n[0], n[1]), pack_bf16(n[2], n[3]), pack_bf16(n[4], n[5]), pack_bf16(n[6], n[7])};
  } else {
    amax = wave_max_u32(amax);
    const bool nan = amax >= 0x7f800000u;
    // 448 = 1.75 * 2^8: the exponent of amax - 8, one more where its mantissa is above 1.75
    const int e0 = (int)((amax + 0x1fffffu) >> 23) - 127 - 8;
    const int e = min(max(e0, -LC_EXP_MAX), LC_EXP_MAX);
    const float inv = __uint_as_float((uint32_t)(127 - e) << 23);
    int w[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float s[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) s[k] = __builtin_amdgcn_fmed3f(n[4 * h + k] * inv, -448.f, 448.f);
      w[h] = __builtin_amdgcn_cvt_pk_fp8_f32(s[0], s[1], 0, false);
      w[h] = __builtin_amdgcn_cvt_pk_fp8_f32(s[2], s[3], w[h], true);
      if (nan) w[h] = 0x7f7f7f7f;
    }
    reinterpret_cast<u32x2 *>(pg.latent)[(size_t)slot * (LC_LORA / 8) + lane] = u32x2{(uint32_t)w[0], (uint32_t)w[1]};
    if (lane == 0) pg.scales[slot] = nan ? 255 : (uint8_t)(e + 127);
  }
}

// LC_ROWS rows a wave: their places are looked up first, so that the loads of all of them are under way together.  e4m3 to
// bf16 is exact.  40001 rows, 72 MB: 15.2 us, 4.7 TB/s, the rate of a large copy; 8111 rows 6.9 us, 1501 of bf16 4.6.
constexpr int LC_ROWS = 4;

template <bool F8>
__global__ __launch_bounds__(64 * LC_WAVES) void latent_read_kernel(LatentPages pg, PackedRows map, int rows,
                                                                    u32x4 *__restrict__ latent,
                                                                    uint32_t *__restrict__ k_pe, int clear_rest) {
  const int lane = threadIdx.x & 63;
  const int i0 = __builtin_amdgcn_readfirstlane((blockIdx.x * LC_WAVES + (threadIdx.x >> 6)) * LC_ROWS);
  int slot[LC_ROWS];
#pragma unroll
  for (int k = 0; k < LC_ROWS; ++k) {
    slot[k] = -1;
    if (i0 + k >= rows) continue;
    const int2 at = map.at(i0 + k);
    if (at.x >= 0) slot[k] = pg.slot(at.x, at.y);
  }
#pragma unroll
  for (int k = 0; k < LC_ROWS; ++k) {
    const size_t i = i0 + k;
    if (i >= (size_t)rows || (slot[k] < 0 && !clear_rest)) continue;
    const size_t s = max(slot[k], 0);
    u32x4 o = {0, 0, 0, 0};
    uint32_t pe = 0;
    if (slot[k] >= 0) {
      pe = reinterpret_cast<const uint32_t *>(pg.k_pe)[s * (LC_ROPE / 2) + (lane & 31)];
      if constexpr (F8) {
        const u32x2 c = reinterpret_cast<const u32x2 *>(pg.latent)[s * (LC_LORA / 8) + lane];
        const uint32_t byte = pg.scales[s];
        const float f = byte == 255 ? __uint_as_float(0x7fc00000u) : __uint_as_float(byte ? byte << 23 : 1u << 22);
        const f32x2 a = fp8x2_to_f32<false>(c.x), b = fp8x2_to_f32<true>(c.x);
        const f32x2 d = fp8x2_to_f32<false>(c.y), e = fp8x2_to_f32<true>(c.y);
        o = u32x4{pack_bf16(a.x * f, a.y * f), pack_bf16(b.x * f, b.y * f), pack_bf16(d.x * f, d.y * f),
                  pack_bf16(e.x * f, e.y * f)};
      } else {
        o = reinterpret_cast<const u32x4 *>(pg.latent)[s * (LC_LORA / 8) + lane];
      }
    }
    latent[i * (LC_LORA / 8) + lane] = o;
    if (lane < 32) k_pe[i * (LC_ROPE / 2) + lane] = pe;
  }
}

// Checks the packed rows of a call and describes them to the kernels.
static int packed_rows(const char *what, int64_t rows, const int32_t *offsets, int64_t seqs, const int32_t *positions,
                       PackedRows *m) {
  if (rows < 0 || seqs < 0) return fail(AMLA_EINVAL, "%s: negative size", what);
  if (rows > INT32_MAX || seqs > AMLA_MAX_SEQS)
    return fail(AMLA_EUNSUPPORTED, "%s: at most 2^31 - 1 rows and %d sequences", what, AMLA_MAX_SEQS);
  if (!offsets && rows && (seqs == 0 || rows % seqs))
    return fail(AMLA_EINVAL, "%s: %lld rows of %lld sequences without offsets", what, (long long)rows, (long long)seqs);
  *m = PackedRows{offsets, positions, (int)seqs, seqs ? (int)(rows / seqs) : 0};
  return AMLA_OK;
}

}  // namespace amla

using namespace amla;

extern "C" {

int amla_latent_cache_write(const amla_latent_cache *cache, const void *kv, int64_t rows, int64_t ldkv,
                            const void *gamma, float eps, const float *rope_table, int64_t rope_rows,
                            const int32_t *offsets, int64_t seqs, const int32_t *positions, void *stream) {
  const char *what = "latent_cache_write";
  LatentPages pg;
  PackedRows map;
  int rc = latent_pages(cache, what, &pg);
  if (!rc) rc = packed_rows(what, rows, offsets, seqs, positions, &map);
  if (rc || rows == 0) return rc;
  if (!kv || !gamma || !rope_table || !positions) return fail(AMLA_EINVAL, "%s: null pointer", what);
  if (rope_rows < 0) return fail(AMLA_EINVAL, "%s: bad shape", what);
  if (ldkv < LC_LORA + LC_ROPE || ldkv % 8 || !aligned16(kv) || !aligned16(gamma))
    return fail(AMLA_EUNSUPPORTED, "%s: rows of 576 values, rows and gamma 16-byte aligned", what);
  if (rows >= 1 << 26) return fail(AMLA_EUNSUPPORTED, "%s: at most 2^26 - 1 rows a call", what);  // 2^32 threads
  const dim3 grid((unsigned)((rows + LC_WAVES - 1) / LC_WAVES));
  const auto fn = pg.scales ? latent_write_kernel<true> : latent_write_kernel<false>;
  fn<<<grid, 64 * LC_WAVES, 0, reinterpret_cast<hipStream_t>(stream)>>>(
      pg, map, static_cast<const uint16_t *>(kv), (int)rows, ldkv, static_cast<const uint16_t *>(gamma), eps,
      reinterpret_cast<const f32x2 *>(rope_table), (int)std::min<int64_t>(rope_rows, INT32_MAX));
  return check_launch(what);
}

int amla_latent_cache_read(const amla_latent_cache *cache, int64_t rows, const int32_t *offsets, int64_t seqs,
                           const int32_t *positions, void *latent, void *k_pe, int clear_rest, void *stream) {
  const char *what = "latent_cache_read";
  LatentPages pg;
  PackedRows map;
  int rc = latent_pages(cache, what, &pg);
  if (!rc) rc = packed_rows(what, rows, offsets, seqs, positions, &map);
  if (rc || rows == 0) return rc;
  if (!latent || !k_pe) return fail(AMLA_EINVAL, "%s: null pointer", what);
  if (!aligned16(latent) || !aligned16(k_pe)) return fail(AMLA_EUNSUPPORTED, "%s: outputs must be 16-byte aligned", what);
  if (rows >= 1 << 28) return fail(AMLA_EUNSUPPORTED, "%s: at most 2^28 - 1 rows a call", what);
  const dim3 grid((unsigned)((rows + LC_WAVES * LC_ROWS - 1) / (LC_WAVES * LC_ROWS)));
  const auto fn = pg.scales ? latent_read_kernel<true> : latent_read_kernel<false>;
  fn<<<grid, 64 * LC_WAVES, 0, reinterpret_cast<hipStream_t>(stream)>>>(pg, map, (int)rows, static_cast<u32x4 *>(latent),
                                                                        static_cast<uint32_t *>(k_pe), clear_rest);
  return check_launch(what);
}

}  // extern "C"
