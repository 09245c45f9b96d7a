// MXFP4 products for gfx950: y = deq(x) deq(w)^T with both operands in 4 bits on
// the scaled MFMA (16x16x128, exact products, fp32 sums).  A skinny kernel for up
// to 64 activation rows, tiles of 256 weight rows x up to 128 activation rows for
// more, each for one weight or for a device schedule of experts, with the output
// rows or silu(gate) * up quantised again as epilogue.
#include <algorithm>
#include <type_traits>

#include "mxfp4.h"
#include "tile_order.h"

namespace amla {

constexpr int MX_ROWS = 128;         // activation rows of a tile
constexpr int MX_MAX_GROUPS = 1024;  // experts of a grouped product

// Operands of a launch.  Two weights (SILU): gate and up.  ent (with count): the
// schedule entries (expert, first position, rows, -), expert -1 for rows to clear;
// null: one entry of M rows.  Position p reads x row xrow[p] and writes y row
// yrow[p] (null: p).
struct MxParams {
  const void *x;       // codes, or bf16 values (xs null; skinny only)
  const uint8_t *xs;
  int64_t ldx;         // bf16 row stride
  const int32_t *xrow, *yrow;
  const uint8_t *w[2], *ws[2];
  int64_t wstride, sstride;  // bytes from expert to expert
  const int32_t *ent, *count;
  int M, N, K;
  void *y;
  int64_t ldy;
  int f32, vec;        // fp32 outputs; four outputs per store
  uint8_t *hc, *hs;    // SILU: codes and exponents by position
};

AMLA_DEV void mx_store4(const MxParams &p, int64_t row, int n, f32x4 v) {
  if (p.f32) {
    float *y = static_cast<float *>(p.y) + row * p.ldy + n;
    if (p.vec) *reinterpret_cast<f32x4 *>(y) = v;
    else
      for (int i = 0; i < 4 && n + i < p.N; ++i) y[i] = v[i];
  } else {
    uint16_t *y = static_cast<uint16_t *>(p.y) + row * p.ldy + n;
    if (p.vec) *reinterpret_cast<u32x2 *>(y) = u32x2{pack_bf16(v.x, v.y), pack_bf16(v.z, v.w)};
    else
      for (int i = 0; i < 4 && n + i < p.N; ++i) y[i] = f2bf(v[i]);
  }
}

AMLA_DEV float mx_silu_mul(float g, float u) { return g / (1.f + expf(-g)) * u; }

// ---------------------------------------------------------------- skinny product

// Up to 16 XT activation rows by 16 WT weight rows per workgroup; the waves take
// runs of the 128-wide K steps and meet in LDS, in wave order.  Weights and
// activations go from memory straight into the operands' registers: 16 rows x 64
// bytes per load, four steps at a time, the exponents of four steps in one 16-byte
// load per row (the lanes of a row share it).  FUSED: bf16 rows, quantised in the
// registers (a lane holds whole blocks), which saves the pass and the launch
// before it.
template <int WT, int XT, bool FUSED, bool SILU>
__global__ __launch_bounds__(512) void mx_skinny_kernel(MxParams p, int ntiles) {
  extern __shared__ __align__(16) float red[];
  const int tid = threadIdx.x, lane = tid & 63, r16 = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), nw = blockDim.x >> 6;
  const int en = blockIdx.x / ntiles, nt = blockIdx.x - en * ntiles;
  int e = 0, r0 = 0, rows = p.M;
  if (p.ent) {
    if (en >= *p.count) return;
    e = p.ent[4 * en];
    r0 = p.ent[4 * en + 1];
    rows = p.ent[4 * en + 2];
  }
  constexpr int COLS = SILU ? 8 * WT : 16 * WT;  // outputs of the workgroup
  if (!SILU && e < 0) {  // rows of no expert
    for (int i = tid; i < rows * 4 * WT; i += blockDim.x) {
      const int r = i / (4 * WT), n = nt * COLS + 4 * (i - r * 4 * WT);
      if (n < p.N) mx_store4(p, p.yrow ? p.yrow[r0 + r] : r0 + r, n, f32x4{0.f, 0.f, 0.f, 0.f});
    }
    return;
  }
  const int64_t kb = p.K >> 1, ksb = p.K >> 5;
  const uint8_t *wp[WT], *sp[WT];
#pragma unroll
  for (int t = 0; t < WT; ++t) {
    const int seg = SILU && t >= WT / 2 ? 1 : 0;
    const int n = min(nt * COLS + 16 * (SILU ? t % (WT / 2) : t) + r16, p.N - 1);  // rows past N repeat the last
    wp[t] = p.w[seg] + e * p.wstride + n * kb + 16 * g;
    sp[t] = p.ws[seg] + e * p.sstride + n * ksb;
  }
  const uint8_t *xp[XT], *xsp[XT];
  bool act[XT];
#pragma unroll
  for (int j = 0; j < XT; ++j) {
    act[j] = 16 * j + r16 < rows;
    const int pos = r0 + min(16 * j + r16, rows - 1);
    const int64_t xr = p.xrow ? p.xrow[pos] : pos;
    xp[j] = static_cast<const uint8_t *>(p.x) + (FUSED ? xr * p.ldx * 2 + 64 * g : xr * kb + 16 * g);
    xsp[j] = FUSED ? nullptr : p.xs + xr * ksb;
  }
  f32x4 acc[WT][XT];
#pragma unroll
  for (int t = 0; t < WT; ++t)
#pragma unroll
    for (int j = 0; j < XT; ++j) acc[t][j] = f32x4{0.f, 0.f, 0.f, 0.f};

  const int steps = p.K >> 7, s1 = steps * (wave + 1) / nw;
  // one run of U steps from step s
  auto run = [&](int s, auto u_c) {
    constexpr int U = decltype(u_c)::value;
    u32x4 wc[U][WT], xc[U][XT], xraw[FUSED ? U : 1][FUSED ? 4 : 1];
    uint32_t wsc[WT][U], xsc[XT][U];
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int t = 0; t < WT; ++t) wc[u][t] = ldg16_nt(wp[t] + (int64_t)(s + u) * 64);
#pragma unroll
    for (int t = 0; t < WT; ++t) {
      if constexpr (U == 4) {
        const u32x4_a4 v = *reinterpret_cast<const u32x4_a4 *>(sp[t] + s * 4);
#pragma unroll
        for (int u = 0; u < 4; ++u) wsc[t][u] = v[u];
      } else {
#pragma unroll
        for (int u = 0; u < U; ++u) wsc[t][u] = *reinterpret_cast<const uint32_t *>(sp[t] + (s + u) * 4);
      }
    }
#pragma unroll
    for (int j = 0; j < XT; ++j) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        xc[u][j] = u32x4{0, 0, 0, 0};
        xsc[j][u] = 0;
      }
      if (act[j]) {
        if constexpr (FUSED) {
#pragma unroll
          for (int u = 0; u < U; ++u) {
            u16x2 am = {0, 0};
#pragma unroll
            for (int q = 0; q < 4; ++q) xraw[u][q] = ldg16(xp[j] + (int64_t)(s + u) * 256 + 16 * q);
#pragma unroll
            for (int q = 0; q < 4; ++q) am = mx_absmax(am, xraw[u][q]);
            const uint32_t byte = mx_byte(mx_amax_bits(am));
            const float sc = mx_scale(byte);
#pragma unroll
            for (int q = 0; q < 4; ++q) xc[u][j][q] = mx_codes8(xraw[u][q], sc);
            xsc[j][u] = byte << (8 * g);
          }
        } else {
#pragma unroll
          for (int u = 0; u < U; ++u) {
            xc[u][j] = ldg16(xp[j] + (int64_t)(s + u) * 64);
            xsc[j][u] = *reinterpret_cast<const uint32_t *>(xsp[j] + (s + u) * 4);
          }
        }
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int t = 0; t < WT; ++t)
#pragma unroll
        for (int j = 0; j < XT; ++j)
          acc[t][j] = mfma_mx<0>(wc[u][t], wsc[t][u] >> (8 * g), xc[u][j], xsc[j][u] >> (8 * g), acc[t][j]);
  };
  int s = steps * wave / nw;
  for (; s + 4 <= s1; s += 4) run(s, std::integral_constant<int, 4>{});
  for (; s < s1; ++s) run(s, std::integral_constant<int, 1>{});

  f32x4 *part = reinterpret_cast<f32x4 *>(red);
#pragma unroll
  for (int t = 0; t < WT; ++t)
#pragma unroll
    for (int j = 0; j < XT; ++j) part[((wave * WT + t) * XT + j) * 64 + lane] = acc[t][j];
  __syncthreads();
  auto total = [&](int t, int j, int l) {
    f32x4 v = part[(t * XT + j) * 64 + l];
    for (int w = 1; w < nw; ++w) v += part[((w * WT + t) * XT + j) * 64 + l];
    return v;
  };
  if constexpr (SILU) {
    // eight lanes hold a block of 32 outputs of a row: four each
    for (int i = tid; i < XT * 16 * 2 * WT; i += blockDim.x) {
      const int c = i % (2 * WT), m = i / (2 * WT), t = c >> 2;
      const int j = m >> 4, l = (c & 3) * 16 + (m & 15);
      const f32x4 gt = total(t, j, l), up = total(t + WT / 2, j, l);
      float h[4];
      uint32_t am = 0;
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        h[q] = mx_silu_mul(gt[q], up[q]);
        am = max(am, __float_as_uint(h[q]) & 0x7fffffffu);
      }
      am = max(am, dpp_u32<0xB1>(am));   // quad_perm [1,0,3,2]
      am = max(am, dpp_u32<0x4E>(am));   // quad_perm [2,3,0,1]
      am = max(am, dpp_u32<0x141>(am));  // row_half_mirror
      const uint32_t byte = mx_byte(am);
      const float sc = mx_scale(byte);
      uint32_t q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0u, h[0], h[1], sc, 0);
      q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, h[2], h[3], sc, 1);
      if (byte == 255) q = 0;
      const int n = nt * COLS + 4 * c;
      if (m < rows) {
        *reinterpret_cast<uint16_t *>(p.hc + (int64_t)(r0 + m) * (p.N >> 1) + (n >> 1)) = (uint16_t)q;
        if ((c & 7) == 0) p.hs[(int64_t)(r0 + m) * (p.N >> 5) + (n >> 5)] = (uint8_t)byte;
      }
    }
  } else {
    for (int i = tid; i < WT * XT * 64; i += blockDim.x) {
      const int l = i & 63, t = (i >> 6) / XT, j = (i >> 6) - t * XT;
      const int n = nt * COLS + 16 * t + 4 * (l >> 4), m = 16 * j + (l & 15);
      if (m < rows && n < p.N) mx_store4(p, p.yrow ? p.yrow[r0 + m] : r0 + m, n, total(t, j, l));
    }
  }
}

// ---------------------------------------------------------------- tiles

// A workgroup is four waves on two 128-row weight segments: wave w multiplies
// rows 32 w .. +31 of both by all activation rows (2 NJ fragments of 16), so with
// gate rows as segment 0 and up rows as segment 1 a lane holds gate and up of the
// same outputs.  Stages of 128 K values (64 bytes a row, chunk c of row r at c ^
// ((r >> 2) & 3): the 16 lanes of a fragment-read pass hit distinct banks) come by
// direct copies into a ring of three, two ahead; two workgroups share a CU.
//
// Exponents: four stages at a time, 16 bytes a row; a lane picks its block's byte of
// each of the four stages into one dword, whose bytes the MFMAs select by number.
constexpr int MX_WST = 256 * 64;  // weight part of a stage
template <int NJ>
struct MxLds {
  static constexpr int XROWS = 32 * NJ;
  static constexpr int STAGE = MX_WST + XROWS * 64;
  static constexpr int SCALES = 3 * STAGE;
  static constexpr int BYTES = SCALES + (256 + XROWS) * 16;
};
static_assert(MxLds<4>::BYTES <= 80 * 1024, "two workgroups per CU");

struct MxTile {
  const uint8_t *w[2], *ws[2];
  int wrows[2];
  const int32_t *xrow;  // of the tile's first position, or null
  int64_t x0;           // x row of the tile's first row (xrow null)
  int rows, it0, it1;   // 128-wide K stages, it0 a multiple of 4
};

template <int NJ>
struct MxSums {
  f32x4 acc[4][2 * NJ];  // [weight fragment][activation fragment]
};

template <int NJ>
struct MxTileMain {
  static AMLA_DEV void run(const MxParams &p, const MxTile &a, MxSums<NJ> &sums) {
  auto &acc = sums.acc;
  extern __shared__ __align__(16) uint8_t lds[];
  using L = MxLds<NJ>;
  constexpr int XC = NJ == 4 ? 2 : 1, C = 4 + XC;  // copies per wave and stage
  const int tid = threadIdx.x, lane = tid & 63, r16 = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int64_t kb = p.K >> 1, ksb = p.K >> 5;
  const int steps = p.K >> 7;
  auto xrow_of = [&](int r) {  // rows past the tile repeat its last row (not stored)
    const int rc = min(r, a.rows - 1);
    return a.xrow ? (int64_t)a.xrow[rc] : a.x0 + rc;
  };

  uint32_t woff[2][2];
#pragma unroll
  for (int s = 0; s < 2; ++s)
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const uint32_t r = 32 * wave + 16 * c + (lane >> 2);
      woff[s][c] = min(r, (uint32_t)a.wrows[s] - 1) * (uint32_t)kb + 16 * ((lane & 3) ^ ((r >> 2) & 3));
    }
  typedef const __attribute__((address_space(1))) uint8_t *gptr;
  gptr xptr[XC];
#pragma unroll
  for (int c = 0; c < XC; ++c) {
    const int r = 8 * NJ * wave + 16 * c + (lane >> 2);
    xptr[c] = (gptr)(static_cast<const uint8_t *>(p.x) + xrow_of(r) * kb + 16 * ((lane & 3) ^ ((r >> 2) & 3)));
  }
  auto opaque = [](uint32_t v) {  // (scalar base + 32-bit lane offset per copy)
    asm volatile("" : "+v"(v));
    return v;
  };
  auto copy = [&](int it, int slot) {
    uint8_t *st = lds + slot * L::STAGE;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      gptr wb = (gptr)(a.w[s] + (size_t)it * 64);
      asm volatile("" : "+s"(wb));
#pragma unroll
      for (int c = 0; c < 2; ++c)
        __builtin_amdgcn_global_load_lds(wb + opaque(woff[s][c]), LDS_PTR(st + (128 * s + 32 * wave + 16 * c) * 64), 16, 0, 0);
    }
#pragma unroll
    for (int c = 0; c < XC; ++c)
      if (NJ > 1 || lane < 32)
        __builtin_amdgcn_global_load_lds(xptr[c] + (size_t)it * 64, LDS_PTR(st + MX_WST + (8 * NJ * wave + 16 * c) * 64), 16, 0, 0);
  };

  // exponents of four stages from stage it: wave w copies those of weight rows 64 w
  // .. +63 and of its quarter of the x rows, 16 bytes a row; where rows are not 16-byte
  // aligned (K % 512), as four planes of one dword a row
  const bool planes = p.K & 511;
  const int seg = wave >> 1;
  const uint32_t swoff = min(64 * (wave & 1) + lane, (seg ? a.wrows[1] : a.wrows[0]) - 1) * (uint32_t)ksb;
  const gptr swp = (gptr)(seg ? a.ws[1] : a.ws[0]);
  const gptr sxp = (gptr)(p.xs + xrow_of(8 * NJ * wave + min(lane, 8 * NJ - 1)) * ksb);
  auto copy_scales = [&](int it) {
    uint8_t *sc = lds + L::SCALES;
    if (!planes) {
      __builtin_amdgcn_global_load_lds(swp + it * 4 + swoff, LDS_PTR(sc + 1024 * wave), 16, 0, 0);
      if (lane < 8 * NJ) __builtin_amdgcn_global_load_lds(sxp + it * 4, LDS_PTR(sc + 4096 + 128 * NJ * wave), 16, 0, 0);
    } else {
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int i = min(it + u, steps - 1) * 4;  // stages past the end are not multiplied
        uint8_t *pl = sc + u * (256 + L::XROWS) * 4;
        __builtin_amdgcn_global_load_lds(swp + i + swoff, LDS_PTR(pl + 256 * wave), 4, 0, 0);
        if (lane < 8 * NJ) __builtin_amdgcn_global_load_lds(sxp + i, LDS_PTR(pl + 1024 + 32 * NJ * wave), 4, 0, 0);
      }
    }
  };
  // the lane's bytes of the four stages of scale row r, in stage order
  const uint32_t gsel = g | (4 + g) << 8;
  auto pick = [&](u32x4 d) {
    return __builtin_amdgcn_perm(__builtin_amdgcn_perm(d.w, d.z, gsel), __builtin_amdgcn_perm(d.y, d.x, gsel), 0x05040100u);
  };
  uint32_t wsc[4], xsc[2 * NJ];
  auto read_scales = [&](auto planes_c) {
    constexpr bool PLANES = decltype(planes_c)::value;
    const uint8_t *sc = lds + L::SCALES + r16 * (PLANES ? 4 : 16);
    auto row = [&](int r) {
      if constexpr (!PLANES) return *reinterpret_cast<const u32x4 *>(sc + 16 * r);
      u32x4 d;
#pragma unroll
      for (int u = 0; u < 4; ++u) d[u] = *reinterpret_cast<const uint32_t *>(sc + (u * (256 + L::XROWS) + r) * 4);
      return d;
    };
#pragma unroll
    for (int f = 0; f < 4; ++f) wsc[f] = pick(row((f >> 1) * 128 + 32 * wave + 16 * (f & 1)));
#pragma unroll
    for (int j = 0; j < 2 * NJ; ++j) xsc[j] = pick(row(256 + 16 * j));
  };

#pragma unroll
  for (int f = 0; f < 4; ++f)
#pragma unroll
    for (int j = 0; j < 2 * NJ; ++j) acc[f][j] = f32x4{0.f, 0.f, 0.f, 0.f};

  copy_scales(a.it0);
  copy(a.it0, 0);
  if (a.it0 + 1 < a.it1) copy(a.it0 + 1, 1);

  const uint32_t frag = 16 * (g ^ ((r16 >> 2) & 3)) + r16 * 64;
  int slot = 0;
  auto stage = [&](int it, auto u_c) {
    constexpr int U = decltype(u_c)::value;
    if (it + 1 < a.it1) wait_vmcnt<C>();  // all but the next stage's copies have landed
    else wait_vmcnt<0>();
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    if constexpr (U == 0) {
      if (!planes) read_scales(std::false_type{});
      else read_scales(std::true_type{});
    }
    // (every wave has read the four stages' exponents before this barrier)
    if constexpr (U == 1)
      if (it + 3 < a.it1) copy_scales(it + 3);
    if (it + 2 < a.it1) copy(it + 2, slot == 0 ? 2 : slot - 1);
    const uint8_t *st = lds + slot * L::STAGE;
    u32x4 wf[4], xf[2 * NJ];
#pragma unroll
    for (int f = 0; f < 4; ++f)
      wf[f] = *reinterpret_cast<const u32x4 *>(st + ((f >> 1) * 128 + 32 * wave + 16 * (f & 1)) * 64 + frag);
#pragma unroll
    for (int j = 0; j < 2 * NJ; ++j) xf[j] = *reinterpret_cast<const u32x4 *>(st + MX_WST + j * 1024 + frag);
#pragma unroll
    for (int j = 0; j < 2 * NJ; ++j)
#pragma unroll
      for (int f = 0; f < 4; ++f) acc[f][j] = mfma_mx<U>(wf[f], wsc[f], xf[j], xsc[j], acc[f][j]);
    slot = slot == 2 ? 0 : slot + 1;
  };
  for (int it = a.it0; it < a.it1; it += 4) {
    stage(it, std::integral_constant<int, 0>{});
    if (it + 1 < a.it1) stage(it + 1, std::integral_constant<int, 1>{});
    if (it + 2 < a.it1) stage(it + 2, std::integral_constant<int, 2>{});
    if (it + 3 < a.it1) stage(it + 3, std::integral_constant<int, 3>{});
  }
}
};

// Outputs of activation row m (from the tile's position r0; n0 first output, ncols
// of them): v[f] as the lane holds them, fragment f of segment f / 2, outputs
// 32 wave + 16 (f % 2) + 4 g .. +3.
template <bool SILU>
AMLA_DEV void mx_tile_store(const MxParams &p, const f32x4 (&v)[4], int wave, int lane, bool live, int pos, int64_t yrow,
                            int n0) {
  const int g = lane >> 4;
  if constexpr (SILU) {
    // the four lanes of a row hold its block of 32: eight values each
    float h[8];
    uint32_t am = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      h[i] = mx_silu_mul(v[i >> 2][i & 3], v[2 + (i >> 2)][i & 3]);
      am = max(am, __float_as_uint(h[i]) & 0x7fffffffu);
    }
    am = max(am, (uint32_t)__shfl_xor((int)am, 16, 64));
    am = max(am, (uint32_t)__shfl_xor((int)am, 32, 64));
    const uint32_t byte = mx_byte(am);
    uint32_t q = mx_codes8(h, mx_scale(byte));
    if (byte == 255) q = 0;
    if (!live) return;
    uint8_t *hc = p.hc + (int64_t)pos * (p.N >> 1) + ((n0 + 32 * wave) >> 1) + 2 * g;
    *reinterpret_cast<uint16_t *>(hc) = (uint16_t)q;
    *reinterpret_cast<uint16_t *>(hc + 8) = (uint16_t)(q >> 16);
    if (g == 0) p.hs[(int64_t)pos * (p.N >> 5) + (n0 >> 5) + wave] = (uint8_t)byte;
  } else {
    if (!live) return;
#pragma unroll
    for (int f = 0; f < 4; ++f) {
      const int n = n0 + (f >> 1) * 128 + 32 * wave + 16 * (f & 1) + 4 * g;
      if (n < p.N) mx_store4(p, yrow, n, v[f]);
    }
  }
}

struct MxSplit {
  int n_tiles, m_tiles;  // one weight: tiles of 256 outputs (SILU: 128) x 128 rows
  int parts;             // K parts of every tile, whole runs of four stages
  float *partial;        // [tile][part][fragment][wave][lane] f32x4
};
constexpr int MX_PART_F32 = 256 * MX_ROWS;

AMLA_DEV int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }

// Column tile nt of `rows` positions from r0 of expert e.
template <int NJ, bool SILU>
AMLA_DEV void mx_tile(const MxParams &p, int e, int r0, int rows, int nt, int it0, int it1, f32x4 *partial) {
  const int tid = threadIdx.x, lane = tid & 63, r16 = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  MxTile a;
  const int n0 = nt * (SILU ? 128 : 256);
#pragma unroll
  for (int s = 0; s < 2; ++s) {
    int n = SILU ? n0 : n0 + 128 * s;
    if (n >= p.N) n = n0;  // no second segment: the first is multiplied twice, not stored
    a.w[s] = p.w[SILU ? s : 0] + e * p.wstride + (int64_t)n * (p.K >> 1);
    a.ws[s] = p.ws[SILU ? s : 0] + e * p.sstride + (int64_t)n * (p.K >> 5);
    a.wrows[s] = min(128, p.N - n);
  }
  a.xrow = p.xrow ? p.xrow + r0 : nullptr;
  a.x0 = r0;
  a.rows = rows;
  a.it0 = it0;
  a.it1 = it1;
  MxSums<NJ> sums;
  MxTileMain<NJ>::run(p, a, sums);
  auto &acc = sums.acc;
#pragma unroll
  for (int j = 0; j < 2 * NJ; ++j) {
    f32x4 v[4] = {acc[0][j], acc[1][j], acc[2][j], acc[3][j]};
    if (partial) {
#pragma unroll
      for (int f = 0; f < 4; ++f) partial[((f * 8 + j) * 4 + wave) * 64 + lane] = v[f];
      continue;
    }
    const int m = 16 * j + r16;
    const bool live = m < rows;
    const int pos = r0 + min(m, rows - 1);
    mx_tile_store<SILU>(p, v, wave, lane, live, pos, p.yrow ? p.yrow[pos] : pos, n0);
  }
}

template <bool SILU>
AMLA_DEV void mx_tile_rows(const MxParams &p, int e, int r0, int rows, int nt, int it0, int it1, f32x4 *partial) {
  if (rows <= 32) mx_tile<1, SILU>(p, e, r0, rows, nt, it0, it1, partial);
  else if (rows <= 64) mx_tile<2, SILU>(p, e, r0, rows, nt, it0, it1, partial);
  else mx_tile<4, SILU>(p, e, r0, rows, nt, it0, it1, partial);
}

// One weight: tile t, K part q.
template <bool SILU>
__global__ __launch_bounds__(256, 2) void mx_linear_kernel(MxParams p, MxSplit sp) {
  const int tiles = sp.n_tiles * sp.m_tiles;
  const int l = xcd_run(blockIdx.x, tiles * sp.parts);
  if (l < 0) return;
  const int q = l / tiles, t = l - q * tiles;
  int nt, mt;
  tile_coords(t, sp.n_tiles, sp.m_tiles, nt, mt);
  const int steps = p.K >> 7, quads = (steps + 3) >> 2;
  const int it0 = 4 * (quads * q / sp.parts), it1 = min(steps, 4 * (quads * (q + 1) / sp.parts));
  f32x4 *partial = sp.parts > 1 ? reinterpret_cast<f32x4 *>(sp.partial) + (size_t)(t * sp.parts + q) * (MX_PART_F32 / 4)
                                : nullptr;
  mt = uniform(mt);
  mx_tile_rows<SILU>(p, 0, mt * MX_ROWS, min(MX_ROWS, p.M - mt * MX_ROWS), uniform(nt), uniform(it0), uniform(it1), partial);
}

// Sums the K parts of row fragment j of a tile in part order.
template <bool SILU>
__global__ __launch_bounds__(256) void mx_finish_kernel(MxParams p, MxSplit sp) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int t = blockIdx.x >> 3, j = blockIdx.x & 7;
  int nt, mt;
  tile_coords(t, sp.n_tiles, sp.m_tiles, nt, mt);
  if (mt * MX_ROWS + 16 * j >= p.M) return;
  const f32x4 *src = reinterpret_cast<const f32x4 *>(sp.partial) + (size_t)t * sp.parts * (MX_PART_F32 / 4) +
                     (j * 4 + wave) * 64 + lane;
  f32x4 v[4];
#pragma unroll
  for (int f = 0; f < 4; ++f) v[f] = src[f * 2048];
  for (int q = 1; q < sp.parts; ++q)
#pragma unroll
    for (int f = 0; f < 4; ++f) v[f] += src[(size_t)q * (MX_PART_F32 / 4) + f * 2048];
  const int m = mt * MX_ROWS + 16 * j + (lane & 15);
  mx_tile_store<SILU>(p, v, wave, lane, m < p.M, m, m, nt * (SILU ? 128 : 256));
}

// The scheduled entries of up to 128 rows: a contiguous run of (entry, column
// tile) per XCD, so that the activation rows of an entry are read from one L2.
template <bool SILU>
__global__ __launch_bounds__(256, 2) void mx_sched_kernel(MxParams p, int ntiles) {
  const int l = xcd_run(blockIdx.x, *p.count * ntiles);
  if (l < 0) return;
  const int t = uniform(l / ntiles), nt = uniform(l) - t * ntiles;
  const int32_t *en = p.ent + 4 * t;
  const int e = uniform(en[0]), r0 = uniform(en[1]), rows = uniform(en[2]);
  if (!SILU && e < 0) {  // rows of no expert
    for (int i = threadIdx.x; i < rows * 64; i += 256) {
      const int r = i >> 6, n = nt * 256 + 4 * (i & 63);
      if (n < p.N) mx_store4(p, p.yrow ? p.yrow[r0 + r] : r0 + r, n, f32x4{0.f, 0.f, 0.f, 0.f});
    }
    return;
  }
  mx_tile_rows<SILU>(p, e, r0, rows, nt, 0, p.K >> 7, nullptr);
}

// ---------------------------------------------------------------- schedules

// Entries of the groups [offsets[e], offsets[e + 1]) of m rows, at most rows_max
// rows each.  Offsets are taken as they come but never past m and never
// backwards: bad ones lose rows, not bounds.  rest: the rows of no group as
// entries of expert -1.
__global__ __launch_bounds__(1024) void mx_group_kernel(const int32_t *__restrict__ offsets, int E, int m, int rows_max,
                                                        int rest, int32_t *__restrict__ count,
                                                        int32_t *__restrict__ ent) {
  __shared__ int32_t start[MX_MAX_GROUPS + 1], wmax[16], wsum[16];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  // start[i] = max of the clamped offsets 0 .. i, i <= E (offset E by the last step below)
  int v = tid <= E ? min(max(offsets[tid], 0), m) : 0;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int u = __shfl_up(v, o, 64);
    if (lane >= o) v = max(v, u);
  }
  if (lane == 63) wmax[wave] = v;
  __syncthreads();
  for (int w = 0; w < wave; ++w) v = max(v, wmax[w]);
  start[tid] = v;
  __syncthreads();
  if (tid == 0 && E == MX_MAX_GROUPS) start[E] = max(start[E - 1], min(max(offsets[E], 0), m));
  __syncthreads();
  int first = 0, rows = 0, id = -1;
  if (tid < E) {
    first = start[tid];
    rows = start[tid + 1] - first;
    id = tid;
  }
  int n = (rows + rows_max - 1) / rows_max;
  const int own = n;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int u = __shfl_up(n, o, 64);
    if (lane >= o) n += u;
  }
  if (lane == 63) wsum[wave] = n;
  __syncthreads();
  for (int w = 0; w < wave; ++w) n += wsum[w];
  for (int i = 0; i < own; ++i) {
    int32_t *en = ent + 4 * (n - own + i);
    en[0] = id; en[1] = first + i * rows_max; en[2] = min(rows_max, rows - i * rows_max); en[3] = 0;
  }
  if (tid == 1023) {
    int c = n;
    if (rest) {
      const int lo[2] = {0, start[E]}, hi[2] = {start[0], m};
      for (int k = 0; k < 2; ++k)
        for (int r = lo[k]; r < hi[k]; r += rows_max, ++c) {
          int32_t *en = ent + 4 * c;
          en[0] = -1; en[1] = r; en[2] = min(rows_max, hi[k] - r); en[3] = 0;
        }
    }
    *count = c;
  }
}

// expert_out rows of slots that no expert computes
__global__ __launch_bounds__(256) void mx_clear_skipped_kernel(const int64_t *__restrict__ idx, int E, int d,
                                                               uint16_t *__restrict__ y) {
  const int64_t v = idx[blockIdx.x];
  if (v >= 0 && v < E) return;
  for (int i = threadIdx.x; i < d / 8; i += 256) *reinterpret_cast<u32x4 *>(y + (int64_t)blockIdx.x * d + 8 * i) = u32x4{0, 0, 0, 0};
}

// ---------------------------------------------------------------- launches

// Waves of a skinny workgroup: K steps to share
static int mx_waves(int K) { return K / 128 >= 16 ? 8 : 4; }

template <int WT, int XT, bool FUSED, bool SILU>
static int launch_skinny(const MxParams &p, int entries, hipStream_t st) {
  const int cols = SILU ? 8 * WT : 16 * WT, ntiles = (p.N + cols - 1) / cols, nw = mx_waves(p.K);
  const int64_t blocks = (int64_t)entries * ntiles;
  if (blocks > INT32_MAX) return fail(AMLA_EUNSUPPORTED, "mxfp4 product: %d entries", entries);
  mx_skinny_kernel<WT, XT, FUSED, SILU><<<dim3((unsigned)blocks), 64 * nw, nw * WT * XT * 1024, st>>>(p, ntiles);
  return check_launch("mxfp4 skinny product");
}

constexpr int MX_SKINNY_FUSED = 16;  // bf16 rows the skinny kernel quantises itself
constexpr int MX_SKINNY = 64;        // most rows of an entry on it

// entries of at most `rows` rows; p.xs null: bf16 rows (rows <= MX_SKINNY_FUSED)
static int launch_mx_skinny(const MxParams &p, int rows, int entries, hipStream_t st) {
  const bool wide = (int64_t)entries * (p.N / 32) >= 400;  // 32 weight rows a workgroup still fill the machine
  if (!p.xs) return wide ? launch_skinny<2, 1, true, false>(p, entries, st) : launch_skinny<1, 1, true, false>(p, entries, st);
  if (rows <= 16) return wide ? launch_skinny<2, 1, false, false>(p, entries, st) : launch_skinny<1, 1, false, false>(p, entries, st);
  if (rows <= 32) return launch_skinny<2, 2, false, false>(p, entries, st);
  return launch_skinny<2, 4, false, false>(p, entries, st);
}
static int launch_mx_skinny_silu(const MxParams &p, int rows, int entries, hipStream_t st) {
  if (!p.xs) return launch_skinny<4, 1, true, true>(p, entries, st);
  return launch_skinny<4, 1, false, true>(p, entries, st);
}

template <typename F>
static int mx_lds(F *fn) {  // dynamic LDS above 64 KB
  const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void *>(fn), hipFuncAttributeMaxDynamicSharedMemorySize,
                                           MxLds<4>::BYTES);
  return e == hipSuccess ? AMLA_OK : fail((int)e, "mxfp4 tiles: LDS size: %s", hipGetErrorString(e));
}

static MxSplit plan_mx_split(int64_t M, int N, int K, bool silu) {
  MxSplit sp = {};
  const int cols = silu ? 128 : 256;
  sp.n_tiles = (N + cols - 1) / cols;
  sp.m_tiles = (int)((M + MX_ROWS - 1) / MX_ROWS);
  const int64_t tiles = (int64_t)sp.n_tiles * sp.m_tiles;
  const int quads = (K / 128 + 3) / 4;
  sp.parts = (int)std::max<int64_t>(1, std::min<int64_t>(quads, 256 / tiles));
  return sp;
}
static size_t mx_split_bytes(const MxSplit &sp) {
  return sp.parts > 1 ? (size_t)sp.n_tiles * sp.m_tiles * sp.parts * MX_PART_F32 * 4 : 0;
}

template <bool SILU>
static int launch_mx_linear(const MxParams &p, MxSplit sp, hipStream_t st) {
  const int64_t blocks = ((int64_t)sp.n_tiles * sp.m_tiles * sp.parts + 7) / 8 * 8;
  if (blocks > INT32_MAX) return fail(AMLA_EUNSUPPORTED, "mxfp4 product: %d x %d outputs", p.M, p.N);
  int rc = mx_lds(mx_linear_kernel<SILU>);
  if (rc) return rc;
  mx_linear_kernel<SILU><<<dim3((unsigned)blocks), 256, MxLds<4>::BYTES, st>>>(p, sp);
  if ((rc = check_launch("mxfp4 product")) || sp.parts == 1) return rc;
  mx_finish_kernel<SILU><<<dim3((unsigned)(sp.n_tiles * sp.m_tiles * 8)), 256, 0, st>>>(p, sp);
  return check_launch("mxfp4 K-part finish");
}

template <bool SILU>
static int launch_mx_sched(const MxParams &p, int max_entries, hipStream_t st) {
  const int cols = SILU ? 128 : 256, ntiles = (p.N + cols - 1) / cols;
  const int64_t blocks = ((int64_t)max_entries * ntiles + 7) / 8 * 8;
  if (blocks > INT32_MAX) return fail(AMLA_EUNSUPPORTED, "mxfp4 product: %d entries", max_entries);
  int rc = mx_lds(mx_sched_kernel<SILU>);
  if (rc) return rc;
  mx_sched_kernel<SILU><<<dim3((unsigned)blocks), 256, MxLds<4>::BYTES, st>>>(p, ntiles);
  return check_launch("mxfp4 grouped product");
}

// ---------------------------------------------------------------- workspaces

struct MxTake {  // 256-byte aligned pieces of a workspace
  size_t off = 0;
  size_t operator()(size_t bytes) {
    const size_t o = off;
    off = align_up(off + bytes, 256);
    return o;
  }
};
static size_t mx_codes_bytes(int64_t rows, int64_t k) { return (size_t)rows * (k / 2); }
static size_t mx_scale_bytes(int64_t rows, int64_t k) { return (size_t)rows * (k / 32); }

struct MxLinearLayout {
  size_t xc, xs, part, total;
  bool skinny;
  MxSplit sp;
};
// held: x comes quantised
static MxLinearLayout mx_linear_layout(int64_t m, int64_t k, int64_t n, bool held) {
  MxLinearLayout L = {};
  MxTake take;
  L.skinny = m <= MX_SKINNY;
  if (!held && m > MX_SKINNY_FUSED) {
    L.xc = take(mx_codes_bytes(m, k));
    L.xs = take(mx_scale_bytes(m, k));
  }
  if (!L.skinny) {
    L.sp = plan_mx_split(m, (int)n, (int)k, false);
    L.part = take(mx_split_bytes(L.sp));
  }
  L.total = take.off;
  return L;
}

struct MxGroupedLayout {
  size_t count, ent, xc, xs, total;
  int rows, max_entries;  // of an entry; entries at most
  bool skinny;
};
static MxGroupedLayout mx_grouped_layout(int64_t m, int64_t k, int64_t E, bool held) {
  MxGroupedLayout L = {};
  MxTake take;
  L.skinny = m <= 16;
  L.rows = L.skinny ? 16 : MX_ROWS;
  L.max_entries = (int)(std::min(E, m) + m / L.rows + 2);
  L.count = take(4);
  L.ent = take((size_t)L.max_entries * 16);
  if (!held && !L.skinny) {
    L.xc = take(mx_codes_bytes(m, k));
    L.xs = take(mx_scale_bytes(m, k));
  }
  L.total = take.off;
  return L;
}

struct MxSwigluLayout {
  size_t xc, xs, hc, hs, lin, total;
  bool skinny;
  MxSplit sp;
  MxLinearLayout down;
};
static MxSwigluLayout mx_swiglu_layout(int64_t m, int64_t k, int64_t n) {
  MxSwigluLayout L = {};
  MxTake take;
  L.skinny = m <= MX_SKINNY_FUSED;
  L.hc = take(mx_codes_bytes(m, n));
  L.hs = take(mx_scale_bytes(m, n));
  if (!L.skinny) {
    L.xc = take(mx_codes_bytes(m, k));
    L.xs = take(mx_scale_bytes(m, k));
    L.sp = plan_mx_split(m, (int)n, (int)k, true);
  }
  L.down = mx_linear_layout(m, n, k, true);
  L.lin = take(std::max(L.skinny ? 0 : mx_split_bytes(L.sp), L.down.total));
  L.total = take.off;
  return L;
}

struct MxMoeLayout {
  size_t hdr, count, gather, scatter, ent, xc, xs, hc, hs, total;
  int rows, max_entries;
  bool skinny;
};
static MxMoeLayout mx_moe_layout(int64_t m, int64_t d, int top_k, int64_t n, int64_t E) {
  MxMoeLayout L = {};
  MxTake take;
  const int64_t S = m * top_k;
  L.skinny = m <= 16;
  L.rows = L.skinny ? 16 : MX_ROWS;
  L.max_entries = (int)std::min<int64_t>(S, std::min<int64_t>(E, S) + S / L.rows);
  L.hdr = take(16);
  L.count = take(4);
  L.gather = take((size_t)S * 4);
  L.scatter = take((size_t)S * 4);
  L.ent = take((size_t)L.max_entries * 16);
  L.hc = take(mx_codes_bytes(S, n));
  L.hs = take(mx_scale_bytes(S, n));
  if (!L.skinny) {
    L.xc = take(mx_codes_bytes(m, d));
    L.xs = take(mx_scale_bytes(m, d));
  }
  L.total = take.off;
  return L;
}

static bool mx_sizes_ok(int64_t m, int64_t n, int64_t k) {
  return m > 0 && n > 0 && k > 0 && m <= INT32_MAX && n <= INT32_MAX / 4 && k <= (1 << 24) && k % 128 == 0;
}

static void mx_outputs(MxParams &p, void *y, int64_t ldy, int dtype) {
  p.y = y;
  p.ldy = ldy;
  p.f32 = dtype == AMLA_FP32;
  p.vec = p.N % 4 == 0 && ldy % 4 == 0 && reinterpret_cast<uintptr_t>(y) % (p.f32 ? 16 : 8) == 0;
}

}  // namespace amla

using namespace amla;

extern "C" {

size_t amla_mxfp4_linear_workspace_bytes(int64_t m, int64_t n, int64_t k, int quantized) {
  if (!mx_sizes_ok(m, n, k)) return 0;
  return mx_linear_layout(m, k, n, quantized != 0).total;
}

int amla_mxfp4_linear(const void *x, const void *x_scales, int64_t m, int64_t k, int64_t ldx, const void *weight,
                      const void *scales, int64_t n, void *y, int dtype, int64_t ldy, void *workspace,
                      size_t workspace_bytes, void *stream) {
  if (!x || !weight || !scales || !y) return fail(AMLA_EINVAL, "mxfp4_linear: null pointer");
  if (m < 0 || n <= 0 || k <= 0) return fail(AMLA_EINVAL, "mxfp4_linear: bad shape m=%lld n=%lld k=%lld", (long long)m,
                                             (long long)n, (long long)k);
  if (dtype != AMLA_BF16 && dtype != AMLA_FP32) return fail(AMLA_EINVAL, "mxfp4_linear: output dtype %d", dtype);
  if ((!x_scales && ldx < k) || ldy < n) return fail(AMLA_EINVAL, "mxfp4_linear: row stride smaller than the row");
  if (m == 0) return AMLA_OK;
  if (!mx_sizes_ok(m, n, k) || !aligned16(x) || !aligned16(weight) || reinterpret_cast<uintptr_t>(scales) % 4 ||
      reinterpret_cast<uintptr_t>(x_scales) % 4 || (!x_scales && ldx % 8))
    return fail(AMLA_EUNSUPPORTED,
                "mxfp4_linear: needs k %% 128 == 0, 16-byte aligned x rows and weight and 4-byte aligned scales "
                "(n=%lld k=%lld)", (long long)n, (long long)k);
  const MxLinearLayout L = mx_linear_layout(m, k, n, x_scales != nullptr);
  if (L.total && (!workspace || workspace_bytes < L.total || !aligned16(workspace)))
    return fail(AMLA_EWORKSPACE, "mxfp4_linear: needs %zu bytes of 16-byte aligned workspace (got %zu)", L.total,
                workspace ? workspace_bytes : (size_t)0);
  uint8_t *ws = static_cast<uint8_t *>(workspace);
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  MxParams p = {};
  p.x = x;
  p.xs = static_cast<const uint8_t *>(x_scales);
  p.ldx = ldx;
  p.w[0] = p.w[1] = static_cast<const uint8_t *>(weight);
  p.ws[0] = p.ws[1] = static_cast<const uint8_t *>(scales);
  p.M = (int)m; p.N = (int)n; p.K = (int)k;
  mx_outputs(p, y, ldy, dtype);
  if (!x_scales && m > MX_SKINNY_FUSED) {
    const int rc = launch_mx_quantize_bf16(static_cast<const uint16_t *>(x), m, k, ldx, ws + L.xc, ws + L.xs, st);
    if (rc) return rc;
    p.x = ws + L.xc;
    p.xs = ws + L.xs;
  }
  if (L.skinny) return launch_mx_skinny(p, (int)m, 1, st);
  MxSplit sp = L.sp;
  sp.partial = reinterpret_cast<float *>(ws + L.part);
  return launch_mx_linear<false>(p, sp, st);
}

size_t amla_mxfp4_grouped_linear_workspace_bytes(int64_t m, int64_t n, int64_t k, int64_t n_experts, int quantized) {
  if (!mx_sizes_ok(m, n, k) || n_experts <= 0 || n_experts > MX_MAX_GROUPS) return 0;
  return mx_grouped_layout(m, k, n_experts, quantized != 0).total;
}

int amla_mxfp4_grouped_linear(const void *x, const void *x_scales, int64_t m, int64_t k, int64_t ldx,
                              const void *weight, const void *scales, int64_t n, int64_t n_experts,
                              const int32_t *offsets, void *y, int dtype, int64_t ldy, int clear_rest, void *workspace,
                              size_t workspace_bytes, void *stream) {
  if (!x || !weight || !scales || !offsets || !y) return fail(AMLA_EINVAL, "mxfp4_grouped_linear: null pointer");
  if (m < 0 || n <= 0 || k <= 0 || n_experts <= 0)
    return fail(AMLA_EINVAL, "mxfp4_grouped_linear: bad shape m=%lld n=%lld k=%lld experts=%lld", (long long)m,
                (long long)n, (long long)k, (long long)n_experts);
  if (dtype != AMLA_BF16 && dtype != AMLA_FP32) return fail(AMLA_EINVAL, "mxfp4_grouped_linear: output dtype %d", dtype);
  if ((!x_scales && ldx < k) || ldy < n) return fail(AMLA_EINVAL, "mxfp4_grouped_linear: row stride smaller than the row");
  if (m == 0) return AMLA_OK;
  if (!mx_sizes_ok(m, n, k) || n_experts > MX_MAX_GROUPS || !aligned16(x) || !aligned16(weight) ||
      reinterpret_cast<uintptr_t>(scales) % 4 || reinterpret_cast<uintptr_t>(x_scales) % 4 || (!x_scales && ldx % 8))
    return fail(AMLA_EUNSUPPORTED,
                "mxfp4_grouped_linear: needs k %% 128 == 0, at most %d experts, 16-byte aligned x rows and weight and "
                "4-byte aligned scales (n=%lld k=%lld)", MX_MAX_GROUPS, (long long)n, (long long)k);
  const MxGroupedLayout L = mx_grouped_layout(m, k, n_experts, x_scales != nullptr);
  if (!workspace || workspace_bytes < L.total || !aligned16(workspace))
    return fail(AMLA_EWORKSPACE, "mxfp4_grouped_linear: needs %zu bytes of 16-byte aligned workspace (got %zu)", L.total,
                workspace ? workspace_bytes : (size_t)0);
  uint8_t *ws = static_cast<uint8_t *>(workspace);
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  int32_t *count = reinterpret_cast<int32_t *>(ws + L.count), *ent = reinterpret_cast<int32_t *>(ws + L.ent);
  mx_group_kernel<<<1, 1024, 0, st>>>(offsets, (int)n_experts, (int)m, L.rows, clear_rest, count, ent);
  int rc = check_launch("mxfp4 group schedule");
  if (rc) return rc;
  MxParams p = {};
  p.x = x;
  p.xs = static_cast<const uint8_t *>(x_scales);
  p.ldx = ldx;
  p.w[0] = p.w[1] = static_cast<const uint8_t *>(weight);
  p.ws[0] = p.ws[1] = static_cast<const uint8_t *>(scales);
  p.wstride = n * (k / 2);
  p.sstride = n * (k / 32);
  p.ent = ent;
  p.count = count;
  p.M = (int)m; p.N = (int)n; p.K = (int)k;
  mx_outputs(p, y, ldy, dtype);
  if (L.skinny) return launch_mx_skinny(p, L.rows, L.max_entries, st);
  if (!x_scales) {
    if ((rc = launch_mx_quantize_bf16(static_cast<const uint16_t *>(x), m, k, ldx, ws + L.xc, ws + L.xs, st))) return rc;
    p.x = ws + L.xc;
    p.xs = ws + L.xs;
  }
  return launch_mx_sched<false>(p, L.max_entries, st);
}

size_t amla_mxfp4_swiglu_workspace_bytes(int64_t m, int64_t k, int64_t n) {
  if (!mx_sizes_ok(m, n, k) || n % 128) return 0;
  return mx_swiglu_layout(m, k, n).total;
}

int amla_mxfp4_swiglu(const void *x, int64_t m, int64_t k, int64_t ldx, const void *gate_w, const void *gate_s,
                      const void *up_w, const void *up_s, int64_t n, const void *down_w, const void *down_s, void *y,
                      void *workspace, size_t workspace_bytes, void *stream) {
  if (!x || !gate_w || !gate_s || !up_w || !up_s || !down_w || !down_s || !y)
    return fail(AMLA_EINVAL, "mxfp4_swiglu: null pointer");
  if (m < 0 || n <= 0 || k <= 0) return fail(AMLA_EINVAL, "mxfp4_swiglu: bad shape m=%lld k=%lld n=%lld", (long long)m,
                                             (long long)k, (long long)n);
  if (ldx < k) return fail(AMLA_EINVAL, "mxfp4_swiglu: row stride smaller than the row");
  if (m == 0) return AMLA_OK;
  bool ok = mx_sizes_ok(m, n, k) && n % 128 == 0 && ldx % 8 == 0 && aligned16(x) && aligned16(y);
  for (const void *w : {gate_w, up_w, down_w}) ok = ok && aligned16(w);
  for (const void *s : {gate_s, up_s, down_s}) ok = ok && reinterpret_cast<uintptr_t>(s) % 4 == 0;
  if (!ok)
    return fail(AMLA_EUNSUPPORTED,
                "mxfp4_swiglu: needs k %% 128 == 0, n %% 128 == 0, 16-byte aligned rows and weights and 4-byte aligned "
                "scales (n=%lld k=%lld)", (long long)n, (long long)k);
  const MxSwigluLayout L = mx_swiglu_layout(m, k, n);
  if (!workspace || workspace_bytes < L.total || !aligned16(workspace))
    return fail(AMLA_EWORKSPACE, "mxfp4_swiglu: needs %zu bytes of 16-byte aligned workspace (got %zu)", L.total,
                workspace ? workspace_bytes : (size_t)0);
  uint8_t *ws = static_cast<uint8_t *>(workspace);
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  MxParams p = {};
  p.x = x;
  p.ldx = ldx;
  p.w[0] = static_cast<const uint8_t *>(gate_w);
  p.w[1] = static_cast<const uint8_t *>(up_w);
  p.ws[0] = static_cast<const uint8_t *>(gate_s);
  p.ws[1] = static_cast<const uint8_t *>(up_s);
  p.M = (int)m; p.N = (int)n; p.K = (int)k;
  p.hc = ws + L.hc;
  p.hs = ws + L.hs;
  int rc;
  if (L.skinny) {
    rc = launch_mx_skinny_silu(p, (int)m, 1, st);
  } else {
    if ((rc = launch_mx_quantize_bf16(static_cast<const uint16_t *>(x), m, k, ldx, ws + L.xc, ws + L.xs, st))) return rc;
    p.x = ws + L.xc;
    p.xs = ws + L.xs;
    MxSplit sp = L.sp;
    sp.partial = reinterpret_cast<float *>(ws + L.lin);
    rc = launch_mx_linear<true>(p, sp, st);
  }
  if (rc) return rc;
  return amla_mxfp4_linear(ws + L.hc, ws + L.hs, m, n, n, down_w, down_s, k, y, AMLA_BF16, k, ws + L.lin, L.down.total,
                           stream);
}

size_t amla_mxfp4_moe_experts_workspace_bytes(int64_t m, int64_t d, int top_k, int64_t n_inter, int64_t n_experts) {
  if (!mx_sizes_ok(m, n_inter, d) || n_inter % 128 || top_k <= 0 || top_k > 64 || n_experts <= 0 || n_experts > 512 ||
      m * top_k > 65536)
    return 0;
  return mx_moe_layout(m, d, top_k, n_inter, n_experts).total;
}

int amla_mxfp4_moe_experts(const void *hidden, int64_t m, int64_t d, int64_t ldh, int top_k, const int64_t *indices,
                           int64_t n_inter, int64_t n_experts, const void *gate_w, const void *gate_s, const void *up_w,
                           const void *up_s, const void *down_w, const void *down_s, void *expert_out,
                           int clear_skipped, void *workspace, size_t workspace_bytes, void *stream) {
  if (!hidden || !indices || !gate_w || !gate_s || !up_w || !up_s || !down_w || !down_s || !expert_out)
    return fail(AMLA_EINVAL, "mxfp4_moe_experts: null pointer");
  if (m < 0 || d <= 0 || top_k <= 0 || n_inter <= 0 || n_experts <= 0 || ldh < d)
    return fail(AMLA_EINVAL, "mxfp4_moe_experts: bad sizes");
  if (m == 0) return AMLA_OK;
  if (top_k > 64 || n_experts > 512 || m > 65536 || m * top_k > 65536)
    return fail(AMLA_EUNSUPPORTED, "mxfp4_moe_experts: needs top_k <= 64, at most 512 experts and 65536 slots per call");
  bool ok = mx_sizes_ok(m, n_inter, d) && n_inter % 128 == 0 && ldh % 8 == 0 && aligned16(hidden) && aligned16(expert_out);
  for (const void *w : {gate_w, up_w, down_w}) ok = ok && aligned16(w);
  for (const void *s : {gate_s, up_s, down_s}) ok = ok && reinterpret_cast<uintptr_t>(s) % 4 == 0;
  if (!ok)
    return fail(AMLA_EUNSUPPORTED,
                "mxfp4_moe_experts: needs hidden %% 128 == 0, intermediate %% 128 == 0, 16-byte aligned rows and "
                "weights and 4-byte aligned scales");
  const MxMoeLayout L = mx_moe_layout(m, d, top_k, n_inter, n_experts);
  if (!workspace || workspace_bytes < L.total || !aligned16(workspace))
    return fail(AMLA_EWORKSPACE, "mxfp4_moe_experts: needs %zu bytes of 16-byte aligned workspace (got %zu)", L.total,
                workspace ? workspace_bytes : (size_t)0);
  uint8_t *ws = static_cast<uint8_t *>(workspace);
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  int32_t *count = reinterpret_cast<int32_t *>(ws + L.count), *ent = reinterpret_cast<int32_t *>(ws + L.ent);
  int32_t *gather = reinterpret_cast<int32_t *>(ws + L.gather), *scatter = reinterpret_cast<int32_t *>(ws + L.scatter);
  const int S = (int)(m * top_k), E = (int)n_experts;
  int rc = launch_moe_sort(indices, S, top_k, E, (int)std::min<int64_t>(m, 64), L.rows, nullptr,
                           reinterpret_cast<int32_t *>(ws + L.hdr), count, gather, scatter, ent, st);
  if (rc) return rc;
  if (clear_skipped) {
    mx_clear_skipped_kernel<<<dim3((unsigned)S), 256, 0, st>>>(indices, E, (int)d, static_cast<uint16_t *>(expert_out));
    if ((rc = check_launch("mxfp4_moe_experts skipped slots"))) return rc;
  }
  MxParams p = {};
  p.x = hidden;
  p.ldx = ldh;
  p.xrow = gather;
  p.w[0] = static_cast<const uint8_t *>(gate_w);
  p.w[1] = static_cast<const uint8_t *>(up_w);
  p.ws[0] = static_cast<const uint8_t *>(gate_s);
  p.ws[1] = static_cast<const uint8_t *>(up_s);
  p.wstride = n_inter * (d / 2);
  p.sstride = n_inter * (d / 32);
  p.ent = ent;
  p.count = count;
  p.M = S; p.N = (int)n_inter; p.K = (int)d;
  p.hc = ws + L.hc;
  p.hs = ws + L.hs;
  MxParams q = p;
  q.x = ws + L.hc;
  q.xs = ws + L.hs;
  q.xrow = nullptr;
  q.yrow = scatter;
  q.w[0] = q.w[1] = static_cast<const uint8_t *>(down_w);
  q.ws[0] = q.ws[1] = static_cast<const uint8_t *>(down_s);
  q.N = (int)d; q.K = (int)n_inter;
  mx_outputs(q, expert_out, d, AMLA_BF16);
  if (L.skinny) {
    if ((rc = launch_mx_skinny_silu(p, L.rows, L.max_entries, st))) return rc;
    return launch_mx_skinny(q, L.rows, L.max_entries, st);
  }
  if ((rc = launch_mx_quantize_bf16(static_cast<const uint16_t *>(hidden), m, d, ldh, ws + L.xc, ws + L.xs, st)))
    return rc;
  p.x = ws + L.xc;
  p.xs = ws + L.xs;
  if ((rc = launch_mx_sched<true>(p, L.max_entries, st))) return rc;
  return launch_mx_sched<false>(q, L.max_entries, st);
}

}  // extern "C"
