// MXFP4 products for gfx950: y = deq(x) deq(w)^T with both operands in 4 bits on
// the scaled MFMA (16x16x128, exact products, fp32 sums).  A stream kernel for up
// to 16 activation rows, bound by the weights' bytes; tiles of 256 weight rows x up
// to 256 activation rows for more, and of 128 x 64 where there are few; each for one
// weight or (but the last) for a device schedule of experts, with the output rows or
// silu(gate) * up quantised again as epilogue.
#include <algorithm>
#include <type_traits>

#include "mxfp4.h"
#include "tile_order.h"

namespace amla {

constexpr int MX_MAX_GROUPS = 1024;  // experts of a grouped product

// Operands of a launch.  Two weights (SILU): gate and up.  ent (with count): the
// schedule entries (expert, first position, rows, -); null: one entry of M rows.
// Position p reads x row xrow[p] and writes y row yrow[p] (null: p).
struct MxParams {
  const void *x;       // codes, or bf16 values (xs null; stream product only)
  const uint8_t *xs;
  int64_t ldx;         // bf16 row stride
  const int32_t *xrow, *yrow;
  const uint8_t *w[2], *ws[2];
  int64_t wstride, sstride;  // bytes from expert to expert
  const int32_t *ent, *count;
  int M, N, K;
  int rest;            // count[1] entries of expert -1 come behind the others
  void *y;
  int64_t ldy;
  int f32, vec, vec16; // fp32 outputs; four outputs, 16 bytes of them per store
  uint8_t *hc, *hs;    // SILU: codes and exponents by position
};

AMLA_DEV int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }

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

// ---------------------------------------------------------------- stream product

// Up to 16 activation rows: the weights stream once, from memory straight into the
// operands' registers, past activations that stay in LDS.
//
// An item is 16 weight rows (SILU: 32 of gate and the same 32 of up) of an entry; a
// workgroup takes a contiguous run of items.  Its waves share the K of every weight
// row by runs of quads (512 K values) and meet in LDS, in wave order.  A wave walks
// the quads of all its items as one sequence, with the next quad's loads in flight
// while it multiplies one, also across items; a quad is 16 rows x 256 bytes, and 16
// bytes of exponents a row more (the lanes of a row share them).
//
// The matrix units want 16 rows x 64 bytes in a register.  A load takes 4 rows x 256
// bytes all the same, and the wave turns the quad over in 4 KB of LDS of its own (no
// barrier: its LDS operations stay in order): memory delivers whole lines faster (8 x
// 65536 x 7168 58 -> 54 us, 8 x 7168 x 18432 22.8 -> 21.5, 4 x 2112 x 7168 7.0 -> 6.3).
// Four waves a SIMD have to fit: with 129 registers instead of 128 the down projections
// of 57 experts took 87 us, 73 so.
//
// Bound by the weights' stream: 1 x 262144 x 7168 in 177 us, 5.6 TB/s, and 4 us for the
// start and the end of a call.  Three quads in flight instead of two, two or four 16-row
// fragments an item and other numbers of workgroups changed that by 2 % at most.
//
// Activations: rows of one entry (at most `mr`, a power of two), bf16 ones quantised on
// the way in, which saves the pass and the launch before it.  Codes at [step][K
// block][row], so that the lanes read 16 rows in a row; exponents as dwords of the
// quad's four steps, which the MFMAs select by number.
struct MxStream {
  int ntiles;      // items of an entry
  int mr;          // activation rows kept
  int xcodes;      // bytes of the codes, and
  int xbytes;      // with the exponents (the partial sums come behind)
  int turn;        // of the waves' 4 KB, behind the partial sums
};

template <bool SILU, bool PLANES>
__global__ __launch_bounds__(512, 4) void mx_stream_kernel(MxParams p, MxStream sp) {
  extern __shared__ __align__(16) uint8_t lds[];
  constexpr int WT = SILU ? 4 : 1;  // 16-row fragments of an item
  constexpr int COLS = SILU ? 32 : 16;
  constexpr bool TURN = !PLANES;
  const int tid = threadIdx.x, lane = tid & 63, r16 = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), nw = blockDim.x >> 6;
  const int steps = p.K >> 7, quads = (steps + 3) >> 2;
  const int q0 = quads * wave / nw, q1 = quads * (wave + 1) / nw;
  const int64_t kb = p.K >> 1, ksb = p.K >> 5;
  // (scalar loads: a vector load among the weights' would be waited for with them)
  typedef const __attribute__((address_space(4))) int32_t *sptr;
  const sptr ent = (sptr)p.ent;
  const int entries = p.ent ? *(sptr)p.count : 1;
  const int64_t total = (int64_t)entries * sp.ntiles;
  const int64_t i0 = total * blockIdx.x / gridDim.x, i1 = total * (blockIdx.x + 1) / gridDim.x;
  if constexpr (!SILU)
    if (p.rest) {  // rows of no expert
      const int rest = p.count[1];
      for (int en = blockIdx.x; en < rest; en += gridDim.x) {
        const int r0 = p.ent[4 * (entries + en) + 1], rows = p.ent[4 * (entries + en) + 2], n4 = (p.N + 3) >> 2;
        for (int i = tid; i < rows * n4; i += blockDim.x) {
          const int r = i / n4;
          mx_store4(p, p.yrow ? p.yrow[r0 + r] : r0 + r, 4 * (i - r * n4), f32x4{0.f, 0.f, 0.f, 0.f});
        }
      }
    }
  if (i0 >= i1) return;

  // the sequence of the loads, one quad ahead of the multiplications
  struct Loads {
    u32x4 w[4], s;
  };
  int64_t ni = i0;
  int nsub = 0, nq = q0;
  const uint8_t *nw_p, *ns_p;
  uint32_t noff[4];  // TURN: of the lane's four rows
  auto row_of = [&](int64_t item, int sub) {  // the lane's weight row
    const int en = (int)(item / sp.ntiles), t = (int)(item - (int64_t)en * sp.ntiles);
    const int e = p.ent ? ent[4 * uniform(en)] : 0;
    const int seg = SILU && sub >= 2;
    const int n = min(t * COLS + 16 * (SILU ? sub & 1 : 0) + r16, p.N - 1);  // rows past N repeat the last
    if constexpr (!TURN) {
      nw_p = (seg ? p.w[1] : p.w[0]) + e * p.wstride + n * kb + 16 * g;
    } else {
      const int n0 = t * COLS + 16 * (SILU ? sub & 1 : 0);
      nw_p = (seg ? p.w[1] : p.w[0]) + e * p.wstride + n0 * kb + 16 * r16;
#pragma unroll
      for (int u = 0; u < 4; ++u) noff[u] = (uint32_t)min(4 * u + g, p.N - 1 - n0) * (uint32_t)kb;
    }
    ns_p = (seg ? p.ws[1] : p.ws[0]) + e * p.sstride + n * ksb;
  };
  row_of(ni, 0);
  auto load = [&](Loads &l) {
#pragma unroll
    for (int u = 0; u < 4; ++u)
      l.w[u] = ldg16(TURN ? nw_p + noff[u] + nq * 256
                          : nw_p + (int64_t)(PLANES ? min(4 * nq + u, steps - 1) : 4 * nq + u) * 64);
    if constexpr (!PLANES) {
      l.s = *reinterpret_cast<const u32x4_a4 *>(ns_p + nq * 16);
    } else {
#pragma unroll
      for (int u = 0; u < 4; ++u) l.s[u] = *reinterpret_cast<const uint32_t *>(ns_p + min(4 * nq + u, steps - 1) * 4);
    }
    if (++nq == q1) {
      nq = q0;
      if (++nsub == WT) {
        nsub = 0;
        ++ni;
      }
      if (ni < i1) row_of(ni, nsub);  // (past the end: the last row again, not multiplied)
    }
  };
  const int mr = sp.mr;
  int rows = 0, r0 = 0;
  auto fill = [&](int en) {  // the activations of an entry
    rows = p.M;
    if (p.ent) {
      r0 = ent[4 * uniform(en) + 1];
      rows = ent[4 * uniform(en) + 2];
    }
    const int count = (p.K >> 5) * rows, step = blockDim.x;
    auto put = [&](int r, int blk, u32x4 c, uint32_t byte) {
      const int st = blk >> 2;
      *reinterpret_cast<u32x4 *>(lds + 16 * (blk * mr + r)) = c;
      lds[sp.xcodes + 4 * (((st >> 2) * 4 + (blk & 3)) * mr + r) + (st & 3)] = (uint8_t)byte;
    };
    auto at = [&](int i, int &r, int &blk) -> int64_t {  // (past the end: the last block again)
      i = min(i, count - 1);
      blk = i / rows;
      r = i - blk * rows;
      return p.xrow ? p.xrow[r0 + r] : r0 + r;
    };
    // (the loads of several blocks in flight: each trip round the loop waits for memory)
    if (p.xs) {
      constexpr int B = 4;
      for (int i = tid; i < count; i += B * step) {
        u32x4 c[B];
        uint8_t byte[B];
        int r[B], blk[B];
#pragma unroll
        for (int k = 0; k < B; ++k) {
          const int64_t xr = at(i + k * step, r[k], blk[k]);
          c[k] = ldg16(static_cast<const uint8_t *>(p.x) + xr * kb + 16 * blk[k]);
          byte[k] = p.xs[xr * ksb + blk[k]];
        }
#pragma unroll
        for (int k = 0; k < B; ++k) put(r[k], blk[k], c[k], byte[k]);
      }
    } else {
      constexpr int B = 2;
      for (int i = tid; i < count; i += B * step) {
        u32x4 v[B][4];
        int r[B], blk[B];
#pragma unroll
        for (int k = 0; k < B; ++k) {
          const int64_t xr = at(i + k * step, r[k], blk[k]);
          const uint16_t *src = static_cast<const uint16_t *>(p.x) + xr * p.ldx + 32 * blk[k];
#pragma unroll
          for (int j = 0; j < 4; ++j) v[k][j] = ldg16(src + 8 * j);
        }
#pragma unroll
        for (int k = 0; k < B; ++k) {
          u16x2 am = {0, 0};
#pragma unroll
          for (int j = 0; j < 4; ++j) am = mx_absmax(am, v[k][j]);
          const uint32_t byte = mx_byte(mx_amax_bits(am));
          const float sc = mx_scale(byte);
          u32x4 c;
#pragma unroll
          for (int j = 0; j < 4; ++j) c[j] = mx_codes8(v[k][j], sc);
          put(r[k], blk[k], c, byte);
        }
      }
    }
  };
  auto meet = [&]() {
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  };

  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  Loads l0, l1;
  load(l0);
  load(l1);
  int64_t item = i0;
  int en = (int)(item / sp.ntiles), tile = (int)(item - (int64_t)en * sp.ntiles);
  fill(en);
  meet();

  const uint32_t gsel = g | (4 + g) << 8;
  const uint8_t *xl = lds + 16 * (g * mr + (r16 & (mr - 1))), *xsl = lds + sp.xcodes + 4 * (g * mr + (r16 & (mr - 1)));
  int sub = 0, q = q0, odd = 0;
  auto finish = [&]() {  // an item's sums, in wave order
    f32x4 *part = reinterpret_cast<f32x4 *>(lds + sp.xbytes) + odd * nw * WT * 64;
    auto total_of = [&](int t, int l) {
      f32x4 v = part[t * 64 + l];
      for (int w = 1; w < nw; ++w) v += part[(w * WT + t) * 64 + l];
      return v;
    };
    if constexpr (SILU) {
      // eight lanes hold a block of 32 outputs of a row: four each
      for (int i = tid; i < 128; i += blockDim.x) {
        const int c = i & 7, m = i >> 3, t = c >> 2;
        const int l = (c & 3) * 16 + m;
        const f32x4 gt = total_of(t, l), up = total_of(t + 2, l);
        float h[4];
        uint32_t am = 0;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          h[k] = mx_silu_mul(gt[k], up[k]);
          am = max(am, __float_as_uint(h[k]) & 0x7fffffffu);
        }
        am = max(am, dpp_u32<0xB1>(am));   // quad_perm [1,0,3,2]
        am = max(am, dpp_u32<0x4E>(am));   // quad_perm [2,3,0,1]
        am = max(am, dpp_u32<0x141>(am));  // row_half_mirror
        const uint32_t byte = mx_byte(am);
        const float sc = mx_scale(byte);
        uint32_t c4 = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0u, h[0], h[1], sc, 0);
        c4 = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c4, h[2], h[3], sc, 1);
        if (byte == 255) c4 = 0;
        if (m < rows) {
          *reinterpret_cast<uint16_t *>(p.hc + (int64_t)(r0 + m) * (p.N >> 1) + 16 * tile + 2 * c) = (uint16_t)c4;
          if (c == 0) p.hs[(int64_t)(r0 + m) * (p.N >> 5) + tile] = (uint8_t)byte;
        }
      }
    } else {
      if (tid < 64) {
        const int n = tile * COLS + 4 * (tid >> 4), m = tid & 15;
        if (m < rows && n < p.N) mx_store4(p, p.yrow ? p.yrow[r0 + m] : r0 + m, n, total_of(0, tid));
      }
    }
  };
  // multiplies the quad in l, then refills l
  auto body = [&](Loads &l) {
    const uint32_t ws = __builtin_amdgcn_perm(__builtin_amdgcn_perm(l.s.w, l.s.z, gsel),
                                              __builtin_amdgcn_perm(l.s.y, l.s.x, gsel), 0x05040100u);
    const uint32_t xs = *reinterpret_cast<const uint32_t *>(xsl + 16 * q * mr);
    u32x4 xc[4];  // (PLANES: steps past the end read the last one's)
#pragma unroll
    for (int u = 0; u < 4; ++u) xc[u] = ldg16(xl + 64 * (PLANES ? min(4 * q + u, steps - 1) : 4 * q + u) * mr);
    const int nst = PLANES ? steps - 4 * q : 4;
    auto multiply = [&](const u32x4 *w) {
      acc = mfma_mx<0>(w[0], ws, xc[0], xs, acc);
      if (!PLANES || nst > 1) acc = mfma_mx<1>(w[1], ws, xc[1], xs, acc);
      if (!PLANES || nst > 2) acc = mfma_mx<2>(w[2], ws, xc[2], xs, acc);
      if (!PLANES || nst > 3) acc = mfma_mx<3>(w[3], ws, xc[3], xs, acc);
    };
    if constexpr (TURN) {
      // 16-byte chunk c of row r at c ^ r: sixteen bank groups both ways
      uint8_t *turn = lds + sp.turn + 4096 * wave;
      u32x4 w[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) *reinterpret_cast<u32x4 *>(turn + 256 * (4 * u + g) + 16 * (r16 ^ (4 * u + g))) = l.w[u];
      __builtin_amdgcn_sched_barrier(0);  // (the registers of l are free: no copies of them)
      load(l);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int u = 0; u < 4; ++u) w[u] = ldg16(turn + 256 * r16 + 16 * ((4 * u + g) ^ r16));
      multiply(w);
    } else {
      multiply(l.w);
      __builtin_amdgcn_sched_barrier(0);
      load(l);
    }
    __builtin_amdgcn_sched_barrier(0);
    if (++q < q1) return;
    q = q0;
    f32x4 *part = reinterpret_cast<f32x4 *>(lds + sp.xbytes) + ((odd * nw + wave) * WT + sub) * 64;
    part[lane] = acc;
    acc = f32x4{0.f, 0.f, 0.f, 0.f};
    if (++sub < WT) return;
    sub = 0;
    meet();
    finish();
    odd ^= 1;
    if (++item == i1 || ++tile < sp.ntiles) return;
    tile = 0;
    meet();  // (every wave is past its last read of the old rows)
    fill(++en);
    meet();
  };
  const int64_t len = (i1 - i0) * WT * (q1 - q0);
  int64_t n = 0;
  for (; n + 2 <= len; n += 2) {
    body(l0);
    body(l1);
  }
  if (n < len) body(l0);
}

// ---------------------------------------------------------------- tiles

// A workgroup is eight waves on two 128-row weight segments and up to 256 activation
// rows: waves w and w + 4 multiply the weight rows 32 (w % 4) .. +31 of both segments
// (fragments f of 16: segment f / 2), so with gate rows as segment 0 and up rows as
// segment 1 a lane holds gate and up of the same outputs.  One workgroup per CU.
//
// Stages of 256 K values are whole 128-byte lines of a row, copied straight into LDS.
// 16-byte chunk c of row r is at c ^ ((r >> 1) & 7): a pass of a 16-byte LDS read
// takes lanes 0-3, 12-15 and 20-27 (and so on), here rows 0-3 and 12-15 of one chunk
// and 4-11 of the next: sixteen distinct bank groups.  (Stages of 64 bytes a row: the
// L2 delivers 20 TB/s in such pieces, 35 TB/s in lines.)
//
// Exponents: four K steps at a time, 16 bytes a row (PLANES: K % 512, rows without
// that alignment: four planes of a dword a row); a lane picks its K block's bytes into
// one dword, whose bytes the MFMAs select by number.
constexpr int MX_WHALF = 256 * 128;       // weight part of a stage
constexpr int MX_SCALE_LDS = 512 * 16;    // exponents of the 256 + 256 rows

struct MxTile {
  const uint8_t *w[2], *ws[2];
  int wrows[2];
  const int32_t *xrow;  // of the tile's first position, or null
  int64_t x0;           // x row of the tile's first row (xrow null)
  int rows, it0, it1;   // 128-wide K steps, it0 a multiple of 4
};

// Copies of 16 bytes a lane into LDS (lane l: dst + 16 l) from `base` + lane offset +
// scalar offset, the offsets below 4 GB.
AMLA_DEV __amdgpu_buffer_rsrc_t mx_rsrc(const uint8_t *base) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t *>(base), 0, 0xffffffffu, 0x00027000);
}
AMLA_DEV void mx_copy16(__amdgpu_buffer_rsrc_t r, uint8_t *dst, uint32_t lane_off, uint32_t off) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, LDS_PTR(dst), 16, lane_off, off, 0, 0);
}

template <int XF>
struct MxSums {
  f32x4 acc[4][XF];  // [weight fragment][activation fragment]
};

// Up to 16 XF <= 128 activation rows: the two halves of the workgroup take the two K
// steps of a stage (and meet in LDS at the end).  Three slots, two stages on their way.
// Bound by the weights' stream for the few rows that an expert gets: gate and up of 256
// experts of 7168 x 2048 for 2000 tokens in 840 us, 4.8 TB/s.  Copies of the weights alone
// take 612; those of the activations add 55, of the exponents (16 of a line's 128 bytes at
// a time) 45, the stores 35, entries of more than 128 rows 55.
template <int XF>
struct MxRowsLds {
  static constexpr int XROWS = XF > 4 ? 128 : 16 * XF;
  static constexpr int STAGE = MX_WHALF + XROWS * 128;
  static constexpr int SCALES = 3 * STAGE;
  static constexpr int BYTES = SCALES + MX_SCALE_LDS;
};
static_assert(MxRowsLds<8>::BYTES <= 160 * 1024, "LDS of a CU");

template <int XF, bool PLANES>
struct MxRowsMain {
  static AMLA_DEV void run(const MxParams &p, const MxTile &a, MxSums<XF> &sums) {
  auto &acc = sums.acc;
  extern __shared__ __align__(16) uint8_t lds[];
  using L = MxRowsLds<XF>;
  constexpr int XC = XF > 4 ? 2 : 1, C = 4 + XC;  // copies per wave and stage
  constexpr int XW = L::XROWS / 8;                // x rows a wave copies
  const int tid = threadIdx.x, lane = tid & 63, r16 = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), wn = wave & 3, wk = wave >> 2;
  const int64_t kb = p.K >> 1, ksb = p.K >> 5;
  const int steps = p.K >> 7;
  const int seg = wave >> 2;
  const int wrows = seg ? a.wrows[1] : a.wrows[0];
  const auto wrsrc = mx_rsrc(seg ? a.w[1] : a.w[0]), xrsrc = mx_rsrc(static_cast<const uint8_t *>(p.x) + (a.xrow ? 0 : a.x0 * kb));
  auto xrow_of = [&](int r) {  // (a gathered x is less than 4 GB); rows past the tile repeat its last row
    const int rc = min(r, a.rows - 1);
    return (uint32_t)(a.xrow ? a.xrow[rc] : rc);
  };
  // wave w copies weight rows 32 w .. +31 (of the 256) and XW x rows, 8 rows a copy
  uint32_t woff[4], xoff[XC];
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    const int r = 8 * c + (lane >> 3);
    woff[c] = (uint32_t)min(32 * wn + r, wrows - 1) * (uint32_t)kb + 16 * ((lane & 7) ^ ((r >> 1) & 7));
  }
#pragma unroll
  for (int c = 0; c < XC; ++c) {
    const int r = XW * wave + 8 * c + (lane >> 3);
    xoff[c] = xrow_of(r) * (uint32_t)kb + 16 * ((lane & 7) ^ ((r >> 1) & 7));
  }
  auto copy = [&](int i, int slot) {  // the stage of the K steps i, i + 1
    uint8_t *st = lds + slot * L::STAGE;
    // (a last stage of one K step: the lanes of the other repeat it)
    auto back = [&](int r) -> uint32_t { return PLANES && i + 1 >= steps && (((lane & 7) ^ (r >> 1)) & 4) ? 64 : 0; };
#pragma unroll
    for (int c = 0; c < 4; ++c)
      mx_copy16(wrsrc, st + (32 * wave + 8 * c) * 128, woff[c] - back(8 * c + (lane >> 3)), i * 64);
#pragma unroll
    for (int c = 0; c < XC; ++c)
      if (XF > 2 || lane < 32)
        mx_copy16(xrsrc, st + MX_WHALF + (XW * wave + 8 * c) * 128, xoff[c] - back(XW * wave + 8 * c + (lane >> 3)), i * 64);
  };
  // exponent rows in LDS 64 w + lane: weight row r at 64 (r / 32) + r % 32, x row r at
  // 64 (r / XW) + 32 + r % XW
  typedef const __attribute__((address_space(1))) uint8_t *gptr;
  const gptr sptr = lane < 32 ? (gptr)((seg ? a.ws[1] : a.ws[0]) + (int64_t)min(32 * wn + lane, wrows - 1) * ksb)
                              : (gptr)(p.xs + ((a.xrow ? 0 : a.x0) + (int64_t)xrow_of(XW * wave + min(lane - 32, XW - 1))) * ksb);
  auto copy_scales = [&](int i) {
    uint8_t *sc = lds + L::SCALES;
    if constexpr (!PLANES) {
      __builtin_amdgcn_global_load_lds(sptr + i * 4, LDS_PTR(sc + 1024 * wave), 16, 0, 0);
    } else {
#pragma unroll
      for (int u = 0; u < 4; ++u)
        __builtin_amdgcn_global_load_lds(sptr + min(i + u, steps - 1) * 4, LDS_PTR(sc + 2048 * u + 256 * wave), 4, 0, 0);
    }
  };
  // bytes of the wave's K step of this stage and of the next
  const uint32_t gsel = g | (4 + g) << 8;
  uint32_t wsc[4], xsc[XF];
  auto read_scales = [&]() {
    const uint8_t *sc = lds + L::SCALES + wk * (PLANES ? 2048 : 4);
    auto row = [&](int r) {
      const uint8_t *at = sc + r * (PLANES ? 4 : 16);
      return __builtin_amdgcn_perm(*reinterpret_cast<const uint32_t *>(at + (PLANES ? 4096 : 8)),
                                   *reinterpret_cast<const uint32_t *>(at), gsel);
    };
    const int x16 = 64 * (r16 / XW) + 32 + r16 % XW;
#pragma unroll
    for (int f = 0; f < 4; ++f) wsc[f] = row(64 * (4 * (f >> 1) + wn) + 16 * (f & 1) + r16);
#pragma unroll
    for (int j = 0; j < XF; ++j) xsc[j] = row(64 * (16 / XW) * j + x16);
  };
#pragma unroll
  for (int f = 0; f < 4; ++f)
#pragma unroll
    for (int j = 0; j < XF; ++j) acc[f][j] = f32x4{0.f, 0.f, 0.f, 0.f};

  const uint32_t frag = r16 * 128 + 16 * ((4 * wk + g) ^ ((r16 >> 1) & 7));
  copy_scales(a.it0);
  copy(a.it0, 0);
  if (a.it0 + 2 < a.it1) copy(a.it0 + 2, 1);
  int slot = 0;
  auto stage = [&](int i, auto u_c) {
    constexpr int U = decltype(u_c)::value;
    if (i + 2 < a.it1) wait_vmcnt<C>();  // all but the next stage's copies have landed
    else wait_vmcnt<0>();
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    if constexpr (U == 0) read_scales();
    if constexpr (U == 1)  // (every wave has read the others before this barrier)
      if (i + 2 < a.it1) copy_scales(i + 2);
    if (i + 4 < a.it1) copy(i + 4, slot == 0 ? 2 : slot - 1);
    const uint8_t *st = lds + slot * L::STAGE + frag;
    slot = slot == 2 ? 0 : slot + 1;
    if (PLANES && i + wk >= a.it1) return;
    u32x4 wf[4], xf[XF];
#pragma unroll
    for (int f = 0; f < 4; ++f)
      wf[f] = *reinterpret_cast<const u32x4 *>(st + ((f >> 1) * 128 + 32 * wn + 16 * (f & 1)) * 128);
#pragma unroll
    for (int j = 0; j < XF; ++j) xf[j] = *reinterpret_cast<const u32x4 *>(st + MX_WHALF + j * 2048);
#pragma unroll
    for (int j = 0; j < XF; ++j)
#pragma unroll
      for (int f = 0; f < 4; ++f) acc[f][j] = mfma_mx<U>(wf[f], wsc[f], xf[j], xsc[j], acc[f][j]);
  };
  for (int i = a.it0; i < a.it1; i += 4) {
    stage(i, std::integral_constant<int, 0>{});
    if (i + 2 < a.it1) stage(i + 2, std::integral_constant<int, 1>{});
  }

  // each half adds up half of the activation fragments (waves w and w + 4 exchange)
  __builtin_amdgcn_s_barrier();  // every wave is past its last fragment read
  asm volatile("" ::: "memory");
  f32x4 *ex = reinterpret_cast<f32x4 *>(lds) + lane;
#pragma unroll
  for (int f = 0; f < 4; ++f)
#pragma unroll
    for (int j = 0; j < XF / 2; ++j)
      ex[((wave * 4 + f) * (XF / 2) + j) * 64] = wk ? acc[f][j] : acc[f][XF / 2 + j];
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
  // (the K step 0 half first in every sum; the wave's own fragments end up in 0 .. XF/2 - 1)
#pragma unroll
  for (int f = 0; f < 4; ++f)
#pragma unroll
    for (int j = 0; j < XF / 2; ++j) {
      const f32x4 o = ex[(((wave ^ 4) * 4 + f) * (XF / 2) + j) * 64];
      acc[f][j] = wk ? o + acc[f][XF / 2 + j] : acc[f][j] + o;
    }
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  __builtin_amdgcn_s_barrier();  // (LDS is free)
}
};

// More rows: waves 0 .. 3 take the first 128 activation rows, the others the rest.  Two
// slots: the second K step's fragments of a stage are read while its first is
// multiplied, so that the slot is free for the stage after next when the second
// begins.
//
// Bound by the power of the matrix units and by whole rounds of tiles.  16384 K values to 7168
// outputs: 4096 rows (448 tiles, two rounds of the 256 CUs with the second three quarters
// full) in 226 - 243 us (4.0 - 4.3 PFLOP/s), on zeros in 195; 4608 rows (504 tiles) in 244 -
// 259, on zeros in 196: idle CUs in the second round cost all of their time on zeros, where
// power does not bound, and half of it on data.
// The multiplications and barriers of 4096 rows alone, on the same data, take 223 us.
// Four slots of 64-byte rows, two stages on their way: 306 us (the L2 delivers 20
// TB/s in such pieces, 35 TB/s in lines).  256 x 128 tiles, two workgroups per CU: 332.
constexpr int MXB_STAGE = 2 * MX_WHALF;
constexpr int MXB_SCALES = 2 * MXB_STAGE;
constexpr int MX_TILE_LDS = MxRowsLds<8>::BYTES;
static_assert(MXB_SCALES + MX_SCALE_LDS <= MX_TILE_LDS, "LDS of either form");

template <bool PLANES>
struct MxBigMain {
  static AMLA_DEV void run(const MxParams &p, const MxTile &a, MxSums<8> &sums) {
  auto &acc = sums.acc;
  extern __shared__ __align__(16) uint8_t lds[];
  const int tid = threadIdx.x, lane = tid & 63, r16 = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), wn = wave & 3, wm = wave >> 2;
  const int64_t kb = p.K >> 1, ksb = p.K >> 5;
  const int steps = p.K >> 7;
  // wave w copies weight rows 32 w .. +31 (of the 256) and x rows 32 w .. +31, 8 rows a
  // copy: lane offsets from a tile's first row, the stage as the scalar offset
  const int seg = wave >> 2;
  const int wrows = seg ? a.wrows[1] : a.wrows[0];
  const auto wrsrc = mx_rsrc(seg ? a.w[1] : a.w[0]), xrsrc = mx_rsrc(static_cast<const uint8_t *>(p.x) + (a.xrow ? 0 : a.x0 * kb));
  auto xrow_of = [&](int r) {  // (a gathered x is less than 4 GB); rows past the tile repeat its last row
    const int rc = min(r, a.rows - 1);
    return (uint32_t)(a.xrow ? a.xrow[rc] : rc);
  };
  uint32_t woff[4], xoff[4];
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    const int r = 8 * c + (lane >> 3), ch = (lane & 7) ^ ((r >> 1) & 7);
    woff[c] = (uint32_t)min(32 * wn + r, wrows - 1) * (uint32_t)kb + 16 * ch;
    xoff[c] = xrow_of(32 * wave + r) * (uint32_t)kb + 16 * ch;
  }
  auto copy = [&](int i, int slot) {  // the stage of the K steps i, i + 1
    uint8_t *st = lds + slot * MXB_STAGE + 32 * wave * 128;
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      // (a last stage of one K step: the lanes of the other repeat it)
      const uint32_t back = PLANES && i + 1 >= steps && (((lane & 7) ^ (4 * c + (lane >> 4))) & 4) ? 64 : 0;
      mx_copy16(wrsrc, st + c * 1024, woff[c] - back, i * 64);
      mx_copy16(xrsrc, st + MX_WHALF + c * 1024, xoff[c] - back, i * 64);
    }
  };
  // exponents: wave w has 32 rows of each half, 16 bytes (or four planes of 4) a row;
  // scale rows in LDS 64 w + lane: weight row r at 64 (r / 32) + r % 32, x row r 32 further
  const int sl = lane & 31;
  typedef const __attribute__((address_space(1))) uint8_t *gptr;
  const gptr sptr = lane < 32 ? (gptr)((seg ? a.ws[1] : a.ws[0]) + (int64_t)min(32 * wn + sl, wrows - 1) * ksb)
                              : (gptr)(p.xs + ((a.xrow ? 0 : a.x0) + (int64_t)xrow_of(32 * wave + sl)) * ksb);
  auto copy_scales = [&](int i) {
    uint8_t *sc = lds + MXB_SCALES;
    if constexpr (!PLANES) {
      __builtin_amdgcn_global_load_lds(sptr + i * 4, LDS_PTR(sc + 1024 * wave), 16, 0, 0);
    } else {
#pragma unroll
      for (int u = 0; u < 4; ++u)
        __builtin_amdgcn_global_load_lds(sptr + min(i + u, steps - 1) * 4, LDS_PTR(sc + 2048 * u + 256 * wave), 4, 0, 0);
    }
  };
  const uint32_t gsel = g | (4 + g) << 8;
  auto pick = [&](u32x4 d) {
    return __builtin_amdgcn_perm(__builtin_amdgcn_perm(d.w, d.z, gsel), __builtin_amdgcn_perm(d.y, d.x, gsel), 0x05040100u);
  };
  uint32_t wsc[4], xsc[8];
  auto read_scales = [&]() {
    const uint8_t *sc = lds + MXB_SCALES + r16 * (PLANES ? 4 : 16);
    auto row = [&](int r) {
      if constexpr (!PLANES) return *reinterpret_cast<const u32x4 *>(sc + 16 * r);
      u32x4 d;
#pragma unroll
      for (int u = 0; u < 4; ++u) d[u] = *reinterpret_cast<const uint32_t *>(sc + 2048 * u + 4 * r);
      return d;
    };
#pragma unroll
    for (int f = 0; f < 4; ++f) wsc[f] = pick(row(64 * (4 * (f >> 1) + wn) + 16 * (f & 1)));
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      xsc[j] = pick(row(64 * (4 * wm + (j >> 1)) + 32 + 16 * (j & 1)));
      if (j & 1) __builtin_amdgcn_sched_barrier(0);
    }
    // (picked here, not in the next body: four registers a row are not there)
#pragma unroll
    for (int f = 0; f < 4; ++f) asm volatile("" : "+v"(wsc[f]));
#pragma unroll
    for (int j = 0; j < 8; ++j) asm volatile("" : "+v"(xsc[j]));
  };
#pragma unroll
  for (int f = 0; f < 4; ++f)
#pragma unroll
    for (int j = 0; j < 8; ++j) acc[f][j] = f32x4{0.f, 0.f, 0.f, 0.f};

  const uint32_t sw = (r16 >> 1) & 7;
  const uint32_t frag[2] = {r16 * 128 + 16 * (g ^ sw), r16 * 128 + 16 * ((4 + g) ^ sw)};
  u32x4 wf[2][4], xf[8];
  auto read_w = [&](int slot, int ks, int f) {
    return *reinterpret_cast<const u32x4 *>(lds + slot * MXB_STAGE + ((f >> 1) * 128 + 32 * wn + 16 * (f & 1)) * 128 + frag[ks]);
  };
  auto read_x = [&](int slot, int ks, int j) {
    return *reinterpret_cast<const u32x4 *>(lds + slot * MXB_STAGE + MX_WHALF + (128 * wm + 16 * j) * 128 + frag[ks]);
  };
  auto landed = [&]() {  // every copy, and every read of the slot that is free now, in all waves
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  };
  copy_scales(a.it0);
  copy(a.it0, 0);
  landed();
  if (a.it0 + 2 < a.it1) copy(a.it0 + 2, 1);
  read_scales();
#pragma unroll
  for (int f = 0; f < 4; ++f) wf[0][f] = read_w(0, 0, f);
#pragma unroll
  for (int j = 0; j < 8; ++j) xf[j] = read_x(0, 0, j);

  // K step U of four: multiplies it, reads the next one's fragments
  auto step = [&](auto u_c) {
    constexpr int U = decltype(u_c)::value, SLOT = ((U + 1) >> 1) & 1, KS = (U + 1) & 1;
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
#pragma unroll
      for (int f = 0; f < 4; ++f) acc[f][j] = mfma_mx<U>(wf[U & 1][f], wsc[f], xf[j], xsc[j], acc[f][j]);
      __builtin_amdgcn_sched_barrier(0);
      xf[j] = read_x(SLOT, KS, j);
      if (j & 1) wf[1 - (U & 1)][j >> 1] = read_w(SLOT, KS, j >> 1);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  std::integral_constant<int, 0> u0;
  std::integral_constant<int, 1> u1;
  std::integral_constant<int, 2> u2;
  std::integral_constant<int, 3> u3;
  // (no branches where four steps are followed by four: the compiler would sink the
  // multiplications behind them, and their operands into memory)
  int i = a.it0;
  for (; i + 8 <= a.it1; i += 4) {
    step(u0);
    landed();
    copy_scales(i + 4);
    copy(i + 4, 0);
    step(u1);
    step(u2);
    landed();
    copy(i + 6, 1);
    step(u3);
    read_scales();
  }
  if constexpr (!PLANES) {  // whole fours: one is left
    step(u0);
    landed();
    step(u1);
    step(u2);
    landed();  // (keeps the steps apart for the compiler)
    step(u3);
  } else {
    for (; i < a.it1; i += 4) {
      const int left = a.it1 - i;
      step(u0);
      landed();
      if (left > 4) {
        copy_scales(i + 4);
        copy(i + 4, 0);
      }
      if (left > 1) step(u1);
      if (left > 2) step(u2);
      landed();
      if (left > 6) copy(i + 6, 1);
      if (left > 3) step(u3);
      if (left > 4) read_scales();
    }
  }
  // (nor sink the last of them into the branches of the stores)
#pragma unroll
  for (int f = 0; f < 4; ++f)
#pragma unroll
    for (int j = 0; j < 8; ++j) asm volatile("" : "+v"(acc[f][j]));
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  __builtin_amdgcn_s_barrier();  // (LDS is free)
}
};

struct MxFrag {
  f32x4 f[4];
};

// Stores a tile of `rows` positions from r0, outputs from n0.  The threads hold it as
// v(j)[f], activation fragment j of j0 .. j0 + XF - 1, weight fragment f: row 16 j +
// lane % 16, outputs 128 (f / 2) + 32 wn + 16 (f % 2) + 4 (lane / 16) .. +3.  Rows go
// through LDS, so that every store is 16 bytes of a run of 512 in one row: stores from
// where the sums are held, 32 bytes in each of 16 rows, reach 1.7 TB/s (down
// projection of 16000 routed rows 505 us, 370 without its stores).
constexpr int MX_PITCH_Y = 512 + 16, MX_PITCH_H = 64 + 16;
template <int XF, bool SILU, int SEGS = 2, typename V>
AMLA_DEV void mx_tile_store(const MxParams &p, V v, int j0, int wn, int rows, int r0, int n0) {
  extern __shared__ __align__(16) uint8_t lds[];
  const int tid = threadIdx.x, threads = blockDim.x, lane = tid & 63, r16 = lane & 15, g = lane >> 4;
  auto meet = [&]() {
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  };
  if constexpr (SILU) {
    // the four lanes of a row hold its block of 32: eight values each
    uint8_t *hs = lds + MX_PITCH_H * 256;
#pragma unroll
    for (int j = 0; j < XF; ++j) {
      const auto t = v(j);
      float h[8];
      uint32_t am = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        h[i] = mx_silu_mul(t.f[i >> 2][i & 3], t.f[2 + (i >> 2)][i & 3]);
        am = max(am, __float_as_uint(h[i]) & 0x7fffffffu);
      }
      am = max(am, (uint32_t)__shfl_xor((int)am, 16, 64));
      am = max(am, (uint32_t)__shfl_xor((int)am, 32, 64));
      const uint32_t byte = mx_byte(am);
      uint32_t q = mx_codes8(h, mx_scale(byte));
      if (byte == 255) q = 0;
      const int m = 16 * (j0 + j) + r16;
      *reinterpret_cast<uint16_t *>(lds + MX_PITCH_H * m + 16 * wn + 2 * g) = (uint16_t)q;
      *reinterpret_cast<uint16_t *>(lds + MX_PITCH_H * m + 16 * wn + 2 * g + 8) = (uint16_t)(q >> 16);
      if (g == 0) hs[4 * m + wn] = (uint8_t)byte;
    }
    meet();
    for (int i = tid; i < rows * 4; i += threads)
      *reinterpret_cast<u32x4 *>(p.hc + (int64_t)(r0 + (i >> 2)) * (p.N >> 1) + (n0 >> 1) + 16 * (i & 3)) =
          ldg16(lds + MX_PITCH_H * (i >> 2) + 16 * (i & 3));
    for (int i = tid; i < rows; i += threads)
      *reinterpret_cast<uint32_t *>(p.hs + (int64_t)(r0 + i) * (p.N >> 5) + (n0 >> 5)) =
          *reinterpret_cast<const uint32_t *>(hs + 4 * i);
  } else if (!p.vec16) {  // any stride and alignment
#pragma unroll
    for (int j = 0; j < XF; ++j) {
      const auto t = v(j);
      const int m = 16 * (j0 + j) + r16;
      if (m >= rows) continue;
      const int64_t yr = p.yrow ? p.yrow[r0 + m] : r0 + m;
#pragma unroll
      for (int f = 0; f < 2 * SEGS; ++f) {
        const int n = n0 + (f >> 1) * 128 + 32 * wn + 16 * (f & 1) + 4 * g;
        if (n < p.N) mx_store4(p, yr, n, t.f[f]);
      }
    }
  } else {
    // bf16: all segments of a row; fp32: one after the other
    for (int s = 0; s < (p.f32 ? SEGS : 1); ++s) {
      if (s) meet();
#pragma unroll
      for (int j = 0; j < XF; ++j) {
        const auto t = v(j);
        uint8_t *row = lds + MX_PITCH_Y * (16 * (j0 + j) + r16);
#pragma unroll
        for (int f = 0; f < 2 * SEGS; ++f) {
          const int c = 32 * wn + 16 * (f & 1) + 4 * g;
          if (!p.f32)
            *reinterpret_cast<u32x2 *>(row + 2 * (128 * (f >> 1) + c)) =
                u32x2{pack_bf16(t.f[f].x, t.f[f].y), pack_bf16(t.f[f].z, t.f[f].w)};
          else if (f >> 1 == s)
            *reinterpret_cast<f32x4 *>(row + 4 * c) = t.f[f];
        }
      }
      meet();
      const int log = p.f32 || SEGS == 2 ? 5 : 4, c = tid & ((1 << log) - 1);  // a row's 16-byte pieces
      const int n = n0 + 128 * s + (p.f32 ? 4 : 8) * c;
      if (n < p.N)
        for (int r = tid >> log; r < rows; r += threads >> log) {
          const int64_t yr = p.yrow ? p.yrow[r0 + r] : r0 + r;
          *reinterpret_cast<u32x4 *>(static_cast<uint8_t *>(p.y) + (yr * p.ldy + n) * (p.f32 ? 4 : 2)) =
              ldg16(lds + MX_PITCH_Y * r + 16 * c);
        }
    }
  }
}

// Few tiles: 128 weight rows (gate and up: 64 + 64) x up to 64 activation rows for sixteen
// waves, wave w on weight rows 32 (w % 4) .. +31 (16 (w % 4) .. +15 of each) and K step
// w / 4 of a stage of 512 K values; the four sums of an output meet in LDS.  Nothing but
// waits bounds such a call (a barrier, the reads and eight multiplications one after the
// other in every wave), so its stages are long and four waves of a SIMD stand in for each other: 777 x 2112 x
// 7168 in 17.3 us, 21.8 with tiles of 256 x 32; eight waves with stages of 256 and five
// of them on their way 19.1, which 24 workgroups alone take 0.44 us a stage for.
//
// A stage: two halves of 128-byte lines as above, rows of exponents behind them (wave w
// copies those of weight rows 8 w .. +7 and x rows 4 w .. +3).  Three slots.
constexpr int MXS_ROWS = 64;
constexpr int MXS_X = 2 * 128 * 128, MXS_SCALES = MXS_X + 2 * MXS_ROWS * 128, MXS_STAGE = MXS_SCALES + 16 * 12 * 16;
constexpr int MXS_LDS = 3 * MXS_STAGE;
static_assert(MXS_LDS <= 160 * 1024 && 16 * 8 * 1024 <= MXS_LDS, "LDS of a CU, the sums");

template <bool SILU, bool PLANES>
AMLA_DEV void mx_small_tile(const MxParams &p, int e, int r0, int rows, int n0) {
  extern __shared__ __align__(16) uint8_t lds[];
  constexpr int C = 3 + (PLANES ? 4 : 1);  // copies of a wave and stage
  const int tid = threadIdx.x, lane = tid & 63, r16 = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), wn = wave & 3, wk = wave >> 2;
  const int64_t kb = p.K >> 1, ksb = p.K >> 5;
  const int steps = p.K >> 7, quads = (steps + 3) >> 2, wrows = min(SILU ? 64 : 128, p.N - n0);
  // wave w copies half w / 8 of weight rows 16 (w % 8) .. +15 and x rows 8 (w % 8) .. +7
  // (rows past the tile repeat its last)
  const int half = wave >> 3, w8 = wave & 7, seg = SILU ? w8 >> 2 : 0, ch = lane & 7;
  const auto wrsrc = mx_rsrc((seg ? p.w[1] : p.w[0]) + e * p.wstride + n0 * kb);
  const auto xrsrc = mx_rsrc(static_cast<const uint8_t *>(p.x) + (p.xrow ? 0 : r0 * kb));
  auto xrow_of = [&](int r) {  // (a gathered x is less than 4 GB)
    const int rc = min(r, rows - 1);
    return (uint32_t)(p.xrow ? p.xrow[r0 + rc] : rc);
  };
  const int wr = 16 * w8 + (lane >> 3), xr = 8 * w8 + (lane >> 3);  // (the second weight copy: row + 8, the same chunk ^ 4)
  const int wch = ch ^ ((wr >> 1) & 7), xch = ch ^ ((xr >> 1) & 7), wl = wr - 64 * seg;
  const uint32_t woff[2] = {(uint32_t)min(wl, wrows - 1) * (uint32_t)kb + 16 * wch,
                            (uint32_t)min(wl + 8, wrows - 1) * (uint32_t)kb + 16 * (wch ^ 4)};
  const uint32_t xoff = xrow_of(xr) * (uint32_t)kb + 16 * xch;
  typedef const __attribute__((address_space(1))) uint8_t *gptr;
  const int sseg = SILU ? wave >> 3 : 0;
  const gptr sptr = lane < 8 ? (gptr)((sseg ? p.ws[1] : p.ws[0]) + e * p.sstride +
                                      (n0 + (int64_t)min(8 * wave - 64 * sseg + lane, wrows - 1)) * ksb)
                             : (gptr)(p.xs + ((p.xrow ? 0 : r0) + (int64_t)xrow_of(4 * wave + (lane & 3))) * ksb);
  auto issue = [&](int q, int slot) {
    uint8_t *st = lds + slot * MXS_STAGE;
    const uint32_t off = q * 256 + 128 * half;
    auto copy = [&](__amdgpu_buffer_rsrc_t r, uint8_t *dst, uint32_t lane_off, int c) {
      if constexpr (!PLANES) mx_copy16(r, dst, lane_off, off);
      else  // steps past the end: the lanes repeat the last one
        mx_copy16(r, dst, lane_off + off - 64 * max(0, 4 * q + 2 * half + (c >> 2) - (steps - 1)), 0);
    };
    copy(wrsrc, st + half * 16384 + 16 * w8 * 128, woff[0], wch);
    copy(wrsrc, st + half * 16384 + (16 * w8 + 8) * 128, woff[1], wch ^ 4);
    copy(xrsrc, st + MXS_X + half * 8192 + 8 * w8 * 128, xoff, xch);
    if (lane < 12) {
      if constexpr (!PLANES) {
        __builtin_amdgcn_global_load_lds(sptr + q * 16, LDS_PTR(st + MXS_SCALES + 192 * wave), 16, 0, 0);
      } else {
#pragma unroll
        for (int u = 0; u < 4; ++u)
          __builtin_amdgcn_global_load_lds(sptr + min(4 * q + u, steps - 1) * 4,
                                           LDS_PTR(st + MXS_SCALES + 768 * u + 48 * wave), 4, 0, 0);
      }
    }
  };
  f32x4 acc[2][4];
#pragma unroll
  for (int f = 0; f < 2; ++f)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[f][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  issue(0, 0);
  if (quads > 1) issue(1, 1);

  const uint32_t frag = r16 * 128 + 16 * ((4 * (wk & 1) + g) ^ ((r16 >> 1) & 7));
  auto wfrag = [&](int f) { return SILU ? 64 * f + 16 * wn : 32 * wn + 16 * f; };  // its first row
  int slot = 0;
  for (int q = 0; q < quads; ++q) {
    if (q + 1 < quads) wait_vmcnt<C>();  // all but the next stage's copies have landed
    else wait_vmcnt<0>();
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    if (q + 2 < quads) issue(q + 2, slot == 0 ? 2 : slot - 1);
    const uint8_t *st = lds + slot * MXS_STAGE;
    slot = slot == 2 ? 0 : slot + 1;
    if (PLANES && 4 * q + wk >= steps) continue;
    uint32_t wsc[2], xsc[4];
    const uint8_t *sc = st + MXS_SCALES + wk * (PLANES ? 768 : 4) + g;
    auto scale = [&](int r) { return (uint32_t)sc[r * (PLANES ? 4 : 16)]; };
#pragma unroll
    for (int f = 0; f < 2; ++f) wsc[f] = scale(12 * (wfrag(f) / 8 + (r16 >> 3)) + (r16 & 7));
#pragma unroll
    for (int j = 0; j < 4; ++j) xsc[j] = scale(12 * (4 * j + (r16 >> 2)) + 8 + (r16 & 3));
    const uint8_t *wp = st + (wk >> 1) * 16384 + frag, *xp = st + MXS_X + (wk >> 1) * 8192 + frag;
    u32x4 wf[2], xf[4];
#pragma unroll
    for (int f = 0; f < 2; ++f) wf[f] = *reinterpret_cast<const u32x4 *>(wp + wfrag(f) * 128);
#pragma unroll
    for (int j = 0; j < 4; ++j) xf[j] = *reinterpret_cast<const u32x4 *>(xp + j * 2048);
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int f = 0; f < 2; ++f) acc[f][j] = mfma_mx<0>(wf[f], wsc[f], xf[j], xsc[j], acc[f][j]);
  }

  auto meet = [&]() {
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  };
  meet();  // every wave is past its last fragment read
  f32x4 *ex = reinterpret_cast<f32x4 *>(lds) + lane;
#pragma unroll
  for (int f = 0; f < 2; ++f)
#pragma unroll
    for (int j = 0; j < 4; ++j) ex[((wave * 2 + f) * 4 + j) * 64] = acc[f][j];
  meet();
  // wave w sums activation fragment w / 4, in the order of the K steps
  MxFrag sum = {};
#pragma unroll
  for (int f = 0; f < 2; ++f) {
    sum.f[f] = ex[((wn * 2 + f) * 4 + wk) * 64];
#pragma unroll
    for (int k = 1; k < 4; ++k) sum.f[f] += ex[(((wn + 4 * k) * 2 + f) * 4 + wk) * 64];
  }
  meet();  // (LDS is free)
  if constexpr (!SILU) {
    mx_tile_store<1, false, 1>(p, [&](int) { return sum; }, wk, wn, rows, r0, n0);
  } else {
    // sum: gate and up of outputs 16 wn + 4 g .. +3 of row 16 wk + r16; then four lanes
    // hold a block of 32 outputs of a row: eight each
    constexpr int PITCH = 64 + 4;
    float *h = reinterpret_cast<float *>(lds);
    f32x4 v;
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] = mx_silu_mul(sum.f[0][k], sum.f[1][k]);
    *reinterpret_cast<f32x4 *>(h + PITCH * (16 * wk + r16) + 16 * wn + 4 * g) = v;
    meet();
    const int m = tid >> 3, c = tid & 7;
    if (m < rows) {  // (tid < 512; the lanes of a row together)
      float o[8];
      uint32_t am = 0;
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        o[k] = h[PITCH * m + 8 * c + k];
        am = max(am, __float_as_uint(o[k]) & 0x7fffffffu);
      }
      am = max(am, dpp_u32<0xB1>(am));  // quad_perm [1,0,3,2]
      am = max(am, dpp_u32<0x4E>(am));  // quad_perm [2,3,0,1]
      const uint32_t byte = mx_byte(am), codes = mx_codes8(o, mx_scale(byte));
      *reinterpret_cast<uint32_t *>(p.hc + (int64_t)(r0 + m) * (p.N >> 1) + (n0 >> 1) + 4 * c) = byte == 255 ? 0u : codes;
      if ((c & 3) == 0) p.hs[(int64_t)(r0 + m) * (p.N >> 5) + (n0 >> 5) + (c >> 2)] = (uint8_t)byte;
    }
  }
}

template <bool SILU, bool PLANES>
__global__ __launch_bounds__(1024, 1) void mx_small_kernel(MxParams p, int n_tiles, int m_tiles) {
  const int t = xcd_run(blockIdx.x, n_tiles * m_tiles);
  if (t < 0) return;
  int nt, mt;
  tile_coords(t, n_tiles, m_tiles, nt, mt, TL_PANEL / 2);
  const int r0 = uniform(mt) * MXS_ROWS;
  mx_small_tile<SILU, PLANES>(p, 0, r0, min(MXS_ROWS, p.M - r0), uniform(nt) * (SILU ? 64 : 128));
}

// The same for the scheduled entries of up to 64 rows.
template <bool SILU, bool PLANES>
__global__ __launch_bounds__(1024, 1) void mx_small_sched_kernel(MxParams p, int ntiles) {
  const int l = xcd_run(blockIdx.x, (p.count[0] + (p.rest ? p.count[1] : 0)) * ntiles);
  if (l < 0) return;
  const int t = uniform(l / ntiles), n0 = (uniform(l) - t * ntiles) * (SILU ? 64 : 128);
  const int32_t *en = p.ent + 4 * t;
  const int e = uniform(en[0]), r0 = uniform(en[1]), rows = uniform(en[2]);
  if (!SILU && e < 0) {  // rows of no expert
    for (int i = threadIdx.x; i < rows * 32; i += 1024) {
      const int r = i >> 5, n = n0 + 4 * (i & 31);
      if (n < p.N) mx_store4(p, p.yrow ? p.yrow[r0 + r] : r0 + r, n, f32x4{0.f, 0.f, 0.f, 0.f});
    }
    return;
  }
  mx_small_tile<SILU, PLANES>(p, e, r0, rows, n0);
}

// One weight: tiles of 256 outputs (SILU: 128) x `rows` activation rows.  The first
// `whole` tiles (rounds of 256) take all of K, the others a K part a workgroup.
struct MxSplit {
  int n_tiles, m_tiles, rows, whole;
  bool small;      // tiles of 128 outputs (SILU: 64) x 64 rows (parts 1)
  int parts;       // K parts of the other tiles, whole runs of four steps
  float *partial;  // [tile][part][activation fragment][weight fragment][wave % 4][lane] f32x4
};
constexpr int MX_ROWS = 256;  // most activation rows of a tile
constexpr int MX_FINISH_LDS = MX_PITCH_H * 256 + 4 * 16;  // exponents behind the most rows' codes
static_assert(MX_FINISH_LDS >= 16 * MX_PITCH_Y && 256 * MX_PITCH_Y <= MX_TILE_LDS, "staged rows");

template <bool SILU>
AMLA_DEV MxTile mx_tile_of(const MxParams &p, int e, int r0, int rows, int n0, int it0, int it1) {
  MxTile a;
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
  return a;
}

// The fragments j0 .. j0 + XF - 1 of a tile, held as acc[.][0 .. XF - 1].
template <int XF, int HELD, bool SILU>
AMLA_DEV void mx_tile_out(const MxParams &p, const MxSums<HELD> &sums, int j0, int r0, int rows, int n0, f32x4 *partial) {
  const int lane = threadIdx.x & 63, wn = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) & 3;
  if (partial) {
#pragma unroll
    for (int j = 0; j < XF; ++j)
#pragma unroll
      for (int f = 0; f < 4; ++f) partial[(((j0 + j) * 4 + f) * 4 + wn) * 64 + lane] = sums.acc[f][j];
    return;
  }
  mx_tile_store<XF, SILU>(
      p, [&](int j) { return MxFrag{{sums.acc[0][j], sums.acc[1][j], sums.acc[2][j], sums.acc[3][j]}}; }, j0, wn, rows, r0, n0);
}

template <int XF, bool SILU, bool PLANES>
AMLA_DEV void mx_rows_tile(const MxParams &p, const MxTile &a, int r0, int n0, f32x4 *partial) {
  MxSums<XF> sums;
  MxRowsMain<XF, PLANES>::run(p, a, sums);
  mx_tile_out<XF / 2, XF, SILU>(p, sums, __builtin_amdgcn_readfirstlane(threadIdx.x >> 8) * (XF / 2), r0, a.rows, n0, partial);
}

// Column tile nt of `rows` <= 256 positions from r0 of expert e, K steps it0 .. it1 - 1.
template <bool SILU, bool PLANES>
AMLA_DEV void mx_tile(const MxParams &p, int e, int r0, int rows, int nt, int it0, int it1, f32x4 *partial) {
  const int n0 = nt * (SILU ? 128 : 256);
  const MxTile a = mx_tile_of<SILU>(p, e, r0, rows, n0, it0, it1);
  if (rows <= 32) mx_rows_tile<2, SILU, PLANES>(p, a, r0, n0, partial);
  else if (rows <= 64) mx_rows_tile<4, SILU, PLANES>(p, a, r0, n0, partial);
  else if (rows <= 96) mx_rows_tile<6, SILU, PLANES>(p, a, r0, n0, partial);
  else if (rows <= 128) mx_rows_tile<8, SILU, PLANES>(p, a, r0, n0, partial);
  else {
    MxSums<8> sums;
    MxBigMain<PLANES>::run(p, a, sums);
    mx_tile_out<8, 8, SILU>(p, sums, __builtin_amdgcn_readfirstlane(threadIdx.x >> 8) * 8, r0, rows, n0, partial);
  }
}

// Column tiles of a panel: an XCD's run of tiles has about as many weight rows as
// activation rows, and reads the fewest.
AMLA_DEV int mx_panel(int rows) { return max(1, TL_PANEL * rows / MX_ROWS); }

// One weight: the whole tiles, then the K parts of the others, each as contiguous runs
// per XCD.
template <bool SILU, bool PLANES>
__global__ __launch_bounds__(512, 1) void mx_linear_kernel(MxParams p, MxSplit sp) {
  const int split = sp.n_tiles * sp.m_tiles - sp.whole, steps = p.K >> 7;
  int t, it0 = 0, it1 = steps;
  f32x4 *partial = nullptr;
  if ((int)blockIdx.x < sp.whole) {
    t = xcd_run(blockIdx.x, sp.whole);
  } else {
    const int l = xcd_run(blockIdx.x - sp.whole, split * sp.parts);
    if (l < 0) return;
    const int q = l / split, quads = (steps + 3) >> 2;
    t = l - q * split;
    if (sp.parts > 1) {
      it0 = 4 * (quads * q / sp.parts);
      it1 = min(steps, 4 * (quads * (q + 1) / sp.parts));
      partial = reinterpret_cast<f32x4 *>(sp.partial) + (size_t)(t * sp.parts + q) * (64 * sp.rows);
    }
    t += sp.whole;
  }
  int nt, mt;
  tile_coords(t, sp.n_tiles, sp.m_tiles, nt, mt, mx_panel(sp.rows));
  const int r0 = uniform(mt) * sp.rows;
  mx_tile<SILU, PLANES>(p, 0, r0, min(sp.rows, p.M - r0), uniform(nt), uniform(it0), uniform(it1), partial);
}

// Sums the K parts of activation fragment j of a tile in part order.
template <bool SILU>
__global__ __launch_bounds__(256) void mx_finish_kernel(MxParams p, MxSplit sp) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int t = blockIdx.x / (sp.rows >> 4), j = blockIdx.x - t * (sp.rows >> 4);
  int nt, mt;
  tile_coords(t + sp.whole, sp.n_tiles, sp.m_tiles, nt, mt, mx_panel(sp.rows));
  const int m0 = mt * sp.rows + 16 * j;
  if (m0 >= p.M) return;
  const size_t part = 64 * sp.rows;
  const f32x4 *src = reinterpret_cast<const f32x4 *>(sp.partial) + t * sp.parts * part + j * 1024 + wave * 64 + lane;
  f32x4 v[4];
#pragma unroll
  for (int f = 0; f < 4; ++f) v[f] = src[f * 256];
#pragma unroll 4
  for (int q = 1; q < sp.parts; ++q)
#pragma unroll
    for (int f = 0; f < 4; ++f) v[f] += src[q * part + f * 256];
  mx_tile_store<1, SILU>(p, [&](int) { return MxFrag{{v[0], v[1], v[2], v[3]}}; }, 0, wave, min(16, p.M - m0), m0,
                         nt * (SILU ? 128 : 256));
}

// The scheduled entries of up to 256 rows: a contiguous run of (entry, column
// tile) per XCD, so that the activation rows of an entry are read from one L2.
// A workgroup a tile: persistent ones that take the next tile's first stages during
// the stores were slower (gate and up of 2000 tokens 930 us against 900, in turn).
template <bool SILU, bool PLANES>
__global__ __launch_bounds__(512, 1) void mx_sched_kernel(MxParams p, int ntiles) {
  const int l = xcd_run(blockIdx.x, (p.count[0] + (p.rest ? p.count[1] : 0)) * ntiles);
  if (l < 0) return;
  const int t = uniform(l / ntiles), nt = uniform(l) - t * ntiles;
  const int32_t *en = p.ent + 4 * t;
  const int e = uniform(en[0]), r0 = uniform(en[1]), rows = uniform(en[2]);
  if (!SILU && e < 0) {  // rows of no expert
    for (int i = threadIdx.x; i < rows * 64; i += 512) {
      const int r = i >> 6, n = nt * 256 + 4 * (i & 63);
      if (n < p.N) mx_store4(p, p.yrow ? p.yrow[r0 + r] : r0 + r, n, f32x4{0.f, 0.f, 0.f, 0.f});
    }
    return;
  }
  mx_tile<SILU, PLANES>(p, e, r0, rows, nt, 0, p.K >> 7, nullptr);
}

// ---------------------------------------------------------------- schedules

// Entries of the groups [offsets[e], offsets[e + 1]) of m rows, at most rows_max
// rows each.  Offsets are taken as they come but never past m and never
// backwards: bad ones lose rows, not bounds.  count: the entries; with rest, the
// rows of no group as count[1] more, of expert -1.
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
    count[0] = n;
    if (rest) {
      const int lo[2] = {0, start[E]}, hi[2] = {start[0], m};
      for (int k = 0; k < 2; ++k)
        for (int r = lo[k]; r < hi[k]; r += rows_max, ++c) {
          int32_t *en = ent + 4 * c;
          en[0] = -1; en[1] = r; en[2] = min(rows_max, hi[k] - r); en[3] = 0;
        }
    }
    count[1] = c - n;
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

constexpr int64_t MX_MAX_BLOCKS = (1 << 22) - 8;  // of 1024 threads, fewer than 2^32 a launch

// Dynamic LDS above 64 KB.  The limit is the process's: it is always the CU's, so that no call
// lowers it between another thread's setting and launch.
template <typename F>
static int mx_lds(F *fn, int bytes) {
  if (bytes <= 64 * 1024) return AMLA_OK;
  const hipError_t e =
      hipFuncSetAttribute(reinterpret_cast<const void *>(fn), hipFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024);
  return e == hipSuccess ? AMLA_OK : fail((int)e, "mxfp4 product: LDS size: %s", hipGetErrorString(e));
}

// Activation rows kept for entries of at most `rows` <= 16 rows
static int mx_keep(int rows) {
  int mr = 1;
  while (mr < rows) mr *= 2;
  return mr;
}
static int64_t mx_stream_bytes(int rows, int64_t K) { return (int64_t)mx_keep(rows) * (K / 2 + (K + 511) / 512 * 16); }
// waves of a workgroup: equal runs of quads where there are any, rather four to seven
// (7168 x 16384, one row: four 17.9 us, eight 19.3)
static int mx_waves(int64_t K) {
  const int quads = (int)((K + 511) / 512);
  int best = 1;
  double cost = 1e9;
  for (int w = 1; w <= std::min(8, quads); ++w) {
    const double c = (double)((quads + w - 1) / w) * w / quads + 0.25 / w + 0.01 * w;
    if (c < cost) {
      cost = c;
      best = w;
    }
  }
  return best;
}

static int64_t mx_stream_sums(int rows, int64_t K, bool silu) {  // with two items' partial sums
  return mx_stream_bytes(rows, K) + 2048 * mx_waves(K) * (silu ? 4 : 1);
}
static int64_t mx_stream_lds(int rows, int64_t K, bool silu) {
  return mx_stream_sums(rows, K, silu) + (K % 512 ? 0 : 4096 * mx_waves(K));
}
// Up to 16 rows, as long as it does not take longer to take them in (each workgroup for
// itself) than a tile's pipeline to start: 16 x 7168 x 12288 19.0 us, tiles 20.0; 12 x 7168
// x 16384 24.3 and 22.6; 5 x 7168 x 32768 40 and 35.  Above, tiles: 32 x 18432 x 7168 24.0
// us, with two fragments of activation rows here 26; 64 x 24576 x 1536 8.6, with four 13.7
// (few outputs lose by it: 20 x 2112 x 7168 12.5, here 10.4).
static bool mx_stream_fits(int64_t rows, int64_t K, bool silu) {
  return rows <= 16 && mx_stream_bytes((int)rows, K) <= 112 * 1024 && mx_stream_lds((int)rows, K, silu) <= 160 * 1024;
}

template <bool SILU>
static int launch_mx_stream(const MxParams &p, int rows, int entries, hipStream_t st) {
  MxStream sp;
  sp.ntiles = (p.N + (SILU ? 31 : 15)) / (SILU ? 32 : 16);
  sp.mr = mx_keep(rows);
  sp.xcodes = sp.mr * (p.K >> 1);
  sp.xbytes = (int)mx_stream_bytes(rows, p.K);
  sp.turn = (int)mx_stream_sums(rows, p.K, SILU);
  const int nw = mx_waves(p.K);
  const int lds = (int)mx_stream_lds(rows, p.K, SILU);
  // Three items or more a workgroup (each takes in the activations for itself), up to 16
  // waves a CU, but more than one workgroup of few waves for few rows.  8 x 24576 x 1536:
  // 512 workgroups 8.6 us, 1280 9.3; 1 x 7168 x 16384, four waves each: 448 of one item
  // 15.9, 224 of two 16.8; 8 x 7168 x 8192: 16.6 and 15.0; 1 x 7168 x 18432, six waves: 19.8
  // and 18.3; down projections of 57 experts of 7168 x 2048: 256 108, 1024 73.
  const int64_t items = (int64_t)entries * sp.ntiles, most = std::min(16 / nw, 160 * 1024 / lds);
  const int per_cu = (int)std::max<int64_t>(1, std::min(most, std::max<int64_t>(items / (3 * 256), nw <= 4 && sp.mr <= 4 ? 2 : 1)));
  const int64_t run = (items + 256 * per_cu - 1) / (256 * per_cu);  // items of the longest run
  const unsigned blocks = (unsigned)((items + run - 1) / run);
  const auto kernel = p.K % 512 ? mx_stream_kernel<SILU, true> : mx_stream_kernel<SILU, false>;
  const int rc = mx_lds(kernel, lds);
  if (rc) return rc;
  kernel<<<dim3(blocks), 64 * nw, lds, st>>>(p, sp);
  return check_launch("mxfp4 stream product");
}

// The tiles of one weight by what they cost: a stage of 256 K values and the rest of a
// tile (us, 32 to 256 rows), rounds of 256 workgroups, the sums of K parts through
// memory.  Few tiles stay small (777 x 2112 x 7168: 128 x 64 17.3 us, 256 x 32 21.6, 256 x
// 64 in two parts 22.8, x 128 in four 25.9, x 256 in five 29.3; 300 x 7168 x 16384: x 128
// in three 42.2, x 256 in four 43.8), long K goes in parts (200 x 7168 x 18432: x 128 in
// four 39, in one 95), and a last round that is far from full is split alone (1000 x
// 36864 x 7168: 64 of 576 tiles in two to four parts 170 - 174 us, in one 183).
static MxSplit plan_mx_split(int64_t M, int N, int K, bool silu) {
  const double stage_us[4] = {0.65, 0.8, 1.3, 1.9}, tile_us[4] = {3.5, 4.5, 5, 10}, finish_us = 5, part_us = 0.23;
  const double small_quad_us = 0.9, small_tile_us = 4.6;
  const int cols = silu ? 128 : 256, quads = (K / 128 + 3) / 4;
  MxSplit best = {};
  double least = 1e30;
  for (int i = 0; i < 4; ++i) {
    MxSplit sp = {};
    sp.rows = 32 << i;
    sp.n_tiles = (N + cols - 1) / cols;
    sp.m_tiles = (int)((M + sp.rows - 1) / sp.rows);
    const int64_t tiles = (int64_t)sp.n_tiles * sp.m_tiles;
    if (tiles > 1 << 30) continue;
    sp.whole = (int)(tiles / 256 * 256);
    const int rest = (int)tiles - sp.whole;
    const double whole = sp.whole / 256 * (quads * 2 * stage_us[i] + tile_us[i]);
    for (sp.parts = 1; sp.parts == 1 || (sp.parts <= quads && sp.parts * rest <= 256); ++sp.parts) {
      double us = whole;
      if (rest) us += (quads + sp.parts - 1) / sp.parts * 2 * stage_us[i] + tile_us[i];
      if (sp.parts > 1) us += finish_us + part_us * sp.parts * rest * sp.rows / 1024;
      if (us < least) {
        least = us;
        best = sp;
      }
      if (!rest) break;
    }
    if (sp.rows >= M) break;
  }
  if (M > 32) {
    MxSplit sp = {};
    sp.small = true;
    sp.parts = 1;
    sp.rows = MXS_ROWS;
    sp.n_tiles = silu ? (N + 63) / 64 : (N + 127) / 128;
    sp.m_tiles = (int)((M + MXS_ROWS - 1) / MXS_ROWS);
    const double rounds = (double)(((int64_t)sp.n_tiles * sp.m_tiles + 255) / 256);
    if (rounds * (quads * small_quad_us + small_tile_us) < least) best = sp;
  }
  if (best.parts == 1) best.whole = 0;  // one run per XCD for all
  return best;
}
static size_t mx_split_bytes(const MxSplit &sp) {
  return sp.parts > 1 ? ((size_t)sp.n_tiles * sp.m_tiles - sp.whole) * sp.parts * 1024 * sp.rows : 0;
}

static int64_t mx_linear_blocks(const MxSplit &sp) {
  return sp.whole + (((int64_t)sp.n_tiles * sp.m_tiles - sp.whole) * sp.parts + 7) / 8 * 8;
}
// (checked by the entries before the first launch)
static bool mx_linear_grid_ok(const MxSplit &sp) { return sp.rows && mx_linear_blocks(sp) <= MX_MAX_BLOCKS; }

template <bool SILU>
static int launch_mx_linear(const MxParams &p, const MxSplit &sp, hipStream_t st) {
  const int64_t split = (int64_t)sp.n_tiles * sp.m_tiles - sp.whole, blocks = mx_linear_blocks(sp);
  const auto kernel = p.K % 512 ? mx_linear_kernel<SILU, true> : mx_linear_kernel<SILU, false>;
  int rc;
  if (sp.small) {
    const auto small = p.K % 512 ? mx_small_kernel<SILU, true> : mx_small_kernel<SILU, false>;
    if ((rc = mx_lds(small, MXS_LDS))) return rc;
    small<<<dim3((unsigned)blocks), 1024, MXS_LDS, st>>>(p, sp.n_tiles, sp.m_tiles);
    return check_launch("mxfp4 product of few tiles");
  }
  if ((rc = mx_lds(kernel, MX_TILE_LDS))) return rc;
  kernel<<<dim3((unsigned)blocks), 512, MX_TILE_LDS, st>>>(p, sp);
  if ((rc = check_launch("mxfp4 product")) || sp.parts == 1) return rc;
  mx_finish_kernel<SILU><<<dim3((unsigned)(split * (sp.rows / 16))), 256, MX_FINISH_LDS, st>>>(p, sp);
  return check_launch("mxfp4 K-part finish");
}

// Whether `slots` rows in groups of E make at most a round of small tiles (of a product
// of `tiles` of them side by side).  The estimate takes the groups as equal: the sizes
// are known to the device alone, and the grid is made for the worst case.  K = 7168 to 2048
// outputs with schedule and quantising: 300 rows in 2 groups 23 us, large tiles 52; 1000 in
// 4 32 and 68; 40 in 16 (256 tiles) 33 and 43.  Two rounds: 150 rows in 32 groups 36.6 and
// 32.4 (the product alone), 40 rows in 8 groups, 2048 to 7168, 24.8 and 20.8.
static bool mx_small_round(int64_t slots, int64_t E, int64_t tiles) {
  const int64_t groups = std::min(E, slots), each = (slots + groups - 1) / groups;
  return groups * ((each + MXS_ROWS - 1) / MXS_ROWS) * tiles <= 256;
}

static int mx_sched_tiles(int64_t n, bool silu, bool small) {  // of an entry
  const int cols = (silu ? 128 : 256) / (small ? 2 : 1);
  return (int)((n + cols - 1) / cols);
}
static int64_t mx_sched_blocks(int max_entries, int ntiles) { return ((int64_t)max_entries * ntiles + 7) / 8 * 8; }
static bool mx_sched_grid_ok(int max_entries, int64_t n, bool silu, bool small) {
  return mx_sched_blocks(max_entries, mx_sched_tiles(n, silu, small)) <= MX_MAX_BLOCKS;
}

template <bool SILU>
static int launch_mx_sched(const MxParams &p, int max_entries, bool small, hipStream_t st) {
  const int ntiles = mx_sched_tiles(p.N, SILU, small);
  const int64_t blocks = mx_sched_blocks(max_entries, ntiles);
  int rc;
  if (small) {
    const auto kernel = p.K % 512 ? mx_small_sched_kernel<SILU, true> : mx_small_sched_kernel<SILU, false>;
    if ((rc = mx_lds(kernel, MXS_LDS))) return rc;
    kernel<<<dim3((unsigned)blocks), 1024, MXS_LDS, st>>>(p, ntiles);
    return check_launch("mxfp4 grouped product of few tiles");
  }
  const auto kernel = p.K % 512 ? mx_sched_kernel<SILU, true> : mx_sched_kernel<SILU, false>;
  if ((rc = mx_lds(kernel, MX_TILE_LDS))) return rc;
  kernel<<<dim3((unsigned)blocks), 512, MX_TILE_LDS, st>>>(p, ntiles);
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
  bool stream, fused;  // fused: the stream product quantises
  MxSplit sp;
};
// Values of x that each workgroup of a linear may quantise for itself: 1 x 7168 x 16384 16.8
// us, with a pass before it 19.0; 8 x 18432 x 7168 20.7 and 21.3; 16 x 2112 x 7168 11.8 and
// 11.0.  SwiGLU, groups and experts always do on the stream product, which has more weight rows
// there: SwiGLU of 7168 to 18432, 1 row 38.6 and 40.7, 8 rows 44.8 and 45.4, 16 rows 49.7 and
// 49.1; 16 rows of 32 groups, 7168 to 2048, 24.9 and 26.8; 8 tokens on 64 experts 209 and 211.5.
constexpr int64_t MX_FUSED = 72 * 1024;
// held: x comes quantised
static MxLinearLayout mx_linear_layout(int64_t m, int64_t k, int64_t n, bool held) {
  MxLinearLayout L = {};
  MxTake take;
  L.stream = mx_stream_fits(m, k, false);
  L.fused = L.stream && m * k <= MX_FUSED;
  if (!held && !L.fused) {
    L.xc = take(mx_codes_bytes(m, k));
    L.xs = take(mx_scale_bytes(m, k));
  }
  if (!L.stream) {
    L.sp = plan_mx_split(m, (int)n, (int)k, false);
    L.part = take(mx_split_bytes(L.sp));
  }
  L.total = take.off;
  return L;
}

struct MxGroupedLayout {
  size_t count, ent, xc, xs, total;
  int rows, max_entries;  // of an entry; entries at most
  bool stream, small;
};
static MxGroupedLayout mx_grouped_layout(int64_t m, int64_t k, int64_t n, int64_t E, bool held) {
  MxGroupedLayout L = {};
  MxTake take;
  L.stream = mx_stream_fits(m, k, false);
  L.small = !L.stream && mx_small_round(m, E, (n + 127) / 128);
  L.rows = L.stream ? 16 : L.small ? MXS_ROWS : MX_ROWS;
  L.max_entries = (int)(std::min(E, m) + m / L.rows + 2);
  L.count = take(8);
  L.ent = take((size_t)L.max_entries * 16);
  if (!held && !L.stream) {
    L.xc = take(mx_codes_bytes(m, k));
    L.xs = take(mx_scale_bytes(m, k));
  }
  L.total = take.off;
  return L;
}

struct MxSwigluLayout {
  size_t xc, xs, hc, hs, lin, total;
  bool stream;
  MxSplit sp;
  MxLinearLayout down;
};
static MxSwigluLayout mx_swiglu_layout(int64_t m, int64_t k, int64_t n) {
  MxSwigluLayout L = {};
  MxTake take;
  L.stream = mx_stream_fits(m, k, true);
  L.hc = take(mx_codes_bytes(m, n));
  L.hs = take(mx_scale_bytes(m, n));
  if (!L.stream) {
    L.xc = take(mx_codes_bytes(m, k));
    L.xs = take(mx_scale_bytes(m, k));
    L.sp = plan_mx_split(m, (int)n, (int)k, true);
  }
  L.down = mx_linear_layout(m, n, k, true);
  L.lin = take(std::max(L.stream ? 0 : mx_split_bytes(L.sp), L.down.total));
  L.total = take.off;
  return L;
}

struct MxMoeLayout {
  size_t hdr, count, gather, scatter, ent, xc, xs, hc, hs, total;
  int rows, max_entries;
  bool stream, small_up, small_down;
};
static MxMoeLayout mx_moe_layout(int64_t m, int64_t d, int top_k, int64_t n, int64_t E) {
  MxMoeLayout L = {};
  MxTake take;
  const int64_t S = m * top_k;
  L.stream = mx_stream_fits(m, d, true) && mx_stream_fits(m, n, false);
  L.small_up = !L.stream && mx_small_round(S, E, (n + 63) / 64);
  L.small_down = !L.stream && mx_small_round(S, E, (d + 127) / 128);
  // One schedule for both products: where only one of them has small tiles, the other runs large ones
  // on entries of 64 rows.  Hidden size 7168, intermediate 2048: 400 rows in 8 ragged groups 69 us, with
  // large tiles for both 82; in 2 groups 45 and 81.  2048 and 7168: 700 in 4 groups 67 and 80 - 104, 900
  // in 16 even ones 126 and 121.  (An entry of the stream product holds m rows at most, also where tokens
  // name an expert several times: more entries then.)
  L.rows = L.stream ? (int)m : L.small_up || L.small_down ? MXS_ROWS : MX_ROWS;
  L.max_entries = (int)std::min<int64_t>(S, std::min<int64_t>(E, S) + S / L.rows);
  L.hdr = take(16);
  L.count = take(4);
  L.gather = take((size_t)S * 4);
  L.scatter = take((size_t)S * 4);
  L.ent = take((size_t)L.max_entries * 16);
  L.hc = take(mx_codes_bytes(S, n));
  L.hs = take(mx_scale_bytes(S, n));
  if (!L.stream) {
    L.xc = take(mx_codes_bytes(m, d));
    L.xs = take(mx_scale_bytes(m, d));
  }
  L.total = take.off;
  return L;
}

static bool mx_sizes_ok(int64_t m, int64_t n, int64_t k) {
  return m > 0 && n > 0 && k > 0 && m <= INT32_MAX && n <= INT32_MAX / 4 && k <= (1 << 24) && k % 128 == 0;
}

// (both products of an FFN: k to n and n to k)
static bool mx_ffn_sizes_ok(int64_t m, int64_t n, int64_t k) { return mx_sizes_ok(m, n, k) && mx_sizes_ok(m, k, n); }
static bool mx_moe_sizes_ok(int64_t m, int64_t d, int64_t top_k, int64_t n, int64_t E) {
  return top_k > 0 && top_k <= 64 && E > 0 && E <= 512 && m <= 65536 && m * top_k <= 65536 && mx_ffn_sizes_ok(m, n, d) &&
         m * (d / 2) <= UINT32_MAX;  // gathered rows: 32-bit offsets
}

static void mx_outputs(MxParams &p, void *y, int64_t ldy, int dtype) {
  p.y = y;
  p.ldy = ldy;
  p.f32 = dtype == AMLA_FP32;
  p.vec16 = p.N % (p.f32 ? 4 : 8) == 0 && ldy % (p.f32 ? 4 : 8) == 0 && aligned16(y);
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
  if (!L.stream && !mx_linear_grid_ok(L.sp))
    return fail(AMLA_EUNSUPPORTED, "mxfp4_linear: %lld x %lld outputs", (long long)m, (long long)n);
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
  if (!x_scales && !L.fused) {
    const int rc = launch_mx_quantize_bf16(static_cast<const uint16_t *>(x), m, k, ldx, ws + L.xc, ws + L.xs, st);
    if (rc) return rc;
    p.x = ws + L.xc;
    p.xs = ws + L.xs;
  }
  if (L.stream) return launch_mx_stream<false>(p, (int)m, 1, st);
  MxSplit sp = L.sp;
  sp.partial = reinterpret_cast<float *>(ws + L.part);
  return launch_mx_linear<false>(p, sp, st);
}

size_t amla_mxfp4_grouped_linear_workspace_bytes(int64_t m, int64_t n, int64_t k, int64_t n_experts, int quantized) {
  if (!mx_sizes_ok(m, n, k) || n_experts <= 0 || n_experts > MX_MAX_GROUPS) return 0;
  return mx_grouped_layout(m, k, n, n_experts, quantized != 0).total;
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
  const MxGroupedLayout L = mx_grouped_layout(m, k, n, n_experts, x_scales != nullptr);
  if (!L.stream && !mx_sched_grid_ok(L.max_entries, n, false, L.small))
    return fail(AMLA_EUNSUPPORTED, "mxfp4_grouped_linear: %lld x %lld outputs", (long long)m, (long long)n);
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
  p.rest = clear_rest != 0;
  p.M = (int)m; p.N = (int)n; p.K = (int)k;
  mx_outputs(p, y, ldy, dtype);
  if (L.stream) return launch_mx_stream<false>(p, (int)m, (int)std::min<int64_t>(n_experts, m), st);
  if (!x_scales) {
    if ((rc = launch_mx_quantize_bf16(static_cast<const uint16_t *>(x), m, k, ldx, ws + L.xc, ws + L.xs, st))) return rc;
    p.x = ws + L.xc;
    p.xs = ws + L.xs;
  }
  return launch_mx_sched<false>(p, L.max_entries, L.small, st);
}

size_t amla_mxfp4_swiglu_workspace_bytes(int64_t m, int64_t k, int64_t n) {
  if (!mx_ffn_sizes_ok(m, n, k)) return 0;
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
  bool ok = mx_ffn_sizes_ok(m, n, k) && ldx % 8 == 0 && aligned16(x) && aligned16(y);
  for (const void *w : {gate_w, up_w, down_w}) ok = ok && aligned16(w);
  for (const void *s : {gate_s, up_s, down_s}) ok = ok && reinterpret_cast<uintptr_t>(s) % 4 == 0;
  if (!ok)
    return fail(AMLA_EUNSUPPORTED,
                "mxfp4_swiglu: needs k %% 128 == 0, n %% 128 == 0, 16-byte aligned rows and weights and 4-byte aligned "
                "scales (n=%lld k=%lld)", (long long)n, (long long)k);
  const MxSwigluLayout L = mx_swiglu_layout(m, k, n);
  if ((!L.stream && !mx_linear_grid_ok(L.sp)) || (!L.down.stream && !mx_linear_grid_ok(L.down.sp)))
    return fail(AMLA_EUNSUPPORTED, "mxfp4_swiglu: %lld x %lld outputs", (long long)m, (long long)std::max(n, k));
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
  if (L.stream) {
    rc = launch_mx_stream<true>(p, (int)m, 1, st);
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
  if (!mx_moe_sizes_ok(m, d, top_k, n_inter, n_experts))
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
  bool ok = mx_moe_sizes_ok(m, d, top_k, n_inter, n_experts) && ldh % 8 == 0 && aligned16(hidden) && aligned16(expert_out);
  for (const void *w : {gate_w, up_w, down_w}) ok = ok && aligned16(w);
  for (const void *s : {gate_s, up_s, down_s}) ok = ok && reinterpret_cast<uintptr_t>(s) % 4 == 0;
  if (!ok)
    return fail(AMLA_EUNSUPPORTED,
                "mxfp4_moe_experts: needs top_k <= 64, at most 512 experts, 65536 slots and 4 GB of codes per call, "
                "hidden and intermediate sizes %% 128 == 0, 16-byte aligned rows and weights and 4-byte aligned scales");
  const MxMoeLayout L = mx_moe_layout(m, d, top_k, n_inter, n_experts);
  if (!L.stream && !(mx_sched_grid_ok(L.max_entries, n_inter, true, L.small_up) &&
                     mx_sched_grid_ok(L.max_entries, d, false, L.small_down)))
    return fail(AMLA_EUNSUPPORTED, "mxfp4_moe_experts: %lld tokens of hidden size %lld and intermediate size %lld",
                (long long)m, (long long)d, (long long)n_inter);
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
  if (L.stream) {
    if ((rc = launch_mx_stream<true>(p, (int)m, L.max_entries, st))) return rc;
    return launch_mx_stream<false>(q, (int)m, L.max_entries, st);
  }
  if ((rc = launch_mx_quantize_bf16(static_cast<const uint16_t *>(hidden), m, d, ldh, ws + L.xc, ws + L.xs, st)))
    return rc;
  p.x = ws + L.xc;
  p.xs = ws + L.xs;
  if ((rc = launch_mx_sched<true>(p, L.max_entries, L.small_up, st))) return rc;
  return launch_mx_sched<false>(q, L.max_entries, L.small_down, st);
}

}  // extern "C"
