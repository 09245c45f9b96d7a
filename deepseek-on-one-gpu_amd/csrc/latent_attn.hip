// Attention of the newest tokens over the paged latent cache (latent.h), in latent space:
//   s_t = scale q . (c_t | r_t),  out = sum_t softmax(s)_t c_t
#include <algorithm>
#include <math.h>

#include "latent.h"

namespace amla {

typedef int i32x8 __attribute__((ext_vector_type(8)));

struct LatentAttnParams {
  LatentPages pg;
  const uint16_t *q;
  int64_t ldq_seq, ldq_token, ldq_head;
  const int32_t *lengths;
  int seqs, seq_len, heads, rows;  // rows = seq_len * heads of one sequence
  int chunks;                      // workgroups of rows per sequence and split
  int cap;                         // rows that a table row can hold
  int slots;                       // workgroups (sequence, chunk, split)
  float scale_log2;
  uint16_t *out;
  float *lse;
  uint16_t *part_o;                // (slots, rows of a chunk, 512) bf16, each split normalised
  float *part_lse;                 // (slots, rows of a chunk) log2 of the split's sum of 2^s
};

AMLA_DEV int lc_ceil_div(int a, int b) { return (a + b - 1) / b; }
AMLA_DEV int wave_isum(int v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}
AMLA_DEV int wave_imax(int v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v = max(v, __shfl_xor(v, o, 64));
  return v;
}

// Split plan, formed by every wave from the lengths (no host synchronisation, no launch of
// its own): a sequence of n tiles gets ceil(n / L) splits, L the smallest length whose
// splits, times the chunks, fit the slots; a launch takes as long as its longest split.
// slots >= chunks * seqs + 128, so the search needs only [total / slots, total / 128].
template <int TILE>
struct SplitPlan {
  const LatentAttnParams &p;
  int len;  // L
  AMLA_DEV int tiles(int b) const {
    return b < p.seqs ? lc_ceil_div(min(max(p.lengths[b], 0), p.cap), TILE) : 0;
  }
  AMLA_DEV int used(int L) const {
    int n = 0;
    for (int b = threadIdx.x & 63; b < p.seqs; b += 64) n += lc_ceil_div(tiles(b), L);
    return wave_isum(n) * p.chunks;
  }
  AMLA_DEV explicit SplitPlan(const LatentAttnParams &p_) : p(p_) {
    int sum = 0, most = 0;
    for (int b = threadIdx.x & 63; b < p.seqs; b += 64) {
      const int n = tiles(b);
      sum += n;
      most = max(most, n);
    }
    const int64_t total = (int64_t)wave_isum(sum) * p.chunks;
    int lo = max(1, (int)((total + p.slots - 1) / p.slots));
    int hi = max(lo, min(wave_imax(most), (int)(total / max(1, p.slots - p.chunks * p.seqs)) + 1));
    for (int probe = lo; lo < hi; probe = (lo + hi) >> 1) {
      if (used(probe) <= p.slots) hi = probe;
      else lo = probe + 1;
    }
    len = __builtin_amdgcn_readfirstlane(lo);
  }
  // (sequence, first slot of it, its splits) of a slot; sequence -1 past the plan
  AMLA_DEV int3 find(int slot) const {
    const int lane = threadIdx.x & 63;
    int base = 0;
    for (int b0 = 0; b0 < p.seqs; b0 += 64) {
      const int s = lc_ceil_div(tiles(b0 + lane), len);
      int incl = s * p.chunks;
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) {
        const int v = __shfl_up(incl, o, 64);
        if (lane >= o) incl += v;
      }
      const uint64_t past = __ballot(base + incl > slot);
      if (past) {
        const int l = __builtin_ctzll(past);
        return int3{b0 + l, base + __builtin_amdgcn_readlane(incl, l) - __builtin_amdgcn_readlane(s, l) * p.chunks,
                    __builtin_amdgcn_readlane(s, l)};
      }
      base += __builtin_amdgcn_readlane(incl, 63);
    }
    return int3{-1, 0, 0};
  }
  // (first slot, splits) of sequence b
  AMLA_DEV int2 of(int b) const {
    int before = 0;
    for (int i = threadIdx.x & 63; i < b; i += 64) before += lc_ceil_div(tiles(i), len);
    return int2{wave_isum(before) * p.chunks, lc_ceil_div(tiles(b), len)};
  }
};

// ---------------------------------------------------------------- tiles in LDS
//
// A stage holds TILE rows as they lie in the pool (latent rows of RB bytes, rope rows of
// 128), 16-byte chunks permuted within a row so that every fragment read is free of bank
// conflicts (16 consecutive lanes of a 16-byte read, and the 32 lanes of one pass of a
// transpose read, differ in address bits 4 - 7), then per row: the exponent as a float
// (-inf where there is no row), 2^-exponent and the exponent byte.
template <bool F8> struct Tile;
template <> struct Tile<true> {
  static constexpr int ROWS = 64, RB = 512, STAGES = 3;
  static AMLA_DEV int swz(int r) { return ((r & 3) << 1) | ((r >> 2) & 1) | (r & 8); }
};
template <> struct Tile<false> {
  static constexpr int ROWS = 32, RB = 1024, STAGES = 4;
  static AMLA_DEV int swz(int r) { return ((r & 3) << 2) | ((r >> 2) & 3); }
};
template <bool F8> struct Stage {
  static constexpr int ROWS = Tile<F8>::ROWS;
  static constexpr int PE = ROWS * Tile<F8>::RB, EXP = PE + ROWS * 128, INV = EXP + ROWS * 4, BYTE = INV + ROWS * 4;
  static constexpr int SIZE = BYTE + ROWS * 4;
  static constexpr int LDS = SIZE * Tile<F8>::STAGES;
};

// The reference m of a query row's sums moves (a multiplication of all of them) only when a score passes
// it by 2^40: fp32 and bf16 have the range, and e4m3 has a scale for each block.  m is a whole number.
constexpr float LAG = 40.f;

template <int OFS>
AMLA_DEV u32x4 lds_read16(uint32_t addr) {
  u32x4 v;
  asm volatile("ds_read_b128 %0, %1 offset:%2" : "=v"(v) : "v"(addr), "i"(OFS) : "memory");
  return v;
}
AMLA_DEV u32x4 lds_read16(uint32_t addr) { return lds_read16<0>(addr); }
AMLA_DEV uint32_t lds_read4(uint32_t addr) {
  uint32_t v;
  asm volatile("ds_read_b32 %0, %1" : "=v"(v) : "v"(addr) : "memory");
  return v;
}
AMLA_DEV u32x2 lds_read_tr8(uint32_t addr) {
  u32x2 v;
  asm volatile("ds_read_b64_tr_b8 %0, %1" : "=v"(v) : "v"(addr) : "memory");
  return v;
}
AMLA_DEV u32x2 lds_read_tr16(uint32_t addr) {
  u32x2 v;
  asm volatile("ds_read_b64_tr_b16 %0, %1" : "=v"(v) : "v"(addr) : "memory");
  return v;
}
// Waits until at most N LDS operations are in flight and ties the registers that the wait guards to it.
template <int N> AMLA_DEV void lds_wait() { asm volatile("s_waitcnt lgkmcnt(%0)" ::"i"(N) : "memory"); }
template <typename T, typename... R> AMLA_DEV void lds_tie(T &v, R &...rest) {
  asm volatile("" : "+v"(v)::"memory");
  if constexpr (sizeof...(rest) > 0) lds_tie(rest...);
}
template <int N, typename... T> AMLA_DEV void lds_wait(T &...v) {
  lds_wait<N>();
  lds_tie(v...);
}

AMLA_DEV f32x16 mfma32(bf16x8 a, bf16x8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
AMLA_DEV i32x8 join(u32x4 a, u32x4 b) {
  return i32x8{(int)a.x, (int)a.y, (int)a.z, (int)a.w, (int)b.x, (int)b.y, (int)b.z, (int)b.w};
}
// A (32 x 64) B (64 x 32) of e4m3 codes, lane l holding 32 codes of row (column) l % 32,
// each operand times 2^(byte - 127) of the low byte of its scale: codes 0 - 15 of both lanes of a row are
// one block, scaled by the byte of lane l % 32, codes 16 - 31 the other, by that of lane l % 32 + 32
AMLA_DEV f32x16 mfma32_f8(i32x8 a, int as, i32x8 b, int bs, f32x16 c) {
  return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(a, b, c, 0, 0, 0, as, 0, bs);
}

AMLA_DEV int pk_fp8x4(float a, float b, float c, float d) {
  const int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  return __builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true);
}
// x = hi + lo / 16 in e4m3: four values, magnitudes up to 448.  hi keeps the four leading
// bits, lo the next four, so a bf16 value comes through whole.
AMLA_DEV void split_fp8x4(const float *x, int &hi, int &lo) {
  hi = pk_fp8x4(x[0], x[1], x[2], x[3]);
  const f32x2 a = fp8x2_to_f32<false>(hi), b = fp8x2_to_f32<true>(hi);
  lo = pk_fp8x4((x[0] - a.x) * 16.f, (x[1] - a.y) * 16.f, (x[2] - b.x) * 16.f, (x[3] - b.y) * 16.f);
}

// Copies a wave's rows of a tile, ROWS / 4 from row r0 on, straight into LDS: lane L holds the
// pool row of row r0 + L % (ROWS / 4) (below 0: row 0 of the pool).
template <bool F8>
AMLA_DEV void copy_rows(const LatentPages &pg, uint8_t *st, int r0, int slot) {
  using T = Tile<F8>;
  constexpr int WR = T::ROWS / 4;
  const int lane = threadIdx.x & 63;
  if constexpr (F8) {
#pragma unroll
    for (int i = 0; i < WR / 2; ++i) {  // two rows of 512 bytes each
      const int r = 2 * i + (lane >> 5);
      const size_t s = max(__shfl(slot, r, 64), 0);
      __builtin_amdgcn_global_load_lds(pg.latent + s * 512 + 16 * ((lane & 31) ^ T::swz(r0 + r)),
                                       LDS_PTR(st + (r0 + 2 * i) * 512), 16, 0, 2);
    }
  } else {
#pragma unroll
    for (int i = 0; i < WR; ++i) {
      const size_t s = max(__shfl(slot, i, 64), 0);
      __builtin_amdgcn_global_load_lds(pg.latent + s * 1024 + 16 * (lane ^ T::swz(r0 + i)), LDS_PTR(st + (r0 + i) * 1024),
                                       16, 0, 2);
    }
  }
#pragma unroll
  for (int i = 0; i < WR / 8; ++i) {
    const int r = 8 * i + (lane >> 3);
    const size_t s = max(__shfl(slot, r, 64), 0);
    __builtin_amdgcn_global_load_lds(pg.k_pe + s * 64 + 8 * ((lane & 7) ^ (((r0 + r) >> 1) & 7)),
                                     LDS_PTR(st + Stage<F8>::PE + (r0 + 8 * i) * 128), 16, 0, 2);
  }
}

// One workgroup of four waves per (sequence, chunk of 32 HG rows, split).  HG waves hold 32
// query rows each; the 4 / HG waves of the same rows compute the same scores and
// accumulate 512 HG / 4 columns each.
template <bool F8, int HG>
__global__ __launch_bounds__(256, 1) void latent_attn_kernel(LatentAttnParams p) {
  extern __shared__ __align__(16) uint8_t sm[];
  using T = Tile<F8>;
  using G = Stage<F8>;
  constexpr int TILE = T::ROWS, NST = T::STAGES, PD = NST - 1;
  constexpr int CG = 4 / HG, NCB = 16 / CG;  // 32-column blocks of a wave
  constexpr int KB = TILE / 32;              // 32-row blocks of a tile
  constexpr int WR = TILE / 4;               // rows that a wave copies
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int j32 = lane & 31, hh = lane >> 5, L16 = lane & 15, g16 = lane >> 4;
  const int hg = wave / CG, cg = wave % CG;

  const SplitPlan<TILE> plan(p);
  const int3 at = plan.find(blockIdx.x);
  if (at.x < 0) return;
  const int b = at.x, splits = at.z;
  const int chunk = ((int)blockIdx.x - at.y) / splits, split = ((int)blockIdx.x - at.y) % splits;
  const int rows_held = min(max(p.lengths[b], 0), p.cap);
  const int n_tiles = lc_ceil_div(rows_held, TILE);
  const int t_first = (int)((int64_t)split * n_tiles / splits), t_end = (int)((int64_t)(split + 1) * n_tiles / splits);

  const uint32_t lds0 = (uint32_t)reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) const uint8_t *)sm);

  const int my_row = WR * wave + lane % WR;
  int slot_of[PD], byte_of[PD];
#pragma unroll
  for (int d = 0; d < PD; ++d) {
    slot_of[d] = -1;
    byte_of[d] = 127;
    if (t_first + d < t_end) {
      slot_of[d] = p.pg.slot(b, min((t_first + d) * TILE + my_row, rows_held - 1));
      if (F8) byte_of[d] = p.pg.scales[max(slot_of[d], 0)];
      copy_rows<F8>(p.pg, sm + d * G::SIZE, WR * wave, slot_of[d]);
    }
  }

  // ---- queries: B fragments, lane = row of the chunk
  const int row = (chunk * HG + hg) * 32 + j32;
  const int rq = min(row, p.rows - 1), tok = rq / p.heads;
  const int limit = rows_held - (p.seq_len - 1 - tok);  // rows [0, limit) are seen
  const uint16_t *qp = p.q + b * p.ldq_seq + tok * p.ldq_token + (rq - tok * p.heads) * p.ldq_head;
  constexpr int QN = F8 ? 8 : 32;
  i32x8 qhi[F8 ? QN : 1], qlo[F8 ? QN : 1];
  bf16x8 qb[F8 ? 1 : QN], qr[4];
  int qs = 127;
  if constexpr (F8) {
    u32x4 raw[QN][4];
    uint32_t amax = 0;
#pragma unroll
    for (int ks = 0; ks < QN; ++ks)
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        raw[ks][c] = ldg16(qp + 64 * ks + 32 * hh + 8 * c);
#pragma unroll
        for (int e = 0; e < 4; ++e)
          amax = max(amax, max((raw[ks][c][e] << 16) & 0x7fffffffu, raw[ks][c][e] & 0x7fff0000u));
      }
    amax = max(amax, (uint32_t)__shfl_xor((int)amax, 32, 64));
    // the exponent that brings the row's largest magnitude into [128, 256)
    const int e = min(max((int)(amax >> 23) - 127 - 7, -100), 100);
    qs = 127 + e;
    const float inv = __uint_as_float((uint32_t)(127 - e) << 23);
#pragma unroll
    for (int ks = 0; ks < QN; ++ks)
#pragma unroll
      for (int c = 0; c < 4; ++c)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint32_t w0 = raw[ks][c][2 * h], w1 = raw[ks][c][2 * h + 1];
          const float x[4] = {lo_bf(w0) * inv, hi_bf(w0) * inv, lo_bf(w1) * inv, hi_bf(w1) * inv};
          int hi, lo;
          split_fp8x4(x, hi, lo);
          qhi[ks][2 * c + h] = hi;
          qlo[ks][2 * c + h] = lo;
        }
  } else {
#pragma unroll
    for (int ks = 0; ks < QN; ++ks) qb[ks] = as_bf16x8(ldg16(qp + 16 * ks + 8 * hh));
  }
#pragma unroll
  for (int ks = 0; ks < 4; ++ks) qr[ks] = as_bf16x8(ldg16(qp + LC_LORA + 16 * ks + 8 * hh));

  f32x16 o[NCB];
#pragma unroll
  for (int c = 0; c < NCB; ++c)
#pragma unroll
    for (int i = 0; i < 16; ++i) o[c][i] = 0.f;
  float m = -1e30f, l = 0.f;  // finite: exp2(-inf - m) is 0 while no row has been seen

  int cur = 0;
  for (int tile = t_first; tile < t_end; ++tile, cur = cur + 1 == NST ? 0 : cur + 1) {
    // ---- this tile's rows have landed in every wave
    if (tile + PD - 1 < t_end) wait_vmcnt<(PD - 1) * (F8 ? WR / 2 + WR / 8 : WR + WR / 8)>();
    else wait_vmcnt<0>();
    uint8_t *st = sm + cur * G::SIZE;
    {
      // rows of no page: zeros in place of what the copy clamped to (a masked NaN would come through 0 * NaN)
      const int sl = slot_of[0], t = tile * TILE + WR * wave + lane;
      const bool none = lane < WR && sl < 0;
      for (uint64_t bad = __ballot(none); bad; bad &= bad - 1) {
        const int r = WR * wave + __builtin_ctzll(bad);
        for (int i = lane; i < T::RB / 16; i += 64) *reinterpret_cast<u32x4 *>(st + r * T::RB + 16 * i) = u32x4{0, 0, 0, 0};
        if (lane < 8) *reinterpret_cast<u32x4 *>(st + G::PE + r * 128 + 16 * lane) = u32x4{0, 0, 0, 0};
      }
      if (lane < WR) {
        const int r = WR * wave + lane, by = none ? 127 : byte_of[0];
        *reinterpret_cast<float *>(st + G::EXP + 4 * r) = none || t >= rows_held ? -INFINITY : (float)(by - 127);
        *reinterpret_cast<float *>(st + G::INV + 4 * r) = __uint_as_float((uint32_t)(254 - by) << 23);
        *reinterpret_cast<int *>(st + G::BYTE + 4 * r) = by;
      }
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
#pragma unroll
    for (int d = 0; d + 1 < PD; ++d) {
      slot_of[d] = slot_of[d + 1];
      byte_of[d] = byte_of[d + 1];
    }
    if (tile + PD < t_end) {
      slot_of[PD - 1] = p.pg.slot(b, min((tile + PD) * TILE + my_row, rows_held - 1));
      if (F8) byte_of[PD - 1] = p.pg.scales[max(slot_of[PD - 1], 0)];
      copy_rows<F8>(p.pg, sm + (cur + PD) % NST * G::SIZE, WR * wave, slot_of[PD - 1]);
    }

    // ---- scores: S^T (rows x 32 queries)
    const uint32_t base = lds0 + cur * G::SIZE;
    f32x16 s[KB];
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) {
      const int r = 32 * kb + j32, sw = T::swz(r);
#pragma unroll
      for (int i = 0; i < 16; ++i) s[kb][i] = 0.f;
      if constexpr (F8) {
        uint32_t ab = lds_read4(base + G::BYTE + 4 * r);
        lds_wait<0>(ab);
#pragma unroll
        for (int ks = 0; ks < QN; ++ks) {
          u32x4 a0 = lds_read16(base + r * 512 + 16 * ((4 * ks + 2 * hh) ^ sw));
          u32x4 a1 = lds_read16(base + r * 512 + 16 * ((4 * ks + 2 * hh + 1) ^ sw));
          lds_wait<0>(a0, a1);
          const i32x8 a = join(a0, a1);
          s[kb] = mfma32_f8(a, (int)ab, qhi[ks], qs, s[kb]);
          s[kb] = mfma32_f8(a, (int)ab, qlo[ks], qs - 4, s[kb]);
        }
      } else {
#pragma unroll
        for (int ks = 0; ks < QN; ++ks) {
          u32x4 a = lds_read16(base + r * 1024 + 16 * ((2 * ks + hh) ^ sw));
          lds_wait<0>(a);
          s[kb] = mfma32(as_bf16x8(a), qb[ks], s[kb]);
        }
      }
#pragma unroll
      for (int ks = 0; ks < 4; ++ks) {
        u32x4 a = lds_read16(base + G::PE + r * 128 + 16 * ((2 * ks + hh) ^ ((r >> 1) & 7)));
        lds_wait<0>(a);
        s[kb] = mfma32(as_bf16x8(a), qr[ks], s[kb]);
      }
    }
    // ---- z = s log2(e) scale + exponent
    float mx[KB];  // of 32 rows
    const bool tail = (tile + 1) * TILE > rows_held - (p.seq_len - 1);
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) {
      mx[kb] = -INFINITY;
#pragma unroll
      for (int q4 = 0; q4 < 4; ++q4) {
        u32x4 ex = lds_read16(base + G::EXP + 4 * (32 * kb + 8 * q4 + 4 * hh));
        lds_wait<0>(ex);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float z = __builtin_fmaf(s[kb][4 * q4 + i], p.scale_log2, __uint_as_float(ex[i]));
          if (tail && tile * TILE + 32 * kb + 8 * q4 + 4 * hh + i >= limit) z = -INFINITY;
          s[kb][4 * q4 + i] = z;
          mx[kb] = __builtin_fmaxf(mx[kb], z);
        }
      }
      mx[kb] = __builtin_fmaxf(mx[kb], __shfl_xor(mx[kb], 32, 64));
    }
    const float top = __builtin_fmaxf(mx[0], mx[KB - 1]);
    if (__ballot(top > m + LAG)) {
      const float mn = top > m + LAG ? ceilf(top) : m;
      const float f = __builtin_amdgcn_exp2f(m - mn);
      m = mn;
      l *= f;
#pragma unroll
      for (int c = 0; c < NCB; ++c) o[c] *= f;
    }
    // ---- P = 2^(z - ref); l sums 2^(s - m) = P 2^(ref - m) 2^-exponent
    // e4m3: 32 rows are one block of the matrix unit with a scale of its own, 2^(ref - m), so that rows far
    // below the sequence's maximum keep their bits: a reference for all would drop those below 2^-22 of
    // it, and thousands of them can outweigh it.
    float ref[KB];
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) ref[kb] = F8 ? floorf(__builtin_fmaxf(mx[kb], -1e30f)) - 7.f : m;
    i32x8 phi, plo;
    u32x4 pb[2];
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) {
      float sum = 0.f;
#pragma unroll
      for (int q4 = 0; q4 < 4; ++q4) {
        float e[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) e[i] = __builtin_amdgcn_exp2f(s[kb][4 * q4 + i] - ref[kb]);
        if constexpr (F8) {
          u32x4 iv = lds_read16(base + G::INV + 4 * (32 * kb + 8 * q4 + 4 * hh));
          lds_wait<0>(iv);
#pragma unroll
          for (int i = 0; i < 4; ++i) sum = __builtin_fmaf(e[i], __uint_as_float(iv[i]), sum);
          int hi, lo;
          split_fp8x4(e, hi, lo);
          phi[4 * kb + q4] = hi;
          plo[4 * kb + q4] = lo;
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i) sum += e[i];
          pb[q4 >> 1][2 * (q4 & 1)] = pack_bf16(e[0], e[1]);
          pb[q4 >> 1][2 * (q4 & 1) + 1] = pack_bf16(e[2], e[3]);
        }
      }
      l += F8 ? sum * __builtin_amdgcn_exp2f(ref[kb] - m) : sum;
    }
    // the scale of block kb comes from the lanes of half kb; 4 .. 160, the low halves' 4 less
    const int ps = (int)__builtin_fmaxf((hh ? ref[KB - 1] : ref[0]) - m, -123.f) + 127;
    // ---- O^T (columns x queries) += C^T P^T
#pragma unroll
    for (int c = 0; c < NCB; ++c) {
      const int cb = cg * NCB + c;
      if constexpr (F8) {
        u32x2 v[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {  // rows 16 i + 4 hh + {0..3, 8..11}
          const int r = 16 * i + 8 * (L16 >> 3) + 4 * hh + ((L16 >> 1) & 3);
          v[i] = lds_read_tr8(base + r * 512 + 16 * ((2 * cb + (g16 & 1)) ^ T::swz(r)) + 8 * (L16 & 1));
        }
        lds_wait<0>(v[0], v[1], v[2], v[3]);
        const i32x8 a = join(u32x4{v[0].x, v[0].y, v[1].x, v[1].y}, u32x4{v[2].x, v[2].y, v[3].x, v[3].y});
        o[c] = mfma32_f8(a, 127, phi, ps, o[c]);
        o[c] = mfma32_f8(a, 127, plo, ps - 4, o[c]);
      } else {
#pragma unroll
        for (int kk = 0; kk < 2; ++kk) {
          u32x2 v[2];
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int r = 16 * kk + 8 * i + 4 * hh + (L16 >> 2);
            v[i] = lds_read_tr16(base + r * 1024 + 16 * ((4 * cb + 2 * (g16 & 1) + ((L16 >> 1) & 1)) ^ T::swz(r)) + 8 * (L16 & 1));
          }
          lds_wait<0>(v[0], v[1]);
          o[c] = mfma32(as_bf16x8(u32x4{v[0].x, v[0].y, v[1].x, v[1].y}), as_bf16x8(pb[kk]), o[c]);
        }
      }
    }
  }

  // ---- the split's sums, normalised: the output itself, or a partial one
  l += __shfl_xor(l, 32, 64);
  const float inv = l == 0.f ? 0.f : 1.f / l;
  const float lse2 = l == 0.f ? -INFINITY : m + __builtin_amdgcn_logf(l);
  if (row >= p.rows) return;
  const size_t dst = splits == 1 ? (size_t)b * p.rows + row : (size_t)blockIdx.x * (32 * HG) + 32 * hg + j32;
  uint16_t *od = (splits == 1 ? p.out : p.part_o) + dst * LC_LORA;
#pragma unroll
  for (int c = 0; c < NCB; ++c)
#pragma unroll
    for (int q4 = 0; q4 < 4; ++q4) {
      const u32x2 w = {pack_bf16(o[c][4 * q4] * inv, o[c][4 * q4 + 1] * inv),
                       pack_bf16(o[c][4 * q4 + 2] * inv, o[c][4 * q4 + 3] * inv)};
      *reinterpret_cast<u32x2 *>(od + 32 * (cg * NCB + c) + 8 * q4 + 4 * hh) = w;
    }
  if (cg == 0 && hh == 0) {
    if (splits > 1) p.part_lse[dst] = lse2;
    else if (p.lse) p.lse[dst] = lse2 * 0.6931471805599453f;
  }
}

// Joins the splits of a query row, one wave per row: sum_j 2^(lse_j - max) O_j / sum_j 2^(lse_j - max).
template <bool F8, int HG>
__global__ __launch_bounds__(256) void latent_join_kernel(LatentAttnParams p) {
  const int lane = threadIdx.x & 63;
  const int b = blockIdx.y, row = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const SplitPlan<Tile<F8>::ROWS> plan(p);
  const int2 at = plan.of(b);
  if (at.y == 1 || row >= p.rows) return;
  const size_t dst = (size_t)b * p.rows + row;
  u32x4 *od = reinterpret_cast<u32x4 *>(p.out + dst * LC_LORA) + lane;
  if (at.y == 0) {
    *od = u32x4{0, 0, 0, 0};
    if (lane == 0 && p.lse) p.lse[dst] = -INFINITY;
    return;
  }
  const int chunk = row / (32 * HG);
  const size_t src = (size_t)(at.x + chunk * at.y) * (32 * HG) + row % (32 * HG);
  float top = -INFINITY;
  for (int j = lane; j < at.y; j += 64) top = __builtin_fmaxf(top, p.part_lse[src + (size_t)j * (32 * HG)]);
  top = wave_max(top);
  const float ref = top == -INFINITY ? 0.f : top;
  float total = 0.f, a[8] = {};
  for (int j0 = 0; j0 < at.y; j0 += 64) {
    const float w = j0 + lane < at.y ? __builtin_amdgcn_exp2f(p.part_lse[src + (size_t)(j0 + lane) * (32 * HG)] - ref) : 0.f;
    total += wave_sum(w);
    for (int j = 0; j < min(64, at.y - j0); ++j) {
      const float wj = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(w), j));
      if (wj == 0.f) continue;
      const u32x4 v = ldg16(p.part_o + (src + (size_t)(j0 + j) * (32 * HG)) * LC_LORA + 8 * lane);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        a[2 * e] += wj * lo_bf(v[e]);
        a[2 * e + 1] += wj * hi_bf(v[e]);
      }
    }
  }
  const float inv = total == 0.f ? 0.f : 1.f / total;
  *od = u32x4{pack_bf16(a[0] * inv, a[1] * inv), pack_bf16(a[2] * inv, a[3] * inv), pack_bf16(a[4] * inv, a[5] * inv),
              pack_bf16(a[6] * inv, a[7] * inv)};
  if (lane == 0 && p.lse) p.lse[dst] = total == 0.f ? -INFINITY : (top + __builtin_amdgcn_logf(total)) * 0.6931471805599453f;
}

constexpr int LA_UNITS = 256;  // workgroups that run at a time (one per CU)

// 32-row groups of a workgroup: as many as the rows of a sequence fill
static int attn_groups(int64_t) { return 1; }
struct AttnSizes {
  int hg;
  int64_t chunks, slots;
};
static AttnSizes attn_sizes(int64_t seqs, int64_t rows, int64_t max_rows) {
  AttnSizes s;
  s.hg = attn_groups(rows);
  s.chunks = (rows + 32 * s.hg - 1) / (32 * s.hg);
  s.slots = std::max<int64_t>(LA_UNITS, s.chunks * seqs + LA_UNITS / 2);
  const int64_t tiles = std::max<int64_t>(1, (max_rows + 31) / 32);  // no split is shorter than a tile
  if (tiles < s.slots / (s.chunks * seqs)) s.slots = s.chunks * seqs * tiles;
  return s;
}

template <bool F8, int HG>
static int launch_attn(const LatentAttnParams &p, hipStream_t st) {
  static const hipError_t attr = hipFuncSetAttribute((const void *)latent_attn_kernel<F8, HG>,
                                                     hipFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024);
  (void)attr;
  latent_attn_kernel<F8, HG><<<dim3((unsigned)p.slots), 256, Stage<F8>::LDS, st>>>(p);
  int rc = check_launch("latent_attention");
  if (rc) return rc;
  latent_join_kernel<F8, HG><<<dim3((unsigned)((p.rows + 3) / 4), (unsigned)p.seqs), 256, 0, st>>>(p);
  return check_launch("latent_attention join");
}

}  // namespace amla

using namespace amla;

extern "C" {

size_t amla_latent_attention_workspace_bytes(int64_t seqs, int64_t seq_len, int64_t heads, int64_t max_rows) {
  if (seqs <= 0 || seq_len <= 0 || heads <= 0 || seqs > AMLA_MAX_SEQS || seq_len > INT32_MAX || heads > INT32_MAX / seq_len)
    return 0;
  const AttnSizes s = attn_sizes(seqs, seq_len * heads, max_rows);
  return (size_t)s.slots * 32 * s.hg * (LC_LORA * 2 + 4);
}

int amla_latent_attention(const amla_latent_cache *cache, const void *q, int64_t seqs, int64_t seq_len, int64_t heads,
                          int64_t ldq_seq, int64_t ldq_token, int64_t ldq_head, const int32_t *lengths, float scale,
                          void *out, float *lse, void *workspace, size_t workspace_bytes, void *stream) {
  const char *what = "latent_attention";
  LatentAttnParams p = {};
  int rc = latent_pages(cache, what, &p.pg);
  if (rc) return rc;
  if (seqs < 0 || seq_len < 0 || heads < 0) return fail(AMLA_EINVAL, "%s: negative size", what);
  if (seqs == 0 || seq_len == 0 || heads == 0) return AMLA_OK;
  if (seqs > AMLA_MAX_SEQS || seq_len > INT32_MAX || heads > INT32_MAX / seq_len)
    return fail(AMLA_EUNSUPPORTED, "%s: at most %d sequences and 2^31 - 1 query rows of each", what, AMLA_MAX_SEQS);
  if (!q || !lengths || !out) return fail(AMLA_EINVAL, "%s: null pointer", what);
  if (ldq_seq % 8 || ldq_token % 8 || ldq_head % 8 || !aligned16(q) || !aligned16(out))
    return fail(AMLA_EUNSUPPORTED, "%s: q rows and out must be 16-byte aligned", what);
  const int64_t cap = cache->cols * cache->page_size;
  const AttnSizes s = attn_sizes(seqs, seq_len * heads, cap);
  if (s.slots > (1 << 24) || (seq_len * heads + 3) / 4 > (1 << 24))
    return fail(AMLA_EUNSUPPORTED, "%s: too many query rows", what);
  if (workspace_bytes < amla_latent_attention_workspace_bytes(seqs, seq_len, heads, cap) || !workspace)
    return fail(AMLA_EWORKSPACE, "%s: workspace too small", what);
  if (!aligned16(workspace)) return fail(AMLA_EUNSUPPORTED, "%s: workspace must be 16-byte aligned", what);
  p.q = static_cast<const uint16_t *>(q);
  p.ldq_seq = ldq_seq; p.ldq_token = ldq_token; p.ldq_head = ldq_head;
  p.lengths = lengths;
  p.seqs = (int)seqs; p.seq_len = (int)seq_len; p.heads = (int)heads; p.rows = (int)(seq_len * heads);
  p.chunks = (int)s.chunks; p.slots = (int)s.slots;
  p.cap = (int)cap;
  p.scale_log2 = scale * 1.4426950408889634f;
  p.out = static_cast<uint16_t *>(out);
  p.lse = lse;
  p.part_o = static_cast<uint16_t *>(workspace);
  p.part_lse = reinterpret_cast<float *>(p.part_o + (size_t)s.slots * 32 * s.hg * LC_LORA);
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  if (p.pg.scales) {

    return launch_attn<true, 1>(p, st);
  }

  return launch_attn<false, 1>(p, st);
}

}  // extern "C"
