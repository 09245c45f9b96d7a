// Attention of the newest tokens over the paged latent cache (latent.h), in latent space:
//   s_t = scale q . (c_t | r_t),  out = sum_t softmax(s)_t c_t
// One pass over the cached rows with a running sum per query row, all in fp32; scores are products of bf16 (e4m3 codes are
// exact in it), probabilities are rounded once for the matrix units: to bf16, or to two e4m3 halves that hold eight bits
// of them (inference/ops.py:179 rounds them to bf16).  Every row of the cache serves all heads, so it is read once from
// memory per 128 query rows and split of the sequence.  Many query rows: latent_attn_kernel, bound by the matrix units
// (8 x 32768 rows, 128 heads, e4m3: 83 - 89 us where 73 GFLOP at a large product's rate take 61; the units are busy 43 % of
// the cycles, conversions, softmax and barriers take the others).  Few: latent_attn_few_kernel, bound by the copies (40
// ragged sequences, 16 heads, bf16: 64 us for 342 MB; the copies alone take nine tenths).  Then latent_join_kernel.
#include <algorithm>
#include <math.h>

#include "latent.h"
#include "latent_plan.h"

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
  // Of each split: its sums, normalised, (slots, rows of a chunk, 512) in fp16 times part_scale, a power of two for each of
  // the up to four waves that hold a row's columns; log2 of its sum of 2^s.  fp16 and not bf16, whose rounding would add as
  // much error as the output's own; fp32 would be twice the bytes, a tenth of a long batch's time.  (Columns below 2^-38 of the
  // row's largest are lost; a row of codes spans 2^18.)
  uint16_t *part_o;
  float *part_lse, *part_scale;    // (slots, rows of a chunk), (slots, rows of a chunk, 4)
  int2 *part_plan;                 // (first slot, splits) of each sequence that has rows: the join need not plan again
};

AMLA_DEV int lc_ceil_div(int a, int b) { return (a + b - 1) / b; }
// Sum, maximum and inclusive prefix sum over the wave by lane moves inside the vector unit (a shuffle goes
// through LDS, about ten times the latency).
AMLA_DEV int wave_isum(int v) {
  return (int)wave_reduce_u32((uint32_t)v, [] __device__(uint32_t x, uint32_t y) { return x + y; });
}
AMLA_DEV int wave_imax(int v) { return (int)wave_max_u32((uint32_t)v); }  // of values >= 0
template <int CTRL, int ROWS> AMLA_DEV int dpp_or_zero(int v) {
  return __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xf, true);
}
AMLA_DEV int wave_iscan(int v) {
  v += dpp_or_zero<0x111, 0xf>(v);  // row_shr 1, 2, 4, 8 within 16 lanes
  v += dpp_or_zero<0x112, 0xf>(v);
  v += dpp_or_zero<0x114, 0xf>(v);
  v += dpp_or_zero<0x118, 0xf>(v);
  v += dpp_or_zero<0x142, 0xa>(v);  // lane 15 of each row to the next (rows 1 and 3)
  v += dpp_or_zero<0x143, 0xc>(v);  // lane 31 to rows 2 and 3
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
    return __builtin_amdgcn_readfirstlane(wave_isum(n)) * p.chunks;  // (scalar: what follows from it is uniform)
  }
  AMLA_DEV explicit SplitPlan(const LatentAttnParams &p_) : p(p_) {
    int64_t sum = 0;
    int most = 0;
    for (int b = threadIdx.x & 63; b < p.seqs; b += 64) {
      const int n = tiles(b);
      sum += n;
      most = max(most, n);
    }
    const int low = __builtin_amdgcn_readfirstlane(wave_isum(plan_low(sum)));
    const int high = __builtin_amdgcn_readfirstlane(wave_isum(plan_high(sum)));
    const PlanRange r = plan_range(plan_total(low, high), __builtin_amdgcn_readfirstlane(wave_imax(most)), p.chunks, p.seqs, p.slots);
    int lo = r.lo, hi = r.hi;
    for (int probe = lo; lo < hi; probe = (lo + hi) >> 1) {
      if (used(probe) <= p.slots) hi = probe;
      else lo = probe + 1;
    }
    len = lo;
  }
  // (sequence, first slot of it, its splits) of a slot; sequence -1 past the plan
  AMLA_DEV int3 find(int slot) const {
    const int lane = threadIdx.x & 63;
    int base = 0;
    for (int b0 = 0; b0 < p.seqs; b0 += 64) {
      const int s = lc_ceil_div(tiles(b0 + lane), len);
      const int incl = wave_iscan(s * p.chunks);
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
};

// ---------------------------------------------------------------- tiles in LDS
//
// A stage holds TILE rows as they lie in the pool (latent rows of RB bytes, rope rows of
// 128), 16-byte chunks permuted within a row so that every fragment read is free of bank
// conflicts (16 consecutive lanes of a 16-byte read, and the 32 lanes of one pass of a
// transpose read, differ in address bits 4 - 7), then per row: the exponent as a float
// (-inf where there is no row), 2^-exponent and 2^exponent.
template <bool F8> struct Tile;
template <> struct Tile<true> {
  static constexpr int ROWS = 64, RB = 512, STAGES = 3;
  static AMLA_DEV constexpr int swz(int r) { return ((r & 3) << 1) | ((r >> 2) & 1) | (r & 8); }
};
template <> struct Tile<false> {
  static constexpr int ROWS = 32, RB = 1024, STAGES = 4;
  static AMLA_DEV constexpr int swz(int r) { return ((r & 3) << 2) | ((r >> 2) & 3); }
};
template <bool F8> struct Stage {
  static constexpr int ROWS = Tile<F8>::ROWS;
  static constexpr int PE = ROWS * Tile<F8>::RB, EXP = PE + ROWS * 128, INV = EXP + ROWS * 4, MUL = INV + ROWS * 4;
  static constexpr int SIZE = (MUL + ROWS * 4 + 1023) / 1024 * 1024;  // chunks enter addresses by xor
  // query fragments that the registers have no room for: QL of the latent ones, e4m3: and the four of the rope key
  static constexpr int Q = SIZE * Tile<F8>::STAGES, QL = F8 ? 5 : 3, QF = QL + (F8 ? 4 : 0);
  static constexpr int LDS = Q + 4 * QF * 1024;
};

// The reference m of a query row's sums is its maximum over the split's first tile, so that the output
// accumulators are never multiplied: fp32 and bf16 have the range, and e4m3 has a scale for each block.  It is the maximum
// itself, not a whole number above it: the probability of the loudest row, all there is of a short sequence, is not rounded.  A
// row whose scores pass m by 2^LAG later on (or that saw nothing in the first tile) has the workgroup do
// its split once more, with m from all of it.
constexpr float LAG = 60.f;
// No row seen yet.  Finite, so that 2^(-inf - M_NONE) is 0, below the scores that are told from none, and their difference
// from it is finite.
constexpr float M_NONE = -0x1p126f;

// The lane, opaque to the compiler: what is derived from it is formed anew instead of held in a register
// throughout the loop (there are none to spare).
AMLA_DEV int fresh_lane() {
  int lane = threadIdx.x & 63;
  asm volatile("" : "+v"(lane));
  return lane;
}

template <int OFS> AMLA_DEV u32x4 lds_read16(uint32_t addr) {
  u32x4 v;
  asm volatile("ds_read_b128 %0, %1 offset:%2" : "=v"(v) : "v"(addr), "i"(OFS) : "memory");
  return v;
}
template <bool F8, int OFS> AMLA_DEV u32x2 lds_read_tr(uint32_t addr) {
  u32x2 v;
  if constexpr (F8) asm volatile("ds_read_b64_tr_b8 %0, %1 offset:%2" : "=v"(v) : "v"(addr), "i"(OFS) : "memory");
  else asm volatile("ds_read_b64_tr_b16 %0, %1 offset:%2" : "=v"(v) : "v"(addr), "i"(OFS) : "memory");
  return v;
}
// Waits until at most N LDS operations are in flight; lds_tie ties registers that a wait guards to it.
template <int N> AMLA_DEV void lds_wait() { asm volatile("s_waitcnt lgkmcnt(%0)" ::"i"(N < 15 ? N : 15) : "memory"); }
template <typename T, typename... R> AMLA_DEV void lds_tie(T &v, R &...rest) {
  asm volatile("" : "+v"(v)::"memory");
  if constexpr (sizeof...(rest) > 0) lds_tie(rest...);
}

// Scores accumulate in vector registers (inline asm): the accumulator registers hold the outputs.  WAIT: an operand may have
// been written just before, which takes two wait states (8 cycles); where none can be, the test of the assembly holds it to that.
template <bool WAIT> AMLA_DEV void mfma_score(f32x16 &c, bf16x8 a, bf16x8 b) {
  if constexpr (WAIT) asm volatile("s_nop 1\n\tv_mfma_f32_32x32x16_bf16 %0, %1, %2, %0" : "+v"(c) : "v"(a), "v"(b));
  else asm volatile("v_mfma_f32_32x32x16_bf16 %0, %1, %2, %0" : "+v"(c) : "v"(a), "v"(b));
}
template <bool WAIT> AMLA_DEV void mfma_score0(f32x16 &c, bf16x8 a, bf16x8 b) {
  if constexpr (WAIT) asm volatile("s_nop 1\n\tv_mfma_f32_32x32x16_bf16 %0, %1, %2, 0" : "=&v"(c) : "v"(a), "v"(b));
  else asm volatile("v_mfma_f32_32x32x16_bf16 %0, %1, %2, 0" : "=&v"(c) : "v"(a), "v"(b));
}
// Outputs accumulate in accumulator registers that nothing else reads inside the loop; settle() covers what follows outside it.
template <bool WAIT> AMLA_DEV void mfma_value(f32x16 &c, bf16x8 a, bf16x8 b) {
  if constexpr (WAIT) asm volatile("s_nop 1\n\tv_mfma_f32_32x32x16_bf16 %0, %1, %2, %0" : "+a"(c) : "v"(a), "v"(b));
  else asm volatile("v_mfma_f32_32x32x16_bf16 %0, %1, %2, %0" : "+a"(c) : "v"(a), "v"(b));
}
AMLA_DEV i32x8 join(u32x2 a, u32x2 b, u32x2 c, u32x2 d) {
  return i32x8{(int)a.x, (int)a.y, (int)b.x, (int)b.y, (int)c.x, (int)c.y, (int)d.x, (int)d.y};
}
// A (32 x 64) B (64 x 32) of e4m3 codes, lane l holding 32 codes of row (column) l % 32, B times
// 2^(byte - 127) of the low byte of its scale: codes 0 - 15 of both lanes of a column are one block, scaled
// by the byte of lane l % 32, codes 16 - 31 the other, by that of lane l % 32 + 32.  one: 127.
template <bool WAIT> AMLA_DEV void mfma_value(f32x16 &c, i32x8 a, int one, i32x8 b, int bs) {
  if constexpr (WAIT)
    asm volatile("s_nop 1\n\tv_mfma_scale_f32_32x32x64_f8f6f4 %0, %1, %2, %0, %3, %4 op_sel_hi:[0,0,0]"
                 : "+a"(c) : "v"(a), "v"(b), "v"(one), "v"(bs));
  else
    asm volatile("v_mfma_scale_f32_32x32x64_f8f6f4 %0, %1, %2, %0, %3, %4 op_sel_hi:[0,0,0]"
                 : "+a"(c) : "v"(a), "v"(b), "v"(one), "v"(bs));
}
// Before vector code reads what the asm MFMAs above wrote, and before they read what it wrote.
template <int N> AMLA_DEV void settle(f32x16 (&o)[N]) {
  asm volatile("s_nop 7\n\ts_nop 7\n\ts_nop 7" ::: "memory");
#pragma unroll
  for (int c = 0; c < N; ++c) asm volatile("" : "+a"(o[c]));
}

AMLA_DEV int pk_fp8x4(float a, float b, float c, float d) {
  // (the first conversion's other half is written by the second: any register will do for it)
  const int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, __float_as_int(a), false);
  return __builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true);
}
AMLA_DEV int pk_fp8x4_16(float a, float b, float c, float d, float sixteenth) {  // of 16 times the values
  int w;  // (the builtin's vector of shorts made the compiler take unrelated registers apart, before they were loaded)
  asm("v_cvt_scalef32_pk_fp8_f32 %0, %1, %2, %3" : "=v"(w) : "v"(a), "v"(b), "v"(sixteenth));
  asm("v_cvt_scalef32_pk_fp8_f32 %0, %1, %2, %3 op_sel:[0,0,0,1]" : "+v"(w) : "v"(c), "v"(d), "v"(sixteenth));
  return w;
}
// x = hi + lo / 16 in e4m3, magnitudes up to 256: hi keeps four leading bits, lo the next four
AMLA_DEV void split_fp8x4(const float *x, float sixteenth, int &hi, int &lo) {
  hi = pk_fp8x4(x[0], x[1], x[2], x[3]);
  const f32x2 a = fp8x2_to_f32<false>(hi), b = fp8x2_to_f32<true>(hi);
  lo = pk_fp8x4_16(x[0] - a.x, x[1] - a.y, x[2] - b.x, x[3] - b.y, sixteenth);
}
// Eight codes times a power of two, exact in bf16
AMLA_DEV bf16x8 codes_to_bf16(uint32_t w0, uint32_t w1, float scale) {
  typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
  const bf16x2_t c0 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w0, scale, false);
  const bf16x2_t c1 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w0, scale, true);
  const bf16x2_t c2 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w1, scale, false);
  const bf16x2_t c3 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w1, scale, true);
  return bf16x8{c0[0], c0[1], c1[0], c1[1], c2[0], c2[1], c3[0], c3[1]};
}

// ---------------------------------------------------------------- copies
//
// A wave copies ROWS / 4 rows of each tile straight into LDS.  Lane L holds the pool row of row
// L % (ROWS / 4) in `slot` and those of rows 8 i + L / 8 in `pe` (below 0: row 0 of the pool is
// copied, its place cleared before use).
template <bool F8> struct Rows {
  static constexpr int WR = Tile<F8>::ROWS / 4, NPE = WR / 8, NLAT = F8 ? WR / 2 : WR, COPIES = NLAT + NPE;
  int slot, pe[NPE];
  AMLA_DEV void spread() {
    const int lane = fresh_lane();
#pragma unroll
    for (int i = 0; i < NPE; ++i) pe[i] = __builtin_amdgcn_ds_bpermute(4 * (8 * i + (lane >> 3)), slot);
  }
  // The shuffle ends before LDS operations are counted by hand.
  AMLA_DEV void landed() {
#pragma unroll
    for (int i = 0; i < NPE; ++i) asm volatile("" : "+v"(pe[i]));
  }
  // The lane's part of the source addresses.
  static AMLA_DEV uint2 lanes(int r0) {
    const int lane = fresh_lane();
    const uint32_t lat = F8 ? 16 * ((lane & 31) ^ Tile<F8>::swz(lane >> 5)) : 16 * (lane ^ Tile<F8>::swz(r0 & 15));
    const uint32_t pe = 16 * ((lane & 7) ^ ((r0 >> 1) & 7) ^ (lane >> 4));
    return uint2{lat, pe};
  }
  // copy I (0 .. COPIES - 1) into the stage at st, r0 = first row of the wave in it (a multiple of 8; the swizzles
  // are xors of bits of the row)
  template <int I> AMLA_DEV void copy(const LatentPages &pg, uint8_t *st, int r0, uint2 lanes) const {
    using T = Tile<F8>;
    const int lane = threadIdx.x & 63;
    if constexpr (I >= NLAT) {
      constexpr int k = I - NLAT;
      copy_lds_nt(reinterpret_cast<const uint8_t *>(pg.k_pe) + (size_t)max(pe[k], 0) * 128 + (lanes.y ^ (64 * k)),
                  st + Stage<F8>::PE + (r0 + 8 * k) * 128);
    } else if constexpr (F8) {  // two rows of 512 bytes
      const int s0 = __builtin_amdgcn_readlane(slot, 2 * I), s1 = __builtin_amdgcn_readlane(slot, 2 * I + 1);
      const int s = max(lane < 32 ? s0 : s1, 0);
      copy_lds_nt(pg.latent + (size_t)s * 512 + (lanes.x ^ (16 * T::swz(2 * I))), st + (r0 + 2 * I) * 512);
    } else {
      const size_t s = max(__builtin_amdgcn_readlane(slot, I), 0);
      copy_lds_nt(pg.latent + s * 1024 + (lanes.x ^ (16 * T::swz(I))), st + (r0 + I) * 1024);
    }
  }
};
template <bool F8, int I = 0> AMLA_DEV void copy_all(const Rows<F8> &rows, const LatentPages &pg, uint8_t *st, int r0) {
  if constexpr (I < Rows<F8>::COPIES) {
    rows.template copy<I>(pg, st, r0, Rows<F8>::lanes(r0));
    copy_all<F8, I + 1>(rows, pg, st, r0);
  }
}

// ---------------------------------------------------------------- the two phases of a tile

// Latent query fragment f: its place in LDS (one every third, or fifth, score step), -1: in registers.
template <bool F8> constexpr int q_place(int f) {
  const int every = F8 ? 6 : 10;
  return f % every == 1 && f / every < Stage<F8>::QL ? f / every : -1;
}
template <bool F8> constexpr int q_reg(int f) {
  int n = 0;
  for (int i = 0; i < f; ++i) n += q_place<F8>(i) < 0;
  return n;
}
static_assert(Stage<true>::LDS <= 160 * 1024 && Stage<false>::LDS <= 160 * 1024);

template <bool F8> struct Wave {
  static constexpr int KB = Tile<F8>::ROWS / 32;  // 32-row blocks of a tile
  static constexpr int NCB = 16;                  // 32-column blocks of a row
  bf16x8 q[32 - Stage<F8>::QL], qr[F8 ? 1 : 4];  // the rest at qra in LDS, 1 KB a fragment
  uint32_t qra;
  f32x16 o[NCB];  // O^T: columns x queries
  f32x16 s[2];    // S^T of the tile in work: rows x queries (bf16: two chains of the one block)
  i32x8 phi, plo; // P of the tile before it: e4m3 halves and their scale,
  int ps, ps_lo, one;
  u32x4 pb[2];    // or bf16
  float m, l, top;  // reference, sum of 2^(s - m), maximum so far
};

// Reads of score step I: two fragments, one of each chain of MFMAs.
template <bool F8, int I> AMLA_DEV void score_read(u32x4 (&d)[3], uint32_t kl, uint32_t kr, uint32_t qra) {
  constexpr int RB = Tile<F8>::RB;
  if constexpr (I >= 16) {  // the rope key, 16 columns a step: of rows j32, 32 + j32, or two steps of one row
    constexpr int ks = I - 16;
    d[0] = lds_read16<0>(kr ^ (F8 ? 32 * ks : 64 * ks));
    d[1] = F8 ? lds_read16<32 * 128>(kr ^ (32 * ks)) : lds_read16<0>(kr ^ (64 * ks + 32));
    if constexpr (F8) d[2] = lds_read16<1024 * (Stage<F8>::QL + ks)>(qra);
  } else if constexpr (F8) {  // codes 32 I + 16 hh .. + 15 of rows j32, 32 + j32
    d[0] = lds_read16<256 * (I >> 3)>(kl ^ (32 * (I & 7)));
    d[1] = lds_read16<256 * (I >> 3) + 32 * RB>(kl ^ (32 * (I & 7)));
  } else {  // values 32 I + 8 hh .. + 7, and those 16 on
    d[0] = lds_read16<256 * (I >> 2)>(kl ^ (32 * ((2 * I) & 7)));
    d[1] = lds_read16<256 * (I >> 2)>(kl ^ (32 * ((2 * I + 1) & 7)));
  }
  if constexpr (I < 16 && q_place<F8>(2 * I + 1) >= 0) d[2] = lds_read16<1024 * q_place<F8>(2 * I + 1)>(qra);
}

template <bool F8> constexpr int score_reads(int i) {
  return i >= 16 + (F8 ? 4 : 2) ? 0 : (i >= 16 ? F8 : q_place<F8>(2 * i + 1) >= 0) ? 3 : 2;
}
// Steps that reads go out ahead: as many as the registers allow (an LDS read returns after 300 - 400 cycles with
// four waves reading; two steps of bf16 are 128 cycles of products)
template <bool F8> constexpr int score_ahead() { return F8 ? 2 : 3; }
template <bool F8> constexpr int score_reads(int first, int last) {
  int n = 0;
  for (int i = first; i <= last; ++i) n += score_reads<F8>(i);
  return n;
}
template <bool F8, int N, int I = 0> AMLA_DEV void score_reads_first(u32x4 (*ka)[3], uint32_t kl, uint32_t kr, uint32_t qra) {
  if constexpr (I < N) {
    score_read<F8, I>(ka[I], kl, kr, qra);
    score_reads_first<F8, N, I + 1>(ka, kl, kr, qra);
  }
}

// x0, y0: the step's first fragments; e4m3: converted in the step before (a conversion of four instructions fits under each
// MFMA; all sixteen of a step in front of its four MFMAs cost 5900 cycles a tile, not 3900, and one right before the product
// that takes it two wait states each time)
template <bool F8, int I>
AMLA_DEV void score_step(Wave<F8> &w, u32x4 (&ka)[score_ahead<F8>() + 1][3], uint32_t kl, uint32_t kr, bf16x8 x0, bf16x8 y0,
                         float f0, float f1, uint2 lanes, const Rows<F8> &next, const LatentPages &pg, uint8_t *st_next, int r0) {
  constexpr int N = 16 + (F8 ? 4 : 2);  // steps over the latent and the rope key
  if constexpr (I < N) {
    constexpr int AHEAD = score_ahead<F8>(), c = I % (AHEAD + 1), n = (I + 1) % (AHEAD + 1);
    if constexpr (I + AHEAD < N) score_read<F8, I + AHEAD>(ka[(I + AHEAD) % (AHEAD + 1)], kl, kr, w.qra);
    constexpr int r0q = q_reg<F8>(I < 16 ? 2 * I : 0), r1q = q_reg<F8>(I < 16 ? 2 * I + 1 : 0);
    const bf16x8 qa = w.q[r0q], qb = score_reads<F8>(I) == 3 ? as_bf16x8(ka[c][2]) : w.q[r1q];
    bf16x8 xn = x0, yn = y0;
    if constexpr (I >= 16) {
      constexpr int k0 = F8 ? I - 16 : 2 * (I - 16), k1 = F8 ? k0 : k0 + 1;
      mfma_score<false>(w.s[0], x0, F8 ? qb : w.qr[F8 ? 0 : k0]);
      mfma_score<false>(w.s[1], y0, F8 ? qb : w.qr[F8 ? 0 : k1]);
    } else if constexpr (F8) {
      const u32x4 x = ka[c][0], y = ka[c][1];
      if constexpr (I == 0) mfma_score0<true>(w.s[0], x0, qa);
      else mfma_score<false>(w.s[0], x0, qa);
      const bf16x8 x1 = codes_to_bf16(x.z, x.w, f0);
      __builtin_amdgcn_sched_barrier(0);
      if constexpr (I == 0) mfma_score0<true>(w.s[1], y0, qa);
      else mfma_score<false>(w.s[1], y0, qa);
      const bf16x8 y1 = codes_to_bf16(y.z, y.w, f1);
      __builtin_amdgcn_sched_barrier(0);
      mfma_score<false>(w.s[0], x1, qb);
      if constexpr (I + 1 < N) {
        lds_wait<score_reads<F8>(I + 2, I + AHEAD)>();
        lds_tie(ka[n][0], ka[n][1]);
        if constexpr (score_reads<F8>(I + 1) == 3) lds_tie(ka[n][2]);
        xn = I + 1 < 16 ? codes_to_bf16(ka[n][0].x, ka[n][0].y, f0) : as_bf16x8(ka[n][0]);
      }
      __builtin_amdgcn_sched_barrier(0);
      mfma_score<false>(w.s[1], y1, qb);
      if constexpr (I + 1 < N) yn = I + 1 < 16 ? codes_to_bf16(ka[n][1].x, ka[n][1].y, f1) : as_bf16x8(ka[n][1]);
    } else if constexpr (I == 0) {
      mfma_score0<true>(w.s[0], x0, qa);
      mfma_score0<true>(w.s[1], y0, qb);
    } else {
      mfma_score<false>(w.s[0], x0, qa);
      mfma_score<false>(w.s[1], y0, qb);
    }
    if constexpr (I > 0 && I <= Rows<F8>::COPIES) next.template copy<I - 1>(pg, st_next, r0, lanes);
    if constexpr (I + 1 < N && (!F8 || I >= 16)) {
      lds_wait<score_reads<F8>(I + 2, I + AHEAD)>();
      lds_tie(ka[n][0], ka[n][1]);
      if constexpr (score_reads<F8>(I + 1) == 3) lds_tie(ka[n][2]);
      xn = as_bf16x8(ka[n][0]);
      yn = as_bf16x8(ka[n][1]);
    }
    __builtin_amdgcn_sched_barrier(0);
    score_step<F8, I + 1>(w, ka, kl, kr, xn, yn, f0, f1, lanes, next, pg, st_next, r0);
  }
}

// S^T of the tile whose stage is at LDS address base, with the copies of a later tile spread between.
// Two chains of MFMAs: one alone runs at two thirds of the rate.
template <bool F8>
AMLA_DEV void score_phase(Wave<F8> &w, uint32_t base, const Rows<F8> &next, const LatentPages &pg, uint8_t *st_next,
                          int r0) {
  using T = Tile<F8>;
  using G = Stage<F8>;
  const int lane = fresh_lane(), j32 = lane & 31, hh = lane >> 5;
  // the lane's row and first chunk; chunk c sits at c ^ swz(row): bits 1 .. 3 of c enter by xor, higher ones by offset
  const uint32_t kl = base + j32 * T::RB + 16 * (hh ^ T::swz(j32));
  const uint32_t kr = base + G::PE + j32 * 128 + 16 * (hh ^ ((j32 >> 1) & 7));
  float f0 = 1.f, f1 = 1.f;
  if constexpr (F8) {  // 2^exponent of rows j32 and 32 + j32
    asm volatile("ds_read_b32 %0, %1 offset:%2" : "=v"(f0) : "v"(base + 4 * j32), "i"(G::MUL) : "memory");
    asm volatile("ds_read_b32 %0, %1 offset:%2" : "=v"(f1) : "v"(base + 4 * j32), "i"(G::MUL + 128) : "memory");
  }
  constexpr int AHEAD = score_ahead<F8>();
  u32x4 ka[AHEAD + 1][3];
  score_reads_first<F8, AHEAD>(ka, kl, kr, w.qra);
  lds_wait<score_reads<F8>(1, AHEAD - 1)>();
  lds_tie(f0, f1, ka[0][0], ka[0][1]);
  if constexpr (score_reads<F8>(0) == 3) lds_tie(ka[0][2]);
  const bf16x8 x0 = F8 ? codes_to_bf16(ka[0][0].x, ka[0][0].y, f0) : as_bf16x8(ka[0][0]);
  const bf16x8 y0 = F8 ? codes_to_bf16(ka[0][1].x, ka[0][1].y, f1) : as_bf16x8(ka[0][1]);
  score_step<F8, 0>(w, ka, kl, kr, x0, y0, f0, f1, Rows<F8>::lanes(r0), next, pg, st_next, r0);
  // the results are read by vector code that the compiler schedules: cover the asm's write-to-read wait states
  asm volatile("s_nop 7\n\ts_nop 7\n\ts_nop 7" : "+v"(w.s[0]), "+v"(w.s[1])::"memory");
}

// The second phase of a tile goes in steps of one 32-column block of the values; each carries some of the
// slices (four rows) of the softmax: first all scaled scores and their maxima, then the probabilities.
template <bool F8> struct Slices {
  static constexpr int KB = Wave<F8>::KB, NCB = Wave<F8>::NCB, NZ = 4 * KB, NS = 8 * KB;
  static constexpr int PER = (NS + NCB - 1) / NCB;  // slices of a step, at most
  static constexpr int first(int c) { return (c * NS + NCB - 1) / NCB; }
  static constexpr int reads(int c) {  // row factors read for step c: bf16's probabilities need none
    if (c >= NCB) return 0;
    int n = 0;
    for (int s = first(c); s < first(c + 1); ++s) n += s < NZ || F8;
    return n;
  }
};
template <bool F8> struct StepReads {
  u32x2 v[4];
  u32x4 ex[Slices<F8>::PER];
};
constexpr int VALUE_AHEAD = 2;
template <bool F8> struct ValueState {
  static constexpr int KB = Wave<F8>::KB;
  uint32_t v0, v1, eb;
  float scale_log2;
  int lim;  // MASK: rows of the tile below lim are seen by the lane's query
  float mx[KB], ref[KB], sum[KB];
  i32x8 phi, plo;
  u32x4 pb[2];
  StepReads<F8> rd[VALUE_AHEAD + 1];
};

template <bool F8, int S, int END, int K = 0> AMLA_DEV void slice_read(ValueState<F8> &x, StepReads<F8> &r) {
  using G = Stage<F8>;
  using L = Slices<F8>;
  if constexpr (S < END) {
    constexpr int t = S % L::NZ;
    if constexpr (S < L::NZ || F8) r.ex[K] = lds_read16<(S < L::NZ ? G::EXP : G::INV) + 4 * (32 * (t >> 2) + 8 * (t & 3))>(x.eb);
    slice_read<F8, S + 1, END, K + 1>(x, r);
  }
}
template <bool F8, bool ZP, int C> AMLA_DEV void value_read(ValueState<F8> &x) {
  using L = Slices<F8>;
  if constexpr (C < L::NCB) {
    StepReads<F8> &r = x.rd[C % (VALUE_AHEAD + 1)];
    if constexpr (F8) {
      const uint32_t a = x.v0 ^ (32 * (C & 7));
      r.v[0] = lds_read_tr<F8, 256 * (C >> 3)>(a);
      r.v[1] = lds_read_tr<F8, 256 * (C >> 3) + 8192>(a);
      r.v[2] = lds_read_tr<F8, 256 * (C >> 3) + 16384>(a);
      r.v[3] = lds_read_tr<F8, 256 * (C >> 3) + 24576>(a);
    } else {
      const uint32_t a = x.v0 ^ (64 * (C & 3)), b = x.v1 ^ (64 * (C & 3));
      r.v[0] = lds_read_tr<F8, 256 * (C >> 2)>(a);
      r.v[1] = lds_read_tr<F8, 256 * (C >> 2)>(b);
      r.v[2] = lds_read_tr<F8, 256 * (C >> 2) + 16384>(a);
      r.v[3] = lds_read_tr<F8, 256 * (C >> 2) + 16384>(b);
    }
    if constexpr (ZP) slice_read<F8, L::first(C), L::first(C + 1)>(x, r);
  }
}

// The reference of a block of e4m3 probabilities, whose largest score is mx: m plus a whole number, so that the block's scale
// is a power of two, and 2^(mx - ref) in 128 .. 256 (m's own row: 128, without rounding).  From mx, not m + floor(mx - m) - 7:
// beyond 2^27 the rounding of that sum alone is more than e4m3 has room for, beyond 2^29 more than an exponential has.
AMLA_DEV float block_ref(float mx, float m) {
  mx = __builtin_fmaxf(mx, M_NONE);
  return mx - (__builtin_amdgcn_fractf(mx - m) + 7.f);
}
// Its scale for the matrix unit: 2^(ref - m), whole but for the rounding of ref
AMLA_DEV int block_scale(float ref, float m) { return (int)__builtin_rintf(__builtin_fmaxf(ref - m, -123.f)) + 127; }
// Slice S of the softmax, its row factors in ex:
//   z = s log2(e) scale + exponent of the row, P = 2^(z - ref), l sums 2^(s - m) = P 2^(ref - m - exponent)
// e4m3: 32 rows are one block of the matrix unit with a scale of its own, 2^(ref - m), so that rows far
// below the sequence's maximum keep their bits: a reference for all would drop those below 2^-22 of it,
// and thousands of them can outweigh it.
template <bool F8, bool MASK, int S> AMLA_DEV void softmax_slice(Wave<F8> &w, ValueState<F8> &x, u32x4 ex) {
  using L = Slices<F8>;
  constexpr int KB = L::KB, t = S % L::NZ, kb = t >> 2, q4 = t & 3;
  f32x16 &z = w.s[kb];
  if constexpr (S < L::NZ) {
    if constexpr (q4 == 0) x.mx[kb] = -INFINITY;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float sc = F8 ? z[4 * q4 + i] : z[4 * q4 + i] + w.s[1][4 * q4 + i];
      z[4 * q4 + i] = __builtin_fmaf(sc, x.scale_log2, __uint_as_float(ex[i]));
    }
    if constexpr (MASK) {
#pragma unroll
      for (int i = 0; i < 4; ++i) z[4 * q4 + i] = 32 * kb + 8 * q4 + i < x.lim ? z[4 * q4 + i] : -INFINITY;
    }
    x.mx[kb] = __builtin_fmaxf(__builtin_fmaxf(x.mx[kb], z[4 * q4]), z[4 * q4 + 1]);
    x.mx[kb] = __builtin_fmaxf(__builtin_fmaxf(x.mx[kb], z[4 * q4 + 2]), z[4 * q4 + 3]);
    if constexpr (S == L::NZ - 1) {
#pragma unroll
      for (int k = 0; k < KB; ++k) {
        const auto sw = __builtin_amdgcn_permlane32_swap(__float_as_uint(x.mx[k]), __float_as_uint(x.mx[k]), false, false);
        x.mx[k] = __builtin_fmaxf(__uint_as_float(sw[0]), __uint_as_float(sw[1]));
      }
      const float top = __builtin_fmaxf(x.mx[0], x.mx[KB - 1]);
      w.top = __builtin_fmaxf(w.top, top);
      w.m = w.m == M_NONE ? __builtin_fmaxf(top, M_NONE) : w.m;
#pragma unroll
      for (int k = 0; k < KB; ++k) {
        x.ref[k] = F8 ? block_ref(x.mx[k], w.m) : w.m;
        x.sum[k] = 0.f;
      }
    }
  } else {
    float e[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) e[i] = __builtin_amdgcn_exp2f(z[4 * q4 + i] - x.ref[kb]);
    if constexpr (F8) {
#pragma unroll
      for (int i = 0; i < 4; ++i) x.sum[kb] = __builtin_fmaf(e[i], __uint_as_float(ex[i]), x.sum[kb]);
      asm volatile("" : "+v"(x.sum[kb]));  // (here: left to itself the compiler sums up at the end, and keeps all terms until then)
      int hi, lo;
      split_fp8x4(e, 0.0625f, hi, lo);
      x.phi[4 * kb + q4] = hi;
      x.plo[4 * kb + q4] = lo;
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) x.sum[kb] += e[i];
      asm volatile("" : "+v"(x.sum[kb]));
      x.pb[q4 >> 1][2 * (q4 & 1)] = pack_bf16(e[0], e[1]);
      x.pb[q4 >> 1][2 * (q4 & 1) + 1] = pack_bf16(e[2], e[3]);
    }
  }
}
template <bool F8, bool MASK, int S, int END, int K = 0>
AMLA_DEV void softmax_slices(Wave<F8> &w, ValueState<F8> &x, StepReads<F8> &r) {
  if constexpr (S < END) {
    u32x4 ex = {0, 0, 0, 0};
    if constexpr (S < Slices<F8>::NZ || F8) {
      ex = r.ex[K];
      lds_tie(ex);
    }
    softmax_slice<F8, MASK, S>(w, x, ex);
    softmax_slices<F8, MASK, S + 1, END, K + 1>(w, x, r);
  }
}

template <bool F8, bool MASK, bool ZP, int C>
AMLA_DEV void value_step(Wave<F8> &w, ValueState<F8> &x) {
  using L = Slices<F8>;
  if constexpr (C < L::NCB) {
    StepReads<F8> &r = x.rd[C % (VALUE_AHEAD + 1)];
    value_read<F8, ZP, C + VALUE_AHEAD>(x);
    // this step's reads have landed: those of the next two steps may be in flight
    lds_wait<4 * ((C + 1 < L::NCB) + (C + 2 < L::NCB)) + (ZP ? L::reads(C + 1) + L::reads(C + 2) : 0)>();
    // (locals, not members: a pass that sees the members in memory loads several at once, and then takes registers
    // apart that are still being loaded)
    u32x2 v0 = r.v[0], v1 = r.v[1], v2 = r.v[2], v3 = r.v[3];
    lds_tie(v0, v1, v2, v3);
    if constexpr (F8) mfma_value<false>(w.o[C], join(v0, v1, v2, v3), w.one, w.phi, w.ps);
    else mfma_value<false>(w.o[C], as_bf16x8(u32x4{v0.x, v0.y, v1.x, v1.y}), as_bf16x8(w.pb[0]));
    if constexpr (ZP) softmax_slices<F8, MASK, L::first(C), L::first(C + 1)>(w, x, r);
    if constexpr (F8) mfma_value<false>(w.o[C], join(v0, v1, v2, v3), w.one, w.plo, w.ps_lo);
    else mfma_value<false>(w.o[C], as_bf16x8(u32x4{v2.x, v2.y, v3.x, v3.y}), as_bf16x8(w.pb[1]));
    __builtin_amdgcn_sched_barrier(0);
    value_step<F8, MASK, ZP, C + 1>(w, x);
  }
}

// O^T += C^T P^T of the tile before (its stage at pv) while the scores of this tile (stage at zb; ZP) become
// probabilities.
template <bool F8, bool MASK, bool ZP>
AMLA_DEV void value_phase(Wave<F8> &w, uint32_t pv, uint32_t zb, float scale_log2, int lim) {
  using T = Tile<F8>;
  using L = Slices<F8>;
  constexpr int KB = L::KB;
  const int lane = fresh_lane(), hh = lane >> 5, L16 = lane & 15, g16 = lane >> 4;
  ValueState<F8> x;
  if constexpr (F8) {  // rows 16 i + 4 hh + {0..3, 8..11} of 16 columns
    const int r = 8 * (L16 >> 3) + 4 * hh + ((L16 >> 1) & 3);
    x.v0 = pv + r * T::RB + 16 * ((g16 & 1) ^ T::swz(r)) + 8 * (L16 & 1);
  } else {   // rows 16 kk + 8 i + 4 hh + 0..3
    const int r = 4 * hh + (L16 >> 2), ch = 2 * (g16 & 1) + ((L16 >> 1) & 1);
    x.v0 = pv + r * T::RB + 16 * (ch ^ T::swz(r)) + 8 * (L16 & 1);
    x.v1 = pv + (r + 8) * T::RB + 16 * (ch ^ T::swz(r + 8)) + 8 * (L16 & 1);
  }
  x.eb = zb + 16 * hh;
  x.scale_log2 = scale_log2;
  x.lim = lim;
  value_read<F8, ZP, 0>(x);
  value_read<F8, ZP, 1>(x);
  value_step<F8, MASK, ZP, 0>(w, x);
  if constexpr (ZP) {
#pragma unroll
    for (int k = 0; k < KB; ++k) w.l += F8 ? x.sum[k] * __builtin_amdgcn_exp2f(x.ref[k] - w.m) : x.sum[k];
    // the scale of block k comes from the lanes of half k; 4 .. 180 (more only in a pass that is made again), the low
    // halves' 4 less
    if constexpr (F8) {
      w.ps = block_scale(hh ? x.ref[KB - 1] : x.ref[0], w.m);
      w.ps_lo = w.ps - 4;
    }
    w.phi = x.phi;
    w.plo = x.plo;
    w.pb[0] = x.pb[0];
    w.pb[1] = x.pb[1];
  }
}

// The copies of a split: which rows of the pool a wave brings, and what is known of those under way.
template <bool F8> struct Feed {
  static constexpr int TILE = Tile<F8>::ROWS, NST = Tile<F8>::STAGES, PD = NST - 2;  // a tile, the one before it, PD to come
  static constexpr int WR = Rows<F8>::WR, COPIES = Rows<F8>::COPIES;
  const LatentPages &pg;
  uint8_t *sm;
  int b, wave, held, last, cur;  // last: rows past it are copied from it (and have no part in anything)
  Rows<F8> next;     // the tile that goes out next
  int page;          // the table's entry for the lane's row of the tile after it
  int tail = 0;      // the newest rows that some token does not see
  int odd = INT32_MAX;  // the first of them with a value that is no number
  int byte[PD + 1];  // the row's exponent, -1 where it has no page; [0]: the tile in work, [PD]: the one going out

  AMLA_DEV int row_of(int tile) const { return min(tile * TILE + WR * wave + fresh_lane() % WR, last); }
  AMLA_DEV int byte_of(int slot) const {
    int v = 127;
    if constexpr (F8) v = pg.scales[max(slot, 0)];
    return slot < 0 ? -1 : v;
  }
  // Rows of the pool for the tile that goes out after `tile`, from the page loaded before; the page of the one behind it.
  // (Each is loaded a tile ahead of its use: a load waits for every copy before it.)
  AMLA_DEV void prepare(int tile) {
    next.slot = pg.row(page, row_of(tile + 1));
    next.spread();
    byte[PD] = byte_of(next.slot);
    page = pg.page(b, row_of(tile + 2));
  }
  // Factors of the rows of tile `tile`, the next in work, beside where they are landing
  AMLA_DEV void factors(int tile) {
    using G = Stage<F8>;
    uint8_t *st = sm + cur * G::SIZE;
    const int lane = fresh_lane();
    if (lane < WR) {
      const int r = WR * wave + lane;
      const bool gone = byte[0] < 0 || tile * TILE + r >= held;
      const int by = gone ? 127 : byte[0];
      *reinterpret_cast<float *>(st + G::EXP + 4 * r) = gone ? -INFINITY : (float)(by - 127);
      if constexpr (F8) {
        *reinterpret_cast<uint32_t *>(st + G::INV + 4 * r) = by == 255 ? 0x00200000u : (uint32_t)(254 - by) << 23;
        *reinterpret_cast<uint32_t *>(st + G::MUL + 4 * r) = by == 255 ? 0x7fc00000u : (uint32_t)by << 23;
      }
    }
  }
  AMLA_DEV void start(int t_first) {
    cur = 0;
    Rows<F8> r[PD];
#pragma unroll
    for (int d = 0; d < PD; ++d) r[d].slot = pg.page(b, row_of(t_first + d));
    page = pg.page(b, row_of(t_first + PD));
#pragma unroll
    for (int d = 0; d < PD; ++d) {
      r[d].slot = pg.row(r[d].slot, row_of(t_first + d));
      r[d].spread();
    }
#pragma unroll
    for (int d = 0; d < PD; ++d) byte[d] = byte_of(r[d].slot);
#pragma unroll
    for (int d = 0; d < PD; ++d) copy_all<F8>(r[d], pg, sm + d * Stage<F8>::SIZE, WR * wave);
    asm volatile("" ::: "memory");
    prepare(t_first + PD - 1);
    factors(t_first);
  }
  // The rows of tile `tile` have landed in every wave
  template <bool MASK> AMLA_DEV void arrive(int tile) {
    using G = Stage<F8>;
    constexpr int RB = Tile<F8>::RB, LOADS = F8 ? 2 : 1;
    const int lane = threadIdx.x & 63;
    // behind its copies: those of PD - 1 tiles, and prepare()'s loads
    wait_vmcnt<(PD - 1) * COPIES + LOADS>();
    uint8_t *st = sm + cur * G::SIZE;
    // rows of no page or past the end: zeros in place of what was copied (a NaN there would come through 0 * NaN)
    const bool gone = lane < WR && (byte[0] < 0 || tile * TILE + WR * wave + lane >= held);
    for (uint64_t bad = __ballot(gone); bad; bad &= bad - 1) {
      const int r = WR * wave + __builtin_ctzll(bad);
      for (int i = lane; i < RB / 16; i += 64) *reinterpret_cast<u32x4 *>(st + r * RB + 16 * i) = u32x4{0, 0, 0, 0};
      if (lane < 8) *reinterpret_cast<u32x4 *>(st + G::PE + r * 128 + 16 * lane) = u32x4{0, 0, 0, 0};
    }
    if constexpr (MASK) {
      // rows that some token does not see: one with an infinity or a NaN becomes zeros too, and the tokens that do see it
      // get their NaN at the end
      const int end = min(held - tile * TILE - WR * wave, WR);
      for (int r = max(held - tail - tile * TILE - WR * wave, 0); r < end; ++r) {
        u32x4 *at = reinterpret_cast<u32x4 *>(st + (WR * wave + r) * RB + 16 * (lane % (RB / 16)));
        const u32x4 v = *at;
        bool bad = false;
#pragma unroll
        for (int k = 0; k < 4; ++k)
          bad |= F8 ? (((v[k] & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) != 0
                    : (((v[k] & 0x7f807f80u) + 0x00800080u) & 0x80008000u) != 0;
        if (!__ballot(bad) && __builtin_amdgcn_readlane(byte[0], r) != 255) continue;
        *at = u32x4{0, 0, 0, 0};
        odd = min(odd, tile * TILE + WR * wave + r);
      }
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    next.landed();
    asm volatile("" ::: "memory");
  }
  AMLA_DEV uint8_t *next_stage() const { return sm + (cur + PD) % NST * Stage<F8>::SIZE; }
  // After tile `tile`: `next` went out during it
  AMLA_DEV void advance(int tile) {
#pragma unroll
    for (int d = 0; d < PD; ++d) byte[d] = byte[d + 1];
    cur = cur + 1 == NST ? 0 : cur + 1;
    prepare(tile + PD);
    factors(tile + 1);
  }
};

// A wave's sums times inv as rows in LDS: of 16 NCB values in each lane's row, chunk c of 16 bytes at c ^ row
template <bool F16, int NCB> AMLA_DEV void turn_rows(uint8_t *turn, const f32x16 (&o)[NCB], float inv) {
  const int lane = threadIdx.x & 63, j32 = lane & 31, hh = lane >> 5;
#pragma unroll
  for (int c = 0; c < NCB; ++c)
#pragma unroll
    for (int q4 = 0; q4 < 4; ++q4) {
      float x[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] = o[c][4 * q4 + i] * inv;
      *reinterpret_cast<u32x2 *>(turn + j32 * 64 * NCB + 16 * ((4 * c + q4) ^ (j32 % (4 * NCB))) + 8 * hh) =
          F16 ? u32x2{pack_f16(x[0], x[1]), pack_f16(x[2], x[3])} : u32x2{pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3])};
    }
}
// A split's sums, normalised: the output itself, or a partial one.  l, m: of the lane's query row (l = 0: it sees no row).
// GROUPS: 32-row groups of a workgroup; hg: this one, cg: the wave's of 16 / NCB column groups.
template <int GROUPS, int NCB>
AMLA_DEV void store_split(LatentAttnParams p, uint8_t *sm, const f32x16 (&o)[NCB], float l, float m, int b, int chunk, int slot,
                          int splits, int wave, int hg, int cg) {
  constexpr int HG = GROUPS, CG = 16 / NCB;
  const int lane = threadIdx.x & 63, j32 = lane & 31, hh = lane >> 5;
  const int row = (chunk * HG + hg) * 32 + j32;
  float inv = l == 0.f ? 0.f : 1.f / l;
  const float lse2 = l == 0.f ? -INFINITY : m + __builtin_amdgcn_logf(l);
  float scale = 1.f;
  // The largest of the row's values in this wave to 2^14 .. 2^15, or as near as inv times that power stays finite: all of them
  // may be 0 where l is far below 1 (it sums 2^(s - m), and m has the exponent of an e4m3 row in it: down to 2^-32).
  if (splits > 1) {
    float top = 0.f;
#pragma unroll
    for (int c = 0; c < NCB; ++c)
#pragma unroll
      for (int i = 0; i < 16; ++i) top = __builtin_fmaxf(top, __builtin_fabsf(o[c][i]));
    const auto sw = __builtin_amdgcn_permlane32_swap(__float_as_uint(top), __float_as_uint(top), false, false);
    top = __builtin_fmaxf(__uint_as_float(sw[0]), __uint_as_float(sw[1])) * inv;
    const int least = max((int)(__float_as_uint(inv) >> 23) - 112, 15);                       // biased; below it: zeros nearly
    const int e = min(max((int)(__float_as_uint(top) >> 23), least), 240);
    scale = __uint_as_float((uint32_t)(e - 14) << 23);                   // 2^(e - 127 - 14)
    inv *= __uint_as_float((uint32_t)(254 - (e - 14)) << 23);
  }
  // rows of 1 KB / CG through LDS, so that a store is whole lines
  constexpr int RBYTES = 1024 / CG;
  uint8_t *turn = sm + wave * 32 * RBYTES;
  if (splits > 1) turn_rows<true>(turn, o, inv);
  else turn_rows<false>(turn, o, inv);
  if (l == 0.f) {  // no row is seen (sees_none)
    for (int i = 0; i < RBYTES / 2; i += 8) *reinterpret_cast<u32x2 *>(turn + j32 * RBYTES + RBYTES / 2 * hh + i) = u32x2{0, 0};
  }
  const int row0 = (chunk * HG + hg) * 32, held = min(32, p.rows - row0);
  const size_t dst0 = splits == 1 ? (size_t)b * p.rows + row0 : (size_t)slot * (32 * HG) + 32 * hg;
  uint16_t *to[2] = {p.part_o, p.out};
  asm volatile("" : "+s"(to[0]), "+s"(to[1]));  // (a choice between the two arguments' places would be made in scratch memory)
  uint8_t *od = reinterpret_cast<uint8_t *>((splits == 1 ? to[1] : to[0]) + dst0 * LC_LORA) + cg * RBYTES;
  constexpr int LPR = RBYTES / 16;  // lanes of a row
#pragma unroll 4
  for (int r0 = 0; r0 < held; r0 += CG) {
    const int r = r0 + lane / LPR, c = lane % LPR;
    if (r < held)
      *reinterpret_cast<u32x4 *>(od + (size_t)r * (LC_LORA * 2) + 16 * c) =
          *reinterpret_cast<const u32x4 *>(turn + r * RBYTES + 16 * (c ^ (r % (4 * NCB))));
  }
  if (splits > 1 && hh == 0 && row < p.rows) p.part_scale[(dst0 + j32) * 4 + cg] = scale;
  if (cg == 0 && hh == 0 && row < p.rows) {
    if (splits > 1) p.part_lse[dst0 + j32] = lse2;
    else if (p.lse) p.lse[dst0 + j32] = lse2 * 0.6931471805599453f;
  }
}

// The work of a workgroup: its split of a sequence.
struct SplitWork {
  int b, chunk, slot, splits, held, t_first, t_end;  // b < 0: none
};
template <bool F8> AMLA_DEV SplitWork split_work(const LatentAttnParams &p) {
  constexpr int TILE = Tile<F8>::ROWS;
  const SplitPlan<TILE> plan(p);
  // workgroup i runs on XCD i % 8: each takes a run of slots, so that a sequence's queries come from its L2
  const int per_xcd = lc_ceil_div(plan.used(plan.len), 8), slot = (int)(blockIdx.x & 7) * per_xcd + (int)(blockIdx.x >> 3);
  const int3 at = plan.find(slot);
  if ((int)(blockIdx.x >> 3) >= per_xcd || at.x < 0) return SplitWork{-1, 0, 0, 0, 0, 0, 0};
  if (slot == at.y && threadIdx.x == 0) p.part_plan[at.x] = int2{at.y, at.z};
  const int split = (slot - at.y) % at.z, held = __builtin_amdgcn_readfirstlane(min(max(p.lengths[at.x], 0), p.cap));
  const int n_tiles = lc_ceil_div(held, TILE);
  return SplitWork{at.x, (slot - at.y) / at.z, slot, at.z, held, (int)((int64_t)split * n_tiles / at.z),
                   (int)((int64_t)(split + 1) * n_tiles / at.z)};
}
// Whether a token of the split, which sees rows below lim, sees none.  Asked where its sum is NaN: a query that is no number
// times the zeros of absent rows is NaN too (their scores have -inf added, not put in their place: that would be two
// instructions more for each), but what has no rows gives zeros.
template <int TILE> AMLA_DEV bool sees_none(const LatentPages &pg, const SplitWork &at, int lim) {
  const int end = min(at.held, at.t_end * TILE);
  for (int t = at.t_first * TILE; t < end; t += 64) {
    const int r = t + (int)(threadIdx.x & 63);
    const uint64_t there = __ballot(r < end && pg.slot(at.b, r) >= 0);
    if (there) return t + __builtin_ctzll(there) >= lim;
  }
  return true;
}

// One workgroup of four waves per (sequence, chunk of 128 rows, split): a wave holds 32
// query rows, all of whose columns it sums up.  O^T fills half of its 512 registers, the queries
// most of the others: one wave a SIMD, whose own products hide its conversions, copies, LDS
// reads and softmax, each placed between two of them (one phase after the other took twice
// as long).  What spills in the loop costs most: a reload waits behind all copies under way.
template <bool F8, bool MASK>
__global__ __launch_bounds__(256, 1) void latent_attn_kernel(LatentAttnParams p) {
  extern __shared__ __align__(1024) uint8_t sm[];
  using T = Tile<F8>;
  using G = Stage<F8>;
  using W = Wave<F8>;
  constexpr int TILE = T::ROWS, NCB = W::NCB;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int j32 = lane & 31, hh = lane >> 5;

  const SplitWork at = split_work<F8>(p);
  if (at.b < 0) return;
  const int b = at.b, chunk = at.chunk, slot = at.slot, splits = at.splits, rows_held = at.held;
  const int t_first = at.t_first, t_end = at.t_end;
  const uint32_t lds0 = (uint32_t)reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) const uint8_t *)sm);

  Feed<F8> feed{p.pg, sm, b, wave, rows_held, min(rows_held, t_end * TILE) - 1};
  if constexpr (MASK) feed.tail = p.seq_len - 1;
  feed.start(t_first);

  // queries: B fragments, lane = row of the chunk, in the order of the score steps' reads
  W w;
  const int row = (chunk * 4 + wave) * 32 + j32;
  const int rq = min(row, p.rows - 1), tok = rq / p.heads;
  const int limit = rows_held - (p.seq_len - 1 - tok) - 4 * hh;  // rows [0, limit + 4 hh) are seen
  const uint16_t *qp = p.q + b * p.ldq_seq + tok * p.ldq_token + (rq - tok * p.heads) * p.ldq_head;
  uint8_t *const ql = sm + G::Q + 1024 * G::QF * wave + 16 * lane;
  w.qra = lds0 + G::Q + 1024 * G::QF * wave + 16 * lane;
#pragma unroll
  for (int i = 0; i < 32; ++i) {
    const u32x4 v = ldg16(qp + (F8 ? 32 * (i >> 1) + 16 * hh + 8 * (i & 1) : 16 * i + 8 * hh));
    if (q_place<F8>(i) >= 0) *reinterpret_cast<u32x4 *>(ql + 1024 * q_place<F8>(i)) = v;  // (the wave's own place)
    else w.q[q_reg<F8>(i)] = as_bf16x8(v);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const u32x4 v = ldg16(qp + LC_LORA + 16 * i + 8 * hh);
    if constexpr (F8) *reinterpret_cast<u32x4 *>(ql + 1024 * (G::QL + i)) = v;
    else w.qr[i] = as_bf16x8(v);
  }
  w.m = M_NONE;
  w.one = 127;
  for (;;) {  // once, or twice where m turned out too low
#pragma unroll
    for (int c = 0; c < NCB; ++c)
#pragma unroll
      for (int i = 0; i < 16; ++i) w.o[c][i] = 0.f;
    settle(w.o);
    w.l = 0.f;
    w.top = -INFINITY;
    // nothing before the first tile: probabilities of 0 times its own values, which saves a second copy of the loop's code
#pragma unroll
    for (int i = 0; i < 8; ++i) w.phi[i] = w.plo[i] = 0;
    w.pb[0] = w.pb[1] = u32x4{0, 0, 0, 0};
    w.ps = w.ps_lo = 127;
    uint32_t base = lds0;
    for (int tile = t_first; tile < t_end; ++tile) {
      const uint32_t before = base;
      feed.template arrive<MASK>(tile);
      base = lds0 + feed.cur * G::SIZE;
      score_phase<F8>(w, base, feed.next, p.pg, feed.next_stage(), Rows<F8>::WR * wave);
      value_phase<F8, MASK, true>(w, before, base, p.scale_log2, limit - tile * TILE);
      feed.advance(tile);
    }
    value_phase<F8, MASK, false>(w, base, base, p.scale_log2, 0);
    settle(w.o);
    wait_vmcnt<0>();  // (copies past the last tile)
    const bool low = w.top > w.m + LAG;
    // the waves agree: their copies and barriers are common
    __syncthreads();
    uint32_t *vote = reinterpret_cast<uint32_t *>(sm);
    const bool any_low = __ballot(low) != 0;
    if (lane == 0) {
      vote[wave] = any_low;
      if constexpr (MASK) vote[4 + wave] = (uint32_t)feed.odd;
    }
    __syncthreads();
    const bool again = (vote[0] | vote[1] | vote[2] | vote[3]) != 0;
    if constexpr (MASK) feed.odd = (int)min(min(vote[4], vote[5]), min(vote[6], vote[7]));
    __syncthreads();
    if (!again) break;
    w.m = low ? w.top : w.m;
    feed.start(t_first);
  }

  float l = w.l;
  l += __shfl_xor(l, 32, 64);
  if constexpr (MASK) l = feed.odd < limit + 4 * hh ? __uint_as_float(0x7fc00000u) : l;
  if (__ballot(l != l)) l = sees_none<TILE>(p.pg, at, MASK ? limit + 4 * hh : INT32_MAX) ? 0.f : l;
  store_split<4>(p, sm, w.o, l, w.m, b, chunk, slot, splits, wave, wave, 0);
}

// ---------------------------------------------------------------- few query rows
//
// One workgroup per (sequence, 32 or 64 query rows, split).  Wave (r, q) scores one half of a tile's rows for half of the
// queries with 16x16x32 products and writes its probabilities to LDS; a tile later, behind the barrier that the tiles have
// anyway, each wave takes all of them for its 128 columns.  So a tile's keys are read, and e4m3 converted, twice, and its
// values once, where four waves that each hold the outputs of some queries and columns read them four times: with 16 heads
// that took 90 us for 40 ragged sequences, not 69, with 32 heads and two tokens (8 x 17540 rows, bf16) 62, not 52.
template <bool F8, int QG> struct FewStage {
  using G = Stage<F8>;
  // probabilities as the value products take them, 16 bytes a lane: bf16: rows 16 k ..; e4m3: high halves, low halves, the
  // scales of both blocks.  Two buffers: a tile's are read while the next one's are written.
  static constexpr int LO = 2048, PS = 4096, PGRP = F8 ? 4352 : 2048, PBUF = QG * PGRP, P = G::Q;
  static constexpr int TOP = P + 2 * PBUF, M = TOP + 256 * QG, SUM = M + 128 * QG, ODD = SUM + 256 * QG, LIM = ODD + 16,
                       LDS = LIM + 128 * QG;
};
static_assert(FewStage<true, 2>::LDS <= 160 * 1024 && FewStage<false, 2>::LDS <= 160 * 1024);

template <bool F8> struct FewSteps {
  static constexpr int N = F8 ? 10 : 18, READS = F8 ? 2 : 1, AHEAD = F8 ? 4 : 8;  // score steps, reads of one, steps ahead
};
template <bool F8, int QG> struct FewWave {  // QG groups of 32 queries: 16 of each are the wave's in the scores
  bf16x8 q[QG][18];  // in the order of the score steps
  f32x16 o[QG][4];   // O^T: the wave's 128 columns x 32 queries
  f32x4 s[QG][2];    // S^T: e4m3: rows 16 u .. of the wave's 32; bf16: two chains of its 16
  float m[QG], l[QG], top[QG];
};
// What a wave reads of a tile besides the keys: factors of the rows of its scores (4 (lane / 16) .. and, e4m3, 16 on)
template <bool F8> struct FewFactors {
  u32x4 ex[2], inv[2];
  float mul[2];
};
// What it needs for the values of the tile before: probabilities and the first columns
template <bool F8, int QG> struct FewValues {
  u32x4 p[QG][4];
  int ps[QG];
  u32x2 v[3][4];
};

// Chunk of 64 (e4m3) or 32 values that lanes 16 g .. read: an order in which the 16 lanes that LDS serves at a time, 0 - 3,
// 12 - 15 and 20 - 27 of each half wave, find their rows' chunks in 16 different places of 256 bytes
template <bool F8> AMLA_DEV constexpr int few_chunk(int g) { return F8 ? (g & 1) << 1 | g >> 1 : (g >> 1) ^ (3 * (g & 1)); }
template <bool F8, int I> AMLA_DEV void few_read(u32x4 (&d)[2], uint32_t kl, uint32_t kr) {
  if constexpr (F8) {
    if constexpr (I < 8) {  // codes 64 I + 16 few_chunk ..
      d[0] = lds_read16<256 * (I >> 2)>(kl ^ (64 * (I & 3)));
      d[1] = lds_read16<256 * (I >> 2) + 16 * 512>(kl ^ (64 * (I & 3)));
    } else {
      d[0] = lds_read16<0>(kr ^ (64 * (I - 8)));
      d[1] = lds_read16<16 * 128>(kr ^ (64 * (I - 8)));
    }
  } else {  // values 32 I + 8 few_chunk ..
    if constexpr (I < 16) d[0] = lds_read16<256 * (I >> 2)>(kl ^ (64 * (I & 3)));
    else d[0] = lds_read16<0>(kr ^ (64 * (I - 16)));
  }
}
template <bool F8, int I> AMLA_DEV void few_reads_first(u32x4 (*ka)[2], uint32_t kl, uint32_t kr) {
  if constexpr (I < FewSteps<F8>::AHEAD) {
    few_read<F8, I>(ka[I], kl, kr);
    few_reads_first<F8, I + 1>(ka, kl, kr);
  }
}
AMLA_DEV f32x4 mfma_few(bf16x8 a, bf16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
template <bool F8, int QG, bool COPY, int I>
AMLA_DEV void few_step(FewWave<F8, QG> &w, u32x4 (&ka)[FewSteps<F8>::AHEAD + 1][2], const float (&mul)[2], uint32_t kl, uint32_t kr,
                       uint2 lanes, const Rows<F8> &next, const LatentPages &pg, uint8_t *st_next, int r0) {
  using W = FewSteps<F8>;
  if constexpr (I < W::N) {
    constexpr int A = W::AHEAD, c = I % (A + 1);
    if constexpr (I + A < W::N) few_read<F8, I + A>(ka[(I + A) % (A + 1)], kl, kr);
    lds_wait<W::READS * (W::N - 1 - I < A ? W::N - 1 - I : A)>();
    u32x4 x = ka[c][0], y = x;
    if constexpr (F8) {
      y = ka[c][1];
      lds_tie(x, y);
    } else {
      lds_tie(x);
    }
    if constexpr (!F8) {
#pragma unroll
      for (int k = 0; k < QG; ++k) w.s[k][I & 1] = mfma_few(as_bf16x8(x), w.q[k][I], w.s[k][I & 1]);
    } else if constexpr (I < 8) {
      const bf16x8 x0 = codes_to_bf16(x.x, x.y, mul[0]), y0 = codes_to_bf16(y.x, y.y, mul[1]);
#pragma unroll
      for (int k = 0; k < QG; ++k) {
        w.s[k][0] = mfma_few(x0, w.q[k][2 * I], w.s[k][0]);
        w.s[k][1] = mfma_few(y0, w.q[k][2 * I], w.s[k][1]);
      }
      const bf16x8 x1 = codes_to_bf16(x.z, x.w, mul[0]), y1 = codes_to_bf16(y.z, y.w, mul[1]);
#pragma unroll
      for (int k = 0; k < QG; ++k) {
        w.s[k][0] = mfma_few(x1, w.q[k][2 * I + 1], w.s[k][0]);
        w.s[k][1] = mfma_few(y1, w.q[k][2 * I + 1], w.s[k][1]);
      }
    } else {
#pragma unroll
      for (int k = 0; k < QG; ++k) {
        w.s[k][0] = mfma_few(as_bf16x8(x), w.q[k][16 + I - 8], w.s[k][0]);
        w.s[k][1] = mfma_few(as_bf16x8(y), w.q[k][16 + I - 8], w.s[k][1]);
      }
    }
    if constexpr (COPY && I < Rows<F8>::COPIES) next.template copy<I>(pg, st_next, r0, lanes);
    few_step<F8, QG, COPY, I + 1>(w, ka, mul, kl, kr, lanes, next, pg, st_next, r0);
  }
}
// Scores of the tile at LDS address base; COPY: with the copies of a later one between
template <bool F8, int QG, bool COPY>
AMLA_DEV void few_scores(FewWave<F8, QG> &w, FewFactors<F8> &f, uint32_t base, int half, const Rows<F8> &next, const LatentPages &pg,
                         uint8_t *st_next, int r0) {
  using G = Stage<F8>;
  const int lane = threadIdx.x & 63, l16 = lane & 15, g = lane >> 4, row = half * (G::ROWS / 2) + l16;
  const uint32_t fr = base + 4 * (half * (G::ROWS / 2) + 4 * g), fm = base + 4 * row;
  f.ex[0] = lds_read16<G::EXP>(fr);
  if constexpr (F8) {
    f.ex[1] = lds_read16<G::EXP + 64>(fr);
    f.inv[0] = lds_read16<G::INV>(fr);
    f.inv[1] = lds_read16<G::INV + 64>(fr);
    asm volatile("ds_read_b32 %0, %1 offset:%2" : "=v"(f.mul[0]) : "v"(fm), "i"(G::MUL) : "memory");
    asm volatile("ds_read_b32 %0, %1 offset:%2" : "=v"(f.mul[1]) : "v"(fm), "i"(G::MUL + 64) : "memory");
  }
  const uint32_t kl = base + row * Tile<F8>::RB + 16 * (few_chunk<F8>(g) ^ Tile<F8>::swz(row));
  const uint32_t kr = base + G::PE + row * 128 + 16 * (g ^ ((row >> 1) & 7));
  u32x4 ka[FewSteps<F8>::AHEAD + 1][2];
  few_reads_first<F8, 0>(ka, kl, kr);
  lds_wait<FewSteps<F8>::READS * FewSteps<F8>::AHEAD>();
  lds_tie(f.ex[0]);
  if constexpr (F8) lds_tie(f.ex[1], f.inv[0], f.inv[1], f.mul[0], f.mul[1]);
  else f.mul[0] = f.mul[1] = 1.f;
#pragma unroll
  for (int k = 0; k < QG; ++k) w.s[k][0] = w.s[k][1] = f32x4{0.f, 0.f, 0.f, 0.f};
  few_step<F8, QG, COPY, 0>(w, ka, f.mul, kl, kr, Rows<F8>::lanes(r0), next, pg, st_next, r0);
}
// z = s log2(e) scale + exponent of the row, in place; rows past lim are not seen
template <bool F8, bool MASK> AMLA_DEV float few_scaled(f32x4 (&s)[2], const FewFactors<F8> &f, float scale_log2, int lim) {
  float top = -INFINITY;
  if constexpr (!F8) s[0] += s[1];
#pragma unroll
  for (int u = 0; u < (F8 ? 2 : 1); ++u)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float z = __builtin_fmaf(s[u][i], scale_log2, __uint_as_float(f.ex[u][i]));
      if constexpr (MASK) z = 16 * u + i < lim ? z : -INFINITY;
      s[u][i] = z;
      top = __builtin_fmaxf(top, z);
    }
  return top;
}
// The largest of the four lanes of a query
AMLA_DEV float few_max(float x) {
  auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = __builtin_fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __builtin_fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
}
AMLA_DEV void few_write(uint32_t addr, uint32_t v) { asm volatile("ds_write_b32 %0, %1" ::"v"(addr), "v"(v) : "memory"); }
// Probabilities of the wave's scores, to LDS: rows 4 (g / 2 + 2 u) .. of query lane / 16 belong to lane query + 32 (g % 2)
// of the value products
template <bool F8>
AMLA_DEV void few_probabilities(const f32x4 (&s)[2], float m, float &l, float &most, const FewFactors<F8> &f, float top, uint32_t pbuf,
                                int half, int qh) {
  const int lane = threadIdx.x & 63, query = 16 * qh + (lane & 15), g = lane >> 4;
  const uint32_t to = pbuf + 1024 * half + 16 * (query + 32 * (g & 1));
  most = __builtin_fmaxf(most, top);
  if constexpr (F8) {
    const float ref = block_ref(few_max(top), m);  // of the 32 rows: a block of the matrix unit
    float sum = 0.f;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      float e[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        e[i] = __builtin_amdgcn_exp2f(s[u][i] - ref);
        sum = __builtin_fmaf(e[i], __uint_as_float(f.inv[u][i]), sum);
      }
      int hi, lo;
      split_fp8x4(e, 0.0625f, hi, lo);
      few_write(to + 4 * (g >> 1) + 8 * u, hi);
      few_write(to + FewStage<F8, 1>::LO + 4 * (g >> 1) + 8 * u, lo);
    }
    l = __builtin_fmaf(sum, __builtin_amdgcn_exp2f(ref - m), l);
    few_write(pbuf + FewStage<F8, 1>::PS + 4 * (32 * half + query), block_scale(ref, m));
  } else {
    float e[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) e[i] = __builtin_amdgcn_exp2f(s[0][i] - m);
    l += (e[0] + e[1]) + (e[2] + e[3]);
    const u32x2 v = {pack_bf16(e[0], e[1]), pack_bf16(e[2], e[3])};
    asm volatile("ds_write_b64 %0, %1" ::"v"(to + 8 * (g >> 1)), "v"(v) : "memory");
  }
}
template <bool F8, int QG, int C> AMLA_DEV void few_value_read(FewValues<F8, QG> &x, uint32_t v0, uint32_t v1) {
  if constexpr (C < 4) {
    u32x2(&v)[4] = x.v[C % 3];
    const uint32_t a = v0 ^ (F8 ? 32 * C : 64 * C), b = v1 ^ (64 * C);
    if constexpr (F8) {
      v[0] = lds_read_tr<F8, 0>(a);
      v[1] = lds_read_tr<F8, 8192>(a);
      v[2] = lds_read_tr<F8, 16384>(a);
      v[3] = lds_read_tr<F8, 24576>(a);
    } else {
      v[0] = lds_read_tr<F8, 0>(a);
      v[1] = lds_read_tr<F8, 0>(b);
      v[2] = lds_read_tr<F8, 16384>(a);
      v[3] = lds_read_tr<F8, 16384>(b);
    }
  }
}
// Where the wave's columns 128 cg .. of the values at pv begin: the addresses of value_phase, so far on
template <bool F8> AMLA_DEV uint2 few_value_addr(uint32_t pv, int cg) {
  using T = Tile<F8>;
  const int lane = threadIdx.x & 63, hh = lane >> 5, L16 = lane & 15, g16 = lane >> 4;
  if constexpr (F8) {
    const int r = 8 * (L16 >> 3) + 4 * hh + ((L16 >> 1) & 3);
    const uint32_t v = pv + r * T::RB + 16 * ((g16 & 1) ^ T::swz(r)) + 8 * (L16 & 1);
    return uint2{(v ^ (32 * ((4 * cg) & 7))) + 256 * ((4 * cg) >> 3), 0};
  } else {
    const int r = 4 * hh + (L16 >> 2), ch = 2 * (g16 & 1) + ((L16 >> 1) & 1);
    const uint32_t v = pv + 8 * (L16 & 1) + 256 * cg;
    return uint2{v + r * T::RB + 16 * (ch ^ T::swz(r)), v + (r + 8) * T::RB + 16 * (ch ^ T::swz(r + 8))};
  }
}
// The probabilities at pbuf and the first values
template <bool F8, int QG> AMLA_DEV void few_values_first(FewValues<F8, QG> &x, uint32_t pbuf, uint2 v) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int k = 0; k < QG; ++k) {
    const uint32_t pk = pbuf + k * FewStage<F8, QG>::PGRP;
    x.p[k][0] = lds_read16<0>(pk + 16 * lane);
    x.p[k][1] = lds_read16<1024>(pk + 16 * lane);
    if constexpr (F8) {
      x.p[k][2] = lds_read16<2048>(pk + 16 * lane);
      x.p[k][3] = lds_read16<3 * 1024>(pk + 16 * lane);
      asm volatile("ds_read_b32 %0, %1 offset:%2" : "=v"(x.ps[k]) : "v"(pk + 4 * lane), "i"(FewStage<F8, QG>::PS) : "memory");
    }
  }
  few_value_read<F8, QG, 0>(x, v.x, v.y);
  few_value_read<F8, QG, 1>(x, v.x, v.y);
}
template <bool F8, int QG, int C> AMLA_DEV void few_value_step(FewWave<F8, QG> &w, FewValues<F8, QG> &x, uint2 v) {
  if constexpr (C < 4) {
    few_value_read<F8, QG, C + 2>(x, v.x, v.y);
    lds_wait<4 * ((C + 1 < 4) + (C + 2 < 4))>();
    if constexpr (C == 0) {
#pragma unroll
      for (int k = 0; k < QG; ++k) {
        u32x4 a = x.p[k][0], b = x.p[k][1];
        lds_tie(a, b);
        x.p[k][0] = a;
        x.p[k][1] = b;
        if constexpr (F8) {
          u32x4 d = x.p[k][2], e = x.p[k][3];
          int ps = x.ps[k];
          lds_tie(d, e, ps);
          x.p[k][2] = d;
          x.p[k][3] = e;
          x.ps[k] = ps;
        }
      }
    }
    u32x2 a = x.v[C % 3][0], b = x.v[C % 3][1], d = x.v[C % 3][2], e = x.v[C % 3][3];
    lds_tie(a, b, d, e);
#pragma unroll
    for (int k = 0; k < QG; ++k) {
      const u32x4(&p)[4] = x.p[k];
      if constexpr (F8) {
        const i32x8 hi = {(int)p[0].x, (int)p[0].y, (int)p[0].z, (int)p[0].w, (int)p[1].x, (int)p[1].y, (int)p[1].z, (int)p[1].w};
        const i32x8 lo = {(int)p[2].x, (int)p[2].y, (int)p[2].z, (int)p[2].w, (int)p[3].x, (int)p[3].y, (int)p[3].z, (int)p[3].w};
        mfma_value<true>(w.o[k][C], join(a, b, d, e), 127, hi, x.ps[k]);
        mfma_value<true>(w.o[k][C], join(a, b, d, e), 127, lo, x.ps[k] - 4);
      } else {
        mfma_value<true>(w.o[k][C], as_bf16x8(u32x4{a.x, a.y, b.x, b.y}), as_bf16x8(p[0]));
        mfma_value<true>(w.o[k][C], as_bf16x8(u32x4{d.x, d.y, e.x, e.y}), as_bf16x8(p[1]));
      }
    }
    few_value_step<F8, QG, C + 1>(w, x, v);
  }
}

template <bool F8, int QG, bool MASK>
__global__ __launch_bounds__(256, 1) void latent_attn_few_kernel(LatentAttnParams p) {
  extern __shared__ __align__(1024) uint8_t sm[];
  using G = Stage<F8>;
  using F = FewStage<F8, QG>;
  constexpr int TILE = Tile<F8>::ROWS, NQ = 32 * QG;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int half = wave & 1, qh = wave >> 1, l16 = lane & 15, g = lane >> 4;
  const SplitWork at = split_work<F8>(p);
  if (at.b < 0) return;
  const uint32_t lds0 = (uint32_t)reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) const uint8_t *)sm);

  Feed<F8> feed{p.pg, sm, at.b, wave, at.held, min(at.held, at.t_end * TILE) - 1};
  if constexpr (MASK) feed.tail = p.seq_len - 1;
  feed.start(at.t_first);

  FewWave<F8, QG> w;
  const int query = 16 * qh + l16;  // of a group
  int limit[QG], lim[QG];           // rows of a tile below lim - TILE tile are seen: of the lane's first, row TILE / 2 half + 4 g
#pragma unroll
  for (int k = 0; k < QG; ++k) {
    const int rq = min(at.chunk * NQ + 32 * k + query, p.rows - 1), tok = rq / p.heads;
    limit[k] = at.held - (p.seq_len - 1 - tok);
    lim[k] = limit[k] - TILE / 2 * half - 4 * g;
    const uint16_t *qp = p.q + at.b * p.ldq_seq + tok * p.ldq_token + (rq - tok * p.heads) * p.ldq_head;
#pragma unroll
    for (int i = 0; i < 16; ++i)
      w.q[k][i] = as_bf16x8(ldg16(qp + (F8 ? 64 * (i >> 1) + 16 * few_chunk<F8>(g) + 8 * (i & 1) : 32 * i + 8 * few_chunk<F8>(g))));
#pragma unroll
    for (int i = 0; i < 2; ++i) w.q[k][16 + i] = as_bf16x8(ldg16(qp + LC_LORA + 32 * i + 8 * g));
    w.m[k] = M_NONE;
  }
  float *const x_top = reinterpret_cast<float *>(sm + F::TOP), *const x_m = reinterpret_cast<float *>(sm + F::M);
  FewFactors<F8> f;
  for (int pass = 0;; ++pass) {  // once, or twice where m turned out too low
#pragma unroll
    for (int k = 0; k < QG; ++k) {
#pragma unroll
      for (int c = 0; c < 4; ++c)
#pragma unroll
        for (int i = 0; i < 16; ++i) w.o[k][c][i] = 0.f;
      settle(w.o[k]);
      w.l[k] = 0.f;
      w.top[k] = -INFINITY;
    }
    // nothing before the first tile: probabilities of 0 times its own values
    for (int o = threadIdx.x * 4; o < F::PBUF; o += 1024)
      *reinterpret_cast<uint32_t *>(sm + F::P + F::PBUF + o) = o % F::PGRP < F::PS ? 0u : 127u;
    if (pass == 0) {  // the waves agree on m: the first tile's maxima, its scores made twice
      feed.template arrive<MASK>(at.t_first);
      few_scores<F8, QG, false>(w, f, lds0, half, feed.next, p.pg, sm, 0);
#pragma unroll
      for (int k = 0; k < QG; ++k)
        x_top[NQ * half + 32 * k + query] = few_max(few_scaled<F8, MASK>(w.s[k], f, p.scale_log2, lim[k] - at.t_first * TILE));
      __syncthreads();
#pragma unroll
      for (int k = 0; k < QG; ++k)
        w.m[k] = __builtin_fmaxf(__builtin_fmaxf(x_top[32 * k + query], x_top[NQ + 32 * k + query]), M_NONE);
    }
    uint32_t base = lds0, pbuf = lds0 + F::P;
    for (int tile = at.t_first; tile < at.t_end; ++tile) {
      const uint32_t before = base, p_before = 2 * lds0 + 2 * F::P + F::PBUF - pbuf;
      feed.template arrive<MASK>(tile);
      base = lds0 + feed.cur * G::SIZE;
      FewValues<F8, QG> x;
      const uint2 v = few_value_addr<F8>(before, wave);
      few_values_first<F8, QG>(x, p_before, v);
      few_scores<F8, QG, true>(w, f, base, half, feed.next, p.pg, feed.next_stage(), Rows<F8>::WR * wave);
      few_value_step<F8, QG, 0>(w, x, v);
#pragma unroll
      for (int k = 0; k < QG; ++k) {
        const float top = few_scaled<F8, MASK>(w.s[k], f, p.scale_log2, lim[k] - tile * TILE);
        few_probabilities<F8>(w.s[k], w.m[k], w.l[k], w.top[k], f, top, pbuf + k * F::PGRP, half, qh);
      }
      pbuf = p_before;
      feed.advance(tile);
    }
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    {
      FewValues<F8, QG> x;
      const uint2 v = few_value_addr<F8>(base, wave);
      few_values_first<F8, QG>(x, 2 * lds0 + 2 * F::P + F::PBUF - pbuf, v);
      few_value_step<F8, QG, 0>(w, x, v);
    }
#pragma unroll
    for (int k = 0; k < QG; ++k) settle(w.o[k]);
    wait_vmcnt<0>();  // (copies past the last tile)
#pragma unroll
    for (int k = 0; k < QG; ++k) {
      x_top[NQ * half + 32 * k + query] = few_max(w.top[k]);
      x_m[32 * k + query] = w.m[k];
    }
    if constexpr (MASK) reinterpret_cast<int *>(sm + F::ODD)[wave] = feed.odd;
    __syncthreads();
    float high[QG];
#pragma unroll
    for (int k = 0; k < QG; ++k) high[k] = __builtin_fmaxf(x_top[32 * k + query], x_top[NQ + 32 * k + query]);
    const int any = lane % NQ;
    const bool again = __ballot(__builtin_fmaxf(x_top[any], x_top[NQ + any]) > x_m[any] + LAG) != 0;
    __syncthreads();
    if (!again) break;
#pragma unroll
    for (int k = 0; k < QG; ++k) w.m[k] = high[k] > w.m[k] + LAG ? high[k] : w.m[k];
    feed.start(at.t_first);
  }
  // sums over the four lanes and both halves of a query, handed to the lanes that hold its outputs
  float *const x_sum = reinterpret_cast<float *>(sm + F::SUM);
  int *const x_lim = reinterpret_cast<int *>(sm + F::LIM);
#pragma unroll
  for (int k = 0; k < QG; ++k) {
    w.l[k] += __shfl_xor(w.l[k], 16, 64);
    w.l[k] += __shfl_xor(w.l[k], 32, 64);
    x_sum[NQ * half + 32 * k + query] = w.l[k];
    x_m[32 * k + query] = w.m[k];
    if constexpr (MASK) x_lim[32 * k + query] = limit[k];
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < QG; ++k) {
    const int j = 32 * k + (lane & 31);
    float l = x_sum[j] + x_sum[NQ + j];
    if constexpr (MASK) {
      const int *odd = reinterpret_cast<const int *>(sm + F::ODD);
      const int first = min(min(odd[0], odd[1]), min(odd[2], odd[3]));
      l = first < x_lim[j] ? __uint_as_float(0x7fc00000u) : l;
    }
    if (__ballot(l != l)) l = sees_none<TILE>(p.pg, at, MASK ? x_lim[j] : INT32_MAX) ? 0.f : l;
    store_split<QG>(p, sm, w.o[k], l, x_m[j], at.b, at.chunk, at.slot, at.splits, wave, k, wave);
  }
}

// Joins the splits of a query row: sum_j 2^(lse_j - max) O_j / sum_j 2^(lse_j - max).  One workgroup a row, wave k
// taking splits k, k + 4, .., eight rows of 1 KB in flight; the waves' sums meet in LDS in wave order.
template <int HG, int CG>  // 32-row groups and column groups of the workgroups before
__global__ __launch_bounds__(256) void latent_join_kernel(LatentAttnParams p) {
  __shared__ float part[3][64][9];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int b = blockIdx.y, row = blockIdx.x;
  const int held = min(max(p.lengths[b], 0), p.cap);
  const int2 at = held ? p.part_plan[b] : int2{0, 0};
  const int n = __builtin_amdgcn_readfirstlane(at.y);
  if (n == 1) return;
  const size_t dst = (size_t)b * p.rows + row;
  u32x4 *od = reinterpret_cast<u32x4 *>(p.out + dst * LC_LORA) + lane;
  if (n == 0) {
    if (wave == 0) *od = u32x4{0, 0, 0, 0};
    if (threadIdx.x == 0 && p.lse) p.lse[dst] = -INFINITY;
    return;
  }
  const size_t src = (size_t)(at.x + row / (32 * HG) * n) * (32 * HG) + row % (32 * HG);
  const float *lse = p.part_lse + src;
  float top = -INFINITY;
  for (int j = lane; j < n; j += 64) top = __builtin_fmaxf(top, lse[(size_t)j * (32 * HG)]);
  top = wave_max(top);
  const float ref = top == -INFINITY ? 0.f : top;
  float total = 0.f, a[8] = {};
  const uint16_t *po = p.part_o + src * LC_LORA + 8 * lane;
  const float *ps = p.part_scale + src * 4 + lane / (64 / CG);
  for (int j0 = wave; j0 < n; j0 += 32) {
    float w[8], s[8];
    u32x4 v[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const int j = min(j0 + 4 * k, n - 1);
      v[k] = ldg16(po + (size_t)j * (32 * HG * LC_LORA));
      s[k] = ps[(size_t)j * (32 * HG * 4)];
      w[k] = j0 + 4 * k < n ? lse[(size_t)j * (32 * HG)] - ref : -INFINITY;
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const float f = __builtin_amdgcn_exp2f(w[k]);
      total += f;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint32_t x = v[k][e];
        a[2 * e] = __builtin_fmaf(f, lo_f16(x) * s[k], a[2 * e]);
        a[2 * e + 1] = __builtin_fmaf(f, hi_f16(x) * s[k], a[2 * e + 1]);
      }
    }
  }
  if (wave > 0) {
#pragma unroll
    for (int e = 0; e < 8; ++e) part[wave - 1][lane][e] = a[e];
    part[wave - 1][lane][8] = total;
  }
  __syncthreads();
  if (wave > 0) return;
#pragma unroll
  for (int k = 0; k < 3; ++k) {
#pragma unroll
    for (int e = 0; e < 8; ++e) a[e] += part[k][lane][e];
    total += part[k][lane][8];
  }
  const float inv = total == 0.f ? 0.f : 1.f / total;
  *od = u32x4{pack_bf16(a[0] * inv, a[1] * inv), pack_bf16(a[2] * inv, a[3] * inv), pack_bf16(a[4] * inv, a[5] * inv),
              pack_bf16(a[6] * inv, a[7] * inv)};
  if (lane == 0 && p.lse) p.lse[dst] = total == 0.f ? -INFINITY : (top + __builtin_amdgcn_logf(total)) * 0.6931471805599453f;
}

constexpr int LA_MAX_ROWS = INT32_MAX - 511;  // of a sequence: rows are counted in 32 bits up to three tiles past the last one
constexpr int LA_UNITS = 256;  // workgroups that run at a time (one per CU)

// 32-row groups of a workgroup: as many as the rows of a sequence fill, since they share each tile's way through LDS, but
// one while the cached rows do not keep all CUs at work for long: then more, shorter workgroups win.  One or two: the kernel
// for few query rows.  Measured with 128 heads and one new token (1 / 2 / 4 groups, us), fp8: 1 x 257 rows 16 / 21 / 22,
// 64 x 512 31 / 43 / 52, 4 x 8192 34 / 39 / 42, 8 x 8192 50 / 49 / 50, 32 x 4096 85 / 74 / 67, 8 x 32768 146 / 115 / 96;
// bf16: 4 x 8192 36 / 38 / 42, 8 x 8192 50 / 46 / 51, 32 x 4096 85 / 70 / 73, 8 x 32768 149 / 108 / 106; 64 heads: 64 x 1024
// fp8 39 / 43, 40 x 4096 65 / 59, bf16 69 / 59 (four groups half empty there).  max_rows is what a table has room for, since
// the lengths are on the device: of 64 x 512 rows 32 us with a table of their size, 47 - 50 with one of 2048 rows or more, of
// 1 x 257 rows 16 up to 32768 and 22 with 163840 (captured; bf16 32, 48, 13.5 and 20).
static int attn_groups(int64_t seqs, int64_t rows, int64_t max_rows) {
  const double pairs = (double)seqs * rows * max_rows / LA_UNITS;  // query rows x cached rows of a CU
  return pairs < 32 * 1024 || rows <= 32 ? 1 : rows <= 64 ? 2 : 4;
}
struct AttnSizes {
  int hg;
  int64_t chunks, slots;
};
static AttnSizes attn_sizes(int64_t seqs, int64_t rows, int64_t max_rows) {
  AttnSizes s;
  s.hg = attn_groups(seqs, rows, max_rows);
  s.chunks = (rows + 32 * s.hg - 1) / (32 * s.hg);
  s.slots = std::max<int64_t>(LA_UNITS, s.chunks * seqs + LA_UNITS / 2);
  const int64_t tiles = std::max<int64_t>(1, (max_rows + 31) / 32);  // no split is shorter than a tile
  if (tiles < s.slots / (s.chunks * seqs)) s.slots = s.chunks * seqs * tiles;
  return s;
}

template <bool F8, int HG>
static int launch_attn(const LatentAttnParams &p, hipStream_t st) {
  void (*kernel)(LatentAttnParams);
  int lds;
  if constexpr (HG <= 2) {
    kernel = p.seq_len > 1 ? latent_attn_few_kernel<F8, HG, true> : latent_attn_few_kernel<F8, HG, false>;
    lds = FewStage<F8, HG>::LDS;
  } else {
    kernel = p.seq_len > 1 ? latent_attn_kernel<F8, true> : latent_attn_kernel<F8, false>;
    lds = Stage<F8>::LDS;
  }
  int rc = latent_lds(kernel, "latent_attention");
  if (rc) return rc;
  kernel<<<dim3((unsigned)(p.slots + 7) / 8 * 8), 256, lds, st>>>(p);  // whole runs of every XCD
  if ((rc = check_launch("latent_attention"))) return rc;
  latent_join_kernel<HG, HG <= 2 ? 4 : 1><<<dim3((unsigned)p.rows, (unsigned)p.seqs), 256, 0, st>>>(p);
  return check_launch("latent_attention join");
}

}  // namespace amla

using namespace amla;

extern "C" {

size_t amla_latent_attention_workspace_bytes(int64_t seqs, int64_t seq_len, int64_t heads, int64_t max_rows) {
  if (seqs <= 0 || seq_len <= 0 || heads <= 0 || seqs > AMLA_MAX_SEQS || seq_len > INT32_MAX || heads > INT32_MAX / seq_len)
    return 0;
  const AttnSizes s = attn_sizes(seqs, seq_len * heads, max_rows);
  return (size_t)s.slots * 32 * s.hg * (LC_LORA * 2 + 4 + 16) + (size_t)seqs * 8;
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
  if (cap > LA_MAX_ROWS) return fail(AMLA_EUNSUPPORTED, "%s: sequences of at most %d rows in their table", what, LA_MAX_ROWS);
  const AttnSizes s = attn_sizes(seqs, seq_len * heads, cap);
  if (s.slots >= (1 << 24) - 8 || seq_len * heads >= 1 << 24)  // grids of fewer than 2^32 threads
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
  p.part_scale = p.part_lse + (size_t)s.slots * 32 * s.hg;
  p.part_plan = reinterpret_cast<int2 *>(p.part_scale + (size_t)s.slots * 32 * s.hg * 4);
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  if (p.pg.scales) {
    if (s.hg == 4) return launch_attn<true, 4>(p, st);
    return s.hg == 2 ? launch_attn<true, 2>(p, st) : launch_attn<true, 1>(p, st);
  }
  if (s.hg == 4) return launch_attn<false, 4>(p, st);
  return s.hg == 2 ? launch_attn<false, 2>(p, st) : launch_attn<false, 1>(p, st);
}

}  // extern "C"
