// Attention of packed prompts: sequences of different lengths one after another, causal or
// not, heads that share keys and values, an optional rope key shared by all heads.
//   s_ij = scale q_i . k_j,  out_i = sum_j softmax(s_i)_j v_j,  lse_i = log sum_j exp(s_ij)
// One pass over the keys with a reference and a sum per query, all in fp32; P is
// rounded to bf16 for the matrix units (as inference/ops.py:179 rounds it).
//
// Bound: the matrix units and their power.  Two prompts of 50 and 950 rows behind 562 and
// 7438 cached ones, 128 heads with rope keys: 618 GFLOP in 617 - 675 us by card, 0.92 - 1.0 PFLOP/s at
// 1.8 GHz (an 8192^3 product of the library reaches 1.2), the units busy 54 % of the cycles; what a wave issues besides is nearly as long as its products.  Five prompts of 4099
// rows together: 332 - 355 us, where starting and ending a block (15000 cycles) and its last,
// masked tiles weigh as much as a third of the products.  64 queries a wave: with 32 each
// fragment read from LDS fed one product and the same two cases took 858 and 413 us.
#include <algorithm>
#include <math.h>

#include "latent.h"

namespace amla {

constexpr int PA_KT = 64;                 // keys per tile
constexpr int PA_QB = 256;                // queries per workgroup: four waves, two groups of 32 each
constexpr int PA_NST = 3;                 // LDS stages: a tile, the one before it (values), the one to come
constexpr int PA_VD = 128;
constexpr int PA_MAX_ROWS = INT32_MAX - 511;  // of queries and of keys: counted in 32 bits up to a block past the last one
constexpr int PA_HALF = PA_KT * 128;      // 64 rows of 128 bytes: 64 key or value columns of a tile

struct PackedParams {
  const uint16_t *q, *k, *v, *k_pe;  // k_pe null: key columns 128.. are k's own
  uint16_t *out;
  float *lse;
  const int32_t *offsets, *k_offsets;
  int q_rows, k_rows, seqs, heads, group, causal;
  int splits;                        // workgroups of a block, at most
  int64_t ldq, ldq_head, ldk, ldk_head, ldv, ldv_head, ld_pe;
  float scale_log2;
  // With splits: of each (block, head, split) 256 rows of 128 sums, normalised, in fp16 times a power of two a row (bf16 would
  // add as much error as the output's rounding), and (log2 of the sum of 2^s, the power) of each row
  uint16_t *part_o;
  float *part_ls;
};

// Offsets are not checked on the host: clamped to the rows there are, and none below its predecessor's.
AMLA_DEV int span_start(const int32_t *off, int b, int rows) { return min(max(off[b], 0), rows); }

// A query block: its number within the sequence (-1: past the end), the sequence's first query and key and their counts.
struct PackedBlock {
  int block, q0, nq, k0, nk;
};
// Query block `tile` of the batch, wave-uniform.  Lane l looks at sequence b0 + l, queries and keys at once: one trip to
// memory for up to 64 sequences.
AMLA_DEV PackedBlock find_block(const PackedParams &p, int tile) {
  const int lane = threadIdx.x & 63;
  int base = 0;
  for (int b0 = 0; b0 < p.seqs; b0 += 64) {
    const int b = min(b0 + lane, p.seqs - 1);
    const int q0 = span_start(p.offsets, b, p.q_rows), k0 = span_start(p.k_offsets, b, p.k_rows);
    const int nq = max(span_start(p.offsets, b + 1, p.q_rows) - q0, 0);
    const int nk = max(span_start(p.k_offsets, b + 1, p.k_rows) - k0, 0);
    const int blocks = b0 + lane < p.seqs ? (nq + PA_QB - 1) / PA_QB : 0;
    int incl = blocks;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int v = __shfl_up(incl, o, 64);
      if (lane >= o) incl += v;
    }
    const uint64_t past = __ballot(base + incl > tile);
    if (past) {
      const int l = __builtin_ctzll(past);
      const int n = __builtin_amdgcn_readlane(blocks, l), before = base + __builtin_amdgcn_readlane(incl, l) - n;
      // a sequence's last blocks see the most keys: they go first
      return PackedBlock{n - 1 - (tile - before), __builtin_amdgcn_readlane(q0, l), __builtin_amdgcn_readlane(nq, l),
                         __builtin_amdgcn_readlane(k0, l), __builtin_amdgcn_readlane(nk, l)};
    }
    base += __builtin_amdgcn_readlane(incl, 63);
  }
  return PackedBlock{-1, 0, 0, 0, 0};
}

// Tiles of 64 keys that one workgroup takes of a block, at most: with few blocks their keys are split, so that all CUs have
// work and no block is much longer than the others: total / 256, but not below PA_LEAST (2 us each; starting and joining take
// 10).  A block of more is split evenly, seven tiles into three and four.
constexpr int PA_LEAST = 6;
AMLA_DEV int split_tiles(const PackedParams &p) {
  const int lane = threadIdx.x & 63;
  float total = 0.f;
  for (int b0 = 0; b0 < p.seqs; b0 += 64) {
    const int b = min(b0 + lane, p.seqs - 1);
    const int nq = max(span_start(p.offsets, b + 1, p.q_rows) - span_start(p.offsets, b, p.q_rows), 0);
    const int nk = max(span_start(p.k_offsets, b + 1, p.k_rows) - span_start(p.k_offsets, b, p.k_rows), 0);
    const float blocks = b0 + lane < p.seqs ? (float)((nq + PA_QB - 1) / PA_QB) : 0.f;
    total += blocks * (p.causal ? max(nk - nq, 0) / (float)PA_KT + 2.f * (blocks + 1.f) : nk / (float)PA_KT);
  }
  const float each = wave_sum(total) * p.heads / 256.f;
  return __builtin_amdgcn_readfirstlane(max(PA_LEAST, (int)__builtin_fminf(each, 1e9f) + 1));
}
// Keys that a block needs, and its splits
AMLA_DEV int block_keys(const PackedParams &p, const PackedBlock &b) {
  return p.causal ? min(b.nk, max(b.nk - b.nq + min((b.block + 1) * PA_QB, b.nq), 0)) : b.nk;
}
AMLA_DEV int block_splits(const PackedParams &p, int keys) {
  if (p.splits == 1) return 1;
  const int tiles = (keys + PA_KT - 1) / PA_KT, each = split_tiles(p);
  return max(1, min(p.splits, (tiles + each - 1) / each));
}

// ---------------------------------------------------------------- one wave's part of a tile
//
// Scores S^T (keys x queries) = K Q^T and outputs O^T (columns x queries) += V^T P^T, 32x32x16
// products; lane l holds column l % 32, so a query's statistics stay in its two lanes and P
// goes from the score registers into the product as it is.  64 queries a wave: each fragment
// read from LDS feeds two products (with 32 the reads alone take as long as the matrix units).

template <bool ROPE> struct PackedWave {
  static constexpr int KS = ROPE ? 12 : 8, NK = ROPE ? 3 : 2;  // 16-wide steps and 64-wide arrays of a key
  static constexpr int VAL = NK * PA_HALF, STAGE = (NK + 2) * PA_HALF, COPIES = 2 * (NK + 2);
  bf16x8 q[2][KS];
  f32x16 o[2][4];  // [group][32 columns]
  f32x16 s[2][2];  // scores of the tile in work: [group][32 keys]
  f32x16 t[2];     // second 32 keys of the tile before, not yet exponentiated
  f32x4 u[2];      // nor the last four of its first 32
  u32x4 p[2][4];   // P of the tile before, 16 keys each
  float x[2][2];   // the last two probabilities, not yet summed and packed
  float m[2], l[2], top[2];  // reference (log2 units), sum of 2^(z - m), largest score so far
};
// The reference m is the maximum of the first tile that shows a row any key (itself, not a whole number above it: the
// probability of the largest score, all there is where few keys are seen, is not rounded): fp32 and bf16 have the range for
// sums up to 2^PA_LAG above it.  A row that passes it has the workgroup start over with m from all keys.  The rounding of m,
// half a unit in its last place, is in every exponent of its row: no more than 16 up to scores of 2^28, where the range ends.
constexpr float PA_LAG = 60.f, PA_NONE = -1e30f;

template <int OFS> AMLA_DEV u32x4 pa_read16(uint32_t addr) {
  u32x4 v;
  asm volatile("ds_read_b128 %0, %1 offset:%2" : "=v"(v) : "v"(addr), "i"(OFS) : "memory");
  return v;
}
template <int OFS> AMLA_DEV u32x2 pa_read_tr(uint32_t addr) {
  u32x2 v;
  asm volatile("ds_read_b64_tr_b16 %0, %1 offset:%2" : "=v"(v) : "v"(addr), "i"(OFS) : "memory");
  return v;
}
template <int N> AMLA_DEV void pa_wait() { asm volatile("s_waitcnt lgkmcnt(%0)" ::"i"(N) : "memory"); }
template <typename T> AMLA_DEV void pa_tie(T &v) { asm volatile("" : "+v"(v)::"memory"); }
// Scores in vector registers, queries and outputs in accumulator registers (inline asm: left to itself the compiler moves
// accumulators between the two every tile).
// WAIT: the step's first product, whose operands the compiler may have moved just before (two wait states); the other
// products of a step read the same registers.
template <bool ZERO, bool WAIT> AMLA_DEV void pa_score(f32x16 &c, bf16x8 a, bf16x8 b) {
  if constexpr (ZERO && WAIT) asm volatile("s_nop 1\n\tv_mfma_f32_32x32x16_bf16 %0, %1, %2, 0" : "=&v"(c) : "v"(a), "a"(b));
  else if constexpr (ZERO) asm volatile("v_mfma_f32_32x32x16_bf16 %0, %1, %2, 0" : "=&v"(c) : "v"(a), "a"(b));
  else if constexpr (WAIT) asm volatile("s_nop 1\n\tv_mfma_f32_32x32x16_bf16 %0, %1, %2, %0" : "+v"(c) : "v"(a), "a"(b));
  else asm volatile("v_mfma_f32_32x32x16_bf16 %0, %1, %2, %0" : "+v"(c) : "v"(a), "a"(b));
}
template <bool WAIT> AMLA_DEV void pa_value(f32x16 &c, bf16x8 a, bf16x8 b) {
  if constexpr (WAIT) asm volatile("s_nop 1\n\tv_mfma_f32_32x32x16_bf16 %0, %1, %2, %0" : "+a"(c) : "v"(a), "v"(b));
  else asm volatile("v_mfma_f32_32x32x16_bf16 %0, %1, %2, %0" : "+a"(c) : "v"(a), "v"(b));
}
// Before vector code reads what the products above wrote, and before they read what it wrote.
AMLA_DEV void pa_settle(f32x16 (&o)[2][4]) {
  asm volatile("s_nop 7\n\ts_nop 7\n\ts_nop 7"
               : "+a"(o[0][0]), "+a"(o[0][1]), "+a"(o[0][2]), "+a"(o[0][3]), "+a"(o[1][0]), "+a"(o[1][1]), "+a"(o[1][2]),
                 "+a"(o[1][3])::"memory");
}

// Where a wave's copies come from: rows 16 w .. + 15 of a tile, as 8-row pieces of 128-byte half-rows.  Bases are
// uniform, each lane adds a fixed offset; chunk c of row r of a key array sits at c ^ ((r >> 1) & 7), the 64-byte
// half g of a value row at g ^ ((r >> 1) & 1), both free of bank conflicts.
struct PackedFeed {
  const char *k, *v, *pe;       // the head's first key, value and rope key of the sequence
  int64_t ldk, ldv, ldpe;       // bytes of a row
  int klim, row0;               // keys in use, the wave's first row of a tile
  uint32_t ok[2], ov, op[2];    // lane offsets
  const char *tk[2], *tv[2], *tp[2];  // rows row0, row0 + 8 of the tile that is copied next
  AMLA_DEV void init(int lane) {
    const int r8 = lane >> 3;
    const uint32_t rr = klim < PA_KT ? 0 : r8;  // fewer keys than a tile: any row in bounds, nothing of it is used
#pragma unroll
    for (int g = 0; g < 2; ++g) {
      const uint32_t kc = 16 * ((lane & 7) ^ ((r8 >> 1) + 4 * g));
      ok[g] = rr * (uint32_t)ldk + kc;
      op[g] = rr * (uint32_t)ldpe + kc;
    }
    ov = rr * (uint32_t)ldv + 16 * ((lane & 7) ^ (4 * ((r8 >> 1) & 1)));
  }
  // First key of the tile that is loaded as tile j: the last one ends with the last key (what it repeats is masked).
  AMLA_DEV int first(int j) const { return max(min(j * PA_KT, klim - PA_KT), 0); }
  AMLA_DEV void aim(int j) {
    const int64_t row = klim < PA_KT ? 0 : first(j) + row0, more = klim < PA_KT ? 0 : 8;
#pragma unroll
    for (int g = 0; g < 2; ++g) {
      tk[g] = k + (row + more * g) * ldk;
      tv[g] = v + (row + more * g) * ldv;
      tp[g] = pe + (row + more * g) * ldpe;
    }
  }
  // copy I of the tile aimed at
  template <bool ROPE, int I> AMLA_DEV void copy(uint8_t *st) const {
    constexpr int NK = ROPE ? 3 : 2, arr = I >> 1, g = I & 1;
    uint8_t *dst = st + arr * PA_HALF + (row0 + 8 * g) * 128;
    if constexpr (arr >= NK) copy_lds(tv[g] + 128 * (arr - NK) + ov, dst);
    else if constexpr (arr == 2) copy_lds(tp[g] + op[g], dst);
    else copy_lds(tk[g] + 128 * arr + ok[g], dst);
  }
  // Tile 0 with every row clamped to the keys there are
  template <bool ROPE> AMLA_DEV void copy_first(uint8_t *st, int lane) const {
    constexpr int NK = ROPE ? 3 : 2;
#pragma unroll
    for (int g = 0; g < 2; ++g) {
      const int r8 = lane >> 3;
      const int64_t row = min(row0 + 8 * g + r8, klim - 1);
      const int kc = 16 * ((lane & 7) ^ ((r8 >> 1) + 4 * g)), vc = 16 * ((lane & 7) ^ (4 * ((r8 >> 1) & 1)));
      uint8_t *dst = st + (row0 + 8 * g) * 128;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        copy_lds(k + row * ldk + 128 * h + kc, dst + h * PA_HALF);
        copy_lds(v + row * ldv + 128 * h + vc, dst + (NK + h) * PA_HALF);
      }
      if constexpr (ROPE) copy_lds(pe + row * ldpe + kc, dst + 2 * PA_HALF);
    }
  }
  // Values of the tile at st that are no numbers become 0 in LDS: a masked probability of 0 would make them NaN.  Each lane
  // looks at what it copied; true if any lane found one.
  template <bool ROPE> AMLA_DEV bool clean(uint8_t *st, int lane) const {
    bool found = false;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      u32x4 *at = reinterpret_cast<u32x4 *>(st + PackedWave<ROPE>::VAL + (i >> 1) * PA_HALF + (row0 + 8 * (i & 1)) * 128 + 16 * lane);
      const u32x4 x = *at;
      u32x4 y = x;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if ((x[k] & 0x7f80u) == 0x7f80u) y[k] &= 0xffff0000u;
        if ((x[k] & 0x7f800000u) == 0x7f800000u) y[k] &= 0xffffu;
      }
      const bool bad = y.x != x.x || y.y != x.y || y.z != x.z || y.w != x.w;
      if (bad) *at = y;
      found |= bad;
    }
    return __ballot(found) != 0;
  }
  template <bool ROPE, int I = 0> AMLA_DEV void copy_all(uint8_t *st) const {
    if constexpr (I < 2 * ((ROPE ? 3 : 2) + 2)) {
      copy<ROPE, I>(st);
      copy_all<ROPE, I + 1>(st);
    }
  }
};

// Softmax, one exponential behind each product.  A group's 32 probabilities a tile are numbered as they follow each other
// in its registers (first 32 keys: 0 .. 15, second: 16 .. 31); the value products take the first PA_EARLY, the next
// scores' products the others, both groups in turn.  A result is summed and packed one turn later: it is not waited for.
constexpr int PA_EARLY = 12;
template <bool ROPE, int G, int N> AMLA_DEV void pa_turn(PackedWave<ROPE> &w, u32x4 (&p)[4], float z, float c) {
  const float y = __builtin_fmaf(z, c, -w.m[G]);
  if constexpr (N > 0 && N % 2 == 0) p[(N - 2) >> 3][((N - 2) >> 1) & 3] = pack_bf16(w.x[G][0], w.x[G][1]);
  w.l[G] += w.x[G][N & 1];
  w.x[G][N & 1] = __builtin_amdgcn_exp2f(y);
}
// I: 0 .. 2 PA_EARLY - 1
template <bool ROPE, int I> AMLA_DEV void pa_soft_early(PackedWave<ROPE> &w, u32x4 (&pn)[2][4], float c) {
  constexpr int g = I & 1, n = I >> 1;
  pa_turn<ROPE, g, n>(w, pn[g], w.s[g][0][n], c);
}
// I: 0 .. 2 (32 - PA_EARLY) - 1
template <bool ROPE, int I> AMLA_DEV void pa_soft_late(PackedWave<ROPE> &w, float c) {
  constexpr int g = I & 1, n = PA_EARLY + (I >> 1);
  if constexpr (n < 16) pa_turn<ROPE, g, n>(w, w.p[g], w.u[g][n - PA_EARLY], c);
  else if constexpr (n < 32) pa_turn<ROPE, g, n>(w, w.p[g], w.t[g][n - 16], c);
}
template <bool ROPE> AMLA_DEV void pa_soft_end(PackedWave<ROPE> &w) {
  w.p[0][3].w = pack_bf16(w.x[0][0], w.x[0][1]);
  w.p[1][3].w = pack_bf16(w.x[1][0], w.x[1][1]);
}

constexpr int PA_AHEAD = 3;  // steps that LDS reads go out ahead, across the phases too: 300 to 400 cycles

template <bool ROPE, int I> AMLA_DEV void pa_key_read(u32x4 (&ka)[2], uint32_t kr) {
  const uint32_t a = kr ^ (32 * (I & 3));
  ka[0] = pa_read16<(I >> 2) * PA_HALF>(a);
  ka[1] = pa_read16<(I >> 2) * PA_HALF + 32 * 128>(a);
}
template <int C> AMLA_DEV void pa_val_read(u32x2 (&v)[4], uint32_t v0) {
  if constexpr (C < 8) {
    const uint32_t a = v0 ^ (64 * ((C >> 1) & 1));
    constexpr int ofs = (C >> 2) * PA_HALF + (C & 1) * 4096;
    v[0] = pa_read_tr<ofs>(a);
    v[1] = pa_read_tr<ofs + 1024>(a);
    v[2] = pa_read_tr<ofs + 2048>(a);
    v[3] = pa_read_tr<ofs + 3 * 1024>(a);
  }
}
// What goes behind product K of score step I: a copy of the tile to come (one a step) or late probabilities
template <bool ROPE, int I, int K> AMLA_DEV void pa_score_slot(PackedWave<ROPE> &w, float c, const PackedFeed &f, uint8_t *st) {
  if constexpr (!ROPE) {  // 40 probabilities and 8 copies behind 32 products
    if constexpr (K == 0) f.copy<ROPE, I>(st);
    if constexpr (K == 1 || K == 2) pa_soft_late<ROPE, 5 * I + 2 * K - 2>(w, c);
    if constexpr (K > 0) pa_soft_late<ROPE, 5 * I + (K == 3 ? 4 : 2 * K - 1)>(w, c);
  } else if constexpr (I == 0 || I == 11) {  // 40 and 10 behind 48: 5 probabilities in the outer steps, 3 in the others
    constexpr int L = I == 0 ? 0 : 35;
    if constexpr (K == 0) pa_soft_late<ROPE, L>(w, c);
    pa_soft_late<ROPE, L + 1 + K>(w, c);
  } else {
    if constexpr (K == 0) f.copy<ROPE, I - 1>(st);
    else pa_soft_late<ROPE, 5 + 3 * (I - 1) + K - 1>(w, c);
  }
  __builtin_amdgcn_sched_barrier(0);
}
template <bool ROPE, int I>
AMLA_DEV void pa_score_step(PackedWave<ROPE> &w, u32x4 (&ka)[PA_AHEAD + 1][2], u32x2 (&vv)[PA_AHEAD + 1][4], uint32_t kr,
                            uint32_t v0, float c, const PackedFeed &f, uint8_t *st) {
  constexpr int KS = PackedWave<ROPE>::KS, A = PA_AHEAD;
  if constexpr (I < KS) {
    if constexpr (I + A < KS) pa_key_read<ROPE, I + A>(ka[(I + A) % (A + 1)], kr);
    else pa_val_read<I + A - KS>(vv[I + A - KS], v0);
    if constexpr (I >= A) pa_wait<I + A < KS ? 2 * A : 2 * (KS - 1 - I) + 4 * (I + A + 1 - KS)>();  // (the first A are there)
    u32x4 x = ka[I % (A + 1)][0], y = ka[I % (A + 1)][1];
    pa_tie(x);
    pa_tie(y);
    pa_score<I == 0, true>(w.s[0][0], as_bf16x8(x), w.q[0][I]);
    pa_score_slot<ROPE, I, 0>(w, c, f, st);
    pa_score<I == 0, false>(w.s[0][1], as_bf16x8(y), w.q[0][I]);
    pa_score_slot<ROPE, I, 1>(w, c, f, st);
    pa_score<I == 0, false>(w.s[1][0], as_bf16x8(x), w.q[1][I]);
    pa_score_slot<ROPE, I, 2>(w, c, f, st);
    pa_score<I == 0, false>(w.s[1][1], as_bf16x8(y), w.q[1][I]);
    pa_score_slot<ROPE, I, 3>(w, c, f, st);
    pa_score_step<ROPE, I + 1>(w, ka, vv, kr, v0, c, f, st);
  }
}
template <bool ROPE> AMLA_DEV uint32_t pa_key_addr(uint32_t stage) {
  const int lane = threadIdx.x & 63, j32 = lane & 31, hh = lane >> 5;
  return stage + j32 * 128 + 16 * (hh ^ ((j32 >> 1) & 7));
}
template <bool ROPE> AMLA_DEV uint32_t pa_val_addr(uint32_t stage) {
  const int lane = threadIdx.x & 63, hh = lane >> 5, L16 = lane & 15, g16 = lane >> 4;
  return stage + PackedWave<ROPE>::VAL + (4 * hh + (L16 >> 2)) * 128 + 64 * (L16 >> 3) + 32 * (g16 & 1) + 8 * (L16 & 3);
}
// The next tile landed in every wave, and no wave reads the stage two tiles back any more
AMLA_DEV void pa_arrive() {
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
}
// The first reads of a tile's keys; complete when the loop turns (a register whose read is on its way must not be moved)
template <bool ROPE> AMLA_DEV void pa_first_keys(u32x4 (&ka)[PA_AHEAD + 1][2], uint32_t kr) {
  pa_key_read<ROPE, 0>(ka[0], kr);
  pa_key_read<ROPE, 1>(ka[1], kr);
  pa_key_read<ROPE, 2>(ka[2], kr);
}
AMLA_DEV void pa_have_keys(u32x4 (&ka)[PA_AHEAD + 1][2]) {
  u32x4 a = ka[0][0], b = ka[0][1], d = ka[1][0], e = ka[1][1], g = ka[2][0], h = ka[2][1];
  asm volatile("s_waitcnt lgkmcnt(0)" : "+v"(a), "+v"(b), "+v"(d), "+v"(e), "+v"(g), "+v"(h)::"memory");
  ka[0][0] = a;
  ka[0][1] = b;
  ka[1][0] = d;
  ka[1][1] = e;
  ka[2][0] = g;
  ka[2][1] = h;
}

// A copy that the compiler does not see through: a score that outlives its tile by another name would be moved right behind
// the product that makes it, before it is there.
AMLA_DEV float pa_copy(float x) {
  float y;
  asm("v_mov_b32 %0, %1" : "=v"(y) : "v"(x));
  return y;
}
// Eight scores of group G in value slot N = 0 .. 7: their mask (keys lo .. lim - 1 of the tile are seen by the lane's query)
// and maximum; the second 32 keys go to t
template <bool ROPE, bool MASK, int N> AMLA_DEV void pa_max(PackedWave<ROPE> &w, int lo, int lim) {
  constexpr int G = N & 1, KEYS = N >> 2, HALF = (N >> 1) & 1;
#pragma unroll
  for (int i = 8 * HALF; i < 8 * HALF + 8; i += 2) {
    float z[2] = {w.s[G][KEYS][i], w.s[G][KEYS][i + 1]};
    if constexpr (MASK) {
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const int key = 32 * KEYS + 8 * (i >> 2) + (i & 3) + k;
        z[k] = key < lim && key >= lo ? z[k] : -INFINITY;
      }
      if constexpr (KEYS == 0) {
        w.s[G][0][i] = z[0];
        w.s[G][0][i + 1] = z[1];
      } else {
        w.t[G][i] = z[0];
        w.t[G][i + 1] = z[1];
      }
    }
    w.top[G] = __builtin_fmaxf(__builtin_fmaxf(w.top[G], z[0]), z[1]);
  }
  if constexpr (!MASK) {
#pragma unroll
    for (int i = 4 * (N >> 1); i < 4 * (N >> 1) + 4; ++i) w.t[G][i] = pa_copy(w.s[G][1][i]);
  }
}
// Both lanes of a query agree on its largest score so far; the first one sets its reference
AMLA_DEV void pa_refer(float &top, float &m, float c) {
  const auto sw = __builtin_amdgcn_permlane32_swap(__float_as_uint(top), __float_as_uint(top), false, false);
  top = __builtin_fmaxf(__uint_as_float(sw[0]), __uint_as_float(sw[1]));
  m = m == PA_NONE ? __builtin_fmaxf(top * c, PA_NONE) : m;
}
// What goes behind value product N: a part of the mask and the maximum of the scores (0 .. 7), the reference, then an early
// probability each
template <bool ROPE, bool MASK, bool SOFT, int N>
AMLA_DEV void pa_value_slot(PackedWave<ROPE> &w, u32x4 (&pn)[2][4], float c, int lo, int lim0, int lim1) {
  if constexpr (SOFT) {
    if constexpr (N < 8) {
      pa_max<ROPE, MASK, N>(w, lo, N & 1 ? lim1 : lim0);
    } else {
      if constexpr (N == 8) {
        pa_refer(w.top[0], w.m[0], c);
        pa_refer(w.top[1], w.m[1], c);
      }
      pa_soft_early<ROPE, N - 8>(w, pn, c);
    }
  }
  __builtin_amdgcn_sched_barrier(0);
}
// Step C of the outputs: 32 columns C / 2, keys 32 (C % 2) .. + 31.  SOFT: the tile to come is met before step 6, and
// its first keys are read.
template <bool ROPE, bool MASK, bool SOFT, int C>
AMLA_DEV void pa_value_step(PackedWave<ROPE> &w, u32x4 (&ka)[PA_AHEAD + 1][2], u32x2 (&vv)[PA_AHEAD + 1][4], u32x4 (&pn)[2][4],
                            uint32_t v0, uint32_t next, float c, int lo, int lim0, int lim1) {
  if constexpr (C < 8) {
    constexpr int A = PA_AHEAD, cb = C >> 1, kk = 2 * (C & 1);
    pa_val_read<C + A>(vv[(C + A) % (A + 1)], v0);
    if constexpr (SOFT && C == 6) pa_arrive();
    else if constexpr (!SOFT || C < 6) pa_wait<4 * (7 - C < A ? 7 - C : A)>();
    u32x2 a = vv[C % (A + 1)][0], b = vv[C % (A + 1)][1], d = vv[C % (A + 1)][2], e = vv[C % (A + 1)][3];
    pa_tie(a);
    pa_tie(b);
    pa_tie(d);
    pa_tie(e);
    if constexpr (SOFT && C == 6) pa_first_keys<ROPE>(ka, pa_key_addr<ROPE>(next));
    const bf16x8 x = as_bf16x8(u32x4{a.x, a.y, b.x, b.y}), y = as_bf16x8(u32x4{d.x, d.y, e.x, e.y});
    pa_value<true>(w.o[0][cb], x, as_bf16x8(w.p[0][kk]));
    pa_value_slot<ROPE, MASK, SOFT, 4 * C>(w, pn, c, lo, lim0, lim1);
    pa_value<false>(w.o[1][cb], x, as_bf16x8(w.p[1][kk]));
    pa_value_slot<ROPE, MASK, SOFT, 4 * C + 1>(w, pn, c, lo, lim0, lim1);
    pa_value<true>(w.o[0][cb], y, as_bf16x8(w.p[0][kk + 1]));
    pa_value_slot<ROPE, MASK, SOFT, 4 * C + 2>(w, pn, c, lo, lim0, lim1);
    pa_value<false>(w.o[1][cb], y, as_bf16x8(w.p[1][kk + 1]));
    pa_value_slot<ROPE, MASK, SOFT, 4 * C + 3>(w, pn, c, lo, lim0, lim1);
    pa_value_step<ROPE, MASK, SOFT, C + 1>(w, ka, vv, pn, v0, next, c, lo, lim0, lim1);
  }
}
// A tile (its keys at now): scores, while what is left of the tile before becomes probabilities and the tile to come (next)
// is copied; then O^T += V^T P^T of the tile before while the scores are masked and the first of them become probabilities
template <bool ROPE, bool MASK>
AMLA_DEV void pa_tile(PackedWave<ROPE> &w, u32x4 (&ka)[PA_AHEAD + 1][2], uint32_t now, uint32_t before, uint32_t next, uint8_t *st,
                      float c, const PackedFeed &f, int lo, int lim0, int lim1) {
  const uint32_t v0 = pa_val_addr<ROPE>(before);
  u32x2 vv[PA_AHEAD + 1][4];
  u32x4 pn[2][4];
  pa_score_step<ROPE, 0>(w, ka, vv, pa_key_addr<ROPE>(now), v0, c, f, st);
  pa_soft_end<ROPE>(w);
  // (one statement: a move of the scores between the wait and them would read them too early)
  asm volatile("s_nop 7\n\ts_nop 7\n\ts_nop 7" : "+v"(w.s[0][0]), "+v"(w.s[0][1]), "+v"(w.s[1][0]), "+v"(w.s[1][1])::"memory");
  pa_value_step<ROPE, MASK, true, 0>(w, ka, vv, pn, v0, next, c, lo, lim0, lim1);
  pa_have_keys(ka);
#pragma unroll
  for (int g = 0; g < 2; ++g) {
    w.p[g][0] = pn[g][0];
    w.p[g][1].x = pn[g][1].x;
    w.u[g] = f32x4{pa_copy(w.s[g][0][12]), pa_copy(w.s[g][0][13]), pa_copy(w.s[g][0][14]), pa_copy(w.s[g][0][15])};
  }
}
// What is left of the last tile's probabilities, and its part of the outputs
template <bool ROPE, int I = 0> AMLA_DEV void pa_last(PackedWave<ROPE> &w, uint32_t before, float c) {
  if constexpr (I < 2 * (32 - PA_EARLY)) {
    pa_soft_late<ROPE, I>(w, c);
    pa_last<ROPE, I + 1>(w, before, c);
  } else {
    pa_soft_end<ROPE>(w);
#pragma unroll
    for (int g = 0; g < 2; ++g) w.l[g] += w.x[g][0] + w.x[g][1];
    const uint32_t v0 = pa_val_addr<ROPE>(before);
    u32x4 ka[PA_AHEAD + 1][2], pn[2][4];
    u32x2 vv[PA_AHEAD + 1][4];
    pa_val_read<0>(vv[0], v0);
    pa_val_read<1>(vv[1], v0);
    pa_val_read<2>(vv[2], v0);
    pa_value_step<ROPE, false, false, 0>(w, ka, vv, pn, v0, 0, c, 0, 0, 0);
  }
}

// The LDS stages in turn: the tile in work, the one before it, the one on its way
template <bool ROPE> struct PackedStages {
  uint32_t first, now, before;
  AMLA_DEV uint32_t next() const {
    const uint32_t n = now + PackedWave<ROPE>::STAGE;
    return n == first + PA_NST * PackedWave<ROPE>::STAGE ? first : n;
  }
  AMLA_DEV void advance() {
    before = now;
    now = next();
  }
};

// A group's sums times inv as rows of 256 bytes in LDS (the lane's at turn): chunk ch of a row at ch ^ (row & 15)
template <bool F16> AMLA_DEV void pa_turn_rows(uint8_t *turn, const f32x16 (&o)[4], float inv, bool none) {
  const int lane = threadIdx.x & 63, j32 = lane & 31, hh = lane >> 5;
#pragma unroll
  for (int cb = 0; cb < 4; ++cb)
#pragma unroll
    for (int q4 = 0; q4 < 4; ++q4) {
      float x[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] = none ? 0.f : o[cb][4 * q4 + i] * inv;  // (no key seen: what the products left does not count)
      *reinterpret_cast<u32x2 *>(turn + 16 * ((4 * cb + q4) ^ (j32 & 15)) + 8 * hh) =
          F16 ? u32x2{pack_f16(x[0], x[1]), pack_f16(x[2], x[3])} : u32x2{pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3])};
    }
}

// ROPE: 64 more key columns beside the first 128.  One workgroup of four waves per head, block of 256 queries and split.
// SPLIT: calls of one split a block keep a shorter kernel (1 % of five prompts of 4099 rows, 352 us after 355 on one card).
template <bool ROPE, bool SPLIT>
__global__ __launch_bounds__(256, 1) void packed_attn_kernel(PackedParams p) {
  extern __shared__ __align__(1024) uint8_t sm[];
  using W = PackedWave<ROPE>;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int j32 = lane & 31, hh = lane >> 5;

  // workgroup i runs on XCD i % 8: a head's blocks, and heads that share keys, come from the same L2 where heads divide
  const int i = blockIdx.x % p.heads, unit = blockIdx.x / p.heads;
  const int h = p.heads % 8 ? i : (i & 7) * (p.heads >> 3) + (i >> 3);
  const int tile0 = SPLIT ? unit / p.splits : unit, split = SPLIT ? unit % p.splits : 0;
  const PackedBlock blk = find_block(p, tile0);
  if (blk.block < 0) return;
  int splits = 1, first_key = 0, last_key = blk.nk;
  if constexpr (SPLIT) {  // the split's keys: as a sequence that begins and ends with them
    const int keys = block_keys(p, blk), all = (keys + PA_KT - 1) / PA_KT;
    splits = block_splits(p, keys);
    if (split >= splits) return;
    first_key = (int)((int64_t)split * all / splits) * PA_KT;
    if (splits > 1) last_key = min(blk.nk, (int)((int64_t)(split + 1) * all / splits) * PA_KT);
  }
  const int q0 = blk.q0, nq = blk.nq, nk = last_key - first_key;
  const int64_t k0 = blk.k0 + first_key;
  const int s_begin = blk.block * PA_QB, s_wave = s_begin + 64 * wave;
  const int past = blk.nk - nq - first_key;  // keys before the first query's own (causal)
  const int klim = p.causal ? min(nk, max(past + min(s_begin + PA_QB, nq), 0)) : nk;  // keys that the block needs
  const int ntiles = (klim + PA_KT - 1) / PA_KT;
  // keys that the wave's first query sees, and its last one
  const int seen_all = s_wave >= nq ? 0 : p.causal ? min(max(past + s_wave + 1, 0), nk) : nk;
  const int seen_any = s_wave >= nq ? 0 : p.causal ? min(max(past + min(s_wave + 64, nq), 0), nk) : nk;
  const int n_any = (seen_any + PA_KT - 1) / PA_KT;
  // tiles wholly seen by all of the wave's queries, and by all of the block's; the last one may be loaded from further ahead
  const int n_all = min(seen_all / PA_KT, klim / PA_KT);
  const int n_block = min((p.causal ? min(max(past + s_begin + 1, 0), nk) : nk) / PA_KT, klim / PA_KT);

  const int kvh = h / p.group;
  PackedFeed f;
  f.k = reinterpret_cast<const char *>(p.k + k0 * p.ldk + kvh * p.ldk_head);
  f.v = reinterpret_cast<const char *>(p.v + k0 * p.ldv + kvh * p.ldv_head);
  f.pe = p.k_pe ? reinterpret_cast<const char *>(p.k_pe + k0 * p.ld_pe) : f.k + 256;
  f.ldk = 2 * p.ldk;
  f.ldv = 2 * p.ldv;
  f.ldpe = p.k_pe ? 2 * p.ld_pe : f.ldk;
  f.klim = klim;
  f.row0 = 16 * wave;
  f.init(lane);
  if (ntiles > 0) f.copy_first<ROPE>(sm, lane);

  W w;
  int lim[2];  // keys [0, lim) are seen by the lane's query of each group
#pragma unroll
  for (int g = 0; g < 2; ++g) {
    const int iq = min(s_wave + 32 * g + j32, nq - 1);
    const uint16_t *qp = p.q + (size_t)(q0 + iq) * p.ldq + h * p.ldq_head + 8 * hh;
#pragma unroll
    for (int ks = 0; ks < W::KS; ++ks) w.q[g][ks] = as_bf16x8(ldg16(qp + 16 * ks));
    lim[g] = (p.causal ? min(past + iq + 1, nk) : nk) - 4 * hh;
    w.m[g] = PA_NONE;
  }
  const uint32_t lds0 = (uint32_t)reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) const uint8_t *)sm);
  const float c = p.scale_log2;

  // Once; again where m turned out too low, or where an output is no number: then without the values that are none in
  // tiles that some query does not see all of (they would come through a probability of 0), which enter at the end.  (Looking
  // at each such tile first cost 5 in 100 of five prompts' time.)
  bool careful = false, odd = false;  // odd: clean() took something out
  for (;;) {
#pragma unroll
    for (int g = 0; g < 2; ++g) {
#pragma unroll
      for (int cb = 0; cb < 4; ++cb) {
#pragma unroll
        for (int r = 0; r < 16; ++r) w.o[g][cb][r] = 0.f;
      }
#pragma unroll
      for (int r = 0; r < 16; ++r) w.t[g][r] = -INFINITY;
      w.u[g] = f32x4{-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
      for (int k = 0; k < 4; ++k) w.p[g][k] = u32x4{0, 0, 0, 0};
      w.l[g] = w.x[g][0] = w.x[g][1] = 0.f;
      w.top[g] = -INFINITY;
    }
    pa_settle(w.o);
    // nothing before the first tile: probabilities and values of 0
    PackedStages<ROPE> at{lds0, lds0, lds0 + (PA_NST - 1) * W::STAGE};
    for (int o = threadIdx.x * 16; o < 2 * PA_HALF; o += 4096)
      *reinterpret_cast<u32x4 *>(sm + (PA_NST - 1) * W::STAGE + W::VAL + o) = u32x4{0, 0, 0, 0};
    u32x4 ka[PA_AHEAD + 1][2];
    pa_arrive();
    pa_first_keys<ROPE>(ka, pa_key_addr<ROPE>(lds0));
    pa_have_keys(ka);
    int j = 0;
    for (; j < (careful ? min(n_block, n_all) : n_all); ++j) {
      f.aim(j + 1);
      pa_tile<ROPE, false>(w, ka, at.now, at.before, at.next(), sm + (at.next() - lds0), c, f, 0, 0, 0);
      at.advance();
    }
    for (; j < n_any; ++j) {
      f.aim(j + 1);
      if (careful) odd |= f.clean<ROPE>(sm + (at.now - lds0), lane);
      const int first = f.first(j);
      pa_tile<ROPE, true>(w, ka, at.now, at.before, at.next(), sm + (at.next() - lds0), c, f, j * PA_KT - first - 4 * hh,
                          lim[0] - first, lim[1] - first);
      at.advance();
    }
    pa_last<ROPE>(w, at.before, c);
    for (; j < ntiles; ++j) {  // the wave's queries see no more: it goes on copying for the others
      f.aim(j + 1);
      if (careful && j >= n_block) odd |= f.clean<ROPE>(sm + (at.now - lds0), lane);
      f.copy_all<ROPE>(sm + (at.next() - lds0));
      pa_arrive();
      at.advance();
    }
    pa_settle(w.o);
    wait_vmcnt<0>();  // (copies past the last tile)
    const bool low0 = w.top[0] * c > w.m[0] + PA_LAG, low1 = w.top[1] * c > w.m[1] + PA_LAG;
    float none[2] = {0.f, 0.f};  // 0, or NaN where an output is infinite or NaN
#pragma unroll
    for (int g = 0; g < 2; ++g)
#pragma unroll
      for (int cb = 0; cb < 4; ++cb)
#pragma unroll
        for (int r = 0; r < 16; ++r) none[g] = __builtin_fmaf(w.o[g][cb][r], 0.f, none[g]);
    // the waves agree: their copies and barriers are common
    const bool low = __ballot(low0 || low1) != 0;
    // of queries that see a key: by either lane's keys, the other one may have the column
    float seen[2];
#pragma unroll
    for (int g = 0; g < 2; ++g) {
      const auto sw = __builtin_amdgcn_permlane32_swap(__float_as_uint(w.l[g]), __float_as_uint(w.l[g]), false, false);
      seen[g] = __uint_as_float(sw[0]) + __uint_as_float(sw[1]);
    }
    const bool strange = __ballot((seen[0] != 0.f && none[0] != 0.f) || (seen[1] != 0.f && none[1] != 0.f)) != 0;
    __syncthreads();
    uint32_t *vote = reinterpret_cast<uint32_t *>(sm);
    if (lane == 0) vote[wave] = (low ? 1 : 0) | (odd ? 2 : 0) | (strange ? 4 : 0);
    __syncthreads();
    const uint32_t votes = vote[0] | vote[1] | vote[2] | vote[3];
    __syncthreads();
    odd = votes & 2;
    if (!(votes & 1) && (careful || !(votes & 4))) break;
    careful |= (votes & 4) != 0;
    w.m[0] = low0 ? w.top[0] * c : w.m[0];
    w.m[1] = low1 ? w.top[1] * c : w.m[1];
    f.copy_first<ROPE>(sm, lane);
  }

  // outputs: rows of 256 bytes through LDS (chunk ch of a row at ch ^ (row & 15)), so that a store is whole rows
  uint8_t *turn = sm + wave * 64 * 256;
  const size_t slot = ((size_t)tile0 * p.heads + h) * p.splits + split;
  const bool part = SPLIT && splits > 1;
#pragma unroll
  for (int g = 0; g < 2; ++g) {
    float l = w.l[g];
    const auto sw = __builtin_amdgcn_permlane32_swap(__float_as_uint(l), __float_as_uint(l), false, false);
    l = __uint_as_float(sw[0]) + __uint_as_float(sw[1]);
    float inv = l == 0.f ? 0.f : 1.f / l;
    const int r = 32 * g + j32;
    const float lse2 = l == 0.f ? -INFINITY : w.m[g] + __builtin_amdgcn_logf(l);
    // the row's largest value to 2^14 .. 2^15, or as near as inv times that power stays finite: all of them may be 0 where l is
    // below 1 (by the rounding of m: down to 2^-16 for scores of 2^28)
    if (part) {
      float top = 0.f;
#pragma unroll
      for (int cb = 0; cb < 4; ++cb)
#pragma unroll
        for (int k = 0; k < 16; ++k) top = __builtin_fmaxf(top, __builtin_fabsf(w.o[g][cb][k]));
      if (__ballot(top == INFINITY)) {  // of the finite ones
        top = 0.f;
#pragma unroll
        for (int cb = 0; cb < 4; ++cb)
#pragma unroll
          for (int k = 0; k < 16; ++k) {
            const float x = __builtin_fabsf(w.o[g][cb][k]);
            top = x < INFINITY ? __builtin_fmaxf(top, x) : top;
          }
      }
      const auto sx = __builtin_amdgcn_permlane32_swap(__float_as_uint(top), __float_as_uint(top), false, false);
      top = __builtin_fmaxf(__uint_as_float(sx[0]), __uint_as_float(sx[1])) * inv;
      const int least = max((int)(__float_as_uint(inv) >> 23) - 112, 15);
      const int e = min(max((int)(__float_as_uint(top) >> 23), least), 240) - 14;
      inv *= __uint_as_float((uint32_t)(254 - e) << 23);
      if (hh == 0) {
        float *ls = p.part_ls + 2 * (slot * PA_QB + 64 * wave + r);
        ls[0] = lse2;
        ls[1] = __uint_as_float((uint32_t)e << 23);
      }
      pa_turn_rows<true>(turn + r * 256, w.o[g], inv, l == 0.f);
    } else {
      if (p.lse && hh == 0 && s_wave + r < nq) p.lse[(size_t)(q0 + s_wave + r) * p.heads + h] = lse2 * 0.6931471805599453f;
      pa_turn_rows<false>(turn + r * 256, w.o[g], inv, l == 0.f);
    }
  }
  const int held = min(64, nq - s_wave);
  if (__builtin_amdgcn_readfirstlane((int)odd)) {  // infinities and NaN enter the outputs of the queries that see them
    for (int key = n_block * PA_KT; key < seen_any; ++key) {
      const uint32_t x = reinterpret_cast<const uint32_t *>(f.v + key * f.ldv)[lane];
      const bool lo = (x & 0x7f80u) == 0x7f80u, hi = (x & 0x7f800000u) == 0x7f800000u;
      if (!__ballot(lo || hi)) continue;
      for (int r = p.causal ? max(key - past - s_wave, 0) : 0; r < held; ++r) {
        uint32_t *at = reinterpret_cast<uint32_t *>(turn + r * 256 + 16 * ((lane >> 2) ^ (r & 15)) + 4 * (lane & 3));
        const uint32_t y = *at;
        const float a = part ? lo_f16(y) : lo_bf(y), b = part ? hi_f16(y) : hi_bf(y);
        const float c0 = lo ? a + lo_bf(x) : a, c1 = hi ? b + hi_bf(x) : b;
        *at = part ? pack_f16(c0, c1) : pack_bf16(c0, c1);
      }
    }
  }
  uint16_t *od = p.out + ((size_t)(q0 + s_wave) * p.heads + h) * PA_VD;
  size_t ld = (size_t)p.heads * PA_VD;
  if (part) {
    od = p.part_o + (slot * PA_QB + 64 * wave) * PA_VD;
    ld = PA_VD;
  }
#pragma unroll 4
  for (int r0 = 0; r0 < 64; r0 += 4) {
    const int r = r0 + (lane >> 4), ch = lane & 15;
    if (r < held)
      *reinterpret_cast<u32x4 *>(od + r * ld + 8 * ch) = *reinterpret_cast<const u32x4 *>(turn + r * 256 + 16 * (ch ^ (r & 15)));
  }
}

// Joins the splits of 32 rows of a block: sum_j 2^(lse_j - max) O_j / sum_j 2^(lse_j - max), 16 lanes a row, in split order.
__global__ __launch_bounds__(256) void packed_join_kernel(PackedParams p) {
  const int h = blockIdx.x % p.heads, tile0 = blockIdx.x / p.heads;
  const PackedBlock blk = find_block(p, tile0);
  if (blk.block < 0) return;
  const int splits = block_splits(p, block_keys(p, blk));
  if (splits == 1) return;
  const size_t slot = ((size_t)tile0 * p.heads + h) * p.splits;
  const int ch = threadIdx.x & 15;
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const int r = 32 * blockIdx.y + 16 * k + (threadIdx.x >> 4), row = blk.block * PA_QB + r;
    if (row >= blk.nq) continue;
    const float *ls = p.part_ls + 2 * (slot * PA_QB + r);
    const uint16_t *po = p.part_o + (slot * PA_QB + r) * PA_VD + 8 * ch;
    float top = -INFINITY;
    for (int j = 0; j < splits; ++j) top = __builtin_fmaxf(top, ls[(size_t)j * 2 * PA_QB]);
    const float ref = top == -INFINITY ? 0.f : top;
    float total = 0.f, a[8] = {};
#pragma unroll 4
    for (int j = 0; j < splits; ++j) {
      const f32x2 l = *reinterpret_cast<const f32x2 *>(ls + (size_t)j * 2 * PA_QB);
      const u32x4 v = ldg16(po + (size_t)j * PA_QB * PA_VD);
      const float f = __builtin_amdgcn_exp2f(l.x - ref);
      total += f;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint32_t x = v[e];
        a[2 * e] = __builtin_fmaf(f, lo_f16(x) * l.y, a[2 * e]);
        a[2 * e + 1] = __builtin_fmaf(f, hi_f16(x) * l.y, a[2 * e + 1]);
      }
    }
    const float inv = total == 0.f ? 0.f : 1.f / total;
    const size_t at = (size_t)(blk.q0 + row) * p.heads + h;
    *reinterpret_cast<u32x4 *>(p.out + at * PA_VD + 8 * ch) =
        u32x4{pack_bf16(a[0] * inv, a[1] * inv), pack_bf16(a[2] * inv, a[3] * inv), pack_bf16(a[4] * inv, a[5] * inv),
              pack_bf16(a[6] * inv, a[7] * inv)};
    if (ch == 0 && p.lse) p.lse[at] = total == 0.f ? -INFINITY : (top + __builtin_amdgcn_logf(total)) * 0.6931471805599453f;
  }
}

template <bool ROPE, bool SPLIT>
static int launch_packed(const PackedParams &p, int64_t blocks, hipStream_t st) {
  constexpr int lds = PackedWave<ROPE>::STAGE * PA_NST;
  const int rc = latent_lds(packed_attn_kernel<ROPE, SPLIT>, "packed_attention");
  if (rc) return rc;
  packed_attn_kernel<ROPE, SPLIT><<<dim3((unsigned)blocks * p.splits), 256, lds, st>>>(p);
  const int err = check_launch("packed_attention");
  if (err || !SPLIT) return err;
  packed_join_kernel<<<dim3((unsigned)blocks, PA_QB / 32), 256, 0, st>>>(p);
  return check_launch("packed_attention join");
}

// Query blocks of a call, at least those there are
static int64_t packed_blocks(int64_t q_rows, int64_t seqs) { return q_rows / PA_QB + std::min(seqs, q_rows); }
// Splits of a block, at most: where blocks times heads leave half of the CUs idle.  One or 64 rows of 16 heads behind 4000
// keys: 111 -> 28 and 114 -> 36 us, 1000 rows 150 -> 94, 16 rows of 128 heads 113 -> 69, 4000 rows of 8 heads 105 -> 78.
// With 256 blocks and heads nothing was won (4000 rows of 16 heads: 121, 124 split), few keys only pay for the join.
static int packed_splits(int64_t units, int64_t k_rows) {
  return units > 128 || k_rows <= PA_LEAST * PA_KT ? 1 : (int)std::min<int64_t>(32, 512 / units);
}

}  // namespace amla

using namespace amla;

extern "C" size_t amla_packed_attention_workspace_bytes(int64_t q_rows, int64_t k_rows, int64_t seqs, int64_t heads) {
  if (q_rows <= 0 || k_rows < 0 || seqs <= 0 || heads <= 0 || q_rows > INT32_MAX || seqs > AMLA_MAX_SEQS || heads > INT32_MAX) return 0;
  const int64_t units = packed_blocks(q_rows, seqs) * heads;
  const int splits = packed_splits(units, k_rows);
  return splits == 1 ? 0 : (size_t)units * splits * PA_QB * (PA_VD * 2 + 8);
}

extern "C" int amla_packed_attention(const amla_packed_args *a, void *stream) {
  const char *what = "packed_attention";
  if (!a) return fail(AMLA_EINVAL, "%s: null pointer", what);
  if (a->q_rows < 0 || a->k_rows < 0 || a->seqs < 0 || a->heads < 0 || a->kv_heads < 0)
    return fail(AMLA_EINVAL, "%s: negative size", what);
  if (a->q_rows == 0 || a->heads == 0 || a->seqs == 0) return AMLA_OK;
  if (!a->q || !a->out || !a->offsets || (a->k_rows && (!a->k || !a->v))) return fail(AMLA_EINVAL, "%s: null pointer", what);
  if (a->kv_heads == 0 || a->heads % a->kv_heads)
    return fail(AMLA_EINVAL, "%s: %d heads do not share %d keys evenly", what, a->heads, a->kv_heads);
  if ((a->dn != 128 && a->dn != 192) || (a->k_pe && a->dn != 128))
    return fail(AMLA_EUNSUPPORTED, "%s: keys of 128 values (with or without k_pe) or of 192 (dn=%d)", what, a->dn);
  if (!(a->scale > 0.f) || !(a->scale < INFINITY)) return fail(AMLA_EINVAL, "%s: scale must be positive", what);
  if (a->q_rows > PA_MAX_ROWS || a->k_rows > PA_MAX_ROWS || a->seqs > AMLA_MAX_SEQS)
    return fail(AMLA_EUNSUPPORTED, "%s: at most %d rows and %d sequences", what, PA_MAX_ROWS, AMLA_MAX_SEQS);
  const int64_t lds[] = {a->ldq, a->ldq_head, a->ldk, a->ldk_head, a->ldv, a->ldv_head, a->k_pe ? a->ld_pe : 0};
  for (int64_t ld : lds)
    if (ld % 8 || ld < 0 || ld > (1 << 27)) return fail(AMLA_EUNSUPPORTED, "%s: strides must be multiples of 8 values up to 2^27", what);
  if (!aligned16(a->q) || !aligned16(a->k) || !aligned16(a->v) || !aligned16(a->k_pe) || !aligned16(a->out))
    return fail(AMLA_EUNSUPPORTED, "%s: tensors must be 16-byte aligned", what);
  const int64_t tiles = packed_blocks(a->q_rows, a->seqs);
  if (tiles * a->heads > (1 << 23)) return fail(AMLA_EUNSUPPORTED, "%s: too many query blocks", what);
  const size_t need = amla_packed_attention_workspace_bytes(a->q_rows, a->k_rows, a->seqs, a->heads);
  if (need && (!a->workspace || a->workspace_bytes < need)) return fail(AMLA_EWORKSPACE, "%s: workspace too small", what);
  if (need && !aligned16(a->workspace)) return fail(AMLA_EUNSUPPORTED, "%s: workspace must be 16-byte aligned", what);
  PackedParams p = {};
  p.splits = packed_splits(tiles * a->heads, a->k_rows);
  p.part_o = static_cast<uint16_t *>(a->workspace);
  p.part_ls = reinterpret_cast<float *>(p.part_o + (size_t)tiles * a->heads * p.splits * PA_QB * PA_VD);
  p.q = static_cast<const uint16_t *>(a->q); p.k = static_cast<const uint16_t *>(a->k);
  p.v = static_cast<const uint16_t *>(a->v); p.k_pe = static_cast<const uint16_t *>(a->k_pe);
  p.out = static_cast<uint16_t *>(a->out); p.lse = a->lse;
  p.offsets = a->offsets; p.k_offsets = a->k_offsets ? a->k_offsets : a->offsets;
  p.q_rows = (int)a->q_rows; p.k_rows = (int)a->k_rows; p.seqs = (int)a->seqs;
  p.heads = a->heads; p.group = a->heads / a->kv_heads; p.causal = a->causal != 0;
  p.ldq = a->ldq; p.ldq_head = a->ldq_head; p.ldk = a->ldk; p.ldk_head = a->ldk_head;
  p.ldv = a->ldv; p.ldv_head = a->ldv_head; p.ld_pe = a->ld_pe;
  p.scale_log2 = a->scale * 1.4426950408889634f;
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  const int64_t blocks = tiles * a->heads;
  if (a->dn == 192 || a->k_pe) return p.splits > 1 ? launch_packed<true, true>(p, blocks, st) : launch_packed<true, false>(p, blocks, st);
  return p.splits > 1 ? launch_packed<false, true>(p, blocks, st) : launch_packed<false, false>(p, blocks, st);
}
