// The paged latent cache: rows, pages and packed sequences, shared by the kernels that
// write, read and attend to it.
//
// A row is 512 latent values and a 64-wide rope key in bf16.  Latents are bf16, or e4m3
// codes with one exponent byte per row: value = code * 2^(byte - 127).  One power of two
// for the row rather than one per block: e4m3 has 17 binades of its own, so a row's
// small values keep their three mantissa bits, and attention can move the factor from
// the values to the probabilities, which leaves the codes themselves as operands of the
// matrix units.  Row i of a sequence is row i % page_size of page table[i / page_size].
#pragma once

#include "amla_common.h"
#include "amla_internal.h"

namespace amla {

constexpr int LC_LORA = 512, LC_ROPE = 64;
constexpr int LC_EXP_MAX = 32;  // exponents are clamped to +-32: attention scales sums by their differences

struct LatentPages {
  uint8_t *latent;   // (pages * page_size, 512) e4m3 or bf16
  uint16_t *k_pe;    // (pages * page_size, 64)
  uint8_t *scales;   // (pages * page_size) exponent bytes; null: bf16 latents
  const int32_t *table;
  int64_t ld_table;
  int32_t pages, cols;
  int page_shift;    // page_size = 1 << page_shift
  // The table's entry for row t >= 0 of sequence b (-1 past the table), and the pool row it means: -1 for none.
  AMLA_DEV int page(int b, int t) const {
    const int c = t >> page_shift;
    return c < cols ? table[b * ld_table + c] : -1;
  }
  AMLA_DEV int row(int page, int t) const {
    return (uint32_t)page < (uint32_t)pages ? (page << page_shift) + (t & ((1 << page_shift) - 1)) : -1;
  }
  AMLA_DEV int slot(int b, int t) const { return row(page(b, t), t); }
};

// 64 lanes x 16 bytes from per-lane addresses to 1 KB of LDS.  Functions of their own, not templates: inside
// one the host pass of the compiler drops the enclosing kernel without a word.
AMLA_DEV void copy_lds(const void *src, void *dst) { __builtin_amdgcn_global_load_lds(src, LDS_PTR(dst), 16, 0, 0); }
AMLA_DEV void copy_lds_nt(const void *src, void *dst) { __builtin_amdgcn_global_load_lds(src, LDS_PTR(dst), 16, 0, 2); }

// Two values in fp16, to nearest even
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
AMLA_DEV uint32_t pack_f16(float a, float b) { return __builtin_bit_cast(uint32_t, f16x2{(_Float16)a, (_Float16)b}); }
AMLA_DEV float lo_f16(uint32_t x) { return (float)__builtin_bit_cast(f16x2, x)[0]; }
AMLA_DEV float hi_f16(uint32_t x) { return (float)__builtin_bit_cast(f16x2, x)[1]; }

// Host checks of a cache shared by its entry points: 0 or the code of fail().
int latent_pages(const amla_latent_cache *c, const char *what, LatentPages *p);

// Lets a kernel have all of a CU's LDS; per call, since it holds for the current device.
template <typename F> inline int latent_lds(F *fn, const char *what) {
  const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void *>(fn), hipFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024);
  return e == hipSuccess ? AMLA_OK : fail((int)e, "%s: LDS size: %s", what, hipGetErrorString(e));
}

// The sequence of packed row i (the same in every lane): the number of b with
// offsets[b + 1] <= i, for ascending offsets; seqs if none holds it.  All loads of 64
// offsets each are independent, so it takes one round trip, not one per halving.
AMLA_DEV int packed_seq(const int32_t *offsets, int seqs, int i) {
  const int lane = threadIdx.x & 63;
  int n = 0;
  for (int b = 0; b < seqs; b += 64) {
    const bool past = b + lane < seqs && offsets[b + lane + 1] <= i;
    n += __popcll(__ballot(past));
  }
  return n;
}

// Where packed rows belong: row i of the packed tensor is row positions[b] + (i - first
// row of b) of sequence b.  offsets null: `each` rows per sequence.
struct PackedRows {
  const int32_t *offsets, *positions;
  int seqs, each;
  // (sequence, row of the sequence) of row i (the same in every lane); sequence -1 for none
  AMLA_DEV int2 at(int i) const {
    int b, first;
    if (offsets) {
      b = packed_seq(offsets, seqs, i);
      if (b >= seqs) return int2{-1, 0};
      first = offsets[b];
    } else {
      b = i / each;
      first = b * each;
    }
    const int64_t t = (positions ? (int64_t)positions[b] : 0) + ((int64_t)i - first);
    return t < 0 || i < first || t > INT32_MAX ? int2{-1, 0} : int2{b, (int)t};
  }
};

}  // namespace amla
