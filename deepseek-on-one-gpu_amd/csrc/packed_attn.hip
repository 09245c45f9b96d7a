// Attention of packed prompts: sequences of different lengths one after another, causal or
// not, heads that share keys and values, an optional rope key shared by all heads.
//   s_ij = scale q_i . k_j,  out_i = sum_j softmax(s_i)_j v_j,  lse_i = log sum_j exp(s_ij)
// One pass over the keys with a running maximum and sum per query, all in fp32; P is
// rounded to bf16 for the matrix units (as inference/ops.py:179 rounds it).
#include <algorithm>
#include <math.h>

#include "latent.h"

namespace amla {

constexpr int PA_KT = 64;                 // keys per tile
constexpr int PA_NW = 8;                  // waves per workgroup, 32 queries each
constexpr int PA_QB = 32 * PA_NW;         // queries per workgroup
constexpr int PA_NST = 3;                 // LDS stages: copies run up to two tiles ahead
constexpr int PA_VD = 128;
constexpr float PA_LAG = 40.f;            // the running maximum moves when a score passes it by 2^40: fp32 and bf16 have the range
constexpr int PA_HALF = PA_KT * 128;      // 64 rows of 128 bytes: 64 key or value columns of a tile

struct PackedParams {
  const uint16_t *q, *k, *v, *k_pe;  // k_pe null: key columns 128.. are k's own
  uint16_t *out;
  float *lse;
  const int32_t *offsets, *k_offsets;
  int q_rows, k_rows, seqs, heads, group, causal;
  int tiles;                         // query blocks of all sequences, at most
  int64_t ldq, ldq_head, ldk, ldk_head, ldv, ldv_head, ld_pe;
  float scale_log2;
};

// Offsets are not checked on the host: clamped to the rows there are, and none below its predecessor's.
struct PackedSpan {
  int q0, nq, k0, nk;
};
AMLA_DEV int span_start(const int32_t *off, int b, int rows) { return min(max(off[b], 0), rows); }

AMLA_DEV f32x16 mfma32(bf16x8 a, bf16x8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }

// Query block `tile` of the batch: (sequence, block of it), wave-uniform; the sequence is -1 past the end.
AMLA_DEV int2 find_block(const PackedParams &p, int tile) {
  const int lane = threadIdx.x & 63;
  int base = 0;
  for (int b0 = 0; b0 < p.seqs; b0 += 64) {
    const int b = b0 + lane;
    int n = 0;
    if (b < p.seqs) n = max(span_start(p.offsets, b + 1, p.q_rows) - span_start(p.offsets, b, p.q_rows), 0);
    const int blocks = (n + PA_QB - 1) / PA_QB;
    int incl = blocks;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int v = __shfl_up(incl, o, 64);
      if (lane >= o) incl += v;
    }
    const uint64_t past = __ballot(base + incl > tile);
    if (past) {
      const int l = __builtin_ctzll(past);
      const int before = base + __builtin_amdgcn_readlane(incl, l) - __builtin_amdgcn_readlane(blocks, l);
      // a sequence's last blocks see the most keys: they go first
      return int2{b0 + l, __builtin_amdgcn_readlane(blocks, l) - 1 - (tile - before)};
    }
    base += __builtin_amdgcn_readlane(incl, 63);
  }
  return int2{-1, 0};
}

// ROPE: 64 more key columns beside the first 128
template <bool ROPE>
__global__ __launch_bounds__(64 * PA_NW, 1) void packed_attn_kernel(PackedParams p) {
  extern __shared__ __align__(16) uint8_t sm[];
  constexpr int KS = ROPE ? 12 : 8;        // 16-wide K steps
  constexpr int NK = ROPE ? 3 : 2;         // half-row arrays of keys
  constexpr int VAL = NK * PA_HALF, STAGE = (NK + 2) * PA_HALF;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int j32 = lane & 31, hh = lane >> 5, L16 = lane & 15, g16 = lane >> 4;

  const int h = blockIdx.x % p.heads;
  const int2 blk = find_block(p, blockIdx.x / p.heads);
  if (blk.x < 0) return;
  PackedSpan sp;
  sp.q0 = span_start(p.offsets, blk.x, p.q_rows);
  sp.nq = span_start(p.offsets, blk.x + 1, p.q_rows) - sp.q0;
  sp.k0 = span_start(p.k_offsets, blk.x, p.k_rows);
  sp.nk = max(span_start(p.k_offsets, blk.x + 1, p.k_rows) - sp.k0, 0);
  const int s_begin = blk.y * PA_QB, s_wave = s_begin + 32 * wave;
  const int past = sp.nk - sp.nq;  // keys before the first query's own (causal)
  const int klim = p.causal ? min(sp.nk, max(past + min(s_begin + PA_QB, sp.nq), 0)) : sp.nk;  // keys the block needs
  const int ntiles = (klim + PA_KT - 1) / PA_KT;
  const int kvh = h / p.group;

  auto copy = [&] __device__(int t0, uint8_t *st) {  // wave w: rows 8w .. 8w+7 of the tile
    const int r8 = lane >> 3, r = 8 * wave + r8;
    const size_t t = sp.k0 + min(t0 + r, klim - 1);
    const int kc = (lane & 7) ^ ((r >> 1) & 7), vc = (lane & 7) ^ (4 * ((r >> 2) & 1));
    const uint16_t *kr = p.k + t * p.ldk + kvh * p.ldk_head + 8 * kc;
    const uint16_t *vr = p.v + t * p.ldv + kvh * p.ldv_head + 8 * vc;
    uint8_t *d = st + 8 * wave * 128;
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      copy_lds(kr + 64 * half, d + half * PA_HALF);
      copy_lds(vr + 64 * half, d + VAL + half * PA_HALF);
    }
    if constexpr (ROPE)
      copy_lds(p.k_pe ? p.k_pe + t * p.ld_pe + 8 * kc : kr + 128, d + 2 * PA_HALF);
  };

  if (ntiles > 0) copy(0, sm);
  const int iq = min(s_wave + j32, sp.nq - 1);
  const uint16_t *qp = p.q + (size_t)(sp.q0 + iq) * p.ldq + h * p.ldq_head + 8 * hh;
  bf16x8 qf[KS];
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) qf[ks] = as_bf16x8(ldg16(qp + 16 * ks));
  f32x16 o[4];
#pragma unroll
  for (int c = 0; c < 4; ++c)
#pragma unroll
    for (int i = 0; i < 16; ++i) o[c][i] = 0.f;
  float m = -1e30f, l = 0.f;  // finite: exp2(-inf - m) is 0 while no key has been seen
  const int limit = p.causal ? min(past + iq + 1, sp.nk) : sp.nk;  // keys [0, limit) are seen
  const int seen_by_all = p.causal ? min(past + s_wave + 1, sp.nk) : sp.nk;

  for (int j = 0; j < ntiles; ++j) {
    uint8_t *st = sm + (j % PA_NST) * STAGE;
    if (j + 1 < ntiles) copy((j + 1) * PA_KT, sm + ((j + 1) % PA_NST) * STAGE);
    if (j + 1 < ntiles) wait_vmcnt<ROPE ? 5 : 4>();
    else wait_vmcnt<0>();
    __syncthreads();
    f32x16 s[2];
#pragma unroll
    for (int kg = 0; kg < 2; ++kg) {
      const int r = 32 * kg + j32;
#pragma unroll
      for (int i = 0; i < 16; ++i) s[kg][i] = 0.f;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        const u32x4 a = *reinterpret_cast<const u32x4 *>(st + (ks >> 2) * PA_HALF + r * 128 +
                                                         16 * ((2 * (ks & 3) + hh) ^ ((r >> 1) & 7)));
        s[kg] = mfma32(as_bf16x8(a), qf[ks], s[kg]);
      }
    }
    float mx = -INFINITY;
    const bool masked = (j + 1) * PA_KT > seen_by_all;
#pragma unroll
    for (int kg = 0; kg < 2; ++kg)
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        float z = s[kg][i] * p.scale_log2;
        if (masked && j * PA_KT + 32 * kg + 8 * (i >> 2) + 4 * hh + (i & 3) >= limit) z = -INFINITY;
        s[kg][i] = z;
        mx = __builtin_fmaxf(mx, z);
      }
    mx = __builtin_fmaxf(mx, __shfl_xor(mx, 32, 64));
    if (__ballot(mx > m + PA_LAG)) {
      const float mn = mx > m + PA_LAG ? mx : m, f = __builtin_amdgcn_exp2f(m - mn);
      m = mn;
      l *= f;
#pragma unroll
      for (int c = 0; c < 4; ++c) o[c] *= f;
    }
    u32x4 pb[4];
#pragma unroll
    for (int kg = 0; kg < 2; ++kg)
#pragma unroll
      for (int i = 0; i < 16; i += 2) {
        const float e0 = __builtin_amdgcn_exp2f(s[kg][i] - m), e1 = __builtin_amdgcn_exp2f(s[kg][i + 1] - m);
        l += e0 + e1;
        pb[2 * kg + (i >> 3)][(i >> 1) & 3] = pack_bf16(e0, e1);
      }
#pragma unroll
    for (int c = 0; c < 4; ++c)
#pragma unroll
      for (int kk = 0; kk < 4; ++kk) {
        u32x2 t[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int r = 16 * kk + 8 * i + 4 * hh + (L16 >> 2);
          const uint8_t *a = st + VAL + (c >> 1) * PA_HALF + r * 128 + 64 * ((c & 1) ^ hh) + 32 * (g16 & 1) + 8 * (L16 & 3);
          typedef short v4s __attribute__((ext_vector_type(4)));
          t[i] = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) v4s *)a));
        }
        o[c] = mfma32(as_bf16x8(u32x4{t[0].x, t[0].y, t[1].x, t[1].y}), as_bf16x8(pb[kk]), o[c]);
      }
  }

  l += __shfl_xor(l, 32, 64);
  if (s_wave + j32 >= sp.nq) return;
  const float inv = l == 0.f ? 0.f : 1.f / l;
  const size_t dst = (size_t)(sp.q0 + s_wave + j32) * p.heads + h;
  if (p.lse && hh == 0) p.lse[dst] = l == 0.f ? -INFINITY : (m + __builtin_amdgcn_logf(l)) * 0.6931471805599453f;
#pragma unroll
  for (int c = 0; c < 4; ++c)
#pragma unroll
    for (int q4 = 0; q4 < 4; ++q4)
      *reinterpret_cast<u32x2 *>(p.out + dst * PA_VD + 32 * c + 8 * q4 + 4 * hh) =
          u32x2{pack_bf16(o[c][4 * q4] * inv, o[c][4 * q4 + 1] * inv), pack_bf16(o[c][4 * q4 + 2] * inv, o[c][4 * q4 + 3] * inv)};
}

template <bool ROPE>
static int launch_packed(const PackedParams &p, int64_t blocks, hipStream_t st) {
  constexpr int lds = (ROPE ? 5 : 4) * PA_HALF * PA_NST;
  static const hipError_t attr =
      hipFuncSetAttribute((const void *)packed_attn_kernel<ROPE>, hipFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024);
  (void)attr;
  packed_attn_kernel<ROPE><<<dim3((unsigned)blocks), 64 * PA_NW, lds, st>>>(p);
  return check_launch("packed_attention");
}

}  // namespace amla

using namespace amla;

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
  if (a->q_rows > INT32_MAX || a->k_rows > INT32_MAX || a->seqs > AMLA_MAX_SEQS)
    return fail(AMLA_EUNSUPPORTED, "%s: at most 2^31 - 1 rows and %d sequences", what, AMLA_MAX_SEQS);
  const int64_t lds[] = {a->ldq, a->ldq_head, a->ldk, a->ldk_head, a->ldv, a->ldv_head, a->k_pe ? a->ld_pe : 0};
  for (int64_t ld : lds)
    if (ld % 8) return fail(AMLA_EUNSUPPORTED, "%s: strides must be multiples of 8 values", what);
  if (!aligned16(a->q) || !aligned16(a->k) || !aligned16(a->v) || !aligned16(a->k_pe) || !aligned16(a->out))
    return fail(AMLA_EUNSUPPORTED, "%s: tensors must be 16-byte aligned", what);
  const int64_t tiles = a->q_rows / PA_QB + std::min(a->seqs, a->q_rows);  // at least the blocks there are
  if (tiles * a->heads > (1 << 23)) return fail(AMLA_EUNSUPPORTED, "%s: too many query blocks", what);
  PackedParams p = {};
  p.q = static_cast<const uint16_t *>(a->q); p.k = static_cast<const uint16_t *>(a->k);
  p.v = static_cast<const uint16_t *>(a->v); p.k_pe = static_cast<const uint16_t *>(a->k_pe);
  p.out = static_cast<uint16_t *>(a->out); p.lse = a->lse;
  p.offsets = a->offsets; p.k_offsets = a->k_offsets ? a->k_offsets : a->offsets;
  p.q_rows = (int)a->q_rows; p.k_rows = (int)a->k_rows; p.seqs = (int)a->seqs;
  p.heads = a->heads; p.group = a->heads / a->kv_heads; p.causal = a->causal != 0; p.tiles = (int)tiles;
  p.ldq = a->ldq; p.ldq_head = a->ldq_head; p.ldk = a->ldk; p.ldk_head = a->ldk_head;
  p.ldv = a->ldv; p.ldv_head = a->ldv_head; p.ld_pe = a->ld_pe;
  p.scale_log2 = a->scale * 1.4426950408889634f;
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  return a->dn == 192 || a->k_pe ? launch_packed<true>(p, tiles * a->heads, st) : launch_packed<false>(p, tiles * a->heads, st);
}
