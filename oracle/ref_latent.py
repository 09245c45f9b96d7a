"""The paged latent cache and packed prompts in 64 bits on the CPU, from their definitions.

What ``amla.ops.latent_cache_write``, ``latent_cache_read``, ``latent_attention`` and
``packed_attention`` compute, one sequence after another: the RMSNorm of
inference/ops.py:10-12 without its intermediate rounding, the rotation of :86-97, the
attention of :162-182, in latent space for the cache (the reference decompresses the
latents through kv_b first; the algebra is the same with kv_b absorbed into the query).
"""
from __future__ import annotations

import torch

F64 = torch.float64
LORA, ROPE = 512, 64


def normed(kv: torch.Tensor, gamma: torch.Tensor, eps: float) -> torch.Tensor:
    x = kv[..., :LORA].to(F64)
    return x / torch.sqrt(x.square().mean(-1, keepdim=True) + eps) * gamma.to(F64)


def rotated(kv: torch.Tensor, freqs: torch.Tensor) -> torch.Tensor:
    """kv (n, 576) and its rows' freqs (n, 32) -> rotated rope keys (n, 64)."""
    z = torch.view_as_complex(kv[..., LORA:].to(F64).reshape(-1, ROPE // 2, 2).contiguous()) * freqs.to(torch.complex128)
    return torch.view_as_real(z).flatten(1)


def exponent(rows: torch.Tensor) -> torch.Tensor:
    """min { e : max |row| <= 448 2^e } in [-32, 32]."""
    top = rows.abs().amax(-1)
    e = torch.full(top.shape, -32, dtype=torch.int64)
    for k in range(-32, 32):
        e = torch.where(top > 448.0 * 2.0 ** k, k + 1, e)
    return e


def e4m3(x: torch.Tensor) -> torch.Tensor:
    """fp64 to the nearest e4m3 value (ties to even), saturating at 448."""
    a = x.abs()
    step = torch.exp2(torch.floor(torch.log2(a.clamp(min=2.0 ** -6))) - 3)
    return torch.copysign((torch.round(a / step) * step).clamp(max=448.0), x)


def code_values(codes: torch.Tensor) -> torch.Tensor:
    """e4m3fn codes (as uint8) -> fp64, from their bits."""
    b = codes.to(torch.int64)
    ef, mf = (b >> 3) & 15, (b & 7).to(F64)
    v = torch.where(ef == 0, mf * 2.0 ** -9, (8.0 + mf) * torch.exp2((ef - 10).to(F64)))
    v = torch.where((b & 127) == 127, torch.full_like(v, float("nan")), v)
    return torch.where(b >= 128, -v, v)


def places(table: torch.Tensor, b: int, t: int, page_size: int, pages: int) -> int:
    """Pool row of row t of sequence b, -1 for none."""
    c = t // page_size
    if t < 0 or c >= table.shape[1] or not 0 <= int(table[b, c]) < pages:
        return -1
    return int(table[b, c]) * page_size + t % page_size


def pool_values(cache: tuple) -> tuple:
    """(latents (rows, 512), rope keys (rows, 64)) of a CPU cache in fp64."""
    if len(cache) == 2:
        lat = cache[0].reshape(-1, LORA).to(F64)
    else:
        lat = code_values(cache[0].view(torch.uint8).reshape(-1, LORA)) * \
            torch.exp2(cache[2].reshape(-1, 1).to(F64) - 127)
    return lat, cache[1].reshape(-1, ROPE).to(F64)


def attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, scale: float, seen: torch.Tensor) -> tuple:
    """q (n, d), k (m, d), v (m, e) in fp64, seen (n, m): (softmax(scale q k^T) v, log of the sum of
    exp); what is not seen has no part in either, whatever its values."""
    s = torch.where(seen, q @ torch.where(seen.any(0)[:, None], k, torch.zeros_like(k)).T * scale,
                    torch.full((), float("-inf"), dtype=F64))
    top = s.amax(-1, keepdim=True) if s.shape[1] else torch.full((s.shape[0], 1), float("-inf"), dtype=F64)
    p = torch.where(seen, torch.exp(s - torch.where(top == float("-inf"), torch.zeros_like(top), top)), torch.zeros((), dtype=F64))
    total = p.sum(-1, keepdim=True)
    terms = torch.where(seen[:, :, None], p[:, :, None] * v[None], torch.zeros((), dtype=F64)).sum(1) \
        if not torch.isfinite(v).all() else p @ v
    out = torch.where(total == 0, torch.zeros_like(terms), terms / total)
    return out, (top + torch.log(total))[:, 0]


def latent_attention(q, cache, table, lengths, scale) -> tuple:
    """q (B, S, H, 576), a CPU cache and table, lengths (B): fp64 (B, S, H, 512) and (B, S, H)."""
    B, S, H, _ = q.shape
    pages, page = cache[0].shape[:2]
    lat, rope = pool_values(cache)
    out = torch.zeros(B, S, H, LORA, dtype=F64)
    lse = torch.full((B, S, H), float("-inf"), dtype=F64)
    for b in range(B):
        n = min(max(int(lengths[b]), 0), table.shape[1] * page)
        at = [places(table, b, t, page, pages) for t in range(n)]
        rows = [max(a, 0) for a in at]
        k, v = torch.cat([lat[rows], rope[rows]], -1), lat[rows]
        for s in range(S):
            seen = torch.tensor([a >= 0 and t < n - (S - 1 - s) for t, a in enumerate(at)], dtype=torch.bool)
            out[b, s], lse[b, s] = attention(q[b, s].to(F64), k, v, scale, seen.expand(H, n))
    return out, lse


def packed_attention(q, k, v, offsets, scale, k_offsets=None, k_pe=None, causal=True) -> tuple:
    """fp64 (T, H, 128) and (T, H) of CPU tensors."""
    k_offsets = offsets if k_offsets is None else k_offsets
    H, G = q.shape[1], k.shape[1]
    out = torch.zeros(q.shape[0], H, v.shape[2], dtype=F64)
    lse = torch.full((q.shape[0], H), float("-inf"), dtype=F64)
    for b in range(len(offsets) - 1):
        q0, q1, k0, k1 = int(offsets[b]), int(offsets[b + 1]), int(k_offsets[b]), int(k_offsets[b + 1])
        n, m = q1 - q0, k1 - k0
        i, j = torch.arange(n)[:, None], torch.arange(m)[None]
        seen = (j <= i + m - n) if causal else torch.ones(n, m, dtype=torch.bool)
        for h in range(H):
            kh = k[k0:k1, h * G // H].to(F64)
            if k_pe is not None:
                kh = torch.cat([kh, k_pe[k0:k1].to(F64)], -1)
            out[q0:q1, h], lse[q0:q1, h] = attention(q[q0:q1, h].to(F64), kh, v[k0:k1, h * G // H].to(F64), scale, seen)
    return out, lse
