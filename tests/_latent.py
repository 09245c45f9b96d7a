"""Inputs and tolerances shared by the tests of the paged latent cache and of packed prompts."""
import math

import torch

from oracle import ref_latent as L

DEV = "cuda:0"
BF16, FP8 = torch.bfloat16, torch.float8_e4m3fn
HALF_BF16 = 2.0 ** -8


def cache_of(lat, rope, fp8, page_size, lengths, g, extra_pages=2, junk=None):
    """A CPU cache whose sequences hold the given rows (lists of (n, 512) and (n, 64)), pages in a
    random order; every other row of the pool is `junk` (None: old rows).  Returns (cache, table)."""
    need = [-(-n // page_size) for n in lengths]
    pages = sum(need) + extra_pages
    order = torch.randperm(pages, generator=g).tolist()
    table = torch.full((len(lengths), max(need + [1])), -1, dtype=torch.int32)
    rows = pages * page_size
    all_lat = torch.randn(rows, 512, generator=g, dtype=torch.float64)
    all_pe = torch.randn(rows, 64, generator=g, dtype=torch.float64)
    used = torch.zeros(rows, dtype=torch.bool)
    at = 0
    for b, n in enumerate(lengths):
        for c in range(need[b]):
            table[b, c] = order[at]
            lo = c * page_size
            k = min(page_size, n - lo)
            dst = order[at] * page_size
            all_lat[dst:dst + k], all_pe[dst:dst + k] = lat[b][lo:lo + k], rope[b][lo:lo + k]
            used[dst:dst + k] = True
            at += 1
    pe = all_pe.to(BF16)
    if junk is not None:
        pe[~used] = junk
    pe = pe.view(pages, page_size, 64)
    if not fp8:
        lb = all_lat.to(BF16)
        if junk is not None:
            lb[~used] = junk
        return (lb.view(pages, page_size, 512), pe), table
    e = L.exponent(all_lat)
    codes = L.e4m3(all_lat / torch.exp2(e.double())[:, None]).float().to(FP8)
    byte = (e + 127).to(torch.uint8)
    if junk is not None:
        codes.view(torch.uint8)[~used] = 0x7F
        byte[~used] = 255
    return (codes.view(pages, page_size, 512), pe, byte.view(pages, page_size)), table


def to_dev(t, dev=DEV):
    if isinstance(t, (tuple, list)):
        return tuple(to_dev(x, dev) for x in t)
    return t.to(dev) if isinstance(t, torch.Tensor) else t


def check_attention(got, want, lse, want_lse, weight, size, what):
    """Outputs of an attention against fp64.  weight: sum_t p_t |v_t| of each output value; size: the
    largest scale sum |q k| of any score.

    A score is an fp32 sum of at most 576 products (q bf16, whole in its two e4m3 halves but for 2^-22 of
    the row's largest), so it is off by at most ds = (576 2^-24 + 2^-21) size, the last part for the
    products with log2 e and the scale.  A probability is off by expm1(2 ds) at most, then rounded to
    bf16 or to two e4m3 halves: 2^-8 at most.  l is the fp32 sum of unrounded probabilities.  A split's
    sums are rounded too (to fp16 times a power of two: far less than the 2^-8 of the weight counted
    here), the joined ones to bf16.  So
    |d out| <= weight (expm1(2 ds) + 2^-7) + 2^-8 |out| + 2^-24, and |d lse| <= ds + 2^-20 (1 + |lse|)."""
    got, lse = got.double().cpu(), lse.double().cpu()
    empty = want_lse == float("-inf")
    assert torch.equal(lse == float("-inf"), empty), what
    assert (got[empty] == 0).all(), f"{what}: rows that see nothing"
    ds = (576 * 2.0 ** -24 + 2.0 ** -21) * size
    bound = (math.expm1(2 * ds) + 2.0 ** -7) * weight + HALF_BF16 * want.abs() + 2.0 ** -24
    worst = ((got - want).abs() / bound)[~empty]
    assert worst.numel() == 0 or worst.max() <= 1.0, f"{what}: {worst.max().item():.2f} x the bound"
    if worst.numel():
        d = (lse - want_lse)[~empty].abs()
        assert (d <= ds + 2.0 ** -20 * (1 + want_lse[~empty].abs())).all(), f"{what}: lse off by {d.max().item():.2e}"
        rms = (got - want)[~empty].square().mean().sqrt() / want[~empty].square().mean().sqrt().clamp_min(1e-30)
        print(f"[latent] {what}: rms {rms.item():.2e}, worst {worst.max().item():.3f} of the bound, lse {d.max().item():.1e}",
              flush=True)
