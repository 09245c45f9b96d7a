"""MXFP4 from its definition, in float64 on the CPU (independent of the amla package).

A block of 32 values along K has the exponent e = clamp(floor(log2(max |x|)) - 2, -127, 127),
stored as the byte e + 127 (a block of zeros: byte 0), and its values x / 2^e rounded to the
nearest of the e2m1 magnitudes, ties to the one with an even mantissa, saturating at 6.  A block
with an infinity or a NaN: byte 255, zero codes, all its values NaN.  Code 2i of a row is the low
half of byte i.
"""
from __future__ import annotations

import torch

E2M1 = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)
BLOCK = 32


def quantize(x: torch.Tensor, exponent: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """(..., k) -> (codes uint8 (..., k/2), exponents uint8 (..., k/32)); ``exponent`` replaces the
    blocks' own."""
    x = x.double()
    k = x.shape[-1]
    b = x.reshape(-1, k // BLOCK, BLOCK)
    finite = torch.isfinite(b).all(-1)
    b = torch.where(finite[..., None], b, 0.0)
    amax = b.abs().amax(-1)
    if exponent is None:
        e = torch.frexp(torch.where(amax == 0, 1.0, amax)).exponent.long() - 1 - 2
        e = torch.where(amax == 0, -127, e.clamp(-127, 127))
    else:
        e = exponent.reshape(amax.shape)
    v = b / torch.pow(torch.tensor(2.0, dtype=torch.float64), e.double())[..., None]
    d = (v.abs()[..., None] - E2M1).abs()
    best = d.amin(-1, keepdim=True)
    near = d == best  # one, or the two neighbours of a tie: the even code
    idx = torch.arange(8)
    even = near & (idx % 2 == 0)
    pick = torch.where(near.sum(-1) == 2, even.double().argmax(-1), near.double().argmax(-1))
    code = (pick + 8 * torch.signbit(v)).to(torch.uint8) * finite[..., None].to(torch.uint8)
    byte = torch.where(finite, e + 127, 255).to(torch.uint8)
    code = code.reshape(*x.shape)
    return code[..., 0::2] | (code[..., 1::2] << 4), byte.reshape(*x.shape[:-1], k // BLOCK)


def values(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """float64 values of a pair."""
    pair = torch.stack([codes & 15, codes >> 4], -1).reshape(*codes.shape[:-1], -1).long()
    v = torch.where(pair >= 8, -E2M1[pair & 7], E2M1[pair & 7])
    s = torch.pow(torch.tensor(2.0, dtype=torch.float64), scales.double() - 127)
    s = torch.where(scales == 255, float("nan"), s)
    return v * s.repeat_interleave(BLOCK, -1)


def rounded(x: torch.Tensor, exponent: torch.Tensor | None = None) -> torch.Tensor:
    return values(*quantize(x, exponent))


def linear(x: torch.Tensor, w: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """x (m, k), w (n, k) values -> x @ w.T and the sums of the products' magnitudes."""
    return x @ w.T, x.abs() @ w.abs().T


def linear_slack(mag: torch.Tensor, k: int, eps: float, y: torch.Tensor) -> torch.Tensor:
    """What a correct fp32 sum of the exact products may be off by.

    A matrix instruction adds 128 products to the sum; with the K parts and the waves' sums there
    are at most k / 128 + 40 additions one after another, each off by at most two roundings of
    2^-24 of the magnitudes summed (the products inside an instruction are aligned to the largest
    and added with at least fp32's bits: one rounding, and one of the result).  ``eps``: half a step of the
    output type, relative to the value."""
    return mag * (k / 128 + 40) * 2.0 ** -23 + y.abs() * eps


def swiglu(x: torch.Tensor, gate: torch.Tensor, up: torch.Tensor, down: torch.Tensor):
    """x (m, k) quantised values, weights' values -> (y, slack without the output rounding).

    silu(gate) * up is computed in fp32 and then rounded to four bits: where its error can cross
    a border of that rounding, the other neighbour is as right.  The slack counts these steps."""
    k, n = gate.shape[1], gate.shape[0]
    g, gm = linear(x, gate)
    u, um = linear(x, up)
    dg, du = linear_slack(gm, k, 0.0, g), linear_slack(um, k, 0.0, u)
    s = torch.sigmoid(g)
    h = g * s * u
    # |d silu| <= 1.1 dg; a dozen fp32 roundings of exp, the quotient and the two products
    dh = 1.1 * dg * (u.abs() + du) + (g * s).abs() * du + h.abs() * 2.0 ** -20
    hb, db = h.reshape(h.shape[0], -1, BLOCK), dh.reshape(h.shape[0], -1, BLOCK)
    amax = hb.abs().amax(-1)
    da = db.amax(-1)
    lo = torch.frexp((amax - da).clamp_min(1e-300)).exponent.long() - 3
    hi = torch.frexp((amax + da).clamp_min(1e-300)).exponent.long() - 3
    cand = []
    for e in (lo.clamp(-127, 127), hi.clamp(-127, 127)):
        for sgn in (-1.0, 1.0):
            cand.append(rounded((hb + sgn * db).reshape(h.shape), e))
    cand = torch.stack(cand)
    hq = rounded(h)
    step = (cand - hq).abs().amax(0)
    y, mag = linear(hq, down)
    return y, linear_slack(mag, n, 0.0, y) + step @ down.abs().T


