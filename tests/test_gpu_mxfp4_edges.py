"""The MXFP4 operators at the ends of their types' range."""
import pytest
import torch

from amla import ops
from oracle import ref_mxfp4 as M

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def _tiny_rows(dtype):
    """Blocks whose largest value is subnormal, or next to where subnormals begin: every step of the
    rounding at the exponent bytes 0, 1 and 2 (fp16: of its subnormals)."""
    steps = torch.tensor([0.0, 0.25, 0.26, 0.5, 0.75, 0.76, 1.0, 1.25, 1.26, 1.5, 1.75, 1.76, 2.0, 2.5, 2.52, 3.0, 3.5, 3.52,
                          4.0, 5.0, 5.04, 6.0, 6.5, 7.0, 7.96, -0.0, -0.25, -0.5, -0.75, -1.0, -3.5, -6.0], dtype=torch.float64)
    tops = [0.25, 0.26, 0.5, 0.76, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, 7.96]
    low = {BF16: -127, F32: -127, F16: -24}[dtype]
    rows = [torch.where(steps.abs() <= top, steps, 0.0) * 2.0 ** (low + e) for e in range(4) for top in tops]
    return torch.stack(rows).to(dtype)  # (the type's own rounding, subnormals kept)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_quantise_subnormal_blocks(dtype):
    x = _tiny_rows(dtype)
    assert (x != 0).any(1).sum() > len(x) // 2
    c, s = ops.mxfp4_quantize(x.to(DEV))
    wc, ws = M.quantize(x)
    assert torch.equal(s.cpu(), ws)
    assert torch.equal(c.cpu(), wc)


def test_quantise_fp8_of_tiny_scales():
    """Products of a weight and its scale in fp32's subnormal range."""
    g = torch.Generator().manual_seed(1)
    w = (torch.randn(256, 256, generator=g) * 30).to(torch.float8_e4m3fn)
    s = torch.tensor([[2.0 ** -133, 3e-39], [2.0 ** -128 * 1.3, 2.0 ** -149]])
    c, b = ops.mxfp4_quantize_fp8(w.to(DEV), s.to(DEV))
    dq = ops.fp8_block_dequant(w.to(DEV), s.to(DEV))
    prod = w.double() * s.double().repeat_interleave(128, 0).repeat_interleave(128, 1)
    assert torch.equal(dq.cpu(), prod.float())  # one fp32 rounding, subnormals kept
    wc, wb = M.quantize(dq.cpu())
    assert torch.equal(b.cpu(), wb) and torch.equal(c.cpu(), wc)
    c2, b2 = ops.mxfp4_quantize(dq)
    assert torch.equal(c, c2) and torch.equal(b, b2)


@pytest.mark.parametrize("m", [2, 5, 40])
def test_linear_of_tiny_activations(m):
    """bf16 rows quantised in the product (up to 16 rows) or before it: the same codes as
    mxfp4_quantize gives, down to subnormals."""
    x = _tiny_rows(BF16)[:40].repeat(1, 8)[:m] if m > 5 else _tiny_rows(BF16)[[9, 10, 20, 21, 31][:m]].repeat(1, 8)
    g = torch.Generator().manual_seed(2)
    w = tuple(t.to(DEV) for t in M.quantize(torch.randn(48, 256, generator=g) * 2.0 ** 60))
    got = ops.mxfp4_linear(x.to(DEV), *w, out_dtype=F32)
    held = ops.mxfp4_linear(ops.mxfp4_quantize(x.to(DEV)), *w, out_dtype=F32)
    assert torch.equal(got, held)
    y, mag = M.linear(M.rounded(x), M.values(w[0].cpu(), w[1].cpu()))
    assert ((got.double().cpu() - y).abs() <= M.linear_slack(mag, 256, 2.0 ** -24, y)).all()
    assert (y != 0).any()


# ------------------------------------------------------------------ NaN blocks

def _weight(g, *shape):
    return tuple(t.to(DEV) for t in M.quantize(torch.randn(*shape, generator=g) * 0.05))


@pytest.mark.parametrize("sizes", [[3, 0, 5], [60, 0, 30, 1], [200, 70, 0, 130, 20]])
def test_grouped_nan_blocks_stay_in_their_rows_and_groups(sizes):
    g = torch.Generator().manual_seed(sum(sizes))
    E, m = len(sizes), sum(sizes)
    off = torch.tensor([0] + torch.tensor(sizes).cumsum(0).tolist(), dtype=torch.int32)
    x = torch.randn(m, 512, generator=g).to(BF16)
    c, s = _weight(g, E, 300, 512)
    clean = ops.mxfp4_grouped_linear(x.to(DEV), c, s, off.to(DEV))
    row, last = m // 2, E - 1
    x[row, 100] = float("inf")
    s[last, 7, 3] = 255
    y = ops.mxfp4_grouped_linear(x.to(DEV), c, s, off.to(DEV))
    bad = torch.zeros(m, 300, dtype=torch.bool)
    bad[row] = True
    bad[off[last]:off[last + 1], 7] = True
    assert torch.isnan(y.cpu()[bad]).all() and torch.equal(y.cpu()[~bad], clean.cpu()[~bad])


@pytest.mark.parametrize("m", [4, 50, 300])
def test_swiglu_nan_rows_stay_rows(m):
    g = torch.Generator().manual_seed(m)
    ff = {"gate_proj": _weight(g, 256, 512), "up_proj": _weight(g, 256, 512), "down_proj": _weight(g, 512, 256)}
    x = torch.randn(m, 512, generator=g).to(BF16).to(DEV)
    clean = ops.dense_ffn(x, ff)
    x[m // 2, 3] = float("nan")
    y = ops.dense_ffn(x, ff)
    keep = torch.arange(m, device=DEV) != m // 2
    assert torch.isnan(y[m // 2]).all() and torch.equal(y[keep], clean[keep])
    # a NaN block of up's row 40: block 1 of every h, and so all outputs
    ff["up_proj"][1][40, 0] = 255
    assert torch.isnan(ops.dense_ffn(x[:1], ff)).all()


@pytest.mark.parametrize("m", [4, 60, 700])
def test_experts_nan_rows_stay_rows(m):
    g = torch.Generator().manual_seed(m)
    w = {"gate_proj": _weight(g, 4, 256, 512), "up_proj": _weight(g, 4, 256, 512), "down_proj": _weight(g, 4, 512, 256)}
    x = torch.randn(m, 512, generator=g).to(BF16).to(DEV)
    idx = torch.stack([torch.randperm(4, generator=g)[:2] for _ in range(m)]).to(DEV)
    idx[0, 1] = -1
    clean = ops.mxfp4_moe_experts(x, idx, w)
    x[m // 2, 3] = float("inf")
    w["down_proj"][1][2, 9, 1] = 255  # expert 2, output 9
    y = ops.mxfp4_moe_experts(x, idx, w)
    bad = torch.zeros(m, 2, 512, dtype=torch.bool, device=DEV)
    bad[m // 2] = True
    bad[..., 9] |= idx == 2
    bad &= (idx >= 0)[..., None]
    assert torch.isnan(y[bad]).all() and torch.equal(y[~bad], clean[~bad])
    assert (y[0, 1] == 0).all()


# ------------------------------------------------------------------ silu at its ends

@pytest.mark.parametrize("m", [3, 40, 200])
def test_swiglu_of_far_gates(m):
    """Gates of large magnitude: silu(-large) is zero and silu(large) the gate, with no NaN from an
    overflowing exponential."""
    k = n = 128
    x = torch.zeros(m, k, dtype=BF16)
    x[:, 0] = torch.linspace(-1, 1, m).to(BF16) * 448
    unit = torch.zeros(n, k)
    unit[:, 0] = 2.0
    up = torch.zeros(n, k)
    up[:, 0] = 0.5
    down = torch.eye(k, n)
    w = [tuple(t.to(DEV) for t in M.quantize(t_)) for t_ in (unit, up, down)]
    got = ops.mxfp4_swiglu(x.to(DEV), *w[0], *w[1], *w[2])
    y, slack = M.swiglu(M.rounded(x), *[M.values(c.cpu(), s.cpu()) for c, s in w])
    assert torch.isfinite(got).all()
    assert ((got.double().cpu() - y).abs() <= slack * (1 + 2.0 ** -8) + 2.0 ** -8 * y.abs()).all()
