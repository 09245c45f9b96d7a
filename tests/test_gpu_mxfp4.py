"""The MXFP4 operators on the GPU against their definition in float64 (oracle/ref_mxfp4.py)."""
import pytest
import torch

from amla import ops
from amla.config import DeepSeekConfig
from oracle import ref_mxfp4 as M

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
HALF_STEP = {BF16: 2.0 ** -8, F32: 2.0 ** -24}


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _weight(g, *shape, std=0.05):
    c, s = M.quantize(torch.randn(*shape, generator=g) * std * torch.exp2(torch.randint(-2, 3, (*shape[:-1], 1), generator=g)))
    return c.to(DEV), s.to(DEV)


def _x(g, m, k):
    return (torch.randn(m, k, generator=g) * torch.exp(torch.randn(m, 1, generator=g))).to(BF16)


def _vals(pair):
    return M.values(pair[0].cpu(), pair[1].cpu())


def _check(got, want, slack, what):
    got = got.double().cpu()
    assert got.shape == want.shape, what
    if not got.numel():
        return
    over = (got - want).abs() - slack
    assert torch.isfinite(got).all() and over.max().item() <= 0, \
        f"{what}: {int((over > 0).sum())} of {over.numel()} past the bound, worst by {over.max().item():.3e}"
    print(f"[ok] {what}: largest share of the bound {((got - want).abs() / slack.clamp_min(1e-300)).max().item():.3f}",
          flush=True)


# ------------------------------------------------------------------ quantise

def _hard_rows(k):
    """Rows at which the rounding can go wrong: ties, borders, saturation, zeros, the ends of the
    range, an infinity and a NaN."""
    x = torch.zeros(12, k)
    mids = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 7.0, 0.0, 0.5, 4.0, 1.0, 2.0, 3.0, 1.5])
    x[1] = mids.repeat(k // 16)
    x[2] = -mids.repeat(k // 16) * 2.0 ** 10
    x[3] = (mids * (1 + 2.0 ** -7)).repeat(k // 16)
    x[4] = (mids * (1 - 2.0 ** -8)).repeat(k // 16)
    x[5, :32] = 2.0 ** -126
    x[6, 3] = 3.3e38
    x[6, 4] = -1.0
    x[7, 0], x[7, k - 1] = float("inf"), 2.0
    x[8, k - 2], x[8, 1] = float("nan"), -3.0
    x[9, 0] = -0.0
    x[10] = 65504.0
    x[11] = torch.linspace(-8, 8, k)
    return x


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("rows,k", [(1, 32), (3, 96), (77, 512), (40, 7168)])
def test_quantize_equals_the_definition(dtype, rows, k):
    g = _gen(rows * k)
    x = (torch.randn(rows, k, generator=g) * torch.exp2(torch.randint(-12, 12, (rows, 1), generator=g))).to(dtype)
    if rows > 12:
        x[:12] = _hard_rows(k).to(dtype)
    c, s = ops.mxfp4_quantize(x.to(DEV))
    wc, wsc = M.quantize(x)
    assert torch.equal(s.cpu(), wsc)
    assert torch.equal(c.cpu(), wc)
    for out in (BF16, F32):
        v = ops.mxfp4_dequantize(c, s, out).cpu().double()
        assert torch.equal(torch.nan_to_num(v, 7.0), torch.nan_to_num(M.values(wc, wsc), 7.0))
        assert torch.equal(torch.isnan(v), torch.isnan(M.values(wc, wsc)))


def test_quantize_strides_shapes_and_empty():
    g = _gen(3)
    big = torch.randn(5, 4, 3 * 64 + 8, generator=g).to(BF16).to(DEV)
    for x in (big[:, :, :64], big[:, 1:3, 8:136], big[..., 1:65], big[..., 0:128:2], big[:0, :, :64],
              big[0, 0, :32], big[:1, :1, :32].expand(3, 2, 32)):
        c, s = ops.mxfp4_quantize(x)
        wc, wsc = M.quantize(x.cpu()) if x.numel() else (torch.empty(0, 4, 32, dtype=torch.uint8), torch.empty(0, 4, 2, dtype=torch.uint8))
        assert torch.equal(c.cpu(), wc) and torch.equal(s.cpu(), wsc)
    odd = torch.randn(3 * 64 + 1, generator=g).to(DEV)[1:].view(3, 64)  # a base off the 16-byte grid
    assert torch.equal(ops.mxfp4_quantize(odd)[0].cpu(), M.quantize(odd.cpu())[0])


@pytest.mark.parametrize("n,k", [(1, 128), (130, 384), (257, 160)])
def test_quantize_fp8_equals_dequantised(n, k):
    g = _gen(n)
    w = (torch.randn(n, k, generator=g) * 80).clamp(-448, 448).to(torch.float8_e4m3fn)
    s = torch.rand(-(-n // 128), -(-k // 128), generator=g) * 1e-3 + 1e-5
    c, b = ops.mxfp4_quantize_fp8(w.to(DEV), s.to(DEV))
    dq = ops.fp8_block_dequant(w.to(DEV), s.to(DEV))
    wc, wb = M.quantize(dq.cpu())
    assert torch.equal(c.cpu(), wc) and torch.equal(b.cpu(), wb)
    c2, b2 = ops.mxfp4_quantize(dq)
    assert torch.equal(c, c2) and torch.equal(b, b2)


def test_dequantize_ends_of_the_range():
    codes = torch.arange(256, dtype=torch.uint8).repeat(256, 1)
    byte = torch.arange(256, dtype=torch.uint8)[:, None].repeat(1, 16)
    v = ops.mxfp4_dequantize(codes.to(DEV), byte.to(DEV), F32).cpu()
    want = M.values(codes, byte).float()  # 2^128 and above: infinite
    assert torch.equal(torch.isnan(v), torch.isnan(want))
    assert torch.equal(torch.nan_to_num(v, 7.0), torch.nan_to_num(want, 7.0))


# ------------------------------------------------------------------ linear

LINEARS = [(1, 16, 128), (1, 1001, 1152), (2, 7168, 2048), (5, 130, 640), (16, 2112, 7168), (17, 576, 1536), (32, 256, 512),
           (33, 999, 768), (64, 1536, 7168), (65, 257, 384), (100, 1536, 7168), (128, 256, 256), (129, 512, 1664),
           (300, 2050, 2048), (1000, 640, 1280), (5, 272, 32768), (16, 144, 13056), (2, 7, 12288)]


@pytest.mark.parametrize("m,n,k", LINEARS)
@pytest.mark.parametrize("out", [BF16, F32])
def test_linear(m, n, k, out):
    g = _gen(m + n + k)
    x, w = _x(g, m, k), _weight(g, n, k)
    xq = M.rounded(x)
    y, mag = M.linear(xq, _vals(w))
    got = ops.mxfp4_linear(x.to(DEV), *w, out_dtype=out)
    assert got.dtype == out
    _check(got, y, M.linear_slack(mag, k, HALF_STEP[out], y), f"linear {m}x{n}x{k} {out}")
    held = ops.mxfp4_linear(ops.mxfp4_quantize(x.to(DEV)), *w, out_dtype=out)
    _check(held, y, M.linear_slack(mag, k, HALF_STEP[out], y), "held activations")
    # the same call again: the same bits
    assert torch.equal(got, ops.mxfp4_linear(x.to(DEV), *w, out_dtype=out))


def test_linear_shapes_strides_and_types():
    g = _gen(9)
    w = _weight(g, 48, 256)
    big = _x(g, 12, 3 * 256).to(DEV)
    x = big.view(3, 4, 768)[:, :, 256:512]
    y, mag = M.linear(M.rounded(x.cpu()).reshape(12, 256), _vals(w))
    slack = M.linear_slack(mag, 256, HALF_STEP[BF16], y)
    got = ops.mxfp4_linear(x, *w)
    assert got.shape == (3, 4, 48)
    _check(got.view(12, 48), y, slack, "strided rows")
    _check(ops.mxfp4_linear(x.transpose(0, 1), *w).transpose(0, 1).reshape(12, 48), y, slack, "transposed batch")
    q = ops.mxfp4_quantize(x)
    assert ops.mxfp4_linear(q, *w).shape == (3, 4, 48)
    f16 = ops.mxfp4_linear(x, *w, out_dtype=F16)
    assert f16.dtype == F16
    assert ops.mxfp4_linear(x[:0], *w).shape == (0, 4, 48)
    odd = torch.empty(256 * 4 + 1, dtype=BF16, device=DEV)[1:].view(4, 256).copy_(x[0])
    _check(ops.mxfp4_linear(odd, *w), y[:4], slack[:4], "base off the 16-byte grid")


@pytest.mark.parametrize("m,n,k", [(4097, 4096, 8192), (200, 1000, 18432), (70, 576, 7168), (1000, 2112, 3712)])
def test_linear_in_k_parts_and_rounds(m, n, k):
    """Sizes whose last round of tiles, or all of them, run in K parts: some rows of each tile."""
    g = _gen(m + k)
    x, w = _x(g, m, k).to(DEV), _weight(g, n, k)
    rows = torch.tensor(sorted({r for r in (0, 15, 16, 31, 32, 63, 64, 65, 127, 128, 255, 256, 900, 4000, m - 2, m - 1) if r < m}))
    xq = ops.mxfp4_dequantize(*ops.mxfp4_quantize(x[rows.to(DEV)]), F32).double()
    wv = ops.mxfp4_dequantize(*w, F32).double()
    y, mag = xq @ wv.T, xq.abs() @ wv.abs().T
    for out in (BF16, F32):
        got = ops.mxfp4_linear(x, *w, out_dtype=out)
        _check(got[rows.to(DEV)], y.cpu(), M.linear_slack(mag.cpu(), k, HALF_STEP[out], y.cpu()), f"{m}x{n}x{k} {out}")
        assert torch.equal(got, ops.mxfp4_linear(x, *w, out_dtype=out))


@pytest.mark.parametrize("m", [1, 70, 130])
@pytest.mark.parametrize("k", [1024, 1152])
def test_linear_with_exponents_off_the_16_byte_grid(m, k):
    g = _gen(m + k)
    x, (c, s) = _x(g, m, k).to(DEV), _weight(g, 300, k)
    moved = torch.empty(s.numel() + 4, dtype=torch.uint8, device=DEV)[4:].view(s.shape).copy_(s)
    assert moved.data_ptr() % 16 == 4 and moved.is_contiguous()
    assert torch.equal(ops.mxfp4_linear(x, c, moved), ops.mxfp4_linear(x, c, s))
    xc, xs = ops.mxfp4_quantize(x)
    for off in (4, 1):
        held = torch.empty(xs.numel() + off, dtype=torch.uint8, device=DEV)[off:].view(xs.shape).copy_(xs)
        assert torch.equal(ops.mxfp4_linear((xc, held), c, moved), ops.mxfp4_linear((xc, xs), c, s))


@pytest.mark.parametrize("m", [1, 40, 200])
def test_linear_nan_blocks_stay_in_their_row_and_column(m):
    g = _gen(m)
    x, w = _x(g, m, 512).to(DEV), _weight(g, 300, 512)
    clean = ops.mxfp4_linear(x, *w)
    x2 = x.clone()
    x2[m // 2, 100] = float("inf")
    s2 = w[1].clone()
    s2[7, 3] = 255
    y = ops.mxfp4_linear(x2, w[0], s2)
    bad = torch.zeros(m, 300, dtype=torch.bool, device=DEV)
    bad[m // 2] = True
    bad[:, 7] = True
    assert torch.isnan(y[bad]).all() and torch.equal(y[~bad], clean[~bad])


# ------------------------------------------------------------------ grouped

def _offsets(sizes):
    return torch.tensor([0] + torch.tensor(sizes).cumsum(0).tolist(), dtype=torch.int32)


GROUPS = [([1], 64, 128), ([0, 3, 0, 1], 100, 256), ([5, 0, 11], 257, 640), ([40, 0, 1, 130, 17], 300, 384),
          ([128, 129, 0, 64, 33, 32], 512, 1664), ([0, 0, 0], 64, 128), ([2] * 70, 48, 256),
          ([128, 129, 0, 64, 33, 32, 300], 8194, 384), ([97, 17, 257, 1, 0, 160], 8192, 512), ([64, 65, 0, 200], 1030, 1024)]


@pytest.mark.parametrize("sizes,n,k", GROUPS)
@pytest.mark.parametrize("out", [BF16, F32])
def test_grouped_linear(sizes, n, k, out):
    E, m = len(sizes), sum(sizes)
    g = _gen(m + n)
    tail = 3
    x, w = _x(g, m + tail, k), _weight(g, E, n, k)
    off = _offsets(sizes)
    xq, wv = M.rounded(x), _vals(w)
    want, slack = torch.zeros(m + tail, n, dtype=torch.float64), torch.zeros(m + tail, n, dtype=torch.float64)
    for e in range(E):
        a, b = off[e].item(), off[e + 1].item()
        y, mag = M.linear(xq[a:b], wv[e])
        want[a:b], slack[a:b] = y, M.linear_slack(mag, k, HALF_STEP[out], y)
    got = ops.mxfp4_grouped_linear(x.to(DEV), *w, off.to(DEV), out_dtype=out)
    _check(got, want, slack, f"grouped {sizes} {n} {k} {out}")  # rows behind the last group: zeros
    assert torch.equal(got, ops.mxfp4_grouped_linear(x.to(DEV), *w, off.to(DEV), out_dtype=out))
    held = torch.full((m + tail, n + 4), 7.0, dtype=out, device=DEV)
    res = ops.mxfp4_grouped_linear(ops.mxfp4_quantize(x.to(DEV)), *w, off.to(DEV), out_dtype=out, out=held[:, :n])
    _check(res[:m], want[:m], slack[:m], "into a strided out")
    assert (held[m:] == 7).all() and (held[:, n:] == 7).all()  # left as they were


@pytest.mark.parametrize("m", [10, 300])
def test_grouped_offsets_past_the_end_or_backwards_stay_in_bounds(m):
    g = _gen(1)
    x, w = _x(g, m, 128).to(DEV), _weight(g, 4, 64, 128)
    canary = torch.full((m + 8, 64), 3.0, dtype=BF16, device=DEV)
    off = torch.tensor([4, 2, 7, 6, m + 1000], dtype=torch.int32, device=DEV)
    ops.mxfp4_grouped_linear(x, *w, off, out=canary[4:m + 4])
    full = [ops.mxfp4_linear(x, w[0][e], w[1][e], out_dtype=F32).cpu() for e in range(4)]
    assert (canary[:8] == 3).all() and (canary[m + 4:] == 3).all()  # rows 0 .. 3 are of no group
    got = canary[4:m + 4].float().cpu()
    for lo, hi, e in ((4, 7, 1), (7, m, 3)):  # starts 4, 4, 7, 7, m
        assert (got[lo:hi] - full[e][lo:hi]).abs().max() <= 2.0 ** -7 * full[e][lo:hi].abs().max()


@pytest.mark.parametrize("E", [1023, 1024])
@pytest.mark.parametrize("m", [9, 600])
def test_grouped_linear_of_the_most_groups(E, m):
    g = _gen(E + m)
    w = _weight(g, E, 16, 128)
    cuts = torch.sort(torch.randint(0, m + 1, (E + 1,), generator=g)).values
    cuts[0], cuts[-1] = 0, m
    cuts[-2] = min(int(cuts[-2]), m - 1)  # (the last group has rows)
    cuts = torch.cummax(torch.minimum(cuts, torch.tensor([m - 1] * E + [m])), 0).values
    x = _x(g, m, 128)
    group = torch.bucketize(torch.arange(m), cuts, right=True) - 1
    wv, xq = _vals(w), M.rounded(x)
    y = (xq[:, None, :] * wv[group]).sum(-1)
    mag = (xq[:, None, :].abs() * wv[group].abs()).sum(-1)
    _check(ops.mxfp4_grouped_linear(x.to(DEV), *w, cuts.int().to(DEV)), y, M.linear_slack(mag, 128, HALF_STEP[BF16], y),
           f"{m} rows in {E} groups")


# ------------------------------------------------------------------ swiglu and experts

def _ffn(g, d, n, E=None):
    lead = () if E is None else (E,)
    return {"gate_proj": _weight(g, *lead, n, d), "up_proj": _weight(g, *lead, n, d), "down_proj": _weight(g, *lead, d, n)}


@pytest.mark.parametrize("m,d,n", [(1, 128, 128), (3, 1152, 640), (16, 256, 384), (17, 512, 256), (70, 384, 128),
                                   (150, 1024, 640), (8, 2048, 1536), (300, 512, 4096),
                                   (1000, 640, 8192), (1000, 512, 8192), (200, 1536, 512)])
def test_swiglu(m, d, n):
    g = _gen(m * d)
    x, w = _x(g, m, d), _ffn(g, d, n)
    y, slack = M.swiglu(M.rounded(x), *[_vals(w[key]) for key in ("gate_proj", "up_proj", "down_proj")])
    got = ops.mxfp4_swiglu(x.to(DEV), *w["gate_proj"], *w["up_proj"], *w["down_proj"])
    _check(got, y, slack + HALF_STEP[BF16] * y.abs() + 2.0 ** -8 * slack, f"swiglu {m} {d} {n}")
    assert torch.equal(got, ops.dense_ffn(x.to(DEV), w)) and torch.equal(got, ops.expert_ffn(x.to(DEV)[None], w)[0])


@pytest.mark.parametrize("m,d,n,E,top_k", [(1, 128, 128, 4, 2), (5, 256, 384, 6, 3), (16, 1152, 640, 8, 2),
                                           (17, 256, 128, 3, 3), (60, 512, 256, 8, 2), (300, 256, 128, 2, 2),
                                           (300, 4096, 2048, 4, 2), (90, 4224, 2176, 4, 4), (200, 640, 4096, 8, 3)])
def test_moe_experts(m, d, n, E, top_k):
    g = _gen(m * E)
    x, w = _x(g, m, d), _ffn(g, d, n, E)
    idx = torch.stack([torch.randperm(E, generator=g)[:top_k] for _ in range(m)])
    idx[0, 0] = -1
    idx[m // 2, top_k - 1] = E
    if m > 2:
        idx[2] = idx[2, 0]  # one expert several times over for a token
    vals = {key: _vals(w[key]) for key in w}
    xq = M.rounded(x)
    want, slack = torch.zeros(m, top_k, d, dtype=torch.float64), torch.zeros(m, top_k, d, dtype=torch.float64)
    for e in range(E):
        t, j = torch.where(idx == e)
        if len(t):
            want[t, j], slack[t, j] = M.swiglu(xq[t], vals["gate_proj"][e], vals["up_proj"][e], vals["down_proj"][e])
    got = ops.mxfp4_moe_experts(x.to(DEV), idx.to(DEV), w)
    _check(got, want, slack + HALF_STEP[BF16] * want.abs() + 2.0 ** -8 * slack, f"experts {m} {d} {n} {E} {top_k}")
    assert torch.equal(got, ops.mxfp4_moe_experts(x.to(DEV), idx.to(DEV), w))


@pytest.mark.parametrize("m,top_k", [(1, 8), (2, 20), (3, 8), (5, 64), (16, 5)])
def test_moe_experts_with_one_expert_for_every_slot(m, top_k):
    """More rows for an expert than there are tokens: the slots of a token are equal rows."""
    g = _gen(m * top_k)
    x, w = _x(g, m, 640).to(DEV), _ffn(g, 640, 256, 3)
    once = ops.mxfp4_moe_experts(x, torch.ones(m, 1, dtype=torch.int64, device=DEV), w)
    vals = {key: _vals((w[key][0][1], w[key][1][1])) for key in w}
    y, slack = M.swiglu(M.rounded(x.cpu()), vals["gate_proj"], vals["up_proj"], vals["down_proj"])
    _check(once[:, 0], y, slack + HALF_STEP[BF16] * y.abs() + 2.0 ** -8 * slack, "one slot a token")
    got = ops.mxfp4_moe_experts(x, torch.ones(m, top_k, dtype=torch.int64, device=DEV), w)
    assert torch.equal(got, once.expand(m, top_k, 640))


def test_moe_experts_of_more_slots_than_a_call_takes():
    """9000 x 8 slots run as two calls (65536 slots each at most): tokens on both sides of the cut."""
    g = _gen(5)
    x, w = _x(g, 9000, 128), _ffn(g, 128, 128, 16)
    idx = torch.rand(9000, 16, generator=g).argsort(1)[:, :8].contiguous()
    idx[8191, 3], idx[8192, 0] = -1, 16
    got = ops.mxfp4_moe_experts(x.to(DEV), idx.to(DEV), w).cpu()
    t = torch.tensor([0, 1, 4095, 8190, 8191, 8192, 8193, 8999])
    vals = {key: _vals(w[key]) for key in w}
    xq = M.rounded(x[t])
    want, slack = torch.zeros(len(t), 8, 128, dtype=torch.float64), torch.zeros(len(t), 8, 128, dtype=torch.float64)
    for i, tok in enumerate(t.tolist()):
        for j, e in enumerate(idx[tok].tolist()):
            if 0 <= e < 16:
                y, s = M.swiglu(xq[i:i + 1], vals["gate_proj"][e], vals["up_proj"][e], vals["down_proj"][e])
                want[i, j], slack[i, j] = y[0], s[0]
    _check(got[t], want, slack + HALF_STEP[BF16] * want.abs() + 2.0 ** -8 * slack, "9000 tokens")


@pytest.mark.parametrize("tokens", [3, 40])
def test_moe_block_on_mxfp4_experts(tokens):
    """route, the shared expert (fp8), the MXFP4 experts and the combine as an engine runs them, also
    captured in a graph and replayed among eager calls."""
    cfg = DeepSeekConfig(hidden_size=512, n_routed_experts=16, num_experts_per_tok=4, n_group=4, topk_group=2,
                         moe_intermediate_size=256)
    g = _gen(tokens)
    h = torch.randn(1, tokens, 512, generator=g).to(BF16).to(DEV)
    gate_w = (torch.randn(16, 512, generator=g) * 0.1).to(BF16).to(DEV)

    def fp8(n, k):
        return ((torch.randn(n, k, generator=g) * 60).clamp(-448, 448).to(torch.float8_e4m3fn).to(DEV),
                torch.full((-(-n // 128), -(-k // 128)), 1e-3, device=DEV))

    shared = {"gate_proj": fp8(256, 512), "up_proj": fp8(256, 512), "down_proj": fp8(512, 256)}
    experts = _ffn(g, 512, 256, 16)
    idx, wt = ops.route(h, gate_w, cfg)
    eo = ops.mxfp4_moe_experts(h, idx, experts)[0].float()
    acc = torch.zeros(tokens, 512, device=DEV)
    for j in range(4):
        acc = (acc + (wt[0, :, j, None].to(BF16).float() * eo[:, j]).to(BF16).float()).to(BF16).float()
    want = ops.expert_ffn(h, shared)[0].float() + (acc * cfg.routed_scaling_factor).to(BF16).float()
    got = ops.moe_block(h, gate_w, shared, experts, cfg)
    assert torch.equal(got[0], want.to(BF16))
    assert torch.equal(got, ops.moe_block(h, gate_w, shared, experts, cfg, routing=(idx, wt)))
    with pytest.raises(ValueError, match="grouped on the device"):
        ops.moe_block(h, gate_w, shared, experts, cfg, device_grouping=False)

    static = h.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.moe_block(static, gate_w, shared, experts, cfg)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.moe_block(static, gate_w, shared, experts, cfg)
    for i in range(4):
        fresh = torch.randn(1, tokens, 512, generator=g).to(BF16).to(DEV)
        static.copy_(fresh)
        graph.replay()
        eager = ops.moe_block(fresh, gate_w, shared, experts, cfg)
        torch.cuda.synchronize()
        assert torch.equal(out, eager), i


def test_checkpoint_weights_to_experts_in_one_run():
    """A block-FP8 expert turned into MXFP4 and run: the output is the fp8 expert's up to the two
    roundings to four bits."""
    g = _gen(11)
    d, n, m = 512, 256, 24
    fp8 = {}
    for key, (a, b) in {"gate_proj": (n, d), "up_proj": (n, d), "down_proj": (d, n)}.items():
        fp8[key] = ((torch.randn(a, b, generator=g) * 60).clamp(-448, 448).to(torch.float8_e4m3fn).to(DEV),
                    torch.rand(-(-a // 128), -(-b // 128), generator=g).to(DEV) * 1e-3 + 5e-4)
    mx = {key: ops.mxfp4_quantize_fp8(*pair) for key, pair in fp8.items()}
    x = torch.randn(m, d, generator=g).to(BF16).to(DEV)
    y8, y4 = ops.expert_ffn(x, fp8).double(), ops.expert_ffn(x, mx).double()
    # four roundings of relative rms at most 2^-2 / sqrt(12) x 1.5 (e2m1 steps of up to half the
    # value, most of them a quarter): below 0.25 together for sums of independent terms
    assert ((y8 - y4).pow(2).mean().sqrt() / y8.pow(2).mean().sqrt()).item() < 0.5
    y, slack = M.swiglu(M.rounded(x.cpu()), *[_vals(mx[key]) for key in ("gate_proj", "up_proj", "down_proj")])
    _check(y4, y, slack + HALF_STEP[BF16] * y.abs() + 2.0 ** -8 * slack, "converted expert")


# ------------------------------------------------------------------ streams, capture, refusals

def test_side_stream_and_capture():
    g = _gen(4)
    w = _weight(g, 512, 1024)
    w3 = _weight(g, 3, 96, 1024)
    ff = _ffn(g, 1024, 256)
    off = torch.tensor([0, 30, 31, 90], dtype=torch.int32, device=DEV)
    x = _x(g, 90, 1024).to(DEV)

    def step(t):
        return (ops.mxfp4_linear(t, *w), ops.mxfp4_linear(t[:7], *w), ops.mxfp4_grouped_linear(t, *w3, off),
                ops.mxfp4_swiglu(t, *ff["gate_proj"], *ff["up_proj"], *ff["down_proj"]), *ops.mxfp4_quantize(t))

    want = step(x)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step(x)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    static = x.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(static)
    for i in range(4):
        fresh = _x(g, 90, 1024).to(DEV)
        static.copy_(fresh)
        graph.replay()
        eager = step(fresh)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, eager)), i


def test_calls_on_two_streams_at_once():
    """Each call has scratch of its own: what runs beside it leaves its result alone."""
    g = _gen(7)
    w, ff = _weight(g, 2048, 1024), _ffn(g, 512, 256, 8)
    xs = [(_x(g, 200, 1024).to(DEV), _x(g, 100, 512).to(DEV), torch.randint(0, 8, (100, 4), generator=g).to(DEV))
          for _ in range(2)]

    def step(a, b, idx):
        return ops.mxfp4_linear(a, *w), ops.mxfp4_linear(a[:5], *w), ops.mxfp4_moe_experts(b, idx, ff)

    want = [step(*x) for x in xs]
    torch.cuda.synchronize()
    sides = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(10):
        for i, side in enumerate(sides):
            with torch.cuda.stream(side):
                got[i].append(step(*xs[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(a, b) for res in got[i] for a, b in zip(res, want[i]))


def test_no_backward_is_said_not_passed_over():
    g = _gen(12)
    w, ff = _weight(g, 64, 256), _ffn(g, 256, 128)
    x = _x(g, 5, 256).to(DEV)
    leaf = x.clone().requires_grad_()
    for f in (lambda t: ops.mxfp4_linear(t, *w), lambda t: ops.dense_ffn(t, ff), lambda t: ops.mxfp4_linear(2 * t, *w)):
        y = f(leaf)
        with pytest.raises(RuntimeError, match="no backward"):
            y.float().sum().backward()
        with torch.no_grad():
            assert torch.equal(f(leaf), y) and not f(leaf).requires_grad
    assert torch.equal(ops.mxfp4_linear(leaf, *w), ops.mxfp4_linear(x, *w))
    assert all(torch.equal(a, b) for a, b in zip(ops.mxfp4_quantize(leaf), ops.mxfp4_quantize(x)))


def test_compiled_calls_equal_eager_ones():
    g = _gen(6)
    w = _weight(g, 256, 512)
    ff = _ffn(g, 512, 256)
    x = _x(g, 9, 512).to(DEV)

    def f(t):
        q = ops.mxfp4_quantize(t)
        return ops.mxfp4_linear(q, *w), ops.mxfp4_linear(t, *w, out_dtype=F32), ops.dense_ffn(t, ff)

    got = torch.compile(f, fullgraph=True, backend="aot_eager")(x)
    assert all(torch.equal(a, b) for a, b in zip(got, f(x)))


def test_refusals():
    g = _gen(8)
    x = _x(g, 4, 256).to(DEV)
    w, s = _weight(g, 64, 256)
    with pytest.raises(TypeError, match="bfloat16, float16 or float32"):
        ops.mxfp4_quantize(x.double())
    with pytest.raises(ValueError, match="multiple of 32"):
        ops.mxfp4_quantize(x[:, :40])
    with pytest.raises(TypeError, match="bfloat16"):
        ops.mxfp4_linear(x.float(), w, s)
    with pytest.raises(ValueError, match="expects 256"):
        ops.mxfp4_linear(x[:, :128], w, s)
    with pytest.raises(ValueError, match="does not match codes"):
        ops.mxfp4_linear(x, w, s[:, :4].contiguous())
    with pytest.raises(TypeError, match="uint8"):
        ops.mxfp4_linear(x, w.to(torch.int8), s)
    with pytest.raises(ValueError, match="contiguous"):
        ops.mxfp4_linear(x, w[:, :64], s)
    with pytest.raises(ValueError, match="multiple of 128"):
        ops.mxfp4_linear(x[:, :96], w[:, :48].contiguous(), s[:, :3].contiguous())
    with pytest.raises(ValueError, match="bfloat16 tensor or a"):
        ops.mxfp4_linear((x,), w, s)
    w3, s3 = _weight(g, 2, 64, 256)
    with pytest.raises(ValueError, match="offsets of shape"):
        ops.mxfp4_grouped_linear(x, w3, s3, torch.zeros(2, dtype=torch.int32, device=DEV))
    with pytest.raises(TypeError, match="int32"):
        ops.mxfp4_grouped_linear(x, w3, s3, torch.zeros(3, dtype=torch.int64, device=DEV))
    with pytest.raises(TypeError, match="out must be"):
        ops.mxfp4_grouped_linear(x, w3, s3, torch.zeros(3, dtype=torch.int32, device=DEV),
                                 out=torch.empty(4, 64, device=DEV))
    with pytest.raises(ValueError, match="multiple of 128"):
        ops.mxfp4_swiglu(x, w, s, w, s, *_weight(g, 256, 64))
    ff = _ffn(g, 256, 128, 2)
    with pytest.raises(ValueError, match="int64"):
        ops.mxfp4_moe_experts(x, torch.zeros(4, 2, dtype=torch.int32, device=DEV), ff)
    with pytest.raises(ValueError, match="do not match hidden"):
        ops.mxfp4_moe_experts(x, torch.zeros(3, 2, dtype=torch.int64, device=DEV), ff)
    with pytest.raises(TypeError, match="out_dtype"):
        ops.mxfp4_dequantize(w, s, F16)
