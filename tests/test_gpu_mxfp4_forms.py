"""MXFP4 products in forms that few sizes take: 128-row tiles in K parts, 65 - 96 rows, exponents
off the 16-byte grid in every kernel."""
import pytest
import torch

from amla import ops
from amla._lib import check, lib
from oracle import ref_mxfp4 as M

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16, F32 = torch.bfloat16, torch.float32
HALF_STEP = {BF16: 2.0 ** -8, F32: 2.0 ** -24}


def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def _weight(g, *shape):
    return ops.mxfp4_quantize(torch.randn(*shape, generator=g, device=DEV) * 0.05)


def _x(g, m, k):
    return (torch.randn(m, k, generator=g, device=DEV) * torch.exp(torch.randn(m, 1, generator=g, device=DEV))).to(BF16)


def _moved(s, off=4):
    """The same bytes at an address ``off`` bytes past a 16-byte boundary."""
    t = torch.empty(s.numel() + off, dtype=torch.uint8, device=DEV)[off:].view(s.shape).copy_(s)
    assert t.data_ptr() % 16 == off and t.is_contiguous()
    return t


def _values(pair):
    return ops.mxfp4_dequantize(*pair, F32).double()


@pytest.mark.parametrize("m,n,k", [(1000, 2112, 10240), (500, 5120, 10240), (1000, 2112, 10368)])
def test_linear_of_128_row_tiles_in_k_parts(m, n, k):
    g = _gen(m + k)
    x, w = _x(g, m, k), _weight(g, n, k)
    xq, wv = _values(ops.mxfp4_quantize(x)), _values(w)
    y, mag = xq @ wv.T, xq.abs() @ wv.abs().T
    for out in (BF16, F32):
        got = ops.mxfp4_linear(x, *w, out_dtype=out)
        assert ((got.double() - y).abs() <= M.linear_slack(mag, k, HALF_STEP[out], y)).all()
        assert torch.equal(got, ops.mxfp4_linear(x, *w, out_dtype=out))


@pytest.mark.parametrize("k", [512, 1024, 640])
def test_grouped_linear_of_65_to_96_rows(k):
    sizes = [70, 96, 80, 300, 65]
    g = _gen(k)
    m, n = sum(sizes), 8192
    off = torch.tensor([0] + torch.tensor(sizes).cumsum(0).tolist(), dtype=torch.int32, device=DEV)
    x, w = _x(g, m, k), _weight(g, len(sizes), n, k)
    xq = _values(ops.mxfp4_quantize(x))
    got = ops.mxfp4_grouped_linear(x, *w, off)
    for e in range(len(sizes)):
        r = slice(int(off[e]), int(off[e + 1]))
        wv = _values((w[0][e], w[1][e]))
        y, mag = xq[r] @ wv.T, xq[r].abs() @ wv.abs().T
        assert ((got[r].double() - y).abs() <= M.linear_slack(mag, k, HALF_STEP[BF16], y)).all(), e


@pytest.mark.parametrize("m,n,k", [(7, 300, 1024), (60, 300, 1024), (100, 1000, 2048), (600, 7168, 1024), (1500, 7168, 512)])
def test_linear_with_exponents_off_the_16_byte_grid(m, n, k):
    """The stream, 32-row tiles, few tiles, 128-row and 256-row tiles."""
    g = _gen(m + n)
    x, (c, s) = _x(g, m, k), _weight(g, n, k)
    want = ops.mxfp4_linear(x, c, s)
    xc, xs = ops.mxfp4_quantize(x)
    for off in (4, 8, 12):
        assert torch.equal(ops.mxfp4_linear(x, c, _moved(s, off)), want)
        assert torch.equal(ops.mxfp4_linear((xc, _moved(xs, off)), c, _moved(s, off)), want)


@pytest.mark.parametrize("m", [6, 100, 2000])
def test_ffn_and_experts_with_exponents_off_the_16_byte_grid(m):
    g = _gen(m)
    d, n, E = 1024, 512, 5
    w = {"gate_proj": _weight(g, E, n, d), "up_proj": _weight(g, E, n, d), "down_proj": _weight(g, E, d, n)}
    w2 = {k: (c, _moved(s)) for k, (c, s) in w.items()}
    one, one2 = ({k: (c[2], s[2]) for k, (c, s) in v.items()} for v in (w, w2))
    x = _x(g, m, d)
    idx = torch.randint(0, E, (m, 3), generator=g, device=DEV)
    assert torch.equal(ops.dense_ffn(x, one2), ops.dense_ffn(x, one))
    assert torch.equal(ops.mxfp4_moe_experts(x, idx, w2), ops.mxfp4_moe_experts(x, idx, w))
    off = torch.tensor([0, m // 4, m // 4, m // 2, m // 2 + 1, m], dtype=torch.int32, device=DEV)
    assert torch.equal(ops.mxfp4_grouped_linear(x, *w2["up_proj"], off), ops.mxfp4_grouped_linear(x, *w["up_proj"], off))


# ------------------------------------------------------------------ C entries: bounds

GUARD = 4096


class _Buffers:
    """Buffers of exact sizes between guard bytes."""

    def __init__(self):
        self.kept = []

    def __call__(self, nbytes, fill=0x5a):
        t = torch.full((nbytes + 2 * GUARD,), 0xa7, dtype=torch.uint8, device=DEV)
        t[GUARD:GUARD + nbytes] = fill
        self.kept.append((t, nbytes))
        return t[GUARD:GUARD + nbytes]

    def whole(self):
        return all((t[:GUARD] == 0xa7).all() and (t[GUARD + n:] == 0xa7).all() for t, n in self.kept)


def _stream():
    return torch.cuda.current_stream().cuda_stream


@pytest.mark.parametrize("m,n,k,ldy", [(1, 100, 1152, 100), (5, 100, 640, 104), (16, 257, 13056, 257), (33, 999, 768, 1024),
                                       (100, 1000, 2048, 1000), (200, 1000, 18432, 1008), (500, 5120, 10240, 5120),
                                       (777, 640, 1664, 640), (1500, 1030, 512, 1030)])
@pytest.mark.parametrize("held", [False, True])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_linear_writes_its_outputs_and_workspace_only(m, n, k, ldy, held, dtype):
    L, g, buf = lib(), _gen(m), _Buffers()
    x, w = _x(g, m, k), _weight(g, n, k)
    xc, xs = ops.mxfp4_quantize(x)
    size = 4 if dtype == F32 else 2
    need = L.amla_mxfp4_linear_workspace_bytes(m, n, k, int(held))
    y, ws = buf(m * ldy * size, 0x33), buf(need)
    p = (xc.data_ptr(), xs.data_ptr()) if held else (x.data_ptr(), None)
    check(L.amla_mxfp4_linear(*p, m, k, k, w[0].data_ptr(), w[1].data_ptr(), n, y.data_ptr(), 2 if dtype == F32 else 0, ldy,
                              ws.data_ptr() if need else None, need, _stream()), "mxfp4_linear")
    got = y.view(dtype).view(m, ldy)
    assert torch.equal(got[:, :n], ops.mxfp4_linear((xc, xs) if held else x, *w, out_dtype=dtype))
    assert (got[:, n:].contiguous().view(torch.uint8) == 0x33).all() and buf.whole()


@pytest.mark.parametrize("sizes,n,k", [([3, 0, 5], 100, 640), ([0, 40, 1, 0, 30], 300, 384), ([300, 70, 0, 200], 8192, 512),
                                       ([1] * 50, 128, 128)])
@pytest.mark.parametrize("held", [False, True])
def test_grouped_linear_writes_its_outputs_and_workspace_only(sizes, n, k, held):
    L, g, buf = lib(), _gen(n), _Buffers()
    E, m = len(sizes), sum(sizes) + 4  # rows of no group behind
    off = torch.tensor([0] + torch.tensor(sizes).cumsum(0).tolist(), dtype=torch.int32, device=DEV)
    x, w = _x(g, m, k), _weight(g, E, n, k)
    xc, xs = ops.mxfp4_quantize(x)
    p = (xc.data_ptr(), xs.data_ptr()) if held else (x.data_ptr(), None)
    need = L.amla_mxfp4_grouped_linear_workspace_bytes(m, n, k, E, int(held))
    for clear in (0, 1):
        y, ws = buf(m * n * 2, 0x33), buf(need)
        check(L.amla_mxfp4_grouped_linear(*p, m, k, k, w[0].data_ptr(), w[1].data_ptr(), n, E, off.data_ptr(), y.data_ptr(),
                                          0, n, clear, ws.data_ptr(), need, _stream()), "mxfp4_grouped_linear")
        got = y.view(BF16).view(m, n)
        want = ops.mxfp4_grouped_linear((xc, xs) if held else x, *w, off)
        assert torch.equal(got[:m - 4], want[:m - 4])
        assert (y.view(m, 2 * n)[m - 4:] == (0 if clear else 0x33)).all() and buf.whole()


@pytest.mark.parametrize("m,k,n", [(1, 128, 128), (16, 1152, 640), (40, 512, 256), (300, 512, 4096), (1000, 640, 8192)])
def test_swiglu_writes_its_outputs_and_workspace_only(m, k, n):
    L, g, buf = lib(), _gen(m), _Buffers()
    x = _x(g, m, k)
    w = [t for shape in ((n, k), (n, k), (k, n)) for t in _weight(g, *shape)]
    need = L.amla_mxfp4_swiglu_workspace_bytes(m, k, n)
    y, ws = buf(m * k * 2), buf(need)
    a = [t.data_ptr() for t in w]
    check(L.amla_mxfp4_swiglu(x.data_ptr(), m, k, k, *a[:4], n, *a[4:], y.data_ptr(), ws.data_ptr(), need, _stream()), "swiglu")
    assert torch.equal(y.view(BF16).view(m, k), ops.mxfp4_swiglu(x, *w)) and buf.whole()


@pytest.mark.parametrize("m,d,n,E,top_k", [(1, 128, 128, 4, 64), (5, 256, 384, 6, 3), (16, 1152, 640, 8, 2), (17, 256, 128, 512, 3),
                                           (300, 256, 128, 2, 2), (300, 4096, 2048, 4, 2), (8000, 128, 128, 16, 8)])
def test_experts_write_their_outputs_and_workspace_only(m, d, n, E, top_k):
    L, g, buf = lib(), _gen(m), _Buffers()
    x = _x(g, m, d)
    w = {"gate_proj": _weight(g, E, n, d), "up_proj": _weight(g, E, n, d), "down_proj": _weight(g, E, d, n)}
    idx = torch.randint(-1, E + 1, (m, top_k), generator=g, device=DEV)
    need = L.amla_mxfp4_moe_experts_workspace_bytes(m, d, top_k, n, E)
    a = [t.data_ptr() for k in ("gate_proj", "up_proj", "down_proj") for t in w[k]]
    want = ops.mxfp4_moe_experts(x, idx, w)
    left = (idx < 0) | (idx >= E)
    for clear in (0, 1):
        y, ws = buf(m * top_k * d * 2, 0x33), buf(need)
        check(L.amla_mxfp4_moe_experts(x.data_ptr(), m, d, d, top_k, idx.data_ptr(), n, E, *a, y.data_ptr(), clear,
                                       ws.data_ptr(), need, _stream()), "moe_experts")
        got = y.view(BF16).view(m, top_k, d)
        assert torch.equal(got[~left], want[~left])
        assert (got[left].view(torch.uint8) == (0 if clear else 0x33)).all() and buf.whole()


# ------------------------------------------------------------------ past 32 bits

def test_linear_of_a_weight_past_four_gigabytes():
    g = _gen(1)
    n, k = 600001, 16384  # 4.9 GB of codes
    part = _weight(g, 4096, k)
    c = torch.empty(n, k // 2, dtype=torch.uint8, device=DEV)
    s = torch.empty(n, k // 32, dtype=torch.uint8, device=DEV)
    for a in range(0, n, 4096):
        b = min(n, a + 4096)
        c[a:b], s[a:b] = part[0][:b - a], part[1][:b - a]
    for m in (2, 40, 150):
        x = _x(g, m, k)
        y = ops.mxfp4_linear(x, c, s)
        xq, wv = _values(ops.mxfp4_quantize(x)), _values(part)
        want, mag = xq @ wv.T, xq.abs() @ wv.abs().T
        slack = M.linear_slack(mag, k, HALF_STEP[BF16], want)
        for a in (0, 4096, 4096 * 64, 4096 * 130, 4096 * 145, 4096 * 146):
            got = y[:, a:a + 4096].double()
            assert ((got - want[:, :got.shape[1]]).abs() <= slack[:, :got.shape[1]]).all(), (m, a)


def test_linear_of_activations_and_outputs_past_four_gigabytes():
    g = _gen(2)
    m, k, n = 1200003, 7168, 2048  # x 17 GB, its codes 4.3 GB, y 4.9 GB
    part, w = _x(g, 4096, k), _weight(g, n, k)
    x = torch.empty(m, k, dtype=BF16, device=DEV)
    for a in range(0, m, 4096):
        x[a:a + 4096] = part[:min(4096, m - a)]
    y = ops.mxfp4_linear(x, *w)
    xq, wv = _values(ops.mxfp4_quantize(part)), _values(w)
    want, mag = xq @ wv.T, xq.abs() @ wv.abs().T
    slack = M.linear_slack(mag, k, HALF_STEP[BF16], want)
    for a in (0, 4096, 4096 * 146, 4096 * 150, 4096 * 256, 4096 * 290, 4096 * 292):
        got = y[a:a + 4096].double()
        assert ((got - want[:len(got)]).abs() <= slack[:len(got)]).all(), a
