"""latent_cache_write and latent_cache_read against the definition in 64 bits (oracle/ref_latent.py)."""
import pytest
import torch

from _latent import BF16, DEV, FP8, HALF_BF16, to_dev
from amla import ops
from amla.config import DeepSeekConfig
from oracle import ref_latent as L
from oracle import ref_ops as R

pytestmark = pytest.mark.gpu
CFG = DeepSeekConfig()


def _freqs(n):
    return R.precompute_rope_freqs(CFG, n)


def _kv(g, *shape):
    x = torch.randn(*shape, 576, generator=g) * torch.exp(torch.randn(*shape, 1, generator=g))
    x[..., 3:512:90] *= 8.0
    return x.to(BF16)


def _gamma(g):
    return (1.0 + 0.3 * torch.randn(512, generator=g)).to(BF16)


def _table(g, B, cols, pages):
    return torch.randperm(pages, generator=g)[:B * cols].view(B, cols).to(torch.int32)


def _check_rows(lat, pe, kv, gamma, freqs, eps, fp8, what):
    """lat, pe (n, .) read back against kv (n, 576).  The norm in fp32: a sum of 512 squares, a rsqrt and two products
    are within 2^-20 of the exact value; one rounding follows, half a step of bf16, or of e4m3 at the row's exponent:
    2^-4 relative, at least half the subnormal step 2^-10 of the scale.  Where the fp32 maximum falls on the other
    side of 448 2^e the step doubles."""
    want = L.normed(kv, gamma, eps)
    slack = 2.0 ** -20 * want.abs()
    if fp8:
        unit = torch.exp2(L.exponent(want * (1 + 2.0 ** -20)).double())[:, None]
        bound = torch.maximum(2.0 ** -4 * want.abs(), 2.0 ** -10 * unit) + 1.01 * slack
    else:
        bound = HALF_BF16 * want.abs() + 1.01 * slack
    d = (lat.double().cpu() - want).abs()
    assert (d <= bound).all(), f"{what}: latent {(d / bound.clamp_min(1e-300)).max().item():.3f} x the bound"
    r = L.rotated(kv, freqs)
    x = kv[:, 512:].double().reshape(-1, 32, 2)
    size = (x.abs().sum(-1, keepdim=True)).expand(-1, -1, 2).reshape(-1, 64)
    d = (pe.double().cpu() - r).abs()
    assert (d <= HALF_BF16 * r.abs() + 2.0 ** -22 * size).all(), f"{what}: rope key"


@pytest.mark.parametrize("fp8", [True, False])
@pytest.mark.parametrize("page_size,B,S", [(1, 3, 1), (16, 5, 7), (64, 2, 130), (128, 1, 1), (4, 70, 2)])
def test_write_then_read_uniform(fp8, page_size, B, S):
    g = torch.Generator().manual_seed(11 + page_size + S)
    cols = 300 // page_size + 1
    table = _table(g, B, cols, B * cols + 3)
    cache = ops.latent_cache(B * cols + 3, page_size, CFG, DEV, FP8 if fp8 else BF16)
    kv, gamma, freqs = _kv(g, B, S), _gamma(g), _freqs(300)
    start = torch.randint(0, 300 - S + 1, (B,), generator=g, dtype=torch.int32)
    print(f"[case] write uniform fp8={fp8} page={page_size} B={B} S={S}", flush=True)
    ops.latent_cache_write(kv.to(DEV), gamma.to(DEV), freqs.to(DEV), cache, table.to(DEV), start.to(DEV), eps=1e-6)
    off = torch.arange(B + 1, dtype=torch.int32) * S
    lat, pe = ops.latent_cache_read(cache, table.to(DEV), off.to(DEV), B * S, position=start.to(DEV))
    rows = torch.cat([freqs[s:s + S] for s in start.tolist()])
    _check_rows(lat, pe, kv.reshape(-1, 576), gamma, rows, 1e-6, fp8, "uniform")
    # nothing else of the pool was written
    own = torch.zeros(cache[0].shape[0] * page_size, dtype=torch.bool)
    for b in range(B):
        for i in range(S):
            own[L.places(table, b, int(start[b]) + i, page_size, cache[0].shape[0])] = True
    assert (cache[0].view(torch.uint8 if fp8 else torch.int16).reshape(own.numel(), -1).cpu()[~own] == 0).all()
    assert (cache[1].reshape(own.numel(), -1).cpu()[~own] == 0).all()
    if fp8:
        assert (cache[2].reshape(-1).cpu()[~own] == 127).all()


@pytest.mark.parametrize("fp8", [True, False])
@pytest.mark.parametrize("lens", [[1], [0, 5, 0, 0, 33, 1], [257, 3], [0, 0]])
def test_packed_rows_and_reading_from_row_zero(fp8, lens):
    g = torch.Generator().manual_seed(5 + sum(lens))
    B, ps, cols = len(lens), 16, 20
    pages = B * cols + 1
    table = _table(g, B, cols, pages)
    cache = ops.latent_cache(pages, ps, CFG, DEV, FP8 if fp8 else BF16)
    T = sum(lens)
    kv, gamma, freqs = _kv(g, T), _gamma(g), _freqs(320)
    off = torch.tensor([sum(lens[:b]) for b in range(B + 1)], dtype=torch.int32)
    print(f"[case] write packed fp8={fp8} lens={lens}", flush=True)
    ops.latent_cache_write(kv.to(DEV), gamma.to(DEV), freqs.to(DEV), cache, table.to(DEV), 0, offsets=off.to(DEV))
    lat, pe = ops.latent_cache_read(cache, table.to(DEV), off.to(DEV), T)
    rows = torch.cat([freqs[:n] for n in lens])
    _check_rows(lat, pe, kv, gamma, rows, 1e-6, fp8, "packed")


def test_codes_and_exponents_of_known_rows():
    """Rows whose norm is the identity (gamma makes up for it): maxima at, just above and below 448 2^e."""
    g = torch.Generator().manual_seed(3)
    cache = ops.latent_cache(8, 1, CFG, DEV)
    gamma = torch.ones(512, dtype=BF16)
    kv = torch.zeros(6, 576, dtype=BF16)
    kv[0, :512] = 1.0                                        # normed: ones
    kv[1, 0] = 3.0                                           # one value: sqrt(512) = 22.6
    kv[2] = 0.0                                              # zeros
    kv[3, :512] = torch.randn(512, generator=g).to(BF16)
    kv[4, 7] = float("inf")
    kv[5, 9] = float("nan")
    table = torch.arange(8, dtype=torch.int32)[None]
    print("[case] known rows", flush=True)
    ops.latent_cache_write(kv[None].to(DEV), gamma.to(DEV), _freqs(8).to(DEV), cache, table.to(DEV), 0)
    codes, scale = cache[0].view(torch.uint8).cpu()[:, 0], cache[2].cpu()[:, 0]
    assert scale[:3].tolist() == [127 - 8, 127 - 4, 127 - 32]     # 1 <= 448 2^-8, 22.6 <= 448 2^-4
    v = L.code_values(codes) * torch.exp2(scale.double()[:, None] - 127)
    assert (v[0] == 1.0).all() and (v[2] == 0).all()
    assert abs(v[1, 0].item() - 512 ** 0.5) <= 2.0 ** -4 * 512 ** 0.5 and (v[1, 1:] == 0).all()
    assert scale[4] == scale[5] == 255 and ((codes[4:6] & 127) == 127).all()
    lat, _ = ops.latent_cache_read(cache, table.to(DEV), torch.tensor([0, 6], dtype=torch.int32, device=DEV), 6)
    assert torch.isnan(lat[4:6].float()).all() and torch.isfinite(lat[:4].float()).all()


@pytest.mark.parametrize("gain", [2.0 ** -60, 2.0 ** -30, 2.0 ** 30, 2.0 ** 60])
def test_exponents_stop_at_32(gain):
    """gamma of 2^-60 .. 2^60: exponents are clamped, values below flush, values above saturate."""
    g = torch.Generator().manual_seed(9)
    cache = ops.latent_cache(1, 4, CFG, DEV)
    kv = torch.randn(1, 4, 576, generator=g).to(BF16)
    gamma = torch.full((512,), gain, dtype=BF16)
    table = torch.zeros(1, 1, dtype=torch.int32, device=DEV)
    print(f"[case] gain {gain}", flush=True)
    ops.latent_cache_write(kv.to(DEV), gamma.to(DEV), _freqs(4).to(DEV), cache, table, 0)
    want = L.normed(kv[0], gamma, 1e-6)
    e = L.exponent(want)
    assert torch.equal(cache[2].cpu()[0].long() - 127, e)
    unit = torch.exp2(e.double())[:, None]
    v = L.code_values(cache[0].view(torch.uint8).cpu()[0]) * unit
    cut = want.clamp(min=-448 * unit, max=448 * unit)
    assert ((v - cut).abs() <= torch.maximum(2.0 ** -4 * cut.abs(), 2.0 ** -10 * unit) * (1 + 2.0 ** -15)).all()


@pytest.mark.parametrize("fp8", [True, False])
def test_rows_without_a_place(fp8):
    """Pages outside the pool, positions past the rope table or the block table, rows of no sequence."""
    g = torch.Generator().manual_seed(21)
    ps, pages = 4, 6
    cache = ops.latent_cache(pages, ps, CFG, DEV, FP8 if fp8 else BF16)
    table = torch.tensor([[2, -1, 5], [7, 0, 2 ** 31 - 1], [3, -2 ** 31, 1]], dtype=torch.int32)
    kv, gamma, freqs = _kv(g, 40), _gamma(g), _freqs(11)
    off = torch.tensor([2, 14, 26, 38], dtype=torch.int32)   # rows 0, 1, 38, 39 belong to no sequence
    print(f"[case] no place fp8={fp8}", flush=True)
    ops.latent_cache_write(kv.to(DEV), gamma.to(DEV), freqs.to(DEV), cache, table.to(DEV), 0, offsets=off.to(DEV))
    held = {(b, t) for b in range(3) for t in range(12) if L.places(table, b, t, ps, pages) >= 0 and t < 11}
    lat, pe = ops.latent_cache_read(cache, table.to(DEV), off.to(DEV), 40)
    want = L.normed(kv, gamma, 1e-6)
    for i in range(40):
        b = (i - 2) // 12 if 2 <= i < 38 else -1
        if b < 0 or (b, i - 2 - 12 * b) not in held:
            assert (lat[i] == 0).all() and (pe[i] == 0).all(), i
        else:
            assert (lat[i].double().cpu() - want[i]).abs().max() <= 2.0 ** -4 * want[i].abs().max()
    out = (torch.full((40, 512), 7.0, dtype=BF16, device=DEV), torch.full((40, 64), 7.0, dtype=BF16, device=DEV))
    got = ops.latent_cache_read(cache, table.to(DEV), off.to(DEV), 40, out=out)
    assert got[0] is out[0] and got[1] is out[1]
    for i in range(40):
        b = (i - 2) // 12 if 2 <= i < 38 else -1
        none = b < 0 or L.places(table, b, i - 2 - 12 * b, ps, pages) < 0
        assert (out[0][i] == 7.0).all() == none and (out[1][i] == 7.0).all() == none, i


def test_strides_alignment_and_offsets_that_run_backwards():
    g = torch.Generator().manual_seed(2)
    cache = ops.latent_cache(40, 8, CFG, DEV)
    table = _table(g, 2, 9, 40)
    wide = torch.full((2, 12), -5, dtype=torch.int32)
    wide[:, 1:10] = table
    kv, gamma, freqs = _kv(g, 2, 9), _gamma(g), _freqs(80)
    store = torch.zeros(2, 18, 640, dtype=BF16, device=DEV)
    view = store[:, ::2, 3:579]                              # odd start, strided rows
    view.copy_(kv)
    odd = torch.zeros(513, dtype=BF16, device=DEV)
    odd[1:].copy_(gamma)
    print("[case] strides", flush=True)
    ops.latent_cache_write(view, odd[1:], freqs.to(DEV), cache, wide.to(DEV)[:, 1:10], [3, 60])
    off = torch.tensor([0, 9, 18], dtype=torch.int32, device=DEV)
    lat, pe = ops.latent_cache_read(cache, table.to(DEV), off, 18, position=torch.tensor([3, 60], dtype=torch.int32, device=DEV))
    _check_rows(lat, pe, kv.reshape(-1, 576), gamma, torch.cat([freqs[3:12], freqs[60:69]]), 1e-6, True, "strides")
    before = [t.clone() for t in (cache[0].view(torch.uint8), cache[1], cache[2])]
    # a list that runs backwards or past the end moves rows to another place or to none, nothing else
    for bad in ([18, 9, 0], [-4, 100, 7], [5, 5, 5]):
        o = torch.tensor(bad, dtype=torch.int32, device=DEV)
        ops.latent_cache_write(view.reshape(18, 576), gamma.to(DEV), freqs.to(DEV), cache, table.to(DEV), -9 + 9, offsets=o)
        ops.latent_cache_read(cache, table.to(DEV), o, 18)
    torch.cuda.synchronize()
    free = torch.ones(40, dtype=torch.bool)
    free[table.flatten().long()] = False
    for t, was in zip((cache[0].view(torch.uint8), cache[1], cache[2]), before):
        assert torch.equal(t.cpu()[free], was.cpu()[free])


def test_graph_replays_follow_the_inputs():
    """A captured write and read: positions, rows and the table are read on the device at each replay."""
    g = torch.Generator().manual_seed(77)
    B, ps = 4, 16
    cache = ops.latent_cache(80, ps, CFG, DEV)
    table = _table(g, B, 20, 80).to(DEV)
    gamma, freqs = _gamma(g).to(DEV), _freqs(320).to(DEV)
    kv = torch.zeros(B, 1, 576, dtype=BF16, device=DEV)
    pos = torch.zeros(B, dtype=torch.int32, device=DEV)
    off = torch.arange(B + 1, dtype=torch.int32, device=DEV)

    def step():
        ops.latent_cache_write(kv, gamma, freqs, cache, table, pos)
        return ops.latent_cache_read(cache, table, off, B, position=pos)

    print("[case] graph", flush=True)
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for i in range(5):
        kv.copy_(_kv(g, B, 1))
        pos.copy_(torch.randint(0, 320, (B,), generator=g, dtype=torch.int32))
        graph.replay()
        want = tuple(t.clone() for t in got)
        again = step()
        torch.cuda.synchronize()
        assert torch.equal(again[0], want[0]) and torch.equal(again[1], want[1]), i


def test_gradients_are_refused():
    cache = ops.latent_cache(4, 4, CFG, DEV)
    table = torch.zeros(1, 1, dtype=torch.int32, device=DEV)
    kv = torch.zeros(1, 2, 576, dtype=BF16, device=DEV, requires_grad=True)
    args = (torch.ones(512, dtype=BF16, device=DEV), _freqs(4).to(DEV), cache, table, 0)
    with pytest.raises(RuntimeError, match="no gradient"):
        ops.latent_cache_write(kv, *args)
    with torch.no_grad():
        ops.latent_cache_write(kv, *args)
