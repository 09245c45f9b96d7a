"""latent_attention against the definition in 64 bits (oracle/ref_latent.py)."""
import pytest
import torch

from _latent import BF16, DEV, cache_of, check_attention, to_dev
from amla import ops
from oracle import ref_latent as L

pytestmark = pytest.mark.gpu
SCALE = 0.0988


def _rows(g, n, spread=0.3):
    return torch.randn(n, 512, generator=g, dtype=torch.float64) * torch.exp(spread * torch.randn(n, 1, generator=g)), \
        torch.randn(n, 64, generator=g, dtype=torch.float64)


def _case(seed, lengths, S, H, fp8, page_size, spread=0.3, qstd=0.5, junk=float("nan")):
    g = torch.Generator().manual_seed(seed)
    parts = [_rows(g, n, spread) for n in lengths]
    cache, table = cache_of([p[0] for p in parts], [p[1] for p in parts], fp8, page_size, lengths, g, junk=junk)
    q = (torch.randn(len(lengths), S, H, 576, generator=g) * qstd).to(BF16)
    return q, cache, table, torch.tensor(lengths, dtype=torch.int32)


def _weight(q, cache, table, lengths, scale):
    """(attention of q over the magnitudes of the values, the largest scale sum |q k|)"""
    B, S, H, _ = q.shape
    pages, page = cache[0].shape[:2]
    lat, rope = L.pool_values(cache)
    out = torch.zeros(B, S, H, 512, dtype=torch.float64)
    size = 0.0
    for b in range(B):
        n = min(max(int(lengths[b]), 0), table.shape[1] * page)
        at = [L.places(table, b, t, page, pages) for t in range(n)]
        rows = [max(a, 0) for a in at]
        k = torch.cat([lat[rows], rope[rows]], -1)
        held = torch.tensor([a >= 0 for a in at], dtype=torch.bool)
        if held.any():
            size = max(size, (q[b].double().abs().flatten(0, 1) @ k[held].abs().T).max().item() * scale)
        for s in range(S):
            seen = torch.tensor([a >= 0 and t < n - (S - 1 - s) for t, a in enumerate(at)], dtype=torch.bool)
            out[b, s], _ = L.attention(q[b, s].double(), k, lat[rows].abs(), scale, seen.expand(H, n))
    return out, size


def _run(q, cache, table, lengths, scale=SCALE, what=""):
    print(f"[case] {what}", flush=True)
    got, lse = ops.latent_attention(to_dev(q), to_dev(cache), to_dev(table), to_dev(lengths), scale, return_lse=True)
    want, want_lse = L.latent_attention(q, cache, table, lengths, scale)
    check_attention(got, want, lse, want_lse, *_weight(q, cache, table, lengths, scale), what)
    return got, lse


@pytest.mark.parametrize("fp8", [True, False])
@pytest.mark.parametrize("lengths,S,H,page_size", [
    ([1], 1, 1, 1), ([1], 1, 128, 64), ([64], 1, 16, 64), ([65], 1, 128, 16), ([31, 33], 1, 8, 32), ([257], 1, 128, 64),
    ([0, 5, 0], 1, 20, 16), ([700, 1, 64, 63], 1, 40, 1), ([300, 129], 2, 33, 128), ([3, 1, 2, 130], 4, 64, 8),
    ([90], 3, 128, 64), ([50, 64, 66], 1, 70, 2),
])
def test_against_the_definition(fp8, lengths, S, H, page_size):
    _run(*_case(sum(lengths) + S * H, lengths, S, H, fp8, page_size), what=f"fp8={fp8} {lengths} S={S} H={H} page={page_size}")


@pytest.mark.parametrize("fp8", [True, False])
def test_long_sequences_are_split_and_joined(fp8):
    """Enough tiles for several splits each, of unequal lengths, and batches with more sequences than slots."""
    _run(*_case(1, [5000, 777, 2049], 1, 16, fp8, 64), what=f"fp8={fp8} split")
    _run(*_case(2, [1 + (37 * i) % 90 for i in range(200)], 1, 4, fp8, 16), what=f"fp8={fp8} 200 sequences")


@pytest.mark.parametrize("fp8", [True, False])
def test_rows_of_unlike_scales(fp8):
    """Rows from 2^-12 to 2^12 of each other's size: the factor rides on the probabilities."""
    g = torch.Generator().manual_seed(4)
    n = 333
    lat = torch.randn(n, 512, generator=g, dtype=torch.float64) * torch.exp2(torch.randint(-12, 13, (n, 1), generator=g).double())
    lat[5] = 0
    pe = torch.randn(n, 64, generator=g, dtype=torch.float64)
    cache, table = cache_of([lat], [pe], fp8, 16, [n], g, junk=float("nan"))
    q = (torch.randn(1, 1, 16, 576, generator=g) * 1e-3).to(BF16)
    _run(q, cache, table, torch.tensor([n], dtype=torch.int32), what=f"fp8={fp8} unlike scales")


@pytest.mark.parametrize("fp8", [True, False])
def test_a_maximum_that_keeps_moving(fp8):
    """Scores that rise along the sequence by more than the lazy maximum allows, and fall."""
    g = torch.Generator().manual_seed(8)
    for rising in (True, False):
        n = 400
        ramp = torch.linspace(0, 60, n, dtype=torch.float64)
        lat = 0.02 * torch.randn(n, 512, generator=g, dtype=torch.float64)
        lat[:, 0] = ramp if rising else ramp.flip(0)
        pe = torch.zeros(n, 64, dtype=torch.float64)
        cache, table = cache_of([lat], [pe], fp8, 64, [n], g)
        q = torch.zeros(1, 1, 32, 576)
        q[..., 0] = torch.linspace(0.1, 10, 32)
        _run(q.to(BF16), cache, table, torch.tensor([n], dtype=torch.int32), scale=0.5, what=f"fp8={fp8} rising={rising}")


@pytest.mark.parametrize("fp8", [True, False])
def test_many_faint_rows_outweigh_one_loud(fp8):
    """One row 2^15 and 2^24 times as probable as each of 5000 others: their part is not lost."""
    g = torch.Generator().manual_seed(18)
    n = 5000
    lat = 0.2 * torch.randn(n, 512, generator=g, dtype=torch.float64)
    lat[:, 1] = 1.0
    lat[:, 0] = 0.0
    for at in (0, 17, 4000):
        lat[at, 0], lat[at, 1] = 8.0, -1.0
        pe = torch.zeros(n, 64, dtype=torch.float64)
        cache, table = cache_of([lat], [pe], fp8, 64, [n], g)
        q = torch.zeros(1, 1, 2, 576)
        q[0, 0, :, 0] = torch.tensor([15.0, 24.0]) * 0.6931 / 8.0
        got, _ = _run(q.to(BF16), cache, table, torch.tensor([n], dtype=torch.int32), scale=1.0, what=f"fp8={fp8} loud row {at}")
        lat[at, 0], lat[at, 1] = 0.0, 1.0


@pytest.mark.parametrize("fp8", [True, False])
def test_pages_outside_the_pool_hold_no_rows(fp8):
    q, cache, table, lengths = _case(31, [200, 90, 40], 1, 16, fp8, 16)
    table[0, 3], table[0, 12], table[1, 0], table[2, :] = -1, cache[0].shape[0], 2 ** 31 - 1, -7
    _run(q, cache, table, lengths, what=f"fp8={fp8} bad pages")
    lengths = torch.tensor([10 ** 9, -3, 5], dtype=torch.int32)       # past the table: its end; below zero: none
    _run(q, cache, table, lengths, what=f"fp8={fp8} bad lengths")


def _wider(table, cols):
    """The table with more columns, of no pages: more rows than there are count for the choice of a workgroup's size."""
    return torch.cat([table, torch.full((table.shape[0], cols - table.shape[1]), -1, dtype=torch.int32)], 1)


@pytest.mark.parametrize("fp8", [True, False])
@pytest.mark.parametrize("S,H,cols", [(1, 128, 530), (3, 40, 560), (2, 17, 2000), (1, 64, 1100)])
def test_workgroups_of_more_query_rows(fp8, S, H, cols):
    """Two and four groups of 32 query rows: taken where sequences x rows x columns' rows pass 256 CUs times 32768."""
    lens = [700, 65]
    q, cache, table, lengths = _case(S + H, lens, S, H, fp8, 64)
    _run(q, cache, _wider(table, cols), lengths, what=f"fp8={fp8} S={S} H={H} {cols} columns")


@pytest.mark.parametrize("fp8", [True, False])
@pytest.mark.parametrize("S,H,cols", [(3, 5, 0), (2, 64, 0), (3, 128, 0), (2, 30, 1100), (3, 128, 200), (70, 4, 0)])
def test_what_a_token_does_not_see_does_not_reach_it(fp8, S, H, cols):
    """An infinity or a NaN in one of the newest rows: the tokens before it keep their bits, the others get NaN."""
    q, cache, table, lengths = _case(71, [200, 129], S, H, fp8, 16)
    table = _wider(table, cols * 4) if cols else table
    run = lambda c: ops.latent_attention(to_dev(q), c, to_dev(table), to_dev(lengths), SCALE, return_lse=True)  # noqa: E731
    print(f"[case] fp8={fp8} S={S} H={H}", flush=True)
    want, want_lse = run(to_dev(cache))
    assert torch.isfinite(want).all()
    for back, kind in ((1, "row"), (1, "one"), (S - 1, "one"), (1, "rope"), (S // 2, "row")):
        dc = to_dev(tuple(t.clone() for t in cache))
        for b, n in ((0, 200), (1, 129)):
            page, at = table[b, (n - back) // 16], (n - back) % 16
            if kind == "rope":
                dc[1][page, at, 7] = float("nan")
            elif fp8 and kind == "row":
                dc[0].view(torch.uint8)[page, at], dc[2][page, at] = 0x7F, 255
            elif fp8:
                dc[0].view(torch.uint8)[page, at, 300] = 0xFF
            else:
                dc[0][page, at, 300 if kind == "one" else slice(None)] = float("inf") if kind == "one" else float("nan")
        got, lse = run(dc)
        sees = S - back  # the first token that sees the row
        assert torch.equal(got[:, :sees], want[:, :sees]) and torch.equal(lse[:, :sees], want_lse[:, :sees]), (back, kind)
        assert torch.isnan(got[:, sees:]).all(), (back, kind)


def test_strides_and_no_lse():
    q, cache, table, lengths = _case(6, [100, 37], 2, 24, True, 16)
    want, _ = _run(q, cache, table, lengths, what="contiguous")
    dq, dc, dt, dl = to_dev(q), to_dev(cache), to_dev(table), to_dev(lengths)
    wide = torch.zeros(2, 24, 2, 584, dtype=BF16, device=DEV)
    wide[..., :576] = dq.transpose(1, 2)
    assert torch.equal(ops.latent_attention(wide[..., :576].transpose(1, 2), dc, dt, dl, SCALE), want)
    odd = torch.zeros(2, 2, 24, 577, dtype=BF16, device=DEV)
    odd[..., 1:] = dq
    assert torch.equal(ops.latent_attention(odd[..., 1:], dc, dt, dl, SCALE), want)
    tw = torch.full((2, table.shape[1] + 5), -1, dtype=torch.int32, device=DEV)
    tw[:, 2:2 + table.shape[1]] = dt
    assert torch.equal(ops.latent_attention(dq, dc, tw[:, 2:2 + table.shape[1]], dl, SCALE), want)
    assert ops.latent_attention(dq[:, :0], dc, dt, dl, SCALE).shape == (2, 0, 24, 512)


@pytest.mark.parametrize("fp8", [True, False])
def test_two_graphs_two_streams_and_repeats(fp8):
    """Two captured graphs replayed in turn and on two streams at once, lengths read at each replay; equal inputs give
    equal bits."""
    q, cache, table, lengths = _case(12, [900, 300, 64], 1, 32, fp8, 64)
    dq, dc, dt, dl = to_dev(q), to_dev(cache), to_dev(table), to_dev(lengths)
    print("[case] graphs", flush=True)
    run = lambda: ops.latent_attention(dq, dc, dt, dl, SCALE, return_lse=True)  # noqa: E731
    run()
    torch.cuda.synchronize()
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(run())
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in range(2)]
    for lens in ([900, 300, 64], [1, 0, 33], [640, 299, 5]):
        dl.copy_(torch.tensor(lens, dtype=torch.int32))
        want = run()
        torch.cuda.synchronize()
        for s, g in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for o in outs:
            assert torch.equal(o[0], want[0]) and torch.equal(o[1], want[1]), lens
        again = run()
        assert torch.equal(again[0], want[0]) and torch.equal(again[1], want[1])


def test_gradients_are_refused():
    q, cache, table, lengths = to_dev(_case(1, [9], 1, 4, True, 16))
    o = ops.latent_attention(q.requires_grad_(), cache, table, lengths, SCALE)
    with pytest.raises(RuntimeError, match="no backward"):
        o.float().sum().backward()
