"""packed_attention against the definition in 64 bits (oracle/ref_latent.py)."""
import pytest
import torch

from _latent import BF16, DEV, check_attention, to_dev
from amla import ops
from oracle import ref_latent as L

pytestmark = pytest.mark.gpu


def _offsets(lens):
    return torch.tensor([sum(lens[:b]) for b in range(len(lens) + 1)], dtype=torch.int32)


def _case(seed, new, lens, H, G, form, std=1.0):
    g = torch.Generator().manual_seed(seed)
    T, N = sum(new), sum(lens)
    r = lambda *s: (torch.randn(*s, generator=g) * std).to(BF16)  # noqa: E731
    dk = 128 if form == "plain" else 192
    q, pe = r(T, H, dk), None
    if form == "mla":
        kvb = r(N, G, 256)
        k, v, pe = kvb[..., :128], kvb[..., 128:], r(N, 64)
    else:
        k, v = r(N, G, dk), r(N, G, 128)
    return q, k, v, pe, _offsets(new), _offsets(lens), 1.0 / dk ** 0.5


def _run(q, k, v, pe, off, koff, scale, causal=True, what=""):
    print(f"[case] {what}", flush=True)
    got, lse = ops.packed_attention(to_dev(q), to_dev(k), to_dev(v), to_dev(off), scale, k_offsets=to_dev(koff), k_pe=to_dev(pe),
                                    causal=causal, return_lse=True)
    want, want_lse = L.packed_attention(q, k, v, off, scale, koff, pe, causal)
    weight, _ = L.packed_attention(q, k, v.abs(), off, scale, koff, pe, causal)
    kk = k if pe is None else torch.cat([k, pe[:, None].expand(-1, k.shape[1], -1)], -1)
    size = scale * max((q[:, h].double().abs() @ kk[:, h * k.shape[1] // q.shape[1]].double().abs().T).max().item()
                       for h in range(q.shape[1]))
    check_attention(got, want, lse, want_lse, weight, size, what)
    return got, lse


@pytest.mark.parametrize("form,H,G", [("mla", 8, 8), ("mla", 16, 2), ("whole", 4, 4), ("whole", 6, 3), ("plain", 8, 2), ("plain", 5, 1)])
@pytest.mark.parametrize("new,past", [([1], [0]), ([33], [0]), ([1, 64, 65], [0, 0, 0]), ([300, 7], [0, 0]), ([5, 1], [200, 63])])
def test_causal_against_the_definition(form, H, G, new, past):
    lens = [a + b for a, b in zip(new, past)]
    _run(*_case(sum(lens) + H, new, lens, H, G, form), what=f"{form} H={H}/{G} new={new} past={past}")


@pytest.mark.parametrize("form", ["mla", "plain"])
def test_not_causal_and_unlike_lengths(form):
    _run(*_case(3, [70, 3], [129, 300], 4, 2, form), causal=False, what=f"{form} not causal")
    # fewer keys than queries: the first queries see nothing; sequences without queries or keys
    _run(*_case(4, [40, 0, 9, 5], [25, 6, 0, 70], 4, 2, form), what=f"{form} empty rows")
    _run(*_case(5, [9, 4], [0, 3], 4, 2, form), causal=False, what=f"{form} no keys")


@pytest.mark.parametrize("new,past,H,G,form", [([1], [3001], 3, 1, "plain"), ([40, 3], [2500, 700], 16, 16, "mla"), ([300], [1500], 6, 3, "whole"),
                                              ([1, 0, 7], [255, 900, 4096], 8, 2, "mla"), ([1100], [0], 2, 2, "plain")])
def test_few_blocks_split_their_keys(new, past, H, G, form):
    lens = [a + b for a, b in zip(new, past)]
    _run(*_case(41 + H, new, lens, H, G, form), what=f"{form} split {new} behind {past}")
    _run(*_case(42 + H, new, lens, H, G, form), causal=False, what=f"{form} split, not causal")


def test_split_keys_that_keep_rising_and_a_captured_call():
    q, k, v, pe, off, koff, scale = _case(43, [5], [2000], 4, 2, "plain")
    k[:] = 0
    k[:, :, 0] = torch.linspace(0, 2000, 2000)[:, None].to(BF16)
    q[:, :, 0] = 4.0
    _run(q, k, v, pe, off, koff, scale, what="split, rising")
    _run(q, k.flip(0), v, pe, off, koff, scale, what="split, falling")
    d = [to_dev(t) for t in (q, k, v, off, koff)]
    run = lambda: ops.packed_attention(d[0], d[1], d[2], d[3], scale, k_offsets=d[4], return_lse=True)  # noqa: E731
    run()
    torch.cuda.synchronize()
    graphs, outs = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(run())
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in range(2)]
    for keys in (2000, 300, 5, 1999):
        d[4].copy_(_offsets([keys]))
        want = run()
        torch.cuda.synchronize()
        for s, graph in zip(streams, graphs):
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        for o in outs:
            assert torch.equal(o[0], want[0]) and torch.equal(o[1], want[1]), keys


def test_many_sequences_and_blocks_of_queries():
    new = [(13 * i) % 40 for i in range(90)]
    _run(*_case(6, new, new, 2, 1, "plain"), what="90 sequences")
    _run(*_case(7, [513, 256, 257], [513, 700, 257], 2, 2, "mla"), what="blocks")


def test_scores_that_keep_rising():
    """Keys along one direction with rising length: the running maximum moves in most tiles."""
    q, k, v, pe, off, koff, scale = _case(8, [400], [400], 2, 2, "plain")
    k[:] = 0
    k[:, :, 0] = torch.linspace(0, 300, 400)[:, None].to(BF16)
    q[:, :, 0] = 4.0
    _run(q, k, v, pe, off, koff, scale, what="rising")
    _run(q, k.flip(0), v, pe, off, koff, scale, causal=False, what="falling")


@pytest.mark.parametrize("new,past,H,G,form", [([40], [0], 2, 1, "plain"), ([300, 70], [0, 90], 4, 4, "mla"), ([513], [100], 2, 2, "whole"),
                                              ([300, 70], [0, 90], 130, 130, "plain"), ([20], [1500], 2, 1, "mla")])
def test_what_a_query_does_not_see_does_not_reach_it(new, past, H, G, form):
    """Infinities and NaN in a later key and in its values: the queries before it keep their bits, and the others the bits
    of every column without one."""
    lens = [a + b for a, b in zip(new, past)]
    q, k, v, pe, off, koff, scale = _case(21, new, lens, H, G, form)
    run = lambda k, v: ops.packed_attention(to_dev(q), to_dev(k), to_dev(v), to_dev(off), scale, k_offsets=to_dev(koff),  # noqa: E731
                                            k_pe=to_dev(pe))
    print(f"[case] {form} {new} {past}", flush=True)
    want = run(k, v)
    assert torch.isfinite(want).all()
    for b in range(len(new)):
        for first in sorted({1, new[b] // 3, new[b] - 1}):  # the first query that sees the key
            key, row = int(koff[b]) + past[b] + first, int(off[b]) + first
            sees = torch.zeros(sum(new), dtype=torch.bool, device=DEV)
            sees[row:int(off[b + 1])] = True
            v2, k2 = v.clone(), k.clone()
            v2[key, :, 3], v2[key, :, 77], v2[key, :, 78] = float("inf"), float("nan"), float("-inf")
            got = run(k, v2)
            assert torch.equal(got[~sees], want[~sees]), (b, first)
            rest = [c for c in range(128) if c not in (3, 77, 78)]
            assert torch.equal(got[sees][..., rest], want[sees][..., rest]), (b, first)
            assert (got[sees][..., 3] == float("inf")).all() and torch.isnan(got[sees][..., 77]).all(), (b, first)
            assert (got[sees][..., 78] == float("-inf")).all(), (b, first)
            k2[key] = float("nan")
            got = run(k2, v)
            assert torch.equal(got[~sees], want[~sees]) and torch.isnan(got[sees]).all(), (b, first)


@pytest.mark.parametrize("col", [3, 77])
def test_a_masked_nan_in_a_column_that_another_lane_holds(col):
    """A lane holds every other four keys of its query, and other columns than theirs: three queries, all keys in one lane."""
    q, k, v, pe, off, koff, scale = _case(22, [3], [3], 2, 2, "plain")
    run = lambda v: ops.packed_attention(to_dev(q), to_dev(k), to_dev(v), to_dev(off), scale)  # noqa: E731
    print(f"[case] column {col}", flush=True)
    want = run(v)
    v2 = v.clone()
    v2[2, :, col] = float("nan")
    got = run(v2)
    rest = [c for c in range(128) if c != col]
    assert torch.equal(got[:2], want[:2]) and torch.equal(got[..., rest], want[..., rest]) and torch.isnan(got[2, :, col]).all()


def test_strides_alignment_and_no_lse():
    q, k, v, pe, off, koff, scale = _case(9, [50, 20], [50, 20], 4, 4, "mla")
    want, _ = _run(q, k, v, pe, off, koff, scale, what="views of kv_b")
    d = lambda t: t.to(DEV)  # noqa: E731
    call = lambda q_, k_, v_, pe_: ops.packed_attention(q_, k_, v_, d(off), scale, k_pe=pe_)  # noqa: E731
    assert torch.equal(call(d(q).transpose(0, 1).contiguous().transpose(0, 1), d(k).contiguous(), d(v).contiguous(), d(pe)), want)
    odd = torch.zeros(70, 4, 195, dtype=BF16, device=DEV)
    odd[..., 3:] = d(q)
    ope = torch.zeros(70, 65, dtype=BF16, device=DEV)
    ope[:, 1:] = d(pe)
    assert torch.equal(call(odd[..., 3:], d(k), d(v), ope[:, 1:]), want)


def test_rows_of_no_sequence_are_left_and_bad_offsets_stay_inside():
    q, k, v, pe, _, _, scale = _case(10, [60], [60], 4, 4, "mla")
    d = [to_dev(t) for t in (q, k, v, pe)]
    for bad in ([0, 20, 10, 60], [-5, 30, 1000, 2000], [60, 0, 60, 0], [7, 7, 7, 7]):
        print(f"[case] offsets {bad}", flush=True)
        o = torch.tensor(bad, dtype=torch.int32, device=DEV)
        ops.packed_attention(d[0], d[1], d[2], o, scale, k_pe=d[3])
        torch.cuda.synchronize()


def test_graph_replays_follow_the_offsets():
    q, k, v, pe, off, koff, scale = _case(11, [100, 60], [100, 60], 4, 2, "mla")
    d = [to_dev(t) for t in (q, k, v, pe, off)]
    run = lambda: ops.packed_attention(d[0], d[1], d[2], d[4], scale, k_pe=d[3], return_lse=True)  # noqa: E731
    print("[case] graph", flush=True)
    run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run()
    for lens in ([100, 60], [3, 157], [160, 0], [80, 80]):
        d[4].copy_(_offsets(lens))
        graph.replay()
        torch.cuda.synchronize()
        one = tuple(t.clone() for t in got)
        want = run()
        assert torch.equal(one[0], want[0]) and torch.equal(one[1], want[1]), lens


def test_gradients_are_refused():
    q, k, v, pe, off, _, scale = to_dev(_case(1, [9], [9], 2, 2, "mla"))
    o = ops.packed_attention(q, k, v.clone().requires_grad_(), off, scale, k_pe=pe)
    with pytest.raises(RuntimeError, match="no backward"):
        o.float().sum().backward()
