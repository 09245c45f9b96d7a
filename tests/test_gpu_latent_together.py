"""The operators of the paged cache as a server runs them together: prompts are stored, read back and attended to, then
tokens are decoded over the same pages, eagerly and in a captured graph."""
import math

import pytest
import torch

from _latent import BF16, DEV, FP8, HALF_BF16, check_attention, to_dev
from amla import ops
from amla.config import DeepSeekConfig
from oracle import ref_latent as L

pytestmark = pytest.mark.gpu
CFG = DeepSeekConfig()
SCALE = ops.softmax_scale(CFG)
H = 16


def _offsets(lens):
    return torch.tensor([sum(lens[:b]) for b in range(len(lens) + 1)], dtype=torch.int32)


class _Server:
    """A pool, two matrices that stand for kv_b (per head 128 key and 128 value columns of the latent), and rows."""

    def __init__(self, seed, dtype, lens, room, page=16):
        g = torch.Generator().manual_seed(seed)
        self.g, self.lens, self.page = g, list(lens), page
        need = [-(-(n + room) // page) for n in lens]
        pages = sum(need) + 3
        self.cache = ops.latent_cache(pages, page, CFG, DEV, dtype)
        order = torch.randperm(pages, generator=g).to(torch.int32)
        self.table = torch.full((len(lens), max(need)), -1, dtype=torch.int32)
        at = 0
        for b, n in enumerate(need):
            self.table[b, :n] = order[at:at + n]
            at += n
        self.freqs = ops.precompute_rope_freqs(CFG, 2048, device=DEV)
        self.gamma = (1 + 0.2 * torch.randn(512, generator=g)).to(BF16).to(DEV)
        self.w = (torch.randn(H, 256, 512, generator=g) / 512 ** 0.5).to(BF16)
        self.dt = self.table.to(DEV)

    def rows(self, *shape):
        return torch.randn(*shape, 576, generator=self.g).to(BF16).to(DEV)

    def kv_b(self, latent):
        return (latent.float() @ self.w.to(DEV).float().flatten(0, 1).T).to(BF16).view(-1, H, 256)

    def check_decode(self, q, lens, got, lse, what):
        cache = to_dev(self.cache, "cpu")
        lens = torch.tensor(lens, dtype=torch.int32)
        want, want_lse = L.latent_attention(q.cpu(), cache, self.table, lens, SCALE)
        lat, rope = L.pool_values(cache)
        weight = torch.zeros_like(want)
        size = 0.0
        for b in range(len(lens)):
            at = [L.places(self.table, b, t, self.page, cache[0].shape[0]) for t in range(int(lens[b]))]
            k = torch.cat([lat[at], rope[at]], -1)
            size = max(size, (q[b].double().cpu().abs().flatten(0, 1) @ k.abs().T).max().item() * SCALE)
            for s in range(q.shape[1]):
                n = int(lens[b]) - (q.shape[1] - 1 - s)
                weight[b, s], _ = L.attention(q[b, s].double().cpu(), k[:n], lat[at][:n].abs(), SCALE,
                                              torch.ones(q.shape[2], n, dtype=torch.bool))
        check_attention(got, want, lse, want_lse, weight, size, what)


@pytest.mark.parametrize("dtype", [FP8, BF16])
def test_prompts_then_tokens(dtype):
    lens = [70, 5, 133]
    s = _Server(3, dtype, lens, room=8)
    off = _offsets(lens).to(DEV)
    zero = torch.zeros(3, dtype=torch.int32, device=DEV)
    print(f"[case] {dtype} prompts", flush=True)
    ops.latent_cache_write(s.rows(sum(lens)), s.gamma, s.freqs, s.cache, s.dt, zero, offsets=off)

    # the prompts' attention, on what the cache holds of them
    latent, k_pe = ops.latent_cache_read(s.cache, s.dt, off, sum(lens))
    kvb = s.kv_b(latent)
    q = (0.5 * torch.randn(sum(lens), H, 192, generator=s.g)).to(BF16).to(DEV)
    out, lse = ops.packed_attention(q, kvb[..., :128], kvb[..., 128:], off, SCALE, k_pe=k_pe, return_lse=True)
    cq, ck, cv, cp, co = (t.cpu() for t in (q, kvb[..., :128], kvb[..., 128:], k_pe, off))
    want, want_lse = L.packed_attention(cq, ck, cv, co, SCALE, co, cp, True)
    weight, _ = L.packed_attention(cq, ck, cv.abs(), co, SCALE, co, cp, True)
    kk = torch.cat([ck, cp[:, None].expand(-1, H, -1)], -1)
    size = SCALE * max((cq[:, h].double().abs() @ kk[:, h].double().abs().T).max().item() for h in range(H))
    check_attention(out, want, lse, want_lse, weight, size, f"{dtype} prompts")

    # a prompt's last token once more, as a decode step: kv_b absorbed into its query and taken out of its result
    last = (off[1:] - 1).long()
    w = s.w.to(DEV).float()
    q_lat = torch.einsum("bhd,hdc->bhc", q[last][..., :128].float(), w[:, :128]).to(BF16)
    qd = torch.cat([q_lat, q[last][..., 128:]], -1)[:, None]
    n = torch.tensor(lens, dtype=torch.int32, device=DEV)
    o_lat, lse_d = ops.latent_attention(qd, s.cache, s.dt, n, SCALE, return_lse=True)
    s.check_decode(qd, lens, o_lat, lse_d, f"{dtype} last tokens")
    o = torch.einsum("bhc,hdc->bhd", o_lat[:, 0].float(), w[:, 128:])
    # the two differ by bf16 roundings, 2^-8 of their products at most: of the absorbed query and of kv_b's keys in the
    # scores (ds), of kv_b's values, of both attentions' probabilities and outputs (2^-6 of the weights for all)
    for b in range(3):
        rows = slice(int(off[b]), int(off[b + 1]))
        ds = SCALE * HALF_BF16 * max(
            (q_lat[b].float().abs() @ latent[rows].float().abs().T).max().item()
            + (torch.einsum("hd,nhd->hn", q[last[b]][..., :128].float().abs(), kvb[rows][..., :128].float().abs())).max().item(), 0.0)
        wt = torch.einsum("hc,hdc->hd", latent[rows].float().abs().max(0).values.expand(H, -1), w[:, 128:].abs())
        bound = wt * (math.expm1(2 * ds) + 2.0 ** -6) + 2.0 ** -20
        assert ((o[b] - out[last[b]].float()).abs() <= bound).all(), b
        assert ((lse_d[b, 0] - lse[last[b]]).abs() <= ds + 1e-4).all(), b

    # follow-up tokens: three at once, then one by one
    pos = list(lens)
    for new in (3, 1, 1):
        ops.latent_cache_write(s.rows(3, new), s.gamma, s.freqs, s.cache, s.dt, torch.tensor(pos, dtype=torch.int32, device=DEV))
        pos = [p + new for p in pos]
        qd = (0.5 * torch.randn(3, new, H, 576, generator=s.g)).to(BF16).to(DEV)
        o, l = ops.latent_attention(qd, s.cache, s.dt, torch.tensor(pos, dtype=torch.int32, device=DEV), SCALE, return_lse=True)
        s.check_decode(qd, pos, o, l, f"{dtype} {new} new")


@pytest.mark.parametrize("dtype", [FP8, BF16])
def test_a_captured_step_advances_by_itself(dtype):
    """Store, attend and count up in one graph: each replay is the next token; a second server's eager steps between."""
    lens = [40, 63]
    a, b = (_Server(4, dtype, lens, room=8) for _ in range(2))
    off = _offsets(lens).to(DEV)
    prompt = a.rows(sum(lens))
    steps = [(a.rows(2, 1), (0.5 * torch.randn(2, 1, H, 576, generator=a.g)).to(BF16).to(DEV)) for _ in range(5)]
    for s in (a, b):
        ops.latent_cache_write(prompt, s.gamma, s.freqs, s.cache, s.dt, torch.zeros(2, dtype=torch.int32, device=DEV), offsets=off)
    n = torch.tensor(lens, dtype=torch.int32, device=DEV)
    kv, q, after = steps[0][0].clone(), steps[0][1].clone(), torch.empty_like(n)
    print(f"[case] {dtype} graph", flush=True)

    def step(s, kv, q, n, after):
        ops.latent_cache_write(kv, s.gamma, s.freqs, s.cache, s.dt, n)
        torch.add(n, 1, out=after)
        o = ops.latent_attention(q, s.cache, s.dt, after, SCALE, return_lse=True)
        n.copy_(after)
        return o

    keep = [t.clone() for t in a.cache]
    step(a, kv, q, n.clone(), after)  # (warm-up on the same rows, undone)
    for t, k in zip(a.cache, keep):
        t.copy_(k)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(a, kv, q, n, after)
    m, m_after = torch.tensor(lens, dtype=torch.int32, device=DEV), torch.empty(2, dtype=torch.int32, device=DEV)
    for kv_i, q_i in steps:
        kv.copy_(kv_i)
        q.copy_(q_i)
        graph.replay()
        torch.cuda.synchronize()
        one = [t.clone() for t in got]
        want = step(b, kv_i, q_i, m, m_after)
        assert torch.equal(one[0], want[0]) and torch.equal(one[1], want[1])
    for t, u in zip(a.cache, b.cache):
        assert torch.equal(t.view(torch.uint8), u.view(torch.uint8))


@pytest.mark.parametrize("dtype", [FP8, BF16])
def test_pools_past_four_gigabytes(dtype):
    """The last pages of a pool whose latents take more than 2^32 bytes, against the same rows in a small one."""
    lens, page = [100, 65], 64
    pages = 2 ** 32 // (page * (512 if dtype == FP8 else 1024)) + 100
    assert pages * page < 2 ** 31
    small = _Server(5, dtype, lens, room=4, page=page)
    big = ops.latent_cache(pages, page, CFG, DEV, dtype)
    table = torch.where(small.dt >= 0, pages - 1 - small.dt, -1)
    off, zero = _offsets(lens).to(DEV), torch.zeros(2, dtype=torch.int32, device=DEV)
    kv, new = small.rows(sum(lens)), small.rows(2, 2)
    q = (0.5 * torch.randn(2, 2, H, 576, generator=small.g)).to(BF16).to(DEV)
    n = torch.tensor(lens, dtype=torch.int32, device=DEV)
    print(f"[case] {dtype} {pages} pages", flush=True)
    got = []
    for cache, t in ((small.cache, small.dt), (big, table)):
        ops.latent_cache_write(kv, small.gamma, small.freqs, cache, t, zero, offsets=off)
        ops.latent_cache_write(new, small.gamma, small.freqs, cache, t, n)
        got.append(ops.latent_cache_read(cache, t, off, sum(lens)) + ops.latent_attention(q, cache, t, n + 2, SCALE, return_lse=True))
    for x, y in zip(*got):
        assert torch.equal(x, y)
    assert torch.isfinite(got[0][2]).all()


def test_packed_rows_past_two_to_31_values():
    """Queries, keys and outputs whose offsets pass 2^31 values and 2^32 bytes: the same sequence at both ends."""
    heads, n, rows = 128, 70, 100000
    g = torch.Generator(device=DEV).manual_seed(6)
    q = torch.zeros(rows, heads, 192, dtype=BF16, device=DEV)
    kvb = torch.zeros(rows, heads, 256, dtype=BF16, device=DEV)
    pe = torch.zeros(rows, 64, dtype=BF16, device=DEV)
    for t in (q, kvb, pe):
        t[:n] = torch.randn(t[:n].shape, generator=g, device=DEV).to(BF16)
        t[-n:] = t[:n]
    off = torch.tensor([0, n, rows - n, rows - n, rows], dtype=torch.int32, device=DEV)
    koff = torch.tensor([0, n, n, rows - n, rows], dtype=torch.int32, device=DEV)  # (the middle: queries without keys)
    print("[case] past 2^31", flush=True)
    o, lse = ops.packed_attention(q, kvb[..., :128], kvb[..., 128:], off, SCALE, k_offsets=koff, k_pe=pe, return_lse=True)
    assert torch.equal(o[:n], o[-n:]) and torch.equal(lse[:n], lse[-n:]) and (o[:n] != 0).any()
    assert (o[n:-n] == 0).all() and (lse[n:-n] == float("-inf")).all()


def test_another_stream_than_the_default():
    lens = [90, 20]
    s = _Server(7, FP8, lens, room=4)
    off, zero = _offsets(lens).to(DEV), torch.zeros(2, dtype=torch.int32, device=DEV)
    kv = s.rows(sum(lens))
    q = (0.5 * torch.randn(sum(lens), H, 192, generator=s.g)).to(BF16).to(DEV)
    qd = (0.5 * torch.randn(2, 1, H, 576, generator=s.g)).to(BF16).to(DEV)
    n = torch.tensor(lens, dtype=torch.int32, device=DEV)

    def run():
        ops.latent_cache_write(kv, s.gamma, s.freqs, s.cache, s.dt, zero, offsets=off)
        latent, k_pe = ops.latent_cache_read(s.cache, s.dt, off, sum(lens))
        kvb = s.kv_b(latent)
        return (ops.packed_attention(q, kvb[..., :128], kvb[..., 128:], off, SCALE, k_pe=k_pe),
                ops.latent_attention(qd, s.cache, s.dt, n, SCALE))

    print("[case] streams", flush=True)
    want = run()
    torch.cuda.synchronize()
    for t in s.cache:
        t.view(torch.uint8).zero_()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = run()
    stream.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_no_sequences_and_no_pages():
    s = _Server(8, FP8, [5], room=0)
    none = torch.empty(0, 4, dtype=torch.int32, device=DEV)
    e = torch.empty(0, dtype=torch.int32, device=DEV)
    print("[case] empty", flush=True)
    ops.latent_cache_write(s.rows(0, 1), s.gamma, s.freqs, s.cache, none, e)
    ops.latent_cache_write(s.rows(0), s.gamma, s.freqs, s.cache, none, e, offsets=torch.zeros(1, dtype=torch.int32, device=DEV))
    lat, pe = ops.latent_cache_read(s.cache, none, torch.zeros(1, dtype=torch.int32, device=DEV), 3)
    assert not lat.any() and not pe.any()
    assert ops.latent_attention(torch.empty(0, 1, H, 576, dtype=BF16, device=DEV), s.cache, none, e, SCALE).shape == (0, 1, H, 512)
    bare = torch.empty(2, 0, dtype=torch.int32, device=DEV)  # two sequences, a table without columns
    before = s.cache[0].view(torch.uint8).clone()
    two = torch.zeros(2, dtype=torch.int32, device=DEV)
    ops.latent_cache_write(s.rows(2, 1), s.gamma, s.freqs, s.cache, bare, two)
    assert torch.equal(s.cache[0].view(torch.uint8), before)
    q = torch.ones(2, 1, H, 576, dtype=BF16, device=DEV)
    o, lse = ops.latent_attention(q, s.cache, bare, two + 9, SCALE, return_lse=True)
    assert not o.any() and (lse == float("-inf")).all()


@pytest.mark.parametrize("dtype", [FP8, BF16])
def test_traced_and_in_inference_mode(dtype):
    """A step that is compiled, with its writes as side effects, and one under inference mode give the eager step's bits."""
    lens = [50, 9]
    n = torch.tensor(lens, dtype=torch.int32, device=DEV)

    def step(s, kv, q, n):
        ops.latent_cache_write(kv, s.gamma, s.freqs, s.cache, s.dt, n)
        return ops.latent_attention(q, s.cache, s.dt, n + 1, SCALE, return_lse=True)

    def fresh():
        s = _Server(9, dtype, lens, room=4)
        ops.latent_cache_write(s.rows(sum(lens)), s.gamma, s.freqs, s.cache, s.dt, torch.zeros_like(n), offsets=_offsets(lens).to(DEV))
        return s, s.rows(2, 1), (0.5 * torch.randn(2, 1, H, 576, generator=s.g)).to(BF16).to(DEV)

    print(f"[case] {dtype} traced", flush=True)
    s, kv, q = fresh()
    want = step(s, kv, q, n)
    for run in (torch.compile(step, backend="aot_eager"), torch.inference_mode()(step)):
        t, kv, q = fresh()
        got = run(t, kv, q, n)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        for a, b in zip(s.cache, t.cache):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
