"""latent_attention where its number formats and its passes over the tiles end: sums far from one, scores far below zero,
references that are set anew, in every kernel that it has."""
import pytest
import torch

from _latent import BF16, cache_of, check_attention, to_dev
from amla import ops
from oracle import ref_latent as L
from test_gpu_latent_attention import SCALE, _case, _run, _weight, _wider

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("e", [4, 9, 20, 32])
@pytest.mark.parametrize("H,cols", [(16, 0), (40, 0), (64, 1100)])
def test_columns_of_zeros_in_split_sequences(e, H, cols):
    """Rows of exponent e whose values are 0 in one run of 128 columns: the sum that the outputs are divided by is 2^-e of a
    usual one, and a wave that holds only these columns has no value to take a power of two from."""
    g = torch.Generator().manual_seed(40 + e + H)
    lens, lat, pe = [5000, 700], [], []
    for n in lens:
        x = torch.randn(n, 512, generator=g, dtype=torch.float64)
        x[:, 128:256] = 0
        lat.append(x / x.abs().amax(1, keepdim=True) * 448 * 2.0 ** e * (0.6 + 0.4 * torch.rand(n, 1, generator=g, dtype=torch.float64)))
        pe.append(torch.randn(n, 64, generator=g, dtype=torch.float64))
    cache, table = cache_of(lat, pe, True, 64, lens, g, junk=float("nan"))
    assert (cache[2].flatten()[(cache[2] != 255).flatten()].int() - 127 == e).float().mean() > 0.8
    q = (torch.randn(2, 1, H, 576, generator=g) * (3.2 / (448 * 2.0 ** e * 384 ** 0.5))).to(BF16)
    _run(q, cache, _wider(table, cols) if cols else table, torch.tensor(lens, dtype=torch.int32), scale=1.0,
         what=f"zero columns, e={e} H={H}")


@pytest.mark.parametrize("fp8", [True, False])
@pytest.mark.parametrize("S,H,cols", [(1, 16, 0), (1, 64, 450), (1, 128, 450), (2, 16, 0), (2, 32, 450), (2, 64, 450)])
def test_no_rows_and_a_query_that_is_no_number(fp8, S, H, cols):
    """A slot of the batch without a sequence: its pages are none, its query is whatever was there.  Zeros, like for any
    token that sees no row, and nothing of it in the others."""
    lens = [100, 70, 5000, 3, 17]
    q, cache, table, lengths = _case(61 + S + H, lens, S, H, fp8, 16)
    table[1], table[2], table[4, 0] = -1, -1, cache[0].shape[0]
    clean = q.clone()
    q[1] = float("nan")
    q[2, ..., 5] = float("inf")
    if S > 1:
        q[4, 0] = float("nan")  # sees the absent page only, where the last token sees a row more
    table = _wider(table, max(cols * 4, table.shape[1]))
    print(f"[case] fp8={fp8} S={S} H={H}", flush=True)
    got, lse = ops.latent_attention(to_dev(q), to_dev(cache), to_dev(table), to_dev(lengths), SCALE, return_lse=True)
    want, want_lse = L.latent_attention(clean, cache, table, lengths, SCALE)
    assert (want_lse[[1, 2]] == float("-inf")).all() and ((want_lse[4] == float("-inf")).sum() == (S - 1) * H)
    check_attention(got, want, lse, want_lse, *_weight(clean, cache, table, lengths, SCALE), f"fp8={fp8} S={S} H={H} no rows")


@pytest.mark.parametrize("fp8", [True, False])
@pytest.mark.parametrize("H", [8, 64, 128])
def test_long_sequences_over_few_pages(fp8, H):
    """More than 2^12 tiles in one lane's sum of the plan: tables that name three pages of 512 rows over and over."""
    g = torch.Generator().manual_seed(27)
    n = 1536
    cache, once = cache_of([torch.randn(n, 512, generator=g, dtype=torch.float64)], [torch.randn(n, 64, generator=g, dtype=torch.float64)],
                           fp8, 512, [n], g, junk=float("nan"))
    lens = [270000, 5, 300007, 131073]
    table = torch.stack([once[0, (torch.arange(600) + b) % 3] for b in range(4)])
    q = (torch.randn(4, 1, H, 576, generator=g) * 0.5).to(BF16)
    print(f"[case] fp8={fp8} H={H} long", flush=True)
    got, lse = ops.latent_attention(to_dev(q), to_dev(cache), to_dev(table), to_dev(torch.tensor(lens, dtype=torch.int32)), SCALE,
                                    return_lse=True)
    lat, rope = L.pool_values(cache)
    rows = torch.tensor([L.places(once, 0, t, 512, cache[0].shape[0]) for t in range(n)])
    k = torch.cat([lat[rows], rope[rows]], -1)
    want, weight = torch.zeros(2, 4, 1, H, 512, dtype=torch.float64)
    want_lse = torch.zeros(4, 1, H, dtype=torch.float64)
    for b, m in enumerate(lens):  # the rows as often as they are held
        often = (m // n + (torch.arange(n) < m % n)).double().roll(512 * b)
        s = q[b, 0].double() @ k.T * SCALE + often.log()
        want_lse[b, 0] = s.logsumexp(-1)
        p = (s - want_lse[b, 0, :, None]).exp()
        want[b, 0], weight[b, 0] = p @ lat[rows], p @ lat[rows].abs()
    size = SCALE * (q.double().abs().flatten(0, 2) @ k.abs().T).max().item()
    check_attention(got, want, lse, want_lse, weight, size, f"fp8={fp8} H={H} long")


@pytest.mark.parametrize("fp8", [True, False])
@pytest.mark.parametrize("B,H,cols", [(2, 3, 0), (100, 33, 0), (100, 64, 30), (100, 128, 30)])
def test_scores_far_below_zero(fp8, B, H, cols):
    """Every score -1e33, of the last rows, which are alike, or -2e33, of those before.  At this size scores a unit in the last
    place apart are worlds apart in probability, and alike ones may differ by one: any mean of the last rows is right, so
    d out is 2^-8 of it and 2^-10 more for the sums in between (and 2^-100 of the largest value: an e4m3 block's probabilities
    end at 2^-123), and d lse 2^-20 of it."""
    g = torch.Generator().manual_seed(H)
    n, first = 300, 260
    lat = torch.randn(n, 512, generator=g, dtype=torch.float64) * (1e12 if fp8 else 2.0 ** 57)
    lat[:, 0] = -448 * 2.0 ** 32 if fp8 else -2.0 ** 57
    lat[:first, 0] *= 1.0 if fp8 else 2.0
    lat[:first, 1] = lat[0, 0]
    lat[first:, 1] = 0
    lat[first:] = lat[first].clone()
    cache, table = cache_of([lat], [torch.zeros(n, 64, dtype=torch.float64)], fp8, 64, [n], g)
    last = L.pool_values(cache)[0][L.places(table, 0, n - 1, 64, cache[0].shape[0])]
    q = torch.zeros(B, 1, H, 576)
    q[..., 0] = 2.0 ** 72 if fp8 else 2.0 ** 56
    q[..., 1] = 2.0 ** 72 if fp8 else 0.0
    table = _wider(table, max(cols, table.shape[1])).repeat(B, 1)
    lengths = torch.full((B,), n, dtype=torch.int32)
    print(f"[case] fp8={fp8} B={B} H={H}", flush=True)
    got, lse = ops.latent_attention(to_dev(q.to(BF16)), to_dev(cache), to_dev(table), to_dev(lengths), 0.1, return_lse=True)
    assert ((got.double().cpu() - last).abs() <= (2.0 ** -8 + 2.0 ** -10) * last.abs() + 2.0 ** -100 * last.abs().max()).all()
    z = 0.1 * (last[0] + last[1]) * q[0, 0, 0, 0]
    assert -1e34 < z < -1e32 and ((lse.double().cpu() - z).abs() <= 2.0 ** -20 * z.abs()).all()


@pytest.mark.parametrize("fp8", [True, False])
@pytest.mark.parametrize("H,cols", [(3, 0), (64, 30), (128, 30)])
def test_scores_far_apart(fp8, H, cols):
    """Blocks of 32 rows of score z, of -1.75 z and of -0.375 z, z from 2^24 to 2^100: the first, which are alike, and nothing of
    the others."""
    g = torch.Generator().manual_seed(3)
    n, B = 500, 100
    lat = torch.randn(n, 512, generator=g, dtype=torch.float64)
    kind = (torch.arange(n) // 32) % 3
    loud = kind == 1
    lat[loud] = lat[40].clone()
    lat[:, 0] = torch.tensor([-1.75, 1.0, -0.375])[kind].double()
    cache, table = cache_of([lat], [torch.zeros(n, 64, dtype=torch.float64)], fp8, 64, [n], g)
    row = L.pool_values(cache)[0][L.places(table, 0, 40, 64, cache[0].shape[0])]
    table = _wider(table, max(cols, table.shape[1])).repeat(B, 1)
    q = torch.zeros(B, 1, H, 576)
    each = torch.arange(B * H).view(B, H)
    powers = each % 76 + 24
    q[:, 0, :, 0] = torch.exp2(powers.float()) * (1 + each * 37 % 128 / 128.0)
    lengths = torch.full((B,), n, dtype=torch.int32)
    print(f"[case] fp8={fp8} H={H} far apart", flush=True)
    got, lse = ops.latent_attention(to_dev(q.to(BF16)), to_dev(cache), to_dev(table), to_dev(lengths), 0.7, return_lse=True)
    far = ((got.double().cpu() - row).abs() / ((2.0 ** -8 + 2.0 ** -10) * row.abs() + 2.0 ** -100)).amax((1, 3))
    assert (far <= 1).all(), f"2^{sorted({int(p) for p in powers[~(far <= 1)]})}: {far.max().item()}"
    z = 0.7 * q[:, 0, :, 0].double()
    assert ((lse[:, 0].double().cpu() - z).abs() <= 2.0 ** -20 * z).all()



def _many(lat, pe, fp8, B, g, cols=0):
    """(cache, table (B, .), lengths, the lengths there are): B sequences over the same pages, so that a workgroup's split has
    several tiles; every third one is shorter by 37 rows, every third by 100."""
    n = lat.shape[0]
    cache, table = cache_of([lat], [pe], fp8, 64, [n], g, junk=float("nan"))
    table = _wider(table, max(cols, table.shape[1]))
    kinds = torch.tensor([n, n - 37, n - 100], dtype=torch.int32)
    return cache, table.repeat(B, 1), kinds[torch.arange(B) % 3], kinds


def _check_many(q, cache, table, lengths, scale, what):
    """The same queries for every sequence: the first three against the definition, the others the same up to where their
    splits begin."""
    B = table.shape[0]
    print(f"[case] {what}", flush=True)
    qs = to_dev(q).expand(B, -1, -1, -1)
    run = lambda: ops.latent_attention(qs, to_dev(cache), to_dev(table), to_dev(lengths), scale, return_lse=True)  # noqa: E731
    got, lse = run()
    few = q.expand(3, -1, -1, -1), cache, table[:3], lengths[:3], scale
    want, want_lse = L.latent_attention(*few)
    weight, size = _weight(*few)
    for b in range(0, B, 90):
        k = min(90, B - b)
        some = torch.arange(k) % 3
        check_attention(got[b:b + k], want[some], lse[b:b + k], want_lse[some], weight[some], size, f"{what}, from {b}")
    again = run()
    assert torch.equal(again[0], got) and torch.equal(again[1], lse), what
    return got


# query rows: one group of the kernel for few of them, several of those, two groups of it, four groups of the other one
KERNELS = [(1, 32, 0), (1, 72, 0), (1, 64, 40), (1, 128, 40), (3, 8, 0), (3, 20, 40), (3, 43, 40)]


@pytest.mark.parametrize("fp8", [True, False])
@pytest.mark.parametrize("S,H,cols", KERNELS)
def test_a_reference_that_is_set_anew(fp8, S, H, cols):
    """Scores that rise by up to 70 in log2 from one tile of a split to the next: sequences of five to 13 tiles, and so many of
    them that a split has up to five."""
    g = torch.Generator().manual_seed(H)
    n = 400
    for rising in (True, False):
        ramp = torch.linspace(0, 60, n, dtype=torch.float64)
        lat = 0.02 * torch.randn(n, 512, generator=g, dtype=torch.float64)
        lat[:, 0] = ramp if rising else ramp.flip(0)
        cache, table, lengths, _ = _many(lat, torch.zeros(n, 64, dtype=torch.float64), fp8, 270 * 64 // min(H * S, 64), g, cols)
        q = torch.zeros(1, S, H, 576)
        q[..., 0] = torch.linspace(0.1, 10, S * H).view(S, H)
        _check_many(q.to(BF16), cache, table, lengths, 0.5, f"fp8={fp8} S={S} H={H} rising={rising}")


@pytest.mark.parametrize("fp8", [True, False])
@pytest.mark.parametrize("S,H,cols", [k for k in KERNELS if k[0] > 1])
def test_a_masked_row_that_is_no_number_where_the_reference_is_set_anew(fp8, S, H, cols):
    g = torch.Generator().manual_seed(5 * H)
    n, B = 400, 270 * 64 // min(H * S, 64)
    lat = 0.02 * torch.randn(n, 512, generator=g, dtype=torch.float64)
    lat[:, 0] = torch.linspace(0, 60, n, dtype=torch.float64)
    cache, table, _, _ = _many(lat, torch.zeros(n, 64, dtype=torch.float64), fp8, B, g, cols)
    lengths = torch.full((B,), n, dtype=torch.int32)
    q = torch.zeros(1, S, H, 576)
    q[..., 0] = torch.linspace(0.1, 10, S * H).view(S, H)
    want = _check_many(q.to(BF16), cache, table, lengths, 0.5, f"fp8={fp8} S={S} H={H}")
    page, at = table[0, (n - 1) // 64], (n - 1) % 64
    if fp8:
        cache[0].view(torch.uint8)[page, at, 300] = 0x7F
    else:
        cache[0][page, at, 300] = float("inf")
    qs = to_dev(q.to(BF16)).expand(B, -1, -1, -1)
    got = ops.latent_attention(qs, to_dev(cache), to_dev(table), to_dev(lengths), 0.5)
    assert torch.equal(got[:, :S - 1], want[:, :S - 1]) and torch.isnan(got[:, S - 1]).all()


@pytest.mark.parametrize("fp8", [True, False])
@pytest.mark.parametrize("S,H,cols", [k for k in KERNELS if k[0] == 1])
def test_rows_of_unlike_scales_in_splits_of_several_tiles(fp8, S, H, cols):
    g = torch.Generator().manual_seed(4 + H)
    n = 433
    lat = torch.randn(n, 512, generator=g, dtype=torch.float64) * torch.exp2(torch.randint(-12, 13, (n, 1), generator=g).double())
    lat[5] = 0
    cache, table, lengths, _ = _many(lat, torch.randn(n, 64, generator=g, dtype=torch.float64), fp8, 270 * 64 // min(H, 64), g, cols)
    q = (torch.randn(1, S, H, 576, generator=g) * 1e-3).to(BF16)
    _check_many(q, cache, table, lengths, SCALE, f"fp8={fp8} H={H} unlike scales")


@pytest.mark.parametrize("fp8", [True, False])
@pytest.mark.parametrize("H,cols", [(32, 0), (64, 200), (128, 200)])
def test_many_faint_rows_outweigh_one_loud_in_splits_of_several_tiles(fp8, H, cols):
    """One row 2^15 and 2^24 times as probable as each of 5000 others, 12 sequences: splits of four tiles and more."""
    g = torch.Generator().manual_seed(18)
    n, B = 5000, 12
    for at in (0, 17, 4000):
        lat = 0.2 * torch.randn(n, 512, generator=g, dtype=torch.float64)
        lat[:, 1], lat[:, 0] = 1.0, 0.0
        lat[at, 0], lat[at, 1] = 8.0, -1.0
        cache, table, lengths, _ = _many(lat, torch.zeros(n, 64, dtype=torch.float64), fp8, B, g, cols)
        q = torch.zeros(1, 1, H, 576)
        q[..., 0] = torch.tensor([15.0, 24.0]).repeat(H // 2) * 0.6931 / 8.0
        _check_many(q.to(BF16), cache, table, lengths, 1.0, f"fp8={fp8} H={H} loud row {at}")


@pytest.mark.parametrize("fp8", [True, False])
@pytest.mark.parametrize("S,H,cols", KERNELS)
def test_the_mean_error_is_that_of_two_roundings(fp8, S, H, cols):
    """The output is rounded to 8 bits, and so is each probability, whose errors are independent of each other: an rms error of
    at most 2^-8 / sqrt(3) of the values from either (half a step is 2^-8 of a power of two, and no value is below its own),
    0.0032 together.  Of values spread evenly over an octave it is 0.0022; one bit less in either place makes that 0.0034."""
    g = torch.Generator().manual_seed(H + S)
    n = 700
    cache, table, lengths, _ = _many(torch.randn(n, 512, generator=g, dtype=torch.float64), torch.randn(n, 64, generator=g, dtype=torch.float64),
                                     fp8, 60, g, cols)
    q = (torch.randn(1, S, H, 576, generator=g) * 0.6).to(BF16)
    got = _check_many(q, cache, table, lengths, SCALE, f"fp8={fp8} S={S} H={H} rms")
    want, _ = L.latent_attention(q.expand(3, -1, -1, -1), cache, table[:3], lengths[:3], SCALE)
    for b in range(0, 60, 3):
        rms = (got[b:b + 3].double().cpu() - want).square().mean().sqrt() / want.square().mean().sqrt()
        assert rms <= 2.0 ** -8 * (2 / 3) ** 0.5, f"{b}: {rms.item():.5f}"


@pytest.mark.parametrize("fp8", [True, False])
@pytest.mark.parametrize("S,H,cols", KERNELS)
def test_a_query_that_is_no_number_stays_alone(fp8, S, H, cols):
    """NaN for it, the bits of a call without it for all others; an infinite one has its workgroup start over."""
    g = torch.Generator().manual_seed(H + 3)
    n, B = 400, 270 * 64 // min(H * S, 64)
    cache, table, lengths, _ = _many(torch.randn(n, 512, generator=g, dtype=torch.float64), torch.randn(n, 64, generator=g, dtype=torch.float64),
                                     fp8, B, g, cols)
    q = (torch.randn(B, S, H, 576, generator=g) * 0.5).to(BF16)
    run = lambda q: ops.latent_attention(to_dev(q), to_dev(cache), to_dev(table), to_dev(lengths), SCALE, return_lse=True)  # noqa: E731
    want, want_lse = run(q)
    bad = torch.zeros(B, S, H, dtype=torch.bool)
    bad[1, 0, 0], bad[2, S - 1, H // 2:], bad[B - 1, 0, H - 1] = True, True, True
    q[bad] = float("nan")
    q[1, 0, 0], q[1, 0, 0, 7] = 0.0, float("inf")
    print(f"[case] fp8={fp8} S={S} H={H}", flush=True)
    got, lse = run(q)
    assert torch.isnan(got.cpu()[bad]).all() and torch.isnan(lse.cpu()[bad]).all()
    assert torch.equal(got.cpu()[~bad], want.cpu()[~bad]) and torch.equal(lse.cpu()[~bad], want_lse.cpu()[~bad])
