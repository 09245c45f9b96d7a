"""packed_attention at its edges: rows of no sequence, many sequences whose keys are split, far strides, scores far from zero."""
import ctypes

import pytest
import torch

from _latent import BF16, DEV, check_attention, to_dev
from amla import _lib, ops
from oracle import ref_latent as L
from test_gpu_packed_attention import _case, _run

pytestmark = pytest.mark.gpu


def _split_keys(T, N, B, H):
    return _lib.lib().amla_packed_attention_workspace_bytes(T, N, B, H) > 0


def _entry(q, k, v, pe, off, koff, scale, out, lse):
    """The C entry, with the caller's outputs."""
    T, H, N, B = q.shape[0], q.shape[1], k.shape[0], off.shape[0] - 1
    need = _lib.lib().amla_packed_attention_workspace_bytes(T, N, B, H)
    ws = torch.empty(max(need, 16), dtype=torch.uint8, device=DEV)
    args = _lib.PackedArgs(q.data_ptr(), k.data_ptr(), v.data_ptr(), None if pe is None else pe.data_ptr(), out.data_ptr(), lse.data_ptr(),
                           off.data_ptr(), koff.data_ptr(), T, N, B, q.stride(0), q.stride(1), k.stride(0), k.stride(1), v.stride(0),
                           v.stride(1), 0 if pe is None else pe.stride(0), H, k.shape[1], k.shape[2], 1, scale, ws.data_ptr(), need)
    assert _lib.lib().amla_packed_attention(ctypes.byref(args), torch.cuda.current_stream().cuda_stream) == 0
    torch.cuda.synchronize()


@pytest.mark.parametrize("form,H,lens,split", [("mla", 4, [20, 300, 0, 5], False), ("plain", 130, [20, 300, 0, 5], False),
                                               ("mla", 4, [20, 300, 0, 5], True), ("whole", 2, [1, 0, 70], True)])
@pytest.mark.parametrize("before,behind", [(0, 9), (7, 0), (33, 300)])
def test_rows_of_no_sequence_keep_their_bits(form, H, lens, split, before, behind):
    """Rows before the first sequence and behind the last, and what lies around the outputs, are not written; the sequences'
    own are what they are without such rows."""
    past = [1500, 100, 800, 64][:len(lens)] if split else [0, 9, 0, 30]
    held = [a + b for a, b in zip(lens, past)]
    q, k, v, pe, off, koff, scale = _case(before + H, lens, held, H, H, form)
    T = before + sum(lens) + behind
    wide = torch.randn(T, H, q.shape[2]).to(BF16)
    wide[before:before + sum(lens)] = q
    assert _split_keys(T, sum(held), len(lens), H) == split
    print(f"[case] {form} {before} + {lens} + {behind} split={split}", flush=True)
    guard = 3 * H
    out = torch.full((guard + T * H + guard, 128), 7.0, dtype=BF16, device=DEV)
    lse = torch.full((guard + T * H + guard,), 7.0, device=DEV)
    _entry(to_dev(wide), to_dev(k), to_dev(v), to_dev(pe), to_dev(off + before), to_dev(koff), scale, out[guard:], lse[guard:])
    at = slice(guard + before * H, guard + (before + sum(lens)) * H)
    outside = torch.ones(out.shape[0], dtype=torch.bool, device=DEV)
    outside[at] = False
    assert (out[outside] == 7.0).all() and (lse[outside] == 7.0).all()
    want, want_lse = L.packed_attention(q, k, v, off, scale, koff, pe)
    weight, _ = L.packed_attention(q, k, v.abs(), off, scale, koff, pe)
    kk = k if pe is None else torch.cat([k, pe[:, None].expand(-1, H, -1)], -1)
    size = scale * max((q[:, h].double().abs() @ kk[:, h].double().abs().T).max().item() for h in range(H))
    check_attention(out[at].view(-1, H, 128), want, lse[at].view(-1, H), want_lse, weight, size, f"{form} {before} {behind}")


@pytest.mark.parametrize("form,H", [("plain", 1), ("mla", 2)])
def test_split_keys_of_more_sequences_than_a_wave_has_lanes(form, H):
    """70 sequences, of one query but for four of none and two of 300, and up to 900 keys."""
    n = 70 if H == 1 else 66
    new = [0 if b in (3, 63, 64, n - 2) else 1 for b in range(n)]
    if H == 1:
        new[20], new[n - 1] = 300, 300
    past = [(131 * b) % 900 for b in range(n)]
    lens = [a + b for a, b in zip(new, past)]
    if H == 2:
        new, lens = new[2:], lens[2:]
    assert len(new) >= 64 and _split_keys(sum(new), sum(lens), len(new), H)
    _run(*_case(51, new, lens, H, H, form), what=f"{form} {len(new)} sequences, split")
    _run(*_case(52, new, lens, H, H, form), causal=False, what=f"{form} {len(new)} sequences, split, not causal")


@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("past", [0, 3000])
@pytest.mark.parametrize("form,H", [("plain", 2), ("mla", 4)])
def test_scores_far_from_zero(form, H, past, sign):
    """Scores of 2^19 to 2^28, those of the first keys lower, of the others alike and with values alike: these values come out,
    and zeros where they are 0.  A probability is 2^(z c - m) with m = z c rounded, so up to 2^16 or its reciprocal and, unlike
    1, no bf16 value: alike for all keys, its rounding does not average out.  |d out| <= 2^-8 of the value for that, 2^-8 for the
    output's and 2^-10 for the sums in between; d lse is 2^-20 of it."""
    n, low = 70, past // 2 + 20
    q, k, v, pe, off, koff, _ = _case(13, [n, n], [n + past, n + past], H, H, form)
    k, q = torch.zeros_like(k), torch.zeros_like(q)
    if pe is not None:
        pe = torch.zeros_like(pe)
    each = torch.arange(2 * n * H).view(2 * n, H)
    q[..., 0] = torch.exp2(8.0 + each % 5) * (1 + each * 37 % 128 / 128.0)
    v = v.clone()
    for b in range(2):
        at = b * (n + past)
        k[at:at + n + past, :, 0] = sign * 2.0 ** 14
        k[at:at + low, :, 0] *= 0.25 if sign > 0 else 1.75
        v[at:at + low] = v[at + 1].clone()
        v[at + low:at + n + past] = v[at + low].clone() if b == 0 else 0
    v[n + past:n + past + low] = 0
    print(f"[case] {form} behind {past} sign {sign}", flush=True)
    got, lse = ops.packed_attention(to_dev(q), to_dev(k), to_dev(v), to_dev(off), 0.9, k_offsets=to_dev(koff), k_pe=to_dev(pe),
                                    return_lse=True)
    first = torch.arange(2 * n) % n + past < low  # sees none of the others
    row = torch.arange(2 * n) // n * (n + past) + torch.where(first, 0, low)
    want = v[row].double()
    assert (want[n:] == 0).all()
    d = (got.double().cpu() - want).abs()
    off = ~(d <= (2.0 ** -7 + 2.0 ** -10) * want.abs()).all(2)
    assert not off.any(), (off.nonzero()[:5].tolist(), d[off].max().item(), q[off][:5, 0].tolist())
    z = 0.9 * q[..., 0].double() * k[row][..., 0].double()
    assert z.abs().max() < 2.0 ** 28 and z.abs().min() >= 2.0 ** 19
    alike = torch.arange(2 * n) % n + past + 1 - torch.where(first, 0, low)
    assert ((lse.double().cpu() - z - alike.double().log()[:, None]).abs() <= 2.0 ** -20 * z.abs()).all()


@pytest.mark.parametrize("which", ["q", "k", "v", "pe"])
def test_rows_further_apart_than_the_kernel_counts(which):
    """Rows 2^27 + 8 values apart, like rows with any other stride that it does not take."""
    q, k, v, pe, off, koff, scale = _case(12, [2, 1], [2, 1], 2, 2, "mla")
    t = {n: to_dev(x) for n, x in zip(("q", "k", "v", "pe"), (q, k, v, pe))}
    call = lambda: ops.packed_attention(t["q"], t["k"], t["v"], to_dev(off), scale, k_pe=t["pe"], k_offsets=to_dev(koff))  # noqa: E731
    want = call()
    rows, apart = t[which], 2 ** 27 + 8
    store = torch.empty(2 * apart + rows[0].numel(), dtype=BF16, device=DEV)
    far = store.as_strided(rows.shape, (apart, *rows[0].contiguous().stride()))
    far.copy_(rows)
    t[which] = far
    print(f"[case] far {which}", flush=True)
    assert torch.equal(call(), want)


@pytest.mark.parametrize("form,H,new,past", [("mla", 4, [600], [0]), ("plain", 8, [300, 7], [0, 90]), ("whole", 2, [5], [4000])])
def test_the_mean_error_is_that_of_two_roundings(form, H, new, past):
    """Of the output and of the probabilities, 2^-8 / sqrt(3) of the values at most each (as in the cache's attention)."""
    lens = [a + b for a, b in zip(new, past)]
    case = _case(15, new, lens, H, H, form)
    got, _ = _run(*case, what=f"{form} rms")
    q, k, v, pe, off, koff, scale = case
    want, _ = L.packed_attention(q, k, v, off, scale, koff, pe)
    rms = (got.double().cpu() - want).square().mean().sqrt() / want.square().mean().sqrt()
    assert rms <= 2.0 ** -8 * (2 / 3) ** 0.5, f"{rms.item():.5f}"


@pytest.mark.parametrize("form,H,new,held", [("plain", 2, [40, 9, 300], [25, 0, 90]), ("mla", 2, [600, 3], [450, 0]), ("whole", 130, [300], [90])])
def test_a_query_that_sees_no_key_and_is_no_number(form, H, new, held):
    """More queries than keys: the first of a causal sequence see none, and give zeros whatever they hold."""
    q, k, v, pe, off, koff, scale = _case(17, new, held, H, H, form)
    clean, blind = q.clone(), torch.cat([torch.arange(n) < n - m for n, m in zip(new, held)])
    q[blind] = float("nan")
    q[blind.nonzero()[::2, 0]] = 0.0
    q[blind.nonzero()[::2, 0], :, 5] = float("inf")
    call = lambda q: ops.packed_attention(to_dev(q), to_dev(k), to_dev(v), to_dev(off), scale, k_offsets=to_dev(koff), k_pe=to_dev(pe),  # noqa: E731
                                          return_lse=True)
    print(f"[case] {form} {new} over {held}", flush=True)
    got, lse = call(q)
    want, want_lse = call(clean)
    assert torch.equal(got, want) and torch.equal(lse, want_lse)
    assert (got.cpu()[blind] == 0).all() and (lse.cpu()[blind] == float("-inf")).all() and torch.isfinite(lse.cpu()[~blind]).all()


@pytest.mark.parametrize("form,H,new,past", [("plain", 2, [40, 300], [0, 90]), ("mla", 4, [600], [0]), ("mla", 4, [20], [2000]), ("whole", 130, [300], [70])])
def test_a_query_that_is_no_number_stays_alone(form, H, new, past):
    """NaN for it, the bits of a call without it for all others, also where its block is done again."""
    q, k, v, pe, off, koff, scale = _case(18, new, [a + b for a, b in zip(new, past)], H, H, form)
    call = lambda q: ops.packed_attention(to_dev(q), to_dev(k), to_dev(v), to_dev(off), scale, k_offsets=to_dev(koff), k_pe=to_dev(pe),  # noqa: E731
                                          return_lse=True)
    want, want_lse = call(q)
    bad = torch.zeros(sum(new), H, dtype=torch.bool)
    bad[3, 1], bad[sum(new) - 1, 0], bad[sum(new) // 2, :] = True, True, True
    q[bad] = float("nan")
    print(f"[case] {form} {new} behind {past}", flush=True)
    got, lse = call(q)
    assert torch.isnan(got.cpu()[bad]).all() and torch.isnan(lse.cpu()[bad]).all()
    assert torch.equal(got.cpu()[~bad], want.cpu()[~bad]) and torch.equal(lse.cpu()[~bad], want_lse.cpu()[~bad])
