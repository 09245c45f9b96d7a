"""packed_attention at its edges."""
import pytest
import torch

from _latent import BF16, DEV, to_dev
from amla import ops
from test_gpu_packed_attention import _case

pytestmark = pytest.mark.gpu


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
