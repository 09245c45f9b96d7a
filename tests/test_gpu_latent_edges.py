"""latent_attention where its number formats and its passes over the tiles end: sums far from one, scores far below zero,
references that are set anew, in every kernel that it has."""
import pytest
import torch

from _latent import BF16, cache_of
from test_gpu_latent_attention import _run, _wider

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

