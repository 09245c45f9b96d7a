"""Inputs of latent_cache_write that torch holds in an unusual way, and rows that are no numbers."""
import pytest
import torch

from _latent import BF16, DEV, FP8
from amla import ops
from amla.config import DeepSeekConfig
from test_gpu_latent_cache import _check_rows, _freqs, _gamma, _kv

pytestmark = pytest.mark.gpu
CFG = DeepSeekConfig()


def _stored(kv, gamma, freqs, fp8, B, rows, **kw):
    """Rows 0 .. rows - 1 of B sequences as they are read back after one write at position 0."""
    cache = ops.latent_cache(B * 4, 8, CFG, DEV, FP8 if fp8 else BF16)
    table = torch.arange(B * 4, dtype=torch.int32, device=DEV).view(B, 4)
    ops.latent_cache_write(kv, gamma, freqs, cache, table, 0, **kw)
    off = torch.arange(B + 1, dtype=torch.int32, device=DEV) * rows
    return ops.latent_cache_read(cache, table, off, B * rows)


@pytest.mark.parametrize("fp8", [True, False])
def test_conjugated_angles(fp8):
    """``freqs.conj()`` is a view with a flag: the rotation is the other way round."""
    g = torch.Generator().manual_seed(6)
    kv, gamma, freqs = _kv(g, 2, 7), _gamma(g), _freqs(32)
    print(f"[case] fp8={fp8} conjugated", flush=True)
    lat, pe = _stored(kv.to(DEV), gamma.to(DEV), freqs.to(DEV).conj(), fp8, 2, 7)
    turned = freqs.conj().resolve_conj()
    _check_rows(lat, pe, kv.reshape(-1, 576), gamma, turned[:7].repeat(2, 1), 1e-6, fp8, "conjugated")


@pytest.mark.parametrize("fp8", [True, False])
def test_rows_that_share_memory(fp8):
    """The same rows for every sequence (an expanded tensor), one row for all, and rows that overlap."""
    g = torch.Generator().manual_seed(5)
    gamma, freqs = _gamma(g).to(DEV), _freqs(32).to(DEV)
    for kv in (_kv(g, 1, 5).to(DEV).expand(3, 5, 576), _kv(g, 1, 1).to(DEV).expand(3, 1, 576), _kv(g, 1, 1).to(DEV).expand(3, 5, 576),
               _kv(g, 1, 3).to(DEV).flatten().as_strided((3, 1, 576), (64, 64, 1))):
        rows = kv.shape[1]
        print(f"[case] fp8={fp8} strides {kv.stride()}", flush=True)
        lat, pe = _stored(kv, gamma, freqs, fp8, 3, rows)
        want = _stored(kv.contiguous(), gamma, freqs, fp8, 3, rows)
        assert torch.equal(lat, want[0]) and torch.equal(pe, want[1])
        packed = kv.flatten(0, 1) if rows == 1 else kv.reshape(-1, 576)
        off = torch.arange(4, dtype=torch.int32, device=DEV) * rows
        lat, pe = _stored(packed, gamma, freqs, fp8, 3, rows, offsets=off)
        assert torch.equal(lat, want[0]) and torch.equal(pe, want[1])


@pytest.mark.parametrize("fp8", [True, False])
def test_rows_with_values_that_are_no_numbers(fp8):
    """e4m3: a row of NaN.  bf16: what the formula gives, 0 beside an infinity (1 / rms is 0) and NaN in its place, a row of
    NaN for a NaN.  Rope keys: the pair of such a value only."""
    g = torch.Generator().manual_seed(9)
    kv, gamma, freqs = _kv(g, 1, 4), _gamma(g).to(DEV), _freqs(32).to(DEV)
    clean = _stored(kv.to(DEV), gamma, freqs, fp8, 1, 4)
    kv[0, 1, 77], kv[0, 2, 300], kv[0, 3, 520] = float("inf"), float("nan"), float("nan")
    print(f"[case] fp8={fp8} no numbers", flush=True)
    lat, pe = _stored(kv.to(DEV), gamma, freqs, fp8, 1, 4)
    assert torch.equal(lat[[0, 3]], clean[0][[0, 3]]) and torch.equal(pe[:3], clean[1][:3])
    assert torch.isnan(pe[3, 8:10]).all() and torch.equal(pe[3, 10:], clean[1][3, 10:]) and torch.equal(pe[3, :8], clean[1][3, :8])
    assert torch.isnan(lat[2]).all() and torch.isnan(lat[1, 77])
    rest = torch.arange(512, device=DEV) != 77
    assert torch.isnan(lat[1, rest]).all() if fp8 else (lat[1, rest] == 0).all()
