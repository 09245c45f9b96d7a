"""What the C entries of the MXFP4 operators refuse on the host (no GPU: nothing is launched)."""
import pytest

from amla import _lib

EINVAL, EWORKSPACE, EUNSUPPORTED = -1, -2, -3
P = 1 << 20  # an aligned address that nothing reads


@pytest.fixture(scope="module")
def L():
    return _lib.lib()


def _linear(L, m=4, k=256, n=64, x=P, xs=None, ldx=None, w=P, s=P, y=P, dtype=0, ldy=None, ws=P, need=1 << 40):
    return L.amla_mxfp4_linear(x, xs, m, k, k if ldx is None else ldx, w, s, n, y, dtype, n if ldy is None else ldy,
                               ws, need, None)


def _grouped(L, m=4, k=256, n=64, E=3, x=P, off=P, w=P, y=P, dtype=0, ldy=None, ws=P, need=1 << 40):
    return L.amla_mxfp4_grouped_linear(x, None, m, k, k, w, P, n, E, off, y, dtype, n if ldy is None else ldy, 1, ws,
                                       need, None)


def _swiglu(L, m=4, k=256, n=128, x=P, up=P, y=P, ldx=None, ws=P, need=1 << 40):
    return L.amla_mxfp4_swiglu(x, m, k, k if ldx is None else ldx, P, P, up, P, n, P, P, y, ws, need, None)


def _moe(L, m=4, d=256, top_k=2, n=128, E=3, hidden=P, ldh=None, out=P, ws=P, need=1 << 40):
    return L.amla_mxfp4_moe_experts(hidden, m, d, d if ldh is None else ldh, top_k, P, n, E, P, P, P, P, P, P, out, 1,
                                    ws, need, None)



@pytest.mark.parametrize("call", [_linear, _grouped, _swiglu, _moe])
def test_empty_calls_and_sizes_below_zero(L, call):
    assert call(L, m=0) == 0
    assert call(L, m=-1) == EINVAL
    assert call(L, **{"d" if call is _moe else "k": 0}) == EINVAL
    assert call(L, n=0) == EINVAL


@pytest.mark.parametrize("call", [_linear, _grouped, _swiglu, _moe])
def test_k_that_the_products_do_not_take(L, call):
    key = "d" if call is _moe else "k"
    for k in (96, 192, (1 << 24) + 128):
        assert call(L, **{key: k}) == EUNSUPPORTED


@pytest.mark.parametrize("call", [_swiglu, _moe])
def test_intermediate_sizes_are_checked_before_anything_runs(L, call):
    """They are the K of the second product."""
    for n in (64, 192, (1 << 24) + 128):
        assert call(L, n=n) == EUNSUPPORTED


@pytest.mark.parametrize("call", [_linear, _grouped, _swiglu, _moe])
def test_addresses_and_strides(L, call):
    x = "hidden" if call is _moe else "x"
    assert call(L, **{x: None}) == EINVAL
    assert call(L, **{x: P + 8}) == EUNSUPPORTED
    y = "out" if call is _moe else "y"
    assert call(L, **{y: None}) == EINVAL
    if call in (_linear, _swiglu):
        assert call(L, ldx=128) == EINVAL
        assert call(L, ldx=260) == EUNSUPPORTED
    if call is _moe:
        assert call(L, ldh=128) == EINVAL
        assert call(L, ldh=260) == EUNSUPPORTED
    if call in (_linear, _grouped):
        assert call(L, ldy=63) == EINVAL
        assert call(L, dtype=1) == EINVAL
        assert call(L, w=P + 8) == EUNSUPPORTED


def test_exponents_of_four_bytes_alignment(L):
    assert _linear(L, s=P + 2) == EUNSUPPORTED
    assert _linear(L, xs=P + 2) == EUNSUPPORTED


@pytest.mark.parametrize("call", [_linear, _grouped, _swiglu, _moe])
def test_workspace_too_small_or_misaligned(L, call):
    big = {"m": 300}
    assert call(L, ws=None, **big) == EWORKSPACE
    assert call(L, need=16, **big) == EWORKSPACE
    assert call(L, ws=P + 8, **big) == EWORKSPACE


def test_experts_beyond_the_limits(L):
    assert _grouped(L, E=1025) == EUNSUPPORTED
    assert _moe(L, E=513) == EUNSUPPORTED
    assert _moe(L, top_k=65) == EUNSUPPORTED
    assert _moe(L, m=65536, top_k=2) == EUNSUPPORTED
    assert L.amla_mxfp4_grouped_linear_workspace_bytes(4, 64, 256, 1025, 0) == 0


def test_gathered_rows_of_four_gigabytes_of_codes(L):
    """A gathered row is addressed with 32 bits: 65536 rows of 131072 values would pass them."""
    assert _moe(L, m=65536, d=131072, top_k=1, ws=None) == EUNSUPPORTED
    assert L.amla_mxfp4_moe_experts_workspace_bytes(65536, 131072, 1, 128, 3) == 0
    assert _moe(L, m=65535, d=131072, top_k=1, ws=None) == EWORKSPACE


def test_outputs_beyond_a_grid(L):
    m, n = 2 ** 31 - 1, 2 ** 29 - 1  # 2^44 tiles
    need = L.amla_mxfp4_linear_workspace_bytes(m, n, 128, 1)
    assert _linear(L, m=m, k=128, n=n, xs=P, ws=P, need=max(need, 16)) == EUNSUPPORTED


def test_workspace_covers_one_expert_named_many_times(L):
    """Few tokens: an entry of the schedule holds at most as many rows as there are tokens, so that
    64 slots of one token on one expert are 64 entries."""
    bytes_of = L.amla_mxfp4_moe_experts_workspace_bytes
    assert bytes_of(1, 128, 64, 128, 4) >= 64 * (16 + 4 + 4 + 64 + 4)
