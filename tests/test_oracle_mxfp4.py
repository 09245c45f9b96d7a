"""The MXFP4 oracle against worked values and a search over every code, and the operators' host
side without a GPU: refusals of the C ABI and of the Python functions, fake implementations."""
import ctypes
import math

import pytest
import torch

from amla import _lib, ops, torch_ops
from oracle import ref_mxfp4 as M


def test_worked_blocks():
    x = torch.zeros(6, 32)
    x[1, 0] = 1.0                                    # exponent -2: 1 is code 4.0 there
    x[2, :4] = torch.tensor([6.0, -2.5, 0.25, 0.75])  # exponent 0, ties to even: 2, 0, 1
    x[3, 0], x[3, 1] = 7.9, 5.0                      # saturates at 6; a tie to 4
    x[4, 5] = float("inf")
    x[5, 0] = 2.0 ** -140                            # below e8m0: byte 0, rounds to zero
    codes, byte = M.quantize(x)
    assert byte[:, 0].tolist() == [0, 125, 127, 127, 255, 0]
    v = M.values(codes, byte)
    assert v[0].abs().sum() == 0 and v[1, 0] == 1.0
    assert v[2, :4].tolist() == [6.0, -2.0, 0.0, 1.0]
    assert v[3, :2].tolist() == [6.0, 4.0]
    assert torch.isnan(v[4]).all() and codes[4].sum() == 0
    assert v[5].abs().sum() == 0
    assert codes[2, 0].item() == (0x7 | (0x8 | 0x4) << 4)  # first value in the low half


def test_nearest_by_search():
    g = torch.Generator().manual_seed(5)
    x = torch.randn(64, 32, generator=g, dtype=torch.float64) * torch.exp2(torch.randint(-30, 30, (64, 1), generator=g))
    codes, byte = M.quantize(x)
    v = M.values(codes, byte)
    grid = torch.cat([M.E2M1, -M.E2M1])
    for r in range(64):
        unit = 2.0 ** (byte[r, 0].item() - 127)
        top = x[r].abs().max().item()
        assert 4 * unit <= top < 8 * unit
        best = (x[r][:, None] - grid * unit).abs().amin(1)
        assert ((x[r] - v[r]).abs() == best).all()


def test_codes_round_trip():
    codes = torch.arange(256, dtype=torch.uint8).repeat(2, 1)  # every pair of codes
    byte = torch.full((2, 16), 120, dtype=torch.uint8)
    v = M.values(codes, byte)
    # every block has a code of 4 or 6 in it: the exponent comes back
    keep = v.reshape(2, 16, 32).abs().amax(-1) >= 4 * 2.0 ** -7
    c2, b2 = M.quantize(v)
    assert keep.all() and torch.equal(b2, byte)
    assert torch.equal(M.values(c2, b2), v)


def _p():
    buf = ctypes.create_string_buffer(4096 + 16)
    a = ctypes.addressof(buf)
    return buf, a + (-a) % 16


def test_c_abi_refuses_before_launch():
    L = _lib.lib()
    buf, p = _p()
    q = p + 8
    bad = [
        (L.amla_mxfp4_quantize(None, 0, 1, 32, 32, p, p, None), -1),
        (L.amla_mxfp4_quantize(p, 3, 1, 32, 32, p, p, None), -1),
        (L.amla_mxfp4_quantize(p, 0, -1, 32, 32, p, p, None), -1),
        (L.amla_mxfp4_quantize(p, 0, 1, 32, 16, p, p, None), -1),
        (L.amla_mxfp4_quantize(p, 0, 1, 48, 48, p, p, None), -3),
        (L.amla_mxfp4_quantize(q, 0, 1, 32, 32, p, p, None), -3),
        (L.amla_mxfp4_quantize(p, 0, 2, 32, 36, p, p, None), -3),
        (L.amla_mxfp4_quantize_fp8(p, None, 1, 32, p, p, None), -1),
        (L.amla_mxfp4_quantize_fp8(p, p, 1, 40, p, p, None), -3),
        (L.amla_mxfp4_dequantize(p, p, 1, 32, 1, p, None), -1),
        (L.amla_mxfp4_dequantize(p, p, 1, 33, 0, p, None), -3),
        (L.amla_mxfp4_linear(p, None, 1, 128, 128, p, p, 8, None, 0, 8, None, 0, None), -1),
        (L.amla_mxfp4_linear(p, None, 1, 128, 64, p, p, 8, p, 0, 8, None, 0, None), -1),
        (L.amla_mxfp4_linear(p, None, 1, 128, 128, p, p, 8, p, 1, 8, None, 0, None), -1),
        (L.amla_mxfp4_linear(p, None, 1, 96, 96, p, p, 8, p, 0, 8, None, 0, None), -3),
        (L.amla_mxfp4_linear(p, None, 1, 128, 128, q, p, 8, p, 0, 8, None, 0, None), -3),
        (L.amla_mxfp4_linear(p, p + 1, 1, 128, 128, p, p, 8, p, 0, 8, None, 0, None), -3),
        (L.amla_mxfp4_linear(p, None, 500, 128, 128, p, p, 8, p, 0, 8, None, 0, None), -2),
        (L.amla_mxfp4_grouped_linear(p, None, 4, 128, 128, p, p, 8, 2, None, p, 0, 8, 1, p, 4096, None), -1),
        (L.amla_mxfp4_grouped_linear(p, None, 4, 128, 128, p, p, 8, 1025, p, p, 0, 8, 1, p, 4096, None), -3),
        (L.amla_mxfp4_grouped_linear(p, None, 4, 128, 128, p, p, 8, 2, p, p, 0, 8, 1, None, 0, None), -2),
        (L.amla_mxfp4_swiglu(p, 1, 128, 128, p, p, p, p, 64, p, p, p, p, 4096, None), -3),
        (L.amla_mxfp4_swiglu(p, 1, 128, 128, p, p, p, p, 128, p, p, p, p, 16, None), -2),
        (L.amla_mxfp4_moe_experts(p, 1, 128, 128, 65, p, 128, 4, p, p, p, p, p, p, p, 1, p, 4096, None), -3),
        (L.amla_mxfp4_moe_experts(p, 1, 128, 128, 2, p, 128, 513, p, p, p, p, p, p, p, 1, p, 4096, None), -3),
        (L.amla_mxfp4_moe_experts(p, 40000, 128, 128, 2, p, 128, 4, p, p, p, p, p, p, p, 1, p, 4096, None), -3),
        (L.amla_mxfp4_moe_experts(p, 1, 128, 128, 2, p, 192, 4, p, p, p, p, p, p, p, 1, p, 4096, None), -3),
        (L.amla_mxfp4_moe_experts(p, 1, 128, 128, 2, p, 128, 4, p, p, p, p, p, p, p, 1, p, 16, None), -2),
    ]
    for i, (rc, want) in enumerate(bad):
        assert rc == want, (i, rc, want)
    # nothing to do: no launch either
    assert L.amla_mxfp4_quantize(p, 0, 0, 32, 32, p, p, None) == 0
    assert L.amla_mxfp4_linear(p, None, 0, 128, 128, p, p, 8, p, 0, 8, None, 0, None) == 0


def test_workspace_grows_with_rows():
    L = _lib.lib()
    assert L.amla_mxfp4_linear_workspace_bytes(1, 7168, 16384, 0) == 0
    for m in (65, 200, 1000, 4096):
        x = m * 16384 // 2 + m * 16384 // 32
        assert L.amla_mxfp4_linear_workspace_bytes(m, 7168, 16384, 0) >= x
    assert L.amla_mxfp4_linear_workspace_bytes(8, 100, 100, 0) == 0  # a K it refuses
    assert L.amla_mxfp4_moe_experts_workspace_bytes(8, 7168, 8, 2048, 256) > 64 * 2048 // 2
    assert L.amla_mxfp4_moe_experts_workspace_bytes(8, 7168, 8, 2048, 513) == 0


def test_python_refuses_tensors_off_the_device():
    w, s = torch.zeros(16, 64, dtype=torch.uint8), torch.zeros(16, 4, dtype=torch.uint8)
    with pytest.raises(ValueError, match="ROCm device"):
        ops.mxfp4_quantize(torch.zeros(2, 32))
    with pytest.raises(ValueError, match="ROCm device"):
        ops.mxfp4_linear(torch.zeros(2, 128, dtype=torch.bfloat16), w, s)
    with pytest.raises(TypeError, match="out_dtype"):
        ops.mxfp4_linear(torch.zeros(2, 128, dtype=torch.bfloat16), w, s, out_dtype=torch.int8)


def test_fake_implementations_give_the_shapes():
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        x = torch.empty(5, 256, dtype=torch.bfloat16, device="cuda")
        w, s = torch.empty(40, 128, dtype=torch.uint8, device="cuda"), torch.empty(40, 8, dtype=torch.uint8, device="cuda")
        q = torch.ops.amla.mxfp4_quantize(x)
        assert q[0].shape == (5, 128) and q[1].shape == (5, 8) and q[0].dtype == torch.uint8
        assert torch.ops.amla.mxfp4_dequantize(*q, True).shape == (5, 256)
        y = torch.ops.amla.mxfp4_linear(x, None, w, s, False)
        assert y.shape == (5, 40) and y.dtype == torch.bfloat16
        assert torch.ops.amla.mxfp4_linear(*q, w, s, True).dtype == torch.float32
        off = torch.empty(3, dtype=torch.int32, device="cuda")
        w3, s3 = w.expand(2, 40, 128), s.expand(2, 40, 8)
        assert torch.ops.amla.mxfp4_grouped_linear(x, None, w3, s3, off, False).shape == (5, 40)
        idx = torch.empty(5, 2, dtype=torch.int64, device="cuda")
        assert torch.ops.amla.mxfp4_moe_experts(x, idx, w3, s3, w3, s3, w3, s3).shape == (5, 2, 256)


def test_slack_counts_the_steps_only():
    """The expert oracle's slack is zero in its rounding part where no value is near a border."""
    g = torch.Generator().manual_seed(2)
    x = M.rounded(torch.randn(3, 128, generator=g))
    w = [M.rounded(torch.randn(128, 128, generator=g) * 0.05) for _ in range(3)]
    y, slack = M.swiglu(x, *w)
    assert y.shape == (3, 128) and (slack >= 0).all()
    assert (slack <= 0.05 * y.abs().mean()).float().mean() > 0.9
    assert math.isfinite(slack.max().item())
