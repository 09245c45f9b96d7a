"""When the operators of the paged cache take the short path past torch's dispatcher (on the CPU, with stand-ins for the kernels)."""
import pytest
import torch
from torch.overrides import TorchFunctionMode

from amla import torch_ops

BF16 = torch.bfloat16


def _x(*shape, dtype=BF16):
    return torch.zeros(*shape, dtype=dtype)


def _calls():
    """name -> arguments as amla.ops hands them on: with scales and without, where they are optional"""
    i32 = torch.int32
    latent, k_pe, scales = _x(9, 16, 512), _x(9, 16, 64), _x(9, 16, dtype=torch.uint8)
    table, off = _x(3, 5, dtype=i32), _x(4, dtype=i32)
    return {
        "latent_cache_write": (_x(6, 576), _x(512), _x(100, 32, dtype=torch.complex64), latent, k_pe, scales, table, off[:3], None, 1e-6),
        "latent_cache_read": (latent, k_pe, None, table, off, None, 70),
        "latent_cache_read_out": (latent, k_pe, scales, table, off, off[:3], _x(70, 512), _x(70, 64)),
        "latent_attention": (_x(3, 1, 4, 576), latent, k_pe, scales, table, off[:3], 0.1, True),
        "packed_attention": (_x(50, 16, 192), _x(80, 8, 128), _x(80, 8, 128), _x(80, 64), off, None, 0.1, True, False),
    }


@pytest.mark.parametrize("name", list(_calls()))
def test_a_default_device_does_not_count_as_a_mode(monkeypatch, name):
    """torch.set_default_device and ``with device`` are function modes that change factories only; numbers among the arguments
    are no subclasses."""
    ran, args = [], _calls()[name]
    lib = torch.library.Library("amla", "IMPL")
    lib.impl(name, lambda *a: (a[0].clone(), a[0].clone()) if name.endswith(("read", "attention")) else None, "CPU")
    try:
        monkeypatch.setitem(torch_ops._mx_impl, name, lambda *a: ran.append(1))
        monkeypatch.setattr(torch_ops, "_on_device", lambda fn, t, *a: fn(t, *a))
        torch_ops.call_latent(name, *args)
        assert len(ran) == 1
        with torch.device("cpu"):
            torch_ops.call_latent(name, *args)
            assert len(ran) == 2

            class Watch(TorchFunctionMode):
                def __torch_function__(self, func, types, args=(), kwargs=None):
                    return func(*args, **(kwargs or {}))

            with Watch():
                torch_ops.call_latent(name, *args)
            torch_ops.call_latent(name, args[0].as_subclass(type("Sub", (torch.Tensor,), {})), *args[1:])
            assert len(ran) == 2
    finally:
        lib._destroy()
