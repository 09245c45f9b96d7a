"""The MXFP4 operators under what watches torch's operators: tracers, transforms, dispatch modes.

On the CPU, with stand-ins for the kernels: a stand-in writes its output behind torch's back, as a
kernel does, so that a trace which misses the operator replays uninitialised memory."""
import ctypes
import dataclasses

import pytest
import torch
from torch.autograd import forward_ad
from torch.fx.experimental.proxy_tensor import make_fx
from torch.overrides import TorchFunctionMode
from torch.utils._python_dispatch import TorchDispatchMode

from amla import ops, torch_ops
from amla.config import DeepSeekConfig

BF16, U8 = torch.bfloat16, torch.uint8


def _write(out, value):
    """The bytes of ``value`` into ``out`` by its address."""
    value = value.to(out.dtype).contiguous()
    if out.numel():
        ctypes.memmove(out.data_ptr(), value.data_ptr(), out.numel() * out.element_size())
    return out


def _linear(x, x_scales, weight, scale, f32):
    y = torch.empty(x.shape[0], weight.shape[0], dtype=torch.float32 if f32 else BF16)
    return _write(y, x.float().sum(1, keepdim=True) + weight.float().sum(1))


def _grouped(x, x_scales, weight, scale, offsets, f32):
    y = torch.empty(x.shape[0], weight.shape[1], dtype=torch.float32 if f32 else BF16)
    return _write(y, x.float().sum(1, keepdim=True) + weight.float().sum((0, 2)))


def _grouped_out(x, x_scales, weight, scale, offsets, out):
    _write(out, x.float().sum(1, keepdim=True) + weight.float().sum((0, 2)))


def _swiglu(x, *w):
    return _write(torch.empty(x.shape, dtype=BF16), x.float() * 3)


def _moe(hidden, indices, *w):
    y = torch.empty(hidden.shape[0], indices.shape[1], hidden.shape[1], dtype=BF16)
    return _write(y, hidden.float()[:, None] + indices[..., None])


def _pair(x, *_):
    rows, k = x.shape
    s = x.float().abs().sum(1, keepdim=True)
    return (_write(torch.empty(rows, k // 2, dtype=U8), (s % 200).expand(rows, k // 2)),
            _write(torch.empty(rows, k // 32, dtype=U8), (s % 100).expand(rows, k // 32)))


def _dequantize(codes, scales, f32):
    y = torch.empty(codes.shape[0], codes.shape[1] * 2, dtype=torch.float32 if f32 else BF16)
    return _write(y, codes.float().repeat_interleave(2, 1))


STAND_INS = {"mxfp4_quantize": _pair, "mxfp4_quantize_fp8": _pair, "mxfp4_dequantize": _dequantize,
             "mxfp4_linear": _linear, "mxfp4_grouped_linear": _grouped, "mxfp4_grouped_linear_out": _grouped_out,
             "mxfp4_swiglu": _swiglu, "mxfp4_moe_experts": _moe}


@pytest.fixture(autouse=True)
def stand_ins(monkeypatch):
    lib = torch.library.Library("amla", "IMPL")
    for name, fn in STAND_INS.items():
        lib.impl(name, fn, "CPU")
        monkeypatch.setitem(torch_ops._mx_impl, name, fn)
    monkeypatch.setattr(torch_ops, "_on_device", lambda fn, t, *args: fn(t, *args))
    yield
    lib._destroy()


def _u8(*shape):
    return torch.randint(0, 200, shape, dtype=U8)


def _x(m=4, k=128):
    return torch.randint(-8, 9, (m, k)).to(BF16)


# name: (the call as a function of its first tensor, that tensor)
def _calls():
    w, s = _u8(6, 64), _u8(6, 4)
    w3, s3 = _u8(2, 6, 64), _u8(2, 6, 4)
    ff = [_u8(128, 64), _u8(128, 4)] * 3
    off = torch.tensor([0, 1, 4], dtype=torch.int32)
    idx = torch.randint(0, 2, (4, 2))
    c = torch_ops.call
    return {
        "mxfp4_quantize": (lambda t: c("mxfp4_quantize", t), _x),
        "mxfp4_quantize_fp8": (lambda t: c("mxfp4_quantize_fp8", t, torch.ones(1, 1)), lambda: _x().to(torch.float8_e4m3fn)),
        "mxfp4_dequantize": (lambda t: c("mxfp4_dequantize", t, s, False), lambda: _u8(6, 64)),
        "mxfp4_linear": (lambda t: c("mxfp4_linear", t, None, w, s, True), _x),
        "mxfp4_grouped_linear": (lambda t: c("mxfp4_grouped_linear", t, None, w3, s3, off, False), _x),
        "mxfp4_swiglu": (lambda t: c("mxfp4_swiglu", t, *ff), _x),
        "mxfp4_moe_experts": (lambda t: c("mxfp4_moe_experts", t, idx, w3, s3, w3, s3, w3, s3), _x),
    }


NAMES = sorted(set(STAND_INS) - {"mxfp4_grouped_linear_out"})


def _equal(a, b):
    if isinstance(a, (tuple, list)):
        return len(a) == len(b) and all(_equal(u, v) for u, v in zip(a, b))
    return a.dtype == b.dtype and torch.equal(a, b)


@pytest.mark.parametrize("how", ["real", "fake", "symbolic", "pre_dispatch"])
@pytest.mark.parametrize("name", NAMES)
def test_make_fx_records_the_operator(name, how):
    f, make = _calls()[name]
    kw = {"pre_dispatch": True} if how == "pre_dispatch" else {"tracing_mode": how, "_allow_non_fake_inputs": True}
    gm = make_fx(f, **kw)(make())
    targets = [str(n.target) for n in gm.graph.nodes if n.op == "call_function"]
    assert f"amla.{name}.default" in targets and not any("empty" in t for t in targets)
    fresh = make()
    assert _equal(gm(fresh), f(fresh))


@pytest.mark.parametrize("name", NAMES)
def test_jit_trace_records_the_operator(name):
    f, make = _calls()[name]
    traced = torch.jit.trace(f, make(), check_trace=False)
    assert f"amla::{name}" in str(traced.graph)
    fresh = make()
    assert _equal(traced(fresh), f(fresh))


@pytest.mark.parametrize("name", NAMES)
def test_dispatch_and_function_modes_see_the_operator(name):
    f, make = _calls()[name]
    seen = []

    class Dispatch(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            seen.append(str(func))
            return func(*args, **(kwargs or {}))

    class Function(TorchFunctionMode):
        def __torch_function__(self, func, types, args=(), kwargs=None):
            seen.append(str(func))
            return func(*args, **(kwargs or {}))

    t = make()
    want = f(t)
    for mode in (Dispatch, Function):
        seen.clear()
        with mode():
            got = f(t)
        assert any(f"amla.{name}" in s for s in seen), (mode, seen)
        assert _equal(got, want)


@pytest.mark.parametrize("name", ["mxfp4_linear", "mxfp4_swiglu", "mxfp4_quantize"])
def test_vmap_runs_the_operator_by_item(name):
    f, make = _calls()[name]
    t = torch.stack([make() for _ in range(3)])
    got = torch.func.vmap(f)(t)
    assert _equal(got, torch.func.vmap(f)(t))
    for i in range(3):
        item = tuple(g[i] for g in got) if isinstance(got, tuple) else got[i]
        assert _equal(item, f(t[i]))


def test_vmap_over_the_weights():
    x, w, s = _x(), _u8(3, 6, 64), _u8(3, 6, 4)
    got = torch.func.vmap(lambda a, b: torch_ops.call("mxfp4_linear", x, None, a, b, True))(w, s)
    assert _equal(got, torch.stack([_linear(x, None, w[i], s[i], True) for i in range(3)]))


@pytest.mark.parametrize("name", NAMES)
def test_compiled_calls_hold_the_operator(name):
    f, make = _calls()[name]
    graphs = []

    def backend(gm, inputs):
        graphs.append(str(gm.graph))
        return gm.forward

    torch._dynamo.reset()
    t = make()
    assert _equal(torch.compile(f, fullgraph=True, backend=backend)(t), f(t))
    assert len(graphs) == 1 and f"amla.{name}" in graphs[0]


def test_a_subclass_behind_the_first_argument_is_seen():
    seen = []

    class Marked(torch.Tensor):
        @classmethod
        def __torch_function__(cls, func, types, args=(), kwargs=None):
            seen.append(str(func))
            return super().__torch_function__(func, types, args, kwargs or {})

    w = _u8(6, 64).as_subclass(Marked)
    torch_ops.call("mxfp4_linear", _x(), None, w, _u8(6, 4), True)
    assert any("amla.mxfp4_linear" in s for s in seen)


def test_eager_calls_do_not_pass_the_dispatcher(monkeypatch):
    """The ordinary call (with and without grad mode, in inference mode) runs its implementation."""
    f, make = _calls()["mxfp4_linear"]
    t = make()
    ran = []
    monkeypatch.setattr(torch_ops, "_on_device", lambda fn, t, *args: ran.append(1) or fn(t, *args))
    for ctx in (torch.enable_grad, torch.no_grad, torch.inference_mode):
        with ctx():
            f(t)
    f(torch.nn.Parameter(t, requires_grad=False))
    assert len(ran) == 4


# ------------------------------------------------------------------ gradients

def _out_call(x, out):
    w, s = _u8(2, 6, 64), _u8(2, 6, 4)
    torch_ops.call("mxfp4_grouped_linear_out", x, None, w, s, torch.tensor([0, 1, 4], dtype=torch.int32), out)
    return out


@pytest.fixture
def real_out(monkeypatch):
    """The package's own implementation of the operator with an ``out``, but for its launch."""
    monkeypatch.undo()
    monkeypatch.setattr(torch_ops, "_on_device", lambda fn, t, *args: fn(t, *args))
    monkeypatch.setattr(torch_ops, "_mx_grouped", lambda x, xs, w, s, off, y, clear: _grouped_out(x, xs, w, s, off, y))


def test_out_has_no_gradient_to_give(real_out):
    """Like torch's own out= variants: an error while a gradient is asked for, not a lost term."""
    leaf = _x().requires_grad_()
    out = torch.zeros(4, 6, dtype=BF16)
    for x in (leaf, leaf * 2):
        with pytest.raises(RuntimeError, match="out= .* gradient"):
            _out_call(x, out)
    with pytest.raises(RuntimeError, match="out= .* gradient"):
        _out_call(_x(), torch.zeros(4, 6, dtype=BF16, requires_grad=True))
    assert not out.any()
    with pytest.raises(RuntimeError, match="out= .* gradient"):
        torch.ops.amla.mxfp4_grouped_linear_out(leaf, None, _u8(2, 6, 64), _u8(2, 6, 4),
                                                torch.tensor([0, 1, 4], dtype=torch.int32), out)
    with torch.no_grad():
        assert _out_call(leaf, out).any()
    with torch.inference_mode():
        assert _out_call(leaf, torch.zeros(4, 6, dtype=BF16)).any()


@pytest.mark.parametrize("through", ["call", "operator"])
def test_out_counts_as_written(real_out, through):
    """Autograd sees that a tensor it saved was overwritten."""
    out = torch.ones(4, 6, dtype=BF16)
    a = torch.ones(4, 6, dtype=BF16, requires_grad=True)
    y = (a * out).sum()
    before = out._version
    if through == "call":
        _out_call(_x(), out)
    else:
        lib = torch.library.Library("amla", "IMPL")
        try:
            lib.impl("mxfp4_grouped_linear_out", torch_ops._mx_impl["mxfp4_grouped_linear_out"], "CPU", allow_override=True)
            torch.ops.amla.mxfp4_grouped_linear_out(_x(), None, _u8(2, 6, 64), _u8(2, 6, 4),
                                                    torch.tensor([0, 1, 4], dtype=torch.int32), out)
        finally:
            lib._destroy()
    assert out._version == before + 1
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


def test_compiled_out():
    def f(x, out):
        w = torch.ones(2, 6, 64, dtype=U8)
        torch_ops.call("mxfp4_grouped_linear_out", x, None, w, w[:, :, :4], torch.tensor([0, 1, 4], dtype=torch.int32), out)
        return out + 1

    x = _x()
    a, b = torch.zeros(4, 6, dtype=BF16), torch.zeros(4, 6, dtype=BF16)
    torch._dynamo.reset()
    got = torch.compile(f, fullgraph=True, backend="aot_eager")(x, a)
    assert _equal(got, f(x, b)) and _equal(a, b) and a.any()


def _moe_parts(monkeypatch):
    """moe_block's parts but for the launches."""
    monkeypatch.setattr(ops, "route", lambda h, gate, cfg: (torch.zeros(*h.shape[:-1], 2, dtype=torch.int64),
                                                            torch.ones(*h.shape[:-1], 2)))
    monkeypatch.setattr(ops, "expert_ffn", lambda h, w: _write(torch.empty(h.shape, dtype=BF16), h * 2))
    monkeypatch.setattr(ops, "mxfp4_moe_experts", lambda h, i, w: _write(torch.empty(*i.shape, h.shape[-1], dtype=BF16), h[:, None].expand(*i.shape, -1)))

    def combine(shared, eout, w, m, top_k, d, config, out, hidden):
        return _write(out, (shared.reshape(m, d) + eout.sum(1)).view(out.shape))

    monkeypatch.setattr(ops, "_moe_combine", combine)
    cfg = DeepSeekConfig(hidden_size=128, n_routed_experts=2, num_experts_per_tok=2, n_group=1, topk_group=1,
                         moe_intermediate_size=128)
    w = _u8(2, 128, 64)
    return cfg, {"gate_proj": (w, w), "up_proj": (w, w), "down_proj": (w, w)}


def test_moe_block_on_mxfp4_experts_has_no_backward(monkeypatch):
    """With a residual beside it, a lost gradient would pass unseen."""
    cfg, experts = _moe_parts(monkeypatch)
    h, gate = _x(), _x(2)
    want = ops.moe_block(h, gate, {}, experts, cfg)
    assert not want.requires_grad
    weights = torch.ones(4, 2, requires_grad=True)
    idx = torch.zeros(4, 2, dtype=torch.int64)
    for hidden, gt, routing in ((h.clone().requires_grad_(), gate, None), (h, gate.clone().requires_grad_(), None),
                                (h, gate, (idx, weights))):
        residual = torch.zeros_like(h, requires_grad=True)
        y = ops.moe_block(hidden, gt, {}, experts, cfg, routing=routing)
        assert torch.equal(y, want)
        y += 0  # (an ordinary tensor: in-place residuals work)
        with pytest.raises(RuntimeError, match="no backward"):
            (residual + y).float().sum().backward()
        with torch.no_grad():
            assert not ops.moe_block(hidden, gt, {}, experts, cfg, routing=routing).requires_grad


def test_a_quantised_pair_carries_no_gradient():
    """Its tensors are whole numbers, as after torch's own casts to them."""
    leaf = _x().requires_grad_()
    pair = torch_ops.call("mxfp4_quantize", leaf)
    assert not any(t.requires_grad for t in pair)
    assert not torch_ops.call("mxfp4_linear", *pair, _u8(6, 64), _u8(6, 4), True).requires_grad


@pytest.mark.parametrize("name", ["mxfp4_linear", "mxfp4_grouped_linear", "mxfp4_swiglu", "mxfp4_moe_experts"])
def test_forward_mode_is_refused_not_passed_over(name):
    f, make = _calls()[name]
    x, t = make(), make()
    with pytest.raises(RuntimeError, match="no derivative"):
        torch.func.jvp(f, (x,), (t,))
    with forward_ad.dual_level():
        with pytest.raises(RuntimeError, match="no derivative"):
            f(forward_ad.make_dual(x, t))
        assert _equal(f(x), f(x.clone()))  # a plain tensor beside dual ones
    out = torch.zeros(4, 6, dtype=BF16)
    with forward_ad.dual_level():
        with pytest.raises(RuntimeError, match="no derivative"):
            _out_call(forward_ad.make_dual(_x(), _x()), out)


# ------------------------------------------------------------------ empty pairs

@pytest.mark.parametrize("shape", [(5, 0), (0, 64), (0, 0)])
def test_dequantise_of_no_values(monkeypatch, shape):
    monkeypatch.undo()
    codes = torch.empty(shape, dtype=U8)
    scales = torch.empty(shape[0], shape[1] // 16, dtype=U8)
    for f32 in (False, True):
        y = torch_ops._mx_impl["mxfp4_dequantize"](codes, scales, f32)
        assert y.shape == (shape[0], 2 * shape[1]) and y.dtype == (torch.float32 if f32 else BF16)


# ------------------------------------------------------------------ moe_block's arguments

def test_moe_block_of_a_permuted_batch(monkeypatch):
    """Hidden states with permuted strides (a batch kept time first): the result is written row by row."""
    cfg, experts = _moe_parts(monkeypatch)
    h = _x(6).view(3, 2, 128).transpose(0, 1)
    assert not h.is_contiguous()
    got = ops.moe_block(h, _x(2), {}, experts, cfg)
    assert got.shape == h.shape and torch.equal(got, ops.moe_block(h.contiguous(), _x(2), {}, experts, cfg))


def test_moe_block_refuses_a_routing_of_other_types(monkeypatch):
    """The combine reads the weights as fp32 and the grouping the indices as int64, by address."""
    cfg, experts = _moe_parts(monkeypatch)
    h, gate = _x(), _x(2)
    idx, w = torch.zeros(4, 2, dtype=torch.int64), torch.ones(4, 2)
    assert ops.moe_block(h, gate, {}, experts, cfg, routing=(idx, w)).shape == h.shape
    for routing in ((idx.int(), w), (idx, w.to(BF16)), (idx, w.double()), (idx, w.to("meta")), (idx[:3], w), (idx, w[:3]),
                    (idx[:, :1], w), (idx, torch.ones(4, 3)), (idx.tolist(), w)):
        for ex in (experts, {0: {}, 1: {}}):
            with pytest.raises((TypeError, ValueError), match="routing"):
                ops.moe_block(h, gate, {}, ex, cfg, routing=routing)


def test_moe_block_says_how_mxfp4_experts_are_held(monkeypatch):
    """A mapping or a callable of per-expert pairs: refused by what it is, not as bad fp8 weights."""
    cfg, experts = _moe_parts(monkeypatch)
    by_expert = {e: {k: (c[e], s[e]) for k, (c, s) in experts.items()} for e in range(2)}
    for given in (by_expert, by_expert.__getitem__):
        with pytest.raises(ValueError, match="MXFP4 experts .* stacked"):
            ops.moe_block(_x(), _x(2), {}, given, cfg)


def test_a_default_device_does_not_count_as_a_mode(monkeypatch):
    """torch.set_default_device and ``with device`` are function modes that change factories only."""
    f, make = _calls()["mxfp4_linear"]
    t = make()
    ran = []
    monkeypatch.setattr(torch_ops, "_on_device", lambda fn, t, *args: ran.append(1) or fn(t, *args))
    with torch.device("cpu"):
        f(t)
        assert len(ran) == 1

        class Watch(TorchFunctionMode):
            def __torch_function__(self, func, types, args=(), kwargs=None):
                return func(*args, **(kwargs or {}))

        with Watch():
            f(t)
        f(t.as_subclass(type("Sub", (torch.Tensor,), {})))
        assert len(ran) == 1


@pytest.mark.parametrize("experts,on_device", [(2, True), (512, True), (513, False)])
def test_moe_block_takes_indices_on_the_host_where_it_groups_there(monkeypatch, experts, on_device):
    """fp8 experts past what the device groups: the indices come to the host, or are there already."""
    cfg, _ = _moe_parts(monkeypatch)
    cfg = dataclasses.replace(cfg, n_routed_experts=experts)
    seen = []

    def check(idx, w, hidden, top_k, where):
        seen.append(where)
        raise StopIteration

    monkeypatch.setattr(ops, "_check_routing", check)
    w8 = torch.zeros(experts, 1, 1, dtype=torch.float8_e4m3fn)
    with pytest.raises(StopIteration):
        ops.moe_block(_x(), _x(2), {}, {k: (w8, w8) for k in ("gate_proj", "up_proj", "down_proj")}, cfg,
                      routing=(torch.zeros(4, 2, dtype=torch.int64), torch.ones(4, 2)))
    assert seen == [on_device]
