"""The public MXFP4 functions on the GPU under tracers, transforms and dispatch modes."""
import threading

import pytest
import torch
from torch.fx.experimental.proxy_tensor import make_fx
from torch.utils._python_dispatch import TorchDispatchMode

from amla import ops
from amla.config import DeepSeekConfig
from oracle import ref_mxfp4 as M

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16, F32 = torch.bfloat16, torch.float32


def _weight(g, *shape):
    return tuple(t.to(DEV) for t in M.quantize(torch.randn(*shape, generator=g) * 0.05))


def _calls():
    """name: (function of x (m, 256), operator it has to show)."""
    g = torch.Generator().manual_seed(1)
    w, w3 = _weight(g, 96, 256), _weight(g, 3, 96, 256)
    ff = {"gate_proj": _weight(g, 128, 256), "up_proj": _weight(g, 128, 256), "down_proj": _weight(g, 256, 128)}
    ex = {"gate_proj": _weight(g, 3, 128, 256), "up_proj": _weight(g, 3, 128, 256), "down_proj": _weight(g, 3, 256, 128)}
    off = torch.tensor([0, 2, 2, 5], dtype=torch.int32, device=DEV)
    idx = torch.randint(0, 3, (5, 2), generator=g).to(DEV)
    return {
        "quantize": (lambda x: ops.mxfp4_quantize(x), "mxfp4_quantize"),
        "round trip": (lambda x: ops.mxfp4_dequantize(*ops.mxfp4_quantize(x), F32), "mxfp4_dequantize"),
        "linear": (lambda x: ops.mxfp4_linear(x, *w), "mxfp4_linear"),
        "held": (lambda x: ops.mxfp4_linear(ops.mxfp4_quantize(x), *w, out_dtype=F32), "mxfp4_linear"),
        "grouped": (lambda x: ops.mxfp4_grouped_linear(x, *w3, off), "mxfp4_grouped_linear"),
        "dense_ffn": (lambda x: ops.dense_ffn(x, ff), "mxfp4_swiglu"),
        "expert_ffn": (lambda x: ops.expert_ffn(x, ff), "mxfp4_swiglu"),
        "experts": (lambda x: ops.mxfp4_moe_experts(x, idx, ex), "mxfp4_moe_experts"),
    }


def _x(seed, *shape):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(BF16).to(DEV)


def _equal(a, b):
    if isinstance(a, (tuple, list)):
        return len(a) == len(b) and all(_equal(u, v) for u, v in zip(a, b))
    return a.dtype == b.dtype and torch.equal(a, b)


NAMES = ["quantize", "round trip", "linear", "held", "grouped", "dense_ffn", "expert_ffn", "experts"]


@pytest.mark.parametrize("name", NAMES)
def test_traces_replay_on_new_inputs(name):
    f, op = _calls()[name]
    a, b = _x(1, 5, 256), _x(2, 5, 256)
    want = f(b)
    gm = make_fx(f)(a)
    assert any(f"amla.{op}." in str(n.target) for n in gm.graph.nodes)
    assert _equal(gm(b), want)
    traced = torch.jit.trace(f, a, check_trace=False)
    assert f"amla::{op}" in str(traced.graph)
    assert _equal(traced(b), want)


@pytest.mark.parametrize("name", NAMES)
def test_modes_see_the_operator(name):
    f, op = _calls()[name]
    seen = []

    class Mode(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            seen.append(str(func))
            return func(*args, **(kwargs or {}))

    x = _x(3, 5, 256)
    want = f(x)
    with Mode():
        got = f(x)
    assert any(f"amla.{op}." in s for s in seen) and _equal(got, want)


@pytest.mark.parametrize("name", [n for n in NAMES if n not in ("grouped", "experts")])
def test_vmap_equals_the_calls_one_by_one(name):
    f, _ = _calls()[name]
    x = _x(4, 3, 5, 256)
    got = torch.func.vmap(f)(x)
    for i in range(3):
        assert _equal(tuple(t[i] for t in got) if isinstance(got, tuple) else got[i], f(x[i]))


def test_vmap_over_experts_of_a_stack():
    g = torch.Generator().manual_seed(5)
    c, s = _weight(g, 4, 96, 256)
    x = _x(6, 5, 256)
    got = torch.func.vmap(lambda a, b: ops.mxfp4_linear(x, a, b))(c, s)
    for e in range(4):
        assert torch.equal(got[e], ops.mxfp4_linear(x, c[e], s[e]))


# ------------------------------------------------------------------ gradients

def test_grouped_out_refuses_gradients_and_counts_as_written():
    g = torch.Generator().manual_seed(7)
    w = _weight(g, 3, 96, 256)
    off = torch.tensor([0, 2, 2, 5], dtype=torch.int32, device=DEV)
    leaf = _x(8, 5, 256).requires_grad_()
    out = torch.ones(5, 96, dtype=BF16, device=DEV)
    for x in (leaf, leaf * 2):
        with pytest.raises(RuntimeError, match="out= .* gradient"):
            ops.mxfp4_grouped_linear(x, *w, off, out=out)
    with pytest.raises(RuntimeError, match="out= .* gradient"):
        ops.mxfp4_grouped_linear(leaf.detach(), *w, off, out=out.clone().requires_grad_())
    assert (out == 1).all()
    saved = torch.ones(5, 96, dtype=BF16, device=DEV, requires_grad=True)
    y = (saved * out).sum()
    with torch.no_grad():
        ops.mxfp4_grouped_linear(leaf, *w, off, out=out)
    assert torch.equal(out, ops.mxfp4_grouped_linear(leaf.detach(), *w, off))
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


def test_moe_block_backward_raises_beside_a_residual():
    g = torch.Generator().manual_seed(9)
    cfg = DeepSeekConfig(hidden_size=512, n_routed_experts=16, num_experts_per_tok=4, n_group=4, topk_group=2,
                         moe_intermediate_size=256)
    experts = {"gate_proj": _weight(g, 16, 256, 512), "up_proj": _weight(g, 16, 256, 512),
               "down_proj": _weight(g, 16, 512, 256)}
    shared = {"gate_proj": _weight(g, 256, 512), "up_proj": _weight(g, 256, 512), "down_proj": _weight(g, 512, 256)}
    h, gate = _x(10, 1, 6, 512), _x(11, 16, 512)
    want = ops.moe_block(h, gate, shared, experts, cfg)
    idx, wt = ops.route(h, gate, cfg)
    for hidden, gt, routing in ((h.clone().requires_grad_(), gate, None), (h, gate.clone().requires_grad_(), None),
                                (h, gate, (idx, wt.clone().requires_grad_()))):
        y = ops.moe_block(hidden, gt, shared, experts, cfg, routing=routing)
        assert torch.equal(y, want)
        with pytest.raises(RuntimeError, match="no backward"):
            (torch.zeros_like(h, requires_grad=True) + y).float().sum().backward()
        with torch.no_grad():
            assert not ops.moe_block(hidden, gt, shared, experts, cfg, routing=routing).requires_grad


def test_calls_of_two_host_threads():
    """Calls of different LDS sizes of one kernel from two threads: each gives what it gives alone."""
    g = torch.Generator().manual_seed(12)
    parts = [(_x(13, 8, 16384), _weight(g, 512, 16384)), (_x(14, 8, 12288), _weight(g, 512, 12288))]
    want = [ops.mxfp4_linear(x, *w) for x, w in parts]
    torch.cuda.synchronize()
    results = [[], []]

    def work(i):
        x, w = parts[i]
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(40):
                results[i].append(ops.mxfp4_linear(x, *w))
            torch.cuda.current_stream().synchronize()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(60)
    for i in range(2):
        assert len(results[i]) == 40 and all(torch.equal(y, want[i]) for y in results[i])


@pytest.mark.parametrize("lead", [(5,), (2, 3), (0,)])
def test_dequantise_of_empty_pairs(lead):
    for k in (0, 64) if 0 in lead else (0,):
        c = torch.empty(*lead, k // 2, dtype=torch.uint8, device=DEV)
        s = torch.empty(*lead, k // 32, dtype=torch.uint8, device=DEV)
        assert ops.mxfp4_dequantize(c, s).shape == (*lead, k)
        assert ops.mxfp4_dequantize(c, s, F32).dtype == F32


def _moe(g, experts_of):
    cfg = DeepSeekConfig(hidden_size=512, n_routed_experts=16, num_experts_per_tok=4, n_group=4, topk_group=2,
                         moe_intermediate_size=256)
    shared = {"gate_proj": _weight(g, 256, 512), "up_proj": _weight(g, 256, 512), "down_proj": _weight(g, 512, 256)}
    return cfg, shared, {k: experts_of(*s) for k, s in {"gate_proj": (16, 256, 512), "up_proj": (16, 256, 512),
                                                        "down_proj": (16, 512, 256)}.items()}


def _fp8_stack(g, E, n, k):
    return ((torch.randn(E, n, k, generator=g) * 60).clamp(-448, 448).to(torch.float8_e4m3fn).to(DEV),
            torch.full((E, -(-n // 128), -(-k // 128)), 1e-3, device=DEV))


@pytest.mark.parametrize("kind", ["mxfp4", "fp8"])
@pytest.mark.parametrize("tokens", [3, 40])
def test_moe_block_of_a_permuted_batch(kind, tokens):
    g = torch.Generator().manual_seed(15)
    cfg, shared, experts = _moe(g, (lambda *s: _weight(g, *s)) if kind == "mxfp4" else (lambda *s: _fp8_stack(g, *s)))
    h = _x(16, tokens, 2, 512).transpose(0, 1)
    gate = _x(17, 16, 512)
    got = ops.moe_block(h, gate, shared, experts, cfg)
    assert torch.equal(got, ops.moe_block(h.contiguous(), gate, shared, experts, cfg))
