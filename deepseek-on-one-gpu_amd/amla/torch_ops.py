"""PyTorch custom operators over libamla.so: the ``torch.ops.amla`` namespace.

Each operator is a ``torch.library.custom_op`` whose CUDA (ROCm) implementation
calls the C ABI of include/amla.h through ctypes, with a fake (meta)
implementation so that FakeTensor tracing, ``torch.compile`` and ``make_fx`` see
the op, its output shape and its in-place writes:

* ``amla::fp8_linear(x, weight, scale_inv)``           inference/ops.py:15-44
* ``amla::fp8_linear_f32(x, weight, scale_inv)``       the same with fp32 output (out_dtype)
* ``amla::swiglu(x, gate, gate_scale, up, up_scale, down, down_scale)``  inference/ops.py:186-192
* ``amla::rms_norm(x, weight, eps)``                   inference/ops.py:10-12
* ``amla::apply_rope(x, freqs)``                       inference/ops.py:86-97
* ``amla::mla_decode(...)`` / ``amla::mla_prefill(...)``  inference/ops.py:100-183;
  both mutate ``ckv_cache`` and ``kpe_cache`` in place (the cache store of
  inference/ops.py:140-141) and, when given, ``attn_out`` (the per-head output
  before o_proj).
* ``amla::mxfp4_*``: the MXFP4 operators of amla.ops, which call their
  implementations directly, and the registered operators where something could
  tell the difference: a tracer, a transform, a mode, a subclass, a gradient
  (the dispatch costs as much host time as the rest of a call).

Tensors only, no dicts or dataclasses (the op schema cannot carry them): the
shims in amla.ops keep the reference's signatures and unpack ``attn_weights``
and ``config`` into these arguments after validating them.

Scratch memory (split-K partials, queries, latent partials) is taken from
torch's caching allocator on every call, on the calling stream: a call inside a
HIP graph capture allocates from the graph's private pool, so a replay never
sees memory that a later call freed or reused, and calls on different streams
never share scratch.
"""
from __future__ import annotations

from functools import lru_cache
from typing import Optional

import torch
from torch import Tensor
from torch.autograd import forward_ad
from torch.overrides import has_torch_function
from torch.utils._device import DeviceContext

from ._lib import MlaArgs, check, lib

BF16 = torch.bfloat16


def _stream(dev: torch.device) -> int:
    return torch.cuda.current_stream(dev).cuda_stream


def _scratch(dev: torch.device, nbytes: int) -> Tensor:
    return torch.empty(max(int(nbytes), 16), dtype=torch.uint8, device=dev)


# ------------------------------------------------------------------ fp8_linear

def _rows16(x: Tensor) -> Tensor:
    """x itself when its base is 16-byte aligned, else an aligned copy (the kernels load 16-byte
    chunks); checked here, inside the operator, where the tensor is real."""
    return x if x.data_ptr() % 16 == 0 else x.clone(memory_format=torch.contiguous_format)


def _linear(x: Tensor, weight: Tensor, scale_inv: Tensor, f32: bool) -> Tensor:
    x = _rows16(x)
    m, k = x.shape
    n = weight.shape[0]
    y = torch.empty(m, n, dtype=torch.float32 if f32 else BF16, device=x.device)
    if m == 0:
        return y
    L = lib()
    need = L.amla_fp8_linear_workspace_bytes(m, n, k)
    ws = _scratch(x.device, need) if need else None
    fn = L.amla_fp8_linear_f32 if f32 else L.amla_fp8_linear
    check(fn(x.data_ptr(), m, k, x.stride(0), weight.data_ptr(), scale_inv.data_ptr(), n, y.data_ptr(), n,
             ws.data_ptr() if ws is not None else None, ws.numel() if ws is not None else 0, _stream(x.device)),
          "fp8_linear_f32" if f32 else "fp8_linear")
    return y


@torch.library.custom_op("amla::fp8_linear", mutates_args=(), device_types="cuda")
def fp8_linear(x: Tensor, weight: Tensor, scale_inv: Tensor) -> Tensor:
    """y (M, N) bf16 = bf16(x (M, K) @ dequant(weight, scale_inv).T); x rows with unit stride."""
    return _linear(x, weight, scale_inv, False)


@fp8_linear.register_fake
def _(x, weight, scale_inv):
    return x.new_empty(x.shape[0], weight.shape[0])


@torch.library.custom_op("amla::fp8_linear_f32", mutates_args=(), device_types="cuda")
def fp8_linear_f32(x: Tensor, weight: Tensor, scale_inv: Tensor) -> Tensor:
    """y (M, N) fp32 = x (M, K) @ dequant(weight, scale_inv).T, fp32 accumulation, no rounding."""
    return _linear(x, weight, scale_inv, True)


@fp8_linear_f32.register_fake
def _(x, weight, scale_inv):
    return x.new_empty(x.shape[0], weight.shape[0], dtype=torch.float32)


@torch.library.custom_op("amla::swiglu", mutates_args=(), device_types="cuda")
def swiglu(x: Tensor, gate_proj: Tensor, gate_scale: Tensor, up_proj: Tensor, up_scale: Tensor, down_proj: Tensor,
           down_scale: Tensor) -> Tensor:
    """(M, K) bf16 -> down(silu(gate(x)) * up(x)) (M, K) bf16, every product rounded as in the reference."""
    x = _rows16(x)
    m, k = x.shape
    n = gate_proj.shape[0]
    y = torch.empty(m, k, dtype=BF16, device=x.device)
    if m == 0:
        return y
    L = lib()
    need = L.amla_swiglu_workspace_bytes(m, k, n)
    ws = _scratch(x.device, need)
    check(L.amla_swiglu(x.data_ptr(), m, k, gate_proj.data_ptr(), gate_scale.data_ptr(), up_proj.data_ptr(),
                        up_scale.data_ptr(), n, down_proj.data_ptr(), down_scale.data_ptr(), y.data_ptr(),
                        ws.data_ptr(), ws.numel(), _stream(x.device)), "swiglu")
    return y


@swiglu.register_fake
def _(x, gate_proj, gate_scale, up_proj, up_scale, down_proj, down_scale):
    return torch.empty_like(x)


# ------------------------------------------------------------------ rms_norm / apply_rope

@torch.library.custom_op("amla::rms_norm", mutates_args=(), device_types="cuda")
def rms_norm(x: Tensor, weight: Tensor, eps: float) -> Tensor:
    """(rows, dim) bf16 -> bf16(bf16(x * rsqrt(mean(x^2) + eps)) * weight)."""
    y = torch.empty_like(x)
    rows, dim = x.shape
    check(lib().amla_rms_norm(x.data_ptr(), rows, dim, dim, weight.data_ptr(), float(eps), y.data_ptr(), dim,
                              _stream(x.device)), "rms_norm")
    return y


@rms_norm.register_fake
def _(x, weight, eps):
    return torch.empty_like(x)


@torch.library.custom_op("amla::apply_rope", mutates_args=(), device_types="cuda")
def apply_rope(x: Tensor, freqs: Tensor) -> Tensor:
    """x (groups, S, dim) bf16 rotated by freqs (S, dim/2) complex64."""
    y = torch.empty_like(x)
    groups, s, dim = x.shape
    f = torch.view_as_real(freqs)
    check(lib().amla_apply_rope(x.data_ptr(), groups, s, dim, f.data_ptr(), y.data_ptr(), _stream(x.device)),
          "apply_rope")
    return y


@apply_rope.register_fake
def _(x, freqs):
    return torch.empty_like(x)


# ------------------------------------------------------------------ MLA

def fill_mla_args(hidden: Tensor, w_q_a: Tensor, s_q_a: Tensor, w_q_b: Tensor, s_q_b: Tensor, w_kv_a: Tensor,
                  s_kv_a: Tensor, w_kv_b: Tensor, s_kv_b: Tensor, w_o: Tensor, s_o: Tensor, gamma_q: Tensor,
                  gamma_kv: Tensor, ckv_cache: Tensor, kpe_cache: Tensor, positions: Tensor, rope_freqs: Tensor,
                  input_gamma: Optional[Tensor], residual: Optional[Tensor], attn_out: Optional[Tensor],
                  out: Tensor, max_context: int, eps: float, softmax_scale: float, heads: int, qk_nope: int,
                  v_dim: int) -> MlaArgs:
    """amla_mla_args for validated tensors (no workspace yet)."""
    B, S, D = hidden.shape
    a = MlaArgs()
    a.batch, a.seq_len, a.hidden = B, S, D
    a.heads, a.q_lora, a.kv_lora = heads, w_q_a.shape[0], ckv_cache.shape[2]
    a.qk_nope, a.qk_rope, a.v_dim = qk_nope, kpe_cache.shape[2], v_dim
    a.max_seq, a.rope_rows, a.max_context = ckv_cache.shape[1], rope_freqs.shape[0], int(max_context)
    a.eps, a.softmax_scale = float(eps), float(softmax_scale)
    a.positions = positions.data_ptr()
    a.hidden_states, a.out = hidden.data_ptr(), out.data_ptr()
    a.input_gamma = input_gamma.data_ptr() if input_gamma is not None else None
    a.residual = residual.data_ptr() if residual is not None else None
    a.w_q_a, a.s_q_a, a.w_q_b, a.s_q_b = w_q_a.data_ptr(), s_q_a.data_ptr(), w_q_b.data_ptr(), s_q_b.data_ptr()
    a.w_kv_a, a.s_kv_a = w_kv_a.data_ptr(), s_kv_a.data_ptr()
    a.w_kv_b, a.s_kv_b = w_kv_b.data_ptr(), s_kv_b.data_ptr()
    a.w_o, a.s_o = w_o.data_ptr(), s_o.data_ptr()
    a.gamma_q, a.gamma_kv = gamma_q.data_ptr(), gamma_kv.data_ptr()
    a.ckv_cache, a.kpe_cache = ckv_cache.data_ptr(), kpe_cache.data_ptr()
    a.rope_table = rope_freqs.data_ptr()
    a.attn_out = attn_out.data_ptr() if attn_out is not None else None
    return a


def _mla_run(decode: bool, hidden, w_q_a, s_q_a, w_q_b, s_q_b, w_kv_a, s_kv_a, w_kv_b, s_kv_b, w_o, s_o, gamma_q,
             gamma_kv, ckv_cache, kpe_cache, positions, rope_freqs, input_gamma, residual, attn_out, max_context,
             eps, softmax_scale, heads, qk_nope, v_dim) -> Tensor:
    out = torch.empty_like(hidden)
    a = fill_mla_args(hidden, w_q_a, s_q_a, w_q_b, s_q_b, w_kv_a, s_kv_a, w_kv_b, s_kv_b, w_o, s_o, gamma_q,
                      gamma_kv, ckv_cache, kpe_cache, positions, rope_freqs, input_gamma, residual, attn_out, out,
                      max_context, eps, softmax_scale, heads, qk_nope, v_dim)
    L = lib()
    need = (L.amla_mla_decode_workspace_bytes if decode else L.amla_mla_prefill_workspace_bytes)(a)
    ws = _scratch(hidden.device, need)
    a.workspace, a.workspace_bytes = ws.data_ptr(), ws.numel()
    rc = (L.amla_mla_decode if decode else L.amla_mla_prefill)(a, _stream(hidden.device))
    check(rc, "mla_decode" if decode else "mla_prefill")
    return out


_MLA_MUTATES = ("ckv_cache", "kpe_cache", "attn_out")


@torch.library.custom_op("amla::mla_decode", mutates_args=_MLA_MUTATES, device_types="cuda")
def mla_decode(hidden: Tensor, w_q_a: Tensor, s_q_a: Tensor, w_q_b: Tensor, s_q_b: Tensor, w_kv_a: Tensor,
               s_kv_a: Tensor, w_kv_b: Tensor, s_kv_b: Tensor, w_o: Tensor, s_o: Tensor, gamma_q: Tensor,
               gamma_kv: Tensor, ckv_cache: Tensor, kpe_cache: Tensor, positions: Tensor, rope_freqs: Tensor,
               input_gamma: Optional[Tensor], residual: Optional[Tensor], attn_out: Optional[Tensor],
               max_context: int, eps: float, softmax_scale: float, heads: int, qk_nope: int,
               v_dim: int) -> Tensor:
    """Absorbed-MLA decode (S == 1): returns (B, 1, hidden) bf16; writes the new cache rows."""
    return _mla_run(True, hidden, w_q_a, s_q_a, w_q_b, s_q_b, w_kv_a, s_kv_a, w_kv_b, s_kv_b, w_o, s_o, gamma_q,
                    gamma_kv, ckv_cache, kpe_cache, positions, rope_freqs, input_gamma, residual, attn_out,
                    max_context, eps, softmax_scale, heads, qk_nope, v_dim)


@torch.library.custom_op("amla::mla_prefill", mutates_args=_MLA_MUTATES, device_types="cuda")
def mla_prefill(hidden: Tensor, w_q_a: Tensor, s_q_a: Tensor, w_q_b: Tensor, s_q_b: Tensor, w_kv_a: Tensor,
                s_kv_a: Tensor, w_kv_b: Tensor, s_kv_b: Tensor, w_o: Tensor, s_o: Tensor, gamma_q: Tensor,
                gamma_kv: Tensor, ckv_cache: Tensor, kpe_cache: Tensor, positions: Tensor, rope_freqs: Tensor,
                input_gamma: Optional[Tensor], residual: Optional[Tensor], attn_out: Optional[Tensor],
                max_context: int, eps: float, softmax_scale: float, heads: int, qk_nope: int,
                v_dim: int) -> Tensor:
    """Causal MLA prefill (S >= 1): returns (B, S, hidden) bf16; writes the new cache rows."""
    return _mla_run(False, hidden, w_q_a, s_q_a, w_q_b, s_q_b, w_kv_a, s_kv_a, w_kv_b, s_kv_b, w_o, s_o, gamma_q,
                    gamma_kv, ckv_cache, kpe_cache, positions, rope_freqs, input_gamma, residual, attn_out,
                    max_context, eps, softmax_scale, heads, qk_nope, v_dim)


def _mla_fake(hidden, *args, **kwargs):
    return torch.empty_like(hidden)


mla_decode.register_fake(_mla_fake)
mla_prefill.register_fake(_mla_fake)


# ------------------------------------------------------------------ MXFP4

_MX_CODES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}  # AMLA_BF16, AMLA_FP16, AMLA_FP32
_mx_lib = torch.library.Library("amla", "FRAGMENT")
_mx_impl: dict = {}


def _on_device(fn, t: Tensor, *args):
    if t.device.index == torch._C._cuda_getDevice():
        return fn(t, *args)
    with torch.cuda.device(t.device):
        return fn(t, *args)


def _mx_no_backward(ctx, *grads):
    raise RuntimeError("the MXFP4 operators have no backward pass")


class _NoBackward(torch.autograd.Function):
    @staticmethod
    def forward(ctx, fn, *sources):
        return fn()

    @staticmethod
    def backward(ctx, *grads):
        _mx_no_backward(ctx, *grads)


def without_backward(fn, *sources: Tensor) -> Tensor:
    """``fn()``, a tensor made of ``sources`` behind autograd's back: a backward through it raises."""
    if torch.is_grad_enabled() and any(s.requires_grad for s in sources):
        return _NoBackward.apply(fn, *sources)
    return fn()


def _mx_op(schema: str, fake):
    """Registers amla::<schema> with its ROCm implementation and its fake one."""
    def wrap(fn):
        name = schema.split("(")[0]
        _mx_lib.define(schema)
        _mx_lib.impl(name, lambda t, *args: _on_device(fn, t, *args), "CUDA")
        torch.library.register_fake(f"amla::{name}", fake, lib=_mx_lib)
        if "!" not in schema:
            torch.library.register_autograd(f"amla::{name}", _mx_no_backward, lib=_mx_lib)
        _mx_impl[name] = fn
        return fn
    return wrap


# Bits of the thread's dispatch keys that are off while nothing watches torch's operators: tracers,
# transforms (vmap, grad, jvp, functionalize), torch.jit.trace and dispatch modes set some of them.
_WATCHED = ~torch._C.DispatchKeySet(torch._C.DispatchKey.BackendSelect).add(
    torch._C.DispatchKey.ADInplaceOrView).raw_repr()
_thread_keys = torch._C._dispatch_tls_local_include_set
_dynamo = torch.compiler.is_dynamo_compiling


def call(name: str, t: Tensor, *args):
    """The implementation of amla::<name>, or the operator itself where the difference shows: something
    traces, transforms or intercepts torch's operators, an argument is a tensor subclass, or a derivative
    is asked for."""
    if _dynamo() or _thread_keys().raw_repr() & _WATCHED or has_torch_function((t, *args)) and _intercepted(t, *args) or \
            t.requires_grad or forward_ad._current_level >= 0 or type(t) is not Tensor and not isinstance(t, torch.nn.Parameter):
        if name not in _MX_WHOLE:
            _no_tangent(t)
        return getattr(torch.ops.amla, name)(t, *args)
    return _on_device(_mx_impl[name], t, *args)


_PLAIN_TYPES = frozenset((Tensor, torch.nn.Parameter, type(None), bool))  # of an operator's arguments


def _intercepted(*args) -> bool:
    """Whether a function mode other than a default device is on, or an argument is a subclass."""
    modes = torch._C._len_torch_function_stack()
    for i in range(modes):
        if type(torch._C._get_function_stack_at(i)) is not DeviceContext:
            return True
    return not modes or not _PLAIN_TYPES.issuperset(map(type, args))


_MX_WHOLE = ("mxfp4_quantize", "mxfp4_quantize_fp8")  # outputs are whole numbers: no derivative passes through


def _no_tangent(t: Tensor) -> None:
    if not _dynamo() and forward_ad._current_level >= 0 and forward_ad.unpack_dual(t).tangent is not None:
        raise RuntimeError("the MXFP4 operators have no derivative in forward mode")


# (the workspaces' sizes are functions of the call's sizes alone)
_mx_linear_bytes = lru_cache(4096)(lambda *a: lib().amla_mxfp4_linear_workspace_bytes(*a))
_mx_grouped_bytes = lru_cache(4096)(lambda *a: lib().amla_mxfp4_grouped_linear_workspace_bytes(*a))
_mx_swiglu_bytes = lru_cache(4096)(lambda *a: lib().amla_mxfp4_swiglu_workspace_bytes(*a))
_mx_moe_bytes = lru_cache(4096)(lambda *a: lib().amla_mxfp4_moe_experts_workspace_bytes(*a))


def _mx_stream(t: Tensor) -> int:
    return torch._C._cuda_getCurrentRawStream(t.device.index)


def _mx_fake_pair(x, *_):
    rows, k = x.shape
    return (x.new_empty(rows, k // 2, dtype=torch.uint8), x.new_empty(rows, k // 32, dtype=torch.uint8))


def _mx_pair_out(rows: int, k: int, dev) -> tuple[Tensor, Tensor]:
    return (torch.empty(rows, k // 2, dtype=torch.uint8, device=dev),
            torch.empty(rows, k // 32, dtype=torch.uint8, device=dev))


def _mx_ldx(x: Tensor, k: int) -> int:
    return x.stride(0) if x.shape[0] > 1 else k


def _mx_x(x, x_scales):
    """The activations with the alignment the kernels need (copies of those that lack it)."""
    if x_scales is not None and x_scales.data_ptr() % 4:
        x_scales = x_scales.clone()
    return _rows16(x), x_scales


def _ptr(t):
    return None if t is None else t.data_ptr()


@_mx_op("mxfp4_quantize(Tensor x) -> (Tensor, Tensor)", _mx_fake_pair)
def _mxfp4_quantize(x):
    x = _rows16(x)
    rows, k = x.shape
    q, s = _mx_pair_out(rows, k, x.device)
    check(lib().amla_mxfp4_quantize(x.data_ptr(), _MX_CODES[x.dtype], rows, k, _mx_ldx(x, k), q.data_ptr(),
                                    s.data_ptr(), _mx_stream(x)) if rows else 0, "mxfp4_quantize")
    return q, s


@_mx_op("mxfp4_quantize_fp8(Tensor weight, Tensor scale_inv) -> (Tensor, Tensor)", _mx_fake_pair)
def _mxfp4_quantize_fp8(weight, scale_inv):
    weight = _rows16(weight)
    n, k = weight.shape
    q, s = _mx_pair_out(n, k, weight.device)
    check(lib().amla_mxfp4_quantize_fp8(weight.data_ptr(), scale_inv.data_ptr(), n, k, q.data_ptr(), s.data_ptr(),
                                        _mx_stream(weight)) if n else 0, "mxfp4_quantize_fp8")
    return q, s


@_mx_op("mxfp4_dequantize(Tensor codes, Tensor scales, bool f32) -> Tensor",
        lambda codes, scales, f32: codes.new_empty(codes.shape[0], codes.shape[1] * 2,
                                                   dtype=torch.float32 if f32 else BF16))
def _mxfp4_dequantize(codes, scales, f32):
    codes = _rows16(codes)
    rows, k = codes.shape[0], codes.shape[1] * 2
    out = torch.empty(rows, k, dtype=torch.float32 if f32 else BF16, device=codes.device)
    check(lib().amla_mxfp4_dequantize(codes.data_ptr(), scales.data_ptr(), rows, k, _MX_CODES[out.dtype],
                                      out.data_ptr(), _mx_stream(codes)) if out.numel() else 0, "mxfp4_dequantize")
    return out


def _mx_linear_fake(x, x_scales, weight, scale, f32):
    return x.new_empty(x.shape[0], weight.shape[0], dtype=torch.float32 if f32 else BF16)


@_mx_op("mxfp4_linear(Tensor x, Tensor? x_scales, Tensor weight, Tensor scale, bool f32) -> Tensor", _mx_linear_fake)
def _mxfp4_linear(x, x_scales, weight, scale, f32):
    x, x_scales = _mx_x(x, x_scales)
    m, n, k = x.shape[0], weight.shape[0], weight.shape[1] * 2
    y = torch.empty(m, n, dtype=torch.float32 if f32 else BF16, device=x.device)
    if m == 0 or n == 0:
        return y
    L = lib()
    need = _mx_linear_bytes(m, n, k, x_scales is not None)
    ws = _scratch(x.device, need) if need else None
    check(L.amla_mxfp4_linear(x.data_ptr(), _ptr(x_scales), m, k, _mx_ldx(x, k), weight.data_ptr(), scale.data_ptr(),
                              n, y.data_ptr(), _MX_CODES[y.dtype], n, _ptr(ws), need, _mx_stream(x)),
          "mxfp4_linear")
    return y


def _mx_grouped(x, x_scales, weight, scale, offsets, y, clear) -> None:
    x, x_scales = _mx_x(x, x_scales)
    m, E, n, k = x.shape[0], weight.shape[0], weight.shape[1], weight.shape[2] * 2
    if m == 0:
        return
    L = lib()
    need = _mx_grouped_bytes(m, n, k, E, x_scales is not None)
    ws = _scratch(x.device, need)
    check(L.amla_mxfp4_grouped_linear(x.data_ptr(), _ptr(x_scales), m, k, _mx_ldx(x, k), weight.data_ptr(),
                                      scale.data_ptr(), n, E, offsets.data_ptr(), y.data_ptr(), _MX_CODES[y.dtype],
                                      y.stride(0) if m > 1 else n, clear, ws.data_ptr(), ws.numel(),
                                      _mx_stream(x)), "mxfp4_grouped_linear")


@_mx_op("mxfp4_grouped_linear(Tensor x, Tensor? x_scales, Tensor weight, Tensor scale, Tensor offsets, bool f32) -> Tensor",
        lambda x, x_scales, weight, scale, offsets, f32: x.new_empty(x.shape[0], weight.shape[1],
                                                                     dtype=torch.float32 if f32 else BF16))
def _mxfp4_grouped_linear(x, x_scales, weight, scale, offsets, f32):
    y = torch.empty(x.shape[0], weight.shape[1], dtype=torch.float32 if f32 else BF16, device=x.device)
    _mx_grouped(x, x_scales, weight, scale, offsets, y, 1)
    return y


@_mx_op("mxfp4_grouped_linear_out(Tensor x, Tensor? x_scales, Tensor weight, Tensor scale, Tensor offsets, "
        "Tensor(a!) out) -> ()", lambda x, x_scales, weight, scale, offsets, out: None)
def _mxfp4_grouped_linear_out(x, x_scales, weight, scale, offsets, out):
    _mx_out_gradient(x, out)
    _mx_grouped(x, x_scales, weight, scale, offsets, out, 0)
    torch.autograd.graph.increment_version(out)


def _mx_out_gradient(x, out) -> None:
    if torch.is_grad_enabled() and (x.requires_grad or out.requires_grad):
        raise RuntimeError("mxfp4_grouped_linear: out= has no gradient, but x or out requires one")


def _mxfp4_grouped_linear_out_autograd(x, x_scales, weight, scale, offsets, out):
    _mx_out_gradient(x, out)
    with torch._C._AutoDispatchBelowAutograd():
        torch.ops.amla.mxfp4_grouped_linear_out(x, x_scales, weight, scale, offsets, out)


_mx_lib.impl("mxfp4_grouped_linear_out", _mxfp4_grouped_linear_out_autograd, "Autograd")


@_mx_op("mxfp4_swiglu(Tensor x, Tensor gate_proj, Tensor gate_scale, Tensor up_proj, Tensor up_scale, "
        "Tensor down_proj, Tensor down_scale) -> Tensor",
        lambda x, gate_proj, *_: x.new_empty(x.shape[0], x.shape[1]))
def _mxfp4_swiglu(x, gate_proj, gate_scale, up_proj, up_scale, down_proj, down_scale):
    x = _rows16(x)
    m, k = x.shape
    n = gate_proj.shape[0]
    y = torch.empty(m, k, dtype=BF16, device=x.device)
    if m == 0:
        return y
    L = lib()
    need = _mx_swiglu_bytes(m, k, n)
    ws = _scratch(x.device, need)
    check(L.amla_mxfp4_swiglu(x.data_ptr(), m, k, _mx_ldx(x, k), gate_proj.data_ptr(), gate_scale.data_ptr(),
                              up_proj.data_ptr(), up_scale.data_ptr(), n, down_proj.data_ptr(), down_scale.data_ptr(),
                              y.data_ptr(), ws.data_ptr(), ws.numel(), _mx_stream(x)), "mxfp4_swiglu")
    return y


_MX_MOE_SLOTS, _MX_MOE_CODES = 65536, 2 ** 32 - 1  # (token, k) slots and bytes of codes of one call


@_mx_op("mxfp4_moe_experts(Tensor hidden, Tensor indices, Tensor gate_proj, Tensor gate_scale, Tensor up_proj, "
        "Tensor up_scale, Tensor down_proj, Tensor down_scale) -> Tensor",
        lambda hidden, indices, *_: hidden.new_empty(hidden.shape[0], indices.shape[1], hidden.shape[1]))
def _mxfp4_moe_experts(hidden, indices, gate_proj, gate_scale, up_proj, up_scale, down_proj, down_scale):
    hidden = _rows16(hidden)
    m, top_k = indices.shape
    E, n, d = gate_proj.shape[0], gate_proj.shape[1], hidden.shape[1]
    out = torch.empty(m, top_k, d, dtype=BF16, device=hidden.device)
    L = lib()
    step = min(_MX_MOE_SLOTS // top_k, _MX_MOE_CODES // (d // 2))
    for t in range(0, m, step):
        c = min(step, m - t)
        need = _mx_moe_bytes(c, d, top_k, n, E)
        ws = _scratch(hidden.device, need)
        check(L.amla_mxfp4_moe_experts(hidden[t:].data_ptr(), c, d, _mx_ldx(hidden, d), top_k, indices[t:].data_ptr(),
                                       n, E, gate_proj.data_ptr(), gate_scale.data_ptr(), up_proj.data_ptr(),
                                       up_scale.data_ptr(), down_proj.data_ptr(), down_scale.data_ptr(),
                                       out[t:].data_ptr(), 1, ws.data_ptr(), ws.numel(), _mx_stream(hidden)),
              "mxfp4_moe_experts")
    return out
