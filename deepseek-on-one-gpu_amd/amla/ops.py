"""MLA-path operators with the reference's signatures, on gfx950 HIP kernels.

Drop-in for the MLA half of inference/ops.py: ``rms_norm`` (:10-12),
``fp8_linear`` (:15-44), ``yarn_get_mscale`` (:47-50), ``precompute_rope_freqs``
(:53-83), ``apply_rope`` (:86-97) and ``mla_attention`` (:100-183), plus the
attention half of ``transformer_layer`` (inference/forward.py:92-94) as
``mla_layer``; and the FFN / MoE functions on the same fp8 kernels: ``swiglu``
(:186-192), ``dense_ffn`` / ``expert_ffn`` (:195-206), ``route`` (:209-257) and
``moe_block`` (inference/forward.py:112-153, experts handed in); and the same
linears, FFN and experts for weights held in MXFP4 (``mxfp4_*``); and, for a
server of many sequences, a paged latent cache (``latent_cache_*``), the attention
over it and that of packed prompts.  Same argument names, tensor layouts and dtypes; tensors must be
on a ROCm device.  Every compute call goes to libamla.so; there is no CPU or
PyTorch fallback (a missing library raises).

Superset over the reference: ``position`` of ``mla_attention`` may also be a
list of per-sequence start positions or an int32 device tensor of them (the
reference's scalar position cannot express a ragged batch).
"""
from __future__ import annotations

import ctypes
import math
from typing import Sequence

import torch

from . import _lib, torch_ops
from ._lib import check, lib

BF16 = torch.bfloat16
FP8 = torch.float8_e4m3fn


def _stream_ptr(t: torch.Tensor) -> int:
    return torch.cuda.current_stream(t.device).cuda_stream


def _need_cuda(t: torch.Tensor, name: str) -> None:
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise ValueError(f"{name} must be a tensor on a ROCm device")


def _need(t: torch.Tensor, name: str, dtype, dev=None) -> None:
    _need_cuda(t, name)
    if t.dtype != dtype:
        raise TypeError(f"{name} must be {dtype} (got {t.dtype})")
    if dev is not None and t.device != dev:
        raise ValueError(f"{name} is on {t.device}, expected {dev}")
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")


# ------------------------------------------------------------------ workspace

def workspace(device: torch.device, nbytes: int) -> torch.Tensor:
    """Scratch for one call, from torch's caching allocator on the current stream.

    A fresh buffer per call: inside a HIP graph capture it comes from the
    graph's private pool (a replay never touches memory another call owns),
    and calls on different streams never share it.
    """
    return torch.empty(max(int(nbytes), 16), dtype=torch.uint8, device=device)


# ------------------------------------------------------------------ elementwise / linear

def rms_norm(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6) -> torch.Tensor:
    """inference/ops.py:10-12: y = bf16(bf16(x * rsqrt(mean(x^2) + eps)) * weight)."""
    _need_cuda(x, "x")
    if x.dtype != BF16 or weight.dtype != BF16:
        raise TypeError("rms_norm: x and weight must be bfloat16")
    dim = x.shape[-1]
    if weight.shape != (dim,):
        raise ValueError(f"rms_norm: weight shape {tuple(weight.shape)} != ({dim},)")
    xc = x.contiguous()
    w = weight.contiguous()
    rows = xc.numel() // dim if dim else 0
    return torch.ops.amla.rms_norm(xc.view(rows, dim), w, float(eps)).view(x.shape)


def fp8_block_dequant(weight: torch.Tensor, scale_inv: torch.Tensor) -> torch.Tensor:
    """inference/ops.py:30-43: fp32 f32(weight) * scale_inv[i//128, j//128], bit-exact."""
    _need(weight, "weight", FP8)
    _need(scale_inv, "scale_inv", torch.float32, weight.device)
    n, k = weight.shape
    if scale_inv.shape != (math.ceil(n / 128), math.ceil(k / 128)):
        raise ValueError(f"scale_inv shape {tuple(scale_inv.shape)} does not match weight {n}x{k}")
    out = torch.empty(n, k, dtype=torch.float32, device=weight.device)
    check(lib().amla_fp8_block_dequant(weight.data_ptr(), scale_inv.data_ptr(), n, k, out.data_ptr(),
                                       _stream_ptr(weight)), "fp8_block_dequant")
    return out


def fp8_linear(x: torch.Tensor, weight: torch.Tensor, scale_inv: torch.Tensor,
               out_dtype: torch.dtype = BF16) -> torch.Tensor:
    """inference/ops.py:15-44: ( x @ dequant(weight, scale_inv).T ).to(out_dtype), fp32 accumulation.

    bf16 rounds in the kernel's epilogue (``torch.ops.amla.fp8_linear``); any other out_dtype
    takes the fp32 result (``torch.ops.amla.fp8_linear_f32``) cast with ``.to(out_dtype)`` as the
    reference does."""
    _need_cuda(x, "x")
    if x.dtype != BF16:
        raise TypeError(f"fp8_linear: x must be bfloat16 (got {x.dtype})")
    if not isinstance(out_dtype, torch.dtype) or not (out_dtype.is_floating_point or out_dtype.is_complex):
        raise TypeError(f"fp8_linear: out_dtype must be a floating-point dtype (got {out_dtype})")
    _need(weight, "weight", FP8, x.device)
    _need(scale_inv, "scale_inv", torch.float32, x.device)
    n, k = weight.shape
    if x.shape[-1] != k:
        raise ValueError(f"fp8_linear: x has {x.shape[-1]} features, weight expects {k}")
    if scale_inv.shape != (math.ceil(n / 128), math.ceil(k / 128)):
        raise ValueError(f"scale_inv shape {tuple(scale_inv.shape)} does not match weight {n}x{k}")
    x2 = x.reshape(-1, k)
    if x2.stride(-1) != 1 or x2.stride(0) % 8:
        x2 = x2.contiguous()
    if out_dtype == BF16:
        return torch.ops.amla.fp8_linear(x2, weight, scale_inv).view(*x.shape[:-1], n)
    y = torch.ops.amla.fp8_linear_f32(x2, weight, scale_inv).view(*x.shape[:-1], n)
    return y if out_dtype == torch.float32 else y.to(out_dtype)


# ------------------------------------------------------------------ RoPE

def yarn_get_mscale(scale: float = 1.0, mscale: float = 1.0) -> float:
    """inference/ops.py:47-50 (host scalar)."""
    if scale <= 1.0:
        return 1.0
    return 0.1 * mscale * math.log(scale) + 1.0


def precompute_rope_freqs(config, seq_len: int, device) -> torch.Tensor:
    """inference/ops.py:53-83: YaRN-blended frequencies, complex64 (seq_len, rope/2).

    One-time table set-up (the engine builds it once, inference/engine.py:63):
    computed with fp32 torch ops in the same order as the reference, so the
    table is bit-identical, then moved to ``device``.
    """
    dim = config.qk_rope_head_dim
    base = config.rope_theta
    inv = 1.0 / (base ** (torch.arange(0, dim, 2, dtype=torch.float32) / dim))

    def edge(beta):
        return dim * math.log(config.original_max_position_embeddings / (beta * 2 * math.pi)) / (2 * math.log(base))

    low = max(math.floor(edge(config.rope_scaling_beta_fast)), 0)
    high = min(math.ceil(edge(config.rope_scaling_beta_slow)), dim // 2 - 1)
    ramp = torch.ones(dim // 2, dtype=torch.float32)
    if high > low:
        ramp = ((torch.arange(dim // 2, dtype=torch.float32) - low) / (high - low)).clamp(0.0, 1.0)
    inv = inv * (1.0 - ramp) + (inv / config.rope_scaling_factor) * ramp
    ang = torch.outer(torch.arange(seq_len, dtype=torch.float32), inv)
    return torch.polar(torch.ones_like(ang), ang).to(device)


def apply_rope(x: torch.Tensor, freqs: torch.Tensor) -> torch.Tensor:
    """inference/ops.py:86-97: x (B, H, S, rope) bf16, freqs (S, rope/2) complex64."""
    _need_cuda(x, "x")
    if x.dtype != BF16:
        raise TypeError("apply_rope: x must be bfloat16")
    if freqs.dtype != torch.complex64 or freqs.device != x.device:
        raise TypeError("apply_rope: freqs must be complex64 on the same device")
    S, dim = x.shape[-2], x.shape[-1]
    if freqs.shape != (S, dim // 2):
        raise ValueError(f"apply_rope: freqs shape {tuple(freqs.shape)} != ({S}, {dim // 2})")
    xc = x.contiguous()
    groups = xc.numel() // (S * dim) if S * dim else 0
    return torch.ops.amla.apply_rope(xc.view(groups, S, dim), freqs.contiguous()).view(x.shape)


# ------------------------------------------------------------------ MLA

def softmax_scale(config) -> float:
    """mscale / sqrt(qk_head_dim), mscale applied once (inference/ops.py:166-167)."""
    return yarn_get_mscale(config.rope_scaling_factor, config.rope_scaling_mscale_all_dim) / math.sqrt(
        config.qk_head_dim)


def _positions(position, B: int, S: int, device, max_context):
    """(int32 device tensor (B,), max position+S or None) from an int, a sequence or a tensor."""
    if isinstance(position, torch.Tensor):
        if position.dtype != torch.int32 or position.device != device or position.shape != (B,):
            raise ValueError("position tensor must be int32 (B,) on the hidden states' device")
        return position, max_context
    if isinstance(position, int):
        if position < 0:
            raise ValueError("position must be >= 0")
        return torch.full((B,), position, dtype=torch.int32, device=device), position + S
    pos = [int(p) for p in position]
    if len(pos) != B or min(pos) < 0:
        raise ValueError("one non-negative position per sequence is required")
    return torch.tensor(pos, dtype=torch.int32, device=device), max(pos) + S


_PROJ = (("q_a_proj", "w_q_a"), ("q_b_proj", "w_q_b"), ("kv_a_proj_with_mqa", "w_kv_a"),
         ("kv_b_proj", "w_kv_b"), ("o_proj", "w_o"))


def _mla_operands(hidden, attn_weights, kv_cache, position, rope_freqs, config, *, input_gamma=None,
                  residual=None, attn_out=None, max_context=None) -> dict:
    """Validates the reference's arguments and unpacks them into the operands of
    ``torch.ops.amla.mla_decode`` / ``mla_prefill`` (raises before any launch)."""
    _need(hidden, "hidden", BF16)
    dev = hidden.device
    if hidden.dim() != 3:
        raise ValueError("hidden must be (B, S, hidden_size)")
    B, S, D = hidden.shape
    if D != config.hidden_size:
        raise ValueError(f"hidden size {D} != config.hidden_size {config.hidden_size}")
    ckv, kpe = kv_cache
    _need(ckv, "compressed_kv_cache", BF16, dev)
    _need(kpe, "k_pe_cache", BF16, dev)
    if ckv.dim() != 3 or kpe.dim() != 3 or ckv.shape[:2] != kpe.shape[:2]:
        raise ValueError("kv caches must be (B_alloc, max_seq, kv_lora) and (B_alloc, max_seq, rope)")
    if ckv.shape[0] < B or ckv.shape[2] != config.kv_lora_rank or kpe.shape[2] != config.qk_rope_head_dim:
        raise ValueError(f"kv cache shapes {tuple(ckv.shape)} / {tuple(kpe.shape)} do not fit batch {B}")
    max_seq = ckv.shape[1]
    if rope_freqs.dtype != torch.complex64 or rope_freqs.device != dev or not rope_freqs.is_contiguous():
        raise TypeError("rope_freqs must be a contiguous complex64 tensor on the same device")
    if rope_freqs.dim() != 2 or rope_freqs.shape[1] != config.qk_rope_head_dim // 2:
        raise ValueError("rope_freqs must have qk_rope_head_dim/2 columns")
    pos_t, mc = _positions(position, B, S, dev, max_context)
    if mc is None:
        mc = min(max_seq, rope_freqs.shape[0])
    if mc > max_seq:
        raise ValueError(f"position + seq_len = {mc} exceeds the cache length {max_seq}")
    if mc > rope_freqs.shape[0]:
        raise ValueError(f"position + seq_len = {mc} exceeds the rope table length {rope_freqs.shape[0]}")
    if mc < S:
        raise ValueError(f"max_context {mc} is below seq_len {S}")
    H = config.num_attention_heads
    shapes = {
        "q_a_proj": (config.q_lora_rank, D),
        "q_b_proj": (H * config.qk_head_dim, config.q_lora_rank),
        "kv_a_proj_with_mqa": (config.kv_lora_rank + config.qk_rope_head_dim, D),
        "kv_b_proj": (H * (config.qk_nope_head_dim + config.v_head_dim), config.kv_lora_rank),
        "o_proj": (D, H * config.v_head_dim),
    }
    ops = {"hidden": hidden}
    for name, field in _PROJ:
        w, sc = attn_weights[name]
        _need(w, f"{name}.weight", FP8, dev)
        _need(sc, f"{name}.weight_scale_inv", torch.float32, dev)
        n, k = shapes[name]
        if tuple(w.shape) != (n, k) or tuple(sc.shape) != (math.ceil(n / 128), math.ceil(k / 128)):
            raise ValueError(f"{name}: weight {tuple(w.shape)} / scale {tuple(sc.shape)} do not match ({n}, {k})")
        ops[field] = w
        ops["s" + field[1:]] = sc
    gq, gkv = attn_weights["q_a_layernorm"], attn_weights["kv_a_layernorm"]
    _need(gq, "q_a_layernorm", BF16, dev)
    _need(gkv, "kv_a_layernorm", BF16, dev)
    if gq.shape != (config.q_lora_rank,) or gkv.shape != (config.kv_lora_rank,):
        raise ValueError("q_a_layernorm / kv_a_layernorm do not match q_lora_rank / kv_lora_rank")
    if input_gamma is not None:
        _need(input_gamma, "input_layernorm", BF16, dev)
        if input_gamma.shape != (D,):
            raise ValueError("input_layernorm must be (hidden_size,)")
    if residual is not None:
        _need(residual, "residual", BF16, dev)
        if residual.shape != hidden.shape:
            raise ValueError("residual must have the hidden states' shape")
    if attn_out is not None:
        _need(attn_out, "attn_out", BF16, dev)
        if tuple(attn_out.shape) != (B, S, H * config.v_head_dim) or attn_out.data_ptr() % 16:
            raise ValueError(f"attn_out must be a 16-byte aligned (B, S, {H * config.v_head_dim}) bf16 tensor")
    ops.update(gamma_q=gq, gamma_kv=gkv, ckv_cache=ckv, kpe_cache=kpe, positions=pos_t, rope_freqs=rope_freqs,
               input_gamma=input_gamma, residual=residual, attn_out=attn_out, max_context=int(mc),
               eps=float(config.rms_norm_eps), softmax_scale=float(softmax_scale(config)), heads=H,
               qk_nope=config.qk_nope_head_dim, v_dim=config.v_head_dim)
    return ops


def _mla(ops: dict) -> torch.Tensor:
    fn = torch.ops.amla.mla_decode if ops["hidden"].shape[1] == 1 else torch.ops.amla.mla_prefill
    return fn(**ops)


def mla_attention(hidden: torch.Tensor, attn_weights: dict, kv_cache: tuple, position, rope_freqs: torch.Tensor,
                  config, *, max_context: int | None = None, attn_out: torch.Tensor | None = None) -> torch.Tensor:
    """inference/ops.py:100-183 on gfx950 (``torch.ops.amla.mla_decode`` / ``mla_prefill``).

    S == 1 runs the absorbed decode; S > 1 the kv_b decompression + causal
    flash prefill, or, for a few new tokens over many cached rows, the same
    attention in latent space as the decode.  Writes the raw new rows into ``kv_cache`` at
    [position, position+S) like the reference.  ``max_context`` (largest
    position+S) is only needed when ``position`` is a device tensor.  When
    ``attn_out`` ((B, S, heads * v_head_dim) bf16) is given, the per-head
    attention output before o_proj is written into it.
    """
    return _mla(_mla_operands(hidden, attn_weights, kv_cache, position, rope_freqs, config,
                              max_context=max_context, attn_out=attn_out))


def mla_layer(hidden: torch.Tensor, input_layernorm: torch.Tensor, attn_weights: dict, kv_cache: tuple,
              position, rope_freqs: torch.Tensor, config, *, max_context: int | None = None,
              attn_out: torch.Tensor | None = None) -> torch.Tensor:
    """Attention half of transformer_layer (inference/forward.py:92-94), fused:
    ``hidden + mla_attention(rms_norm(hidden, input_layernorm), ...)`` with the
    norm as the layer's first launch and the bf16 residual add in o_proj's
    epilogue."""
    return _mla(_mla_operands(hidden, attn_weights, kv_cache, position, rope_freqs, config,
                              input_gamma=input_layernorm, residual=hidden, max_context=max_context,
                              attn_out=attn_out))


# ------------------------------------------------------------------ FFN / MoE

def _fp8_pair(w: torch.Tensor, s: torch.Tensor, name: str, shape: tuple, dev) -> None:
    _need(w, name, FP8, dev)
    _need(s, name + " scale", torch.float32, dev)
    if tuple(w.shape) != shape:
        raise ValueError(f"{name}: shape {tuple(w.shape)}, expected {shape}")
    if tuple(s.shape) != (math.ceil(shape[0] / 128), math.ceil(shape[1] / 128)):
        raise ValueError(f"{name} scale: shape {tuple(s.shape)} does not match {shape}")


def swiglu(x: torch.Tensor, gate_proj: torch.Tensor, gate_scale: torch.Tensor, up_proj: torch.Tensor,
           up_scale: torch.Tensor, down_proj: torch.Tensor, down_scale: torch.Tensor) -> torch.Tensor:
    """inference/ops.py:186-192: down_proj(silu(gate_proj(x)) * up_proj(x)), every fp8 linear,
    the silu and the product rounded to bf16 as in the reference."""
    _need_cuda(x, "x")
    if x.dtype != BF16:
        raise TypeError(f"swiglu: x must be bfloat16 (got {x.dtype})")
    if gate_proj.dim() != 2:
        raise ValueError("swiglu: gate_proj must be (intermediate, hidden)")
    n, k = gate_proj.shape
    if x.shape[-1] != k:
        raise ValueError(f"swiglu: x has {x.shape[-1]} features, gate_proj expects {k}")
    _fp8_pair(gate_proj, gate_scale, "gate_proj", (n, k), x.device)
    _fp8_pair(up_proj, up_scale, "up_proj", (n, k), x.device)
    _fp8_pair(down_proj, down_scale, "down_proj", (k, n), x.device)
    x2 = x.reshape(-1, k)
    if not x2.is_contiguous():
        x2 = x2.contiguous()
    y = torch.ops.amla.swiglu(x2, gate_proj, gate_scale, up_proj, up_scale, down_proj, down_scale)
    return y.view(*x.shape[:-1], k)


def dense_ffn(hidden: torch.Tensor, mlp_weights: dict) -> torch.Tensor:
    """inference/ops.py:195-199; uint8 weights are MXFP4 pairs (``mxfp4_swiglu``)."""
    fn = mxfp4_swiglu if _is_mxfp4(mlp_weights) else swiglu
    return fn(hidden, *mlp_weights["gate_proj"], *mlp_weights["up_proj"], *mlp_weights["down_proj"])


def expert_ffn(hidden: torch.Tensor, expert_weights: dict) -> torch.Tensor:
    """inference/ops.py:202-206; uint8 weights are MXFP4 pairs (``mxfp4_swiglu``)."""
    fn = mxfp4_swiglu if _is_mxfp4(expert_weights) else swiglu
    return fn(hidden, *expert_weights["gate_proj"], *expert_weights["up_proj"], *expert_weights["down_proj"])


def route(hidden: torch.Tensor, gate_weight: torch.Tensor, config) -> tuple[torch.Tensor, torch.Tensor]:
    """inference/ops.py:209-257: sigmoid scores, group-limited top-k, optional normalisation.

    Returns (indices int64, weights fp32), each (*hidden.shape[:-1], num_experts_per_tok).
    """
    _need_cuda(hidden, "hidden")
    if hidden.dtype != BF16:
        raise TypeError(f"route: hidden must be bfloat16 (got {hidden.dtype})")
    _need(gate_weight, "gate_weight", BF16, hidden.device)
    E, d = gate_weight.shape
    if hidden.shape[-1] != d:
        raise ValueError(f"route: hidden has {hidden.shape[-1]} features, gate_weight expects {d}")
    if E != config.n_routed_experts:
        raise ValueError(f"route: gate_weight has {E} experts, config says {config.n_routed_experts}")
    top_k = config.num_experts_per_tok
    h2 = hidden.reshape(-1, d)
    if not h2.is_contiguous() or h2.data_ptr() % 16:
        h2 = h2.contiguous()
    m = h2.shape[0]
    idx = torch.empty(m, top_k, dtype=torch.int64, device=hidden.device)
    w = torch.empty(m, top_k, dtype=torch.float32, device=hidden.device)
    if m:
        ws = workspace(hidden.device, lib().amla_moe_route_workspace_bytes(m, E))
        check(lib().amla_moe_route(h2.data_ptr(), m, d, gate_weight.data_ptr(), E, config.n_group,
                                   config.topk_group, top_k, int(bool(config.norm_topk_prob)), idx.data_ptr(),
                                   w.data_ptr(), ws.data_ptr(), ws.numel(), _stream_ptr(hidden)), "route")
    shape = (*hidden.shape[:-1], top_k)
    return idx.view(shape), w.view(shape)


_stacked_cache: dict = {}


def _stacked_key(experts: dict, E: int, d: int) -> tuple:
    return tuple((experts[k][0].data_ptr(), experts[k][1].data_ptr(), tuple(experts[k][0].shape),
                  tuple(experts[k][1].shape), experts[k][0].dtype, experts[k][1].dtype, experts[k][0].stride(),
                  experts[k][1].stride(), str(experts[k][0].device)) for k in ("gate_proj", "up_proj", "down_proj")) + (E, d)


def _stacked_expert_tables(experts: dict, E: int, d: int, dev):
    """Pointer tables of stacked expert weights (validated once per set of tensors)."""
    key = _stacked_key(experts, E, d)
    hit = _stacked_cache.get(key)
    if hit is not None:
        return hit[0], hit[1]
    tabs = []
    n_inter = experts["gate_proj"][0].shape[1]
    for key_name, shape in (("gate_proj", (E, n_inter, d)), ("up_proj", (E, n_inter, d)), ("down_proj", (E, d, n_inter))):
        wt, sc = experts[key_name]
        if wt.dtype != FP8 or sc.dtype != torch.float32 or wt.device != dev or sc.device != dev or \
                not (wt.is_contiguous() and sc.is_contiguous()):
            raise ValueError(f"moe_block: stacked {key_name} must be contiguous e4m3fn weights with fp32 scales on {dev}")
        if tuple(wt.shape) != shape or tuple(sc.shape) != (E, math.ceil(shape[1] / 128), math.ceil(shape[2] / 128)):
            raise ValueError(f"moe_block: stacked {key_name} has shape {tuple(wt.shape)} / {tuple(sc.shape)}, "
                             f"expected {shape}")
        for t in (wt, sc):
            step = t[0].numel() * t.element_size()
            tabs.append((ctypes.c_void_p * E)(*[t.data_ptr() + e * step for e in range(E)]))
    if len(_stacked_cache) > 64:
        _stacked_cache.clear()
    # [host tables, n_inter, device table (made on first use)]: one entry per full key
    # (pointers, shapes, strides, dtypes, device, E, d), so a device table is never reused for
    # other tensors that happen to start at the same addresses
    _stacked_cache[key] = [tabs, n_inter, None]
    return tabs, n_inter


def _stacked_device_table(experts: dict, E: int, d: int, dev):
    """Device pointer table [gate_w | gate_s | up_w | up_s | down_w | down_s] x E of stacked
    expert weights (amla_moe_experts_dev), made once per set of tensors and kept with the
    host tables of the same key."""
    tabs, n_inter = _stacked_expert_tables(experts, E, d, dev)
    entry = _stacked_cache[_stacked_key(experts, E, d)]
    if entry[2] is None:
        flat = [int(t[e] or 0) for t in tabs for e in range(E)]
        entry[2] = torch.tensor(flat, dtype=torch.int64).to(dev)
    return entry[2], n_inter


def moe_block(hidden: torch.Tensor, gate_weight: torch.Tensor, shared_weights: dict, experts, config, *,
              layer: int | None = None, routing=None, device_grouping: bool = True) -> torch.Tensor:
    """inference/forward.py:112-153 with the routed experts handed in.

    ``experts`` is one of:

    * a mapping (or a callable) from expert index to its weight dict on the same device;
    * one dict of stacked weights ``{"gate_proj": (w (E, n, k), s (E, ceil(n/128),
      ceil(k/128))), ...}`` (all experts of the layer contiguous: no per-expert host work);
      with uint8 tensors, stacked MXFP4 weights ``(codes (E, n, k/2), exponents (E, n, k/32))``
      (``mxfp4_moe_experts``; the shared expert may be of either form; MXFP4 experts are taken in
      this form only);
    * an ``amla.experts.ExpertStreamer`` (with ``layer=``): the chosen experts are streamed
      from host memory in waves of at most the pool size, each wave computed before the
      next one is copied, so any batch runs on any pool (gpu_transfer.py:50-89 plus
      forward.py:140-151 without the per-token host synchronisation).

    ``routing=(indices, weights)`` reuses a routing already computed (``route``), so a caller
    that routed to prefetch experts does not route twice.  With stacked weights (and
    ``device_grouping``, the default) the slots are grouped by expert on the device
    (amla_moe_experts_dev): no host copy of the indices and no synchronisation, so the whole
    block can be captured in a HIP graph.  Otherwise, as in the reference, the chosen indices
    come to the host once (one synchronisation) for amla_moe_experts.  Either way each chosen
    expert runs once over all tokens that chose it (the reference loops over (token, k)
    pairs), and the combine keeps the reference's order and bf16 roundings: per token,
    k = 0.. accumulates bf16(bf16(w_k) * expert_k(x)) into a bf16 sum, then shared + sum * 2.5.
    """
    from .experts import ExpertStreamer

    streamed = isinstance(experts, ExpertStreamer)
    if streamed and layer is None:
        raise ValueError("moe_block: an ExpertStreamer needs layer=")
    stacked = not streamed and isinstance(experts, dict) and "gate_proj" in experts and \
        experts["gate_proj"][0].dim() == 3
    get = None if stacked or streamed else (experts if callable(experts) else experts.__getitem__)
    if routing is not None:
        idx, w = routing
        on_device = stacked and device_grouping and (config.n_routed_experts <= MOE_DEV_MAX_EXPERTS or _is_mxfp4(experts))
        _check_routing(idx, w, hidden, config.num_experts_per_tok, on_device)
    else:
        idx, w = route(hidden, gate_weight, config)
    shared_out = expert_ffn(hidden, shared_weights)
    d = hidden.shape[-1]
    top_k = config.num_experts_per_tok
    E = config.n_routed_experts
    h2 = hidden.reshape(-1, d)
    if not h2.is_contiguous() or h2.data_ptr() % 16:
        h2 = h2.contiguous()
    m = h2.shape[0]
    out = torch.empty(hidden.shape, dtype=hidden.dtype, device=hidden.device)  # rows in order, whatever hidden's strides
    if m == 0:
        return out
    dev = hidden.device
    if stacked and _is_mxfp4(experts):
        if not device_grouping:
            raise ValueError("moe_block: MXFP4 experts are grouped on the device only")
        if experts["gate_proj"][0].shape[0] != E:
            raise ValueError(f"moe_block: {experts['gate_proj'][0].shape[0]} stacked experts, config says {E}")
        eout = mxfp4_moe_experts(h2, idx.reshape(m, top_k), experts)
        return torch_ops.without_backward(
            lambda: _moe_combine(shared_out, eout, w, m, top_k, d, config, out, hidden), hidden, gate_weight, w, shared_out)
    if stacked and device_grouping and E <= MOE_DEV_MAX_EXPERTS:
        table, n_inter = _stacked_device_table(experts, E, d, dev)
        eout = torch.empty(m, top_k, d, dtype=BF16, device=dev)
        _moe_experts_dev_call(h2, idx.reshape(m, top_k).contiguous(), table, n_inter, E, eout)
        return _moe_combine(shared_out, eout, w, m, top_k, d, config, out, hidden)
    idx_host = idx.reshape(m, top_k).cpu().contiguous()
    if streamed:
        eout = _moe_experts_streamed(h2, idx_host, experts, layer, config)
        return _moe_combine(shared_out, eout, w, m, top_k, d, config, out, hidden)
    if stacked:
        tables, n_inter = _stacked_expert_tables(experts, E, d, dev)
        keep = []
        chosen = []
    else:
        tables = [(ctypes.c_void_p * E)() for _ in range(6)]
        n_inter = None
        keep = []
        chosen = torch.unique(idx_host).tolist()
    for e in chosen:
        ew = get(int(e))
        for j, key in enumerate(("gate_proj", "up_proj", "down_proj")):
            wt, sc = ew[key]
            if wt.dtype == torch.uint8:
                raise ValueError("moe_block: MXFP4 experts are given as one dict of stacked weights")
            if wt.dtype != FP8 or sc.dtype != torch.float32 or wt.device != dev or sc.device != dev or \
                    not (wt.is_contiguous() and sc.is_contiguous()):
                raise ValueError(f"moe_block: expert {e} {key} must be contiguous e4m3fn weights with fp32 "
                                 f"scales on {dev}")
            tables[2 * j][e] = wt.data_ptr()
            tables[2 * j + 1][e] = sc.data_ptr()
            keep.append((wt, sc))
        ni = ew["gate_proj"][0].shape[0]
        if n_inter is None:
            n_inter = ni
        elif ni != n_inter:
            raise ValueError("moe_block: experts of different intermediate sizes")
        if tuple(ew["gate_proj"][0].shape) != (ni, d) or tuple(ew["up_proj"][0].shape) != (ni, d) or \
                tuple(ew["down_proj"][0].shape) != (d, ni):
            raise ValueError(f"moe_block: expert {e} weights do not match hidden size {d}")
    eout = torch.empty(m, top_k, d, dtype=BF16, device=hidden.device)
    _moe_experts_call(h2, idx_host, tables, n_inter, E, eout)
    del keep
    return _moe_combine(shared_out, eout, w, m, top_k, d, config, out, hidden)


def _check_routing(idx, w, hidden, top_k: int, on_device: bool) -> None:
    """A routing as ``route`` gives it; the indices may be on the host where the slots are grouped there."""
    for t, name, dtype in ((idx, "indices", torch.int64), (w, "weights", torch.float32)):
        if not isinstance(t, torch.Tensor) or t.dtype != dtype:
            raise TypeError(f"moe_block: the routing's {name} must be a {dtype} tensor")
        if t.numel() != hidden.shape[:-1].numel() * top_k:
            raise ValueError(f"moe_block: routing {name} {tuple(t.shape)} for hidden {tuple(hidden.shape)}, {top_k} "
                             "experts a token")
    if w.device != hidden.device or idx.device != hidden.device and (on_device or idx.device.type != "cpu"):
        raise ValueError(f"moe_block: the routing is on {idx.device} and {w.device}, hidden on {hidden.device}")


def _moe_experts_call(h2, idx_host, tables, n_inter, E, eout) -> None:
    """amla_moe_experts over the (token, k) slots whose index is >= 0."""
    m, top_k = idx_host.shape
    d = h2.shape[1]
    ws = workspace(h2.device, lib().amla_moe_experts_workspace_bytes(m, d, top_k, n_inter))
    check(lib().amla_moe_experts(h2.data_ptr(), m, d, top_k, idx_host.data_ptr(), n_inter, E,
                                 *[ctypes.cast(t, ctypes.c_void_p) for t in tables], eout.data_ptr(),
                                 ws.data_ptr(), ws.numel(), _stream_ptr(h2)), "moe_experts")


MOE_DEV_MAX_EXPERTS = 512
MOE_DEV_MAX_SLOTS = 65536


def _moe_experts_dev_call(h2, idx_dev, table, n_inter, E, eout) -> None:
    """amla_moe_experts_dev over token chunks of at most 65536 (token, k) slots each."""
    m, top_k = idx_dev.shape
    d = h2.shape[1]
    tpc = max(1, MOE_DEV_MAX_SLOTS // top_k)
    for t0 in range(0, m, tpc):
        mc = min(tpc, m - t0)
        ws = workspace(h2.device, lib().amla_moe_experts_dev_workspace_bytes(mc, d, top_k, n_inter, E))
        check(lib().amla_moe_experts_dev(h2[t0:t0 + mc].data_ptr(), mc, d, top_k, idx_dev[t0:t0 + mc].data_ptr(),
                                         n_inter, E, table.data_ptr(), eout[t0:t0 + mc].data_ptr(), ws.data_ptr(),
                                         ws.numel(), _stream_ptr(h2)), "moe_experts_dev")


def _moe_combine(shared_out, eout, w, m, top_k, d, config, out, hidden):
    sh = shared_out.reshape(m, d).contiguous()
    wc = w.reshape(m, top_k).contiguous()
    check(lib().amla_moe_combine(sh.data_ptr(), eout.data_ptr(), wc.data_ptr(), m, top_k, d,
                                 float(config.routed_scaling_factor), out.data_ptr(), _stream_ptr(hidden)),
          "moe_combine")
    return out


def _moe_experts_streamed(h2, idx_host, streamer, layer, config) -> torch.Tensor:
    """Routed experts streamed in waves of at most ``streamer.slots`` distinct experts: the
    wave's copies (ordered on the device before its compute), then amla_moe_experts over the
    slots of that wave only (the others carry index -1); the next wave's copies reuse slots
    only after this wave's compute (``ExpertStreamer`` releases on the next call)."""
    m, top_k = idx_host.shape
    d = h2.shape[1]
    E = config.n_routed_experts
    chosen = torch.unique(idx_host).tolist()
    eout = torch.empty(m, top_k, d, dtype=BF16, device=h2.device)
    n_inter = None
    for w0 in range(0, len(chosen), streamer.slots):
        wave = chosen[w0:w0 + streamer.slots]
        table = streamer.experts_for(layer, wave)
        tables = [(ctypes.c_void_p * E)() for _ in range(6)]
        for e, ew in table.items():
            for j, key in enumerate(("gate_proj", "up_proj", "down_proj")):
                wt, sc = ew[key]
                tables[2 * j][e] = wt.data_ptr()
                tables[2 * j + 1][e] = sc.data_ptr()
            n_inter = ew["gate_proj"][0].shape[0]
        in_wave = torch.zeros(E, dtype=torch.bool)
        in_wave[wave] = True
        idx_w = torch.where(in_wave[idx_host], idx_host, torch.full_like(idx_host, -1)).contiguous()
        _moe_experts_call(h2, idx_w, tables, n_inter, E, eout)
    streamer.release()
    return eout


# ------------------------------------------------------------------ MXFP4

MX_BLOCK = 32  # values of a row that share an exponent
_MX_IN = {BF16: 0, torch.float16: 1, torch.float32: 2}
_MX_OUT = (BF16, torch.float32)


def _is_mxfp4(weights: dict) -> bool:
    return weights["gate_proj"][0].dtype == torch.uint8


def _mx_pair(codes: torch.Tensor, scales: torch.Tensor, name: str, dev=None) -> torch.Size:
    """Checks an MXFP4 pair (codes (..., k/2), exponents (..., k/32)) and returns the codes' shape."""
    _need(codes, name, torch.uint8, dev)
    _need(scales, name + " scale", torch.uint8, codes.device)
    shape = codes.shape
    if not shape or shape[-1] % (MX_BLOCK // 2):
        raise ValueError(f"{name}: rows of {tuple(shape)} codes are not blocks of {MX_BLOCK} values")
    if scales.shape != shape[:-1] + (shape[-1] * 2 // MX_BLOCK,):
        raise ValueError(f"{name} scale: shape {tuple(scales.shape)} does not match codes {tuple(shape)}")
    return shape


def _mx_weight(codes, scales, name, dims, dev) -> None:
    """Checks a pair against the dimensions it has to have, the last one in values."""
    if _mx_pair(codes, scales, name, dev) != dims[:-1] + (dims[-1] // 2,):
        raise ValueError(f"{name}: codes {tuple(codes.shape)}, expected the values of {tuple(dims)}")


def _mx_rows(x: torch.Tensor, k: int) -> torch.Tensor:
    """x as (rows, k) with unit column stride and row strides of whole 16 bytes."""
    x2 = x if x.dim() == 2 else x.reshape(-1, k)
    if x2.is_contiguous():
        return x2
    if x2.stride(1) != 1 or x2.stride(0) < k or x2.stride(0) % (16 // x.element_size()):
        x2 = x2.contiguous()
    return x2


def _mx_x(x, what: str, k: int, dev) -> tuple:
    """(x or codes as (rows, .), exponents or None, x's shape but for the last) of the activations of
    a product: a bf16 tensor, or the pair that ``mxfp4_quantize`` returned for one."""
    if isinstance(x, (tuple, list)):
        if len(x) != 2:
            raise ValueError(f"{what}: x must be a bfloat16 tensor or a (codes, scales) pair")
        shape = _mx_pair(x[0], x[1], f"{what}: x", dev)
        if shape[-1] * 2 != k:
            raise ValueError(f"{what}: x has {shape[-1] * 2} features, weight expects {k}")
        if len(shape) == 2:
            return x[0], x[1], shape[:-1]
        return x[0].reshape(-1, k // 2), x[1].reshape(-1, k // MX_BLOCK), shape[:-1]
    _need_cuda(x, "x")
    if x.dtype != BF16:
        raise TypeError(f"{what}: x must be bfloat16 (got {x.dtype})")
    if x.device != dev:
        raise ValueError(f"{what}: x is on {x.device}, the weight on {dev}")
    shape = x.shape
    if not shape or shape[-1] != k:
        raise ValueError(f"{what}: x of shape {tuple(shape)}, weight expects {k} features")
    return _mx_rows(x, k), None, shape[:-1]


def _mx_k(k: int, what: str) -> None:
    if k == 0 or k % 128:
        raise ValueError(f"{what}: K = {k} is not a multiple of 128")


def _mx_out_dtype(out_dtype, what: str) -> torch.dtype:
    """The dtype the kernel writes: bf16 rounds in its epilogue, any other is the fp32 result cast."""
    if not isinstance(out_dtype, torch.dtype) or not (out_dtype.is_floating_point or out_dtype.is_complex):
        raise TypeError(f"{what}: out_dtype must be a floating-point dtype (got {out_dtype})")
    return out_dtype if out_dtype == BF16 else torch.float32


def mxfp4_quantize(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """MXFP4 form of the rows of ``x`` (..., k) bf16, fp16 or fp32, k % 32 == 0: codes uint8
    (..., k/2), two e2m1 values a byte, the first in its low half, and exponents uint8 (..., k/32),
    one e8m0 byte per block of 32 values.

    The exponent of a block is floor(log2(max |x|)) - 2 (a block of zeros: byte 0); values are
    rounded to nearest even and saturate at 6 times the scale.  A block that holds an infinity or
    a NaN is a block of NaN (byte 255).  Codes and exponents are whole numbers: no gradient passes
    through a pair, while a backward through a product of the values themselves raises."""
    _need_cuda(x, "x")
    if x.dtype not in _MX_IN:
        raise TypeError(f"mxfp4_quantize: x must be bfloat16, float16 or float32 (got {x.dtype})")
    if x.dim() == 0 or x.shape[-1] % MX_BLOCK or x.shape[-1] == 0:
        raise ValueError(f"mxfp4_quantize: the last dimension of {tuple(x.shape)} is not a multiple of {MX_BLOCK}")
    k = x.shape[-1]
    codes, scales = torch_ops.call("mxfp4_quantize", _mx_rows(x, k))
    if x.dim() == 2:
        return codes, scales
    return codes.view(*x.shape[:-1], k // 2), scales.view(*x.shape[:-1], k // MX_BLOCK)


def mxfp4_quantize_fp8(weight: torch.Tensor, scale_inv: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """``mxfp4_quantize(fp8_block_dequant(weight, scale_inv))`` without the fp32 matrix between: the
    MXFP4 form of a block-FP8 weight (n, k) of the checkpoint, k % 32 == 0."""
    _need(weight, "weight", FP8)
    _need(scale_inv, "scale_inv", torch.float32, weight.device)
    if weight.dim() != 2 or weight.shape[1] % MX_BLOCK or weight.shape[1] == 0:
        raise ValueError(f"mxfp4_quantize_fp8: weight {tuple(weight.shape)} must be (n, k) with k % {MX_BLOCK} == 0")
    n, k = weight.shape
    if scale_inv.shape != (math.ceil(n / 128), math.ceil(k / 128)):
        raise ValueError(f"scale_inv shape {tuple(scale_inv.shape)} does not match weight {n}x{k}")
    return torch_ops.call("mxfp4_quantize_fp8", weight, scale_inv)


def mxfp4_dequantize(codes: torch.Tensor, scales: torch.Tensor, out_dtype: torch.dtype = BF16) -> torch.Tensor:
    """The values of an MXFP4 pair, exact in bf16 and in fp32 (the two out_dtypes)."""
    shape = _mx_pair(codes, scales, "codes")
    if out_dtype not in _MX_OUT:
        raise TypeError(f"mxfp4_dequantize: out_dtype must be bfloat16 or float32 (got {out_dtype})")
    f32 = out_dtype == torch.float32
    if len(shape) == 2:
        return torch_ops.call("mxfp4_dequantize", codes, scales, f32)
    k = shape[-1] * 2
    if k == 0:
        return torch.empty(*shape[:-1], 0, dtype=out_dtype, device=codes.device)
    y = torch_ops.call("mxfp4_dequantize", codes.view(-1, k // 2), scales.view(-1, k // MX_BLOCK), f32)
    return y.view(*shape[:-1], k)


def mxfp4_linear(x, weight: torch.Tensor, scale: torch.Tensor, out_dtype: torch.dtype = BF16) -> torch.Tensor:
    """``( x @ mxfp4_dequantize(weight, scale).T ).to(out_dtype)`` on the 4-bit matrix units, the
    linear (inference/ops.py:15-44) for MXFP4 weights: x rounded to MXFP4 like the weight, exact
    products, fp32 sums.

    ``x`` (..., k): bf16, quantised in the call, or the ``(codes, scales)`` pair of
    ``mxfp4_quantize``, for activations that several linears share.  ``weight`` (n, k/2) and
    ``scale`` (n, k/32) uint8, k % 128 == 0, any n."""
    wdt = _mx_out_dtype(out_dtype, "mxfp4_linear")
    shape = _mx_pair(weight, scale, "weight")
    if len(shape) != 2:
        raise ValueError("mxfp4_linear: weight must be (n, k/2)")
    n, k = shape[0], shape[1] * 2
    _mx_k(k, "mxfp4_linear")
    x2, xs, lead = _mx_x(x, "mxfp4_linear", k, weight.device)
    y = torch_ops.call("mxfp4_linear", x2, xs, weight, scale, wdt == torch.float32)
    if len(lead) != 1:
        y = y.view(*lead, n)
    return y if wdt == out_dtype else y.to(out_dtype)


def mxfp4_grouped_linear(x, weight: torch.Tensor, scale: torch.Tensor, offsets: torch.Tensor,
                         out_dtype: torch.dtype = BF16, out: torch.Tensor | None = None) -> torch.Tensor:
    """``mxfp4_linear`` by expert over rows sorted by expert: rows offsets[e] .. offsets[e + 1] - 1 of
    ``x`` (m, k) times expert e of ``weight`` (E, n, k/2), ``scale`` (E, n, k/32), E <= 1024.

    ``offsets`` (E + 1,) int32 on the device, ascending; groups may be empty.  They are not checked
    on the host: one above m counts as m, one below its predecessor as that.  Rows of no group are
    zeros in a new output; with ``out`` ((m, n), bf16 or fp32 as out_dtype says, unit column
    stride) they stay as they were.  ``x``: as for ``mxfp4_linear``.  With ``out``, an x or out that
    requires a gradient is refused while grad mode is on."""
    wdt = _mx_out_dtype(out_dtype, "mxfp4_grouped_linear")
    shape = _mx_pair(weight, scale, "weight")
    if len(shape) != 3:
        raise ValueError("mxfp4_grouped_linear: weight must be (experts, n, k/2)")
    E, n, k = shape[0], shape[1], shape[2] * 2
    _mx_k(k, "mxfp4_grouped_linear")
    dev = weight.device
    if not 0 < E <= 1024 or n == 0:
        raise ValueError(f"mxfp4_grouped_linear: {E} experts of {n} outputs (1 to 1024 experts)")
    _need(offsets, "offsets", torch.int32, dev)
    if tuple(offsets.shape) != (E + 1,):
        raise ValueError(f"mxfp4_grouped_linear: offsets of shape {tuple(offsets.shape)}, expected ({E + 1},)")
    x2, xs, lead = _mx_x(x, "mxfp4_grouped_linear", k, dev)
    if len(lead) != 1:
        raise ValueError("mxfp4_grouped_linear: x must be (m, k)")
    if out is None:
        y = torch_ops.call("mxfp4_grouped_linear", x2, xs, weight, scale, offsets, wdt == torch.float32)
        return y if wdt == out_dtype else y.to(out_dtype)
    _need_cuda(out, "out")
    if out.dtype != out_dtype or out_dtype not in _MX_OUT:
        raise TypeError(f"mxfp4_grouped_linear: out must be bfloat16 or float32 as out_dtype (got {out.dtype})")
    if out.device != dev or tuple(out.shape) != (x2.shape[0], n) or (n > 1 and out.stride(1) != 1) or \
            (out.shape[0] > 1 and out.stride(0) < n):
        raise ValueError(f"mxfp4_grouped_linear: out must be ({x2.shape[0]}, {n}) on {dev} with rows of unit stride")
    torch_ops.call("mxfp4_grouped_linear_out", x2, xs, weight, scale, offsets, out)
    return out


def mxfp4_swiglu(x: torch.Tensor, gate_proj: torch.Tensor, gate_scale: torch.Tensor, up_proj: torch.Tensor,
                 up_scale: torch.Tensor, down_proj: torch.Tensor, down_scale: torch.Tensor) -> torch.Tensor:
    """``swiglu`` (inference/ops.py:186-192) with MXFP4 weights: silu(gate(x)) * up(x) in fp32,
    rounded to MXFP4 only, times down_proj.  ``x`` (..., k) bf16; gate_proj, up_proj (n, k/2), their
    exponents (n, k/32), down_proj (k, n/2), (k, n/32); k and n multiples of 128."""
    shape = _mx_pair(gate_proj, gate_scale, "gate_proj")
    if len(shape) != 2:
        raise ValueError("mxfp4_swiglu: gate_proj must be (intermediate, hidden/2)")
    n, k = shape[0], shape[1] * 2
    _mx_k(k, "mxfp4_swiglu")
    _mx_k(n, "mxfp4_swiglu")
    dev = gate_proj.device
    _mx_weight(up_proj, up_scale, "up_proj", (n, k), dev)
    _mx_weight(down_proj, down_scale, "down_proj", (k, n), dev)
    if isinstance(x, (tuple, list)):
        raise TypeError("mxfp4_swiglu: x must be a bfloat16 tensor")
    x2, _, lead = _mx_x(x, "mxfp4_swiglu", k, dev)
    y = torch_ops.call("mxfp4_swiglu", x2, gate_proj, gate_scale, up_proj, up_scale, down_proj, down_scale)
    return y if len(lead) == 1 else y.view(*lead, k)


def mxfp4_moe_experts(hidden: torch.Tensor, indices: torch.Tensor, experts: dict) -> torch.Tensor:
    """Routed experts (the loop of inference/forward.py:139-151) with stacked MXFP4 weights: row
    (t, j) of the result (..., top_k, d) bf16 is ``mxfp4_swiglu(hidden[t], expert indices[t, j])``.

    ``hidden`` (..., d) bf16, ``indices`` (..., top_k) int64 on the device (``route``), ``experts``
    ``{"gate_proj": (codes (E, n, d/2), exponents (E, n, d/32)), "up_proj": ..., "down_proj":
    (codes (E, d, n/2), exponents (E, d, n/32))}``, E <= 512, d and n multiples of 128.  The slots
    are grouped by expert on the device: no host copy, no synchronisation.  A slot whose index is
    no expert's gives a row of zeros."""
    _need_cuda(hidden, "hidden")
    if hidden.dtype != BF16:
        raise TypeError(f"mxfp4_moe_experts: hidden must be bfloat16 (got {hidden.dtype})")
    shape = _mx_pair(*experts["gate_proj"], "gate_proj", hidden.device)
    if len(shape) != 3:
        raise ValueError("mxfp4_moe_experts: gate_proj must be (experts, intermediate, hidden/2)")
    E, n, d = shape[0], shape[1], shape[2] * 2
    _mx_k(d, "mxfp4_moe_experts")
    _mx_k(n, "mxfp4_moe_experts")
    if not 0 < E <= MOE_DEV_MAX_EXPERTS:
        raise ValueError(f"mxfp4_moe_experts: {E} experts (1 to {MOE_DEV_MAX_EXPERTS})")
    _mx_weight(*experts["up_proj"], "up_proj", (E, n, d), hidden.device)
    _mx_weight(*experts["down_proj"], "down_proj", (E, d, n), hidden.device)
    if hidden.dim() == 0 or hidden.shape[-1] != d:
        raise ValueError(f"mxfp4_moe_experts: hidden of shape {tuple(hidden.shape)}, the experts expect {d} features")
    if not isinstance(indices, torch.Tensor) or indices.dtype != torch.int64 or indices.device != hidden.device:
        raise ValueError("mxfp4_moe_experts: indices must be an int64 tensor on the hidden states' device")
    if indices.dim() == 0 or indices.shape[:-1] != hidden.shape[:-1] or not 0 < indices.shape[-1] <= 64:
        raise ValueError(f"mxfp4_moe_experts: indices {tuple(indices.shape)} do not match hidden {tuple(hidden.shape)} "
                         "with 1 to 64 experts a token")
    top_k = indices.shape[-1]
    h2 = _mx_rows(hidden, d)
    idx = indices if indices.dim() == 2 else indices.reshape(-1, top_k)
    out = torch_ops.call("mxfp4_moe_experts", h2, idx.contiguous(), *experts["gate_proj"], *experts["up_proj"],
                         *experts["down_proj"])
    return out if hidden.dim() == 2 else out.view(*hidden.shape[:-1], top_k, d)


# ------------------------------------------------------------------ paged latent cache

def latent_cache(pages: int, page_size: int, config, device, dtype: torch.dtype = FP8) -> tuple:
    """An empty pool of rows for ``latent_cache_write``: ``(latent (pages, page_size, kv_lora_rank),
    k_pe (pages, page_size, qk_rope_head_dim) bf16)`` with bf16 latents, and for e4m3 latents (``dtype``
    float8_e4m3fn, the default) also ``scales (pages, page_size)`` uint8, the exponent byte of each row:
    value = code * 2^(byte - 127).  641 bytes a row instead of 1152.  page_size: a power of two."""
    if dtype not in (FP8, BF16):
        raise TypeError(f"latent_cache: dtype must be float8_e4m3fn or bfloat16 (got {dtype})")
    if config.kv_lora_rank != LATENT or config.qk_rope_head_dim != LATENT_ROPE:
        raise ValueError(f"latent_cache: rows are {LATENT} + {LATENT_ROPE} values (the configuration's: {config.kv_lora_rank} + "
                         f"{config.qk_rope_head_dim})")
    if pages <= 0 or page_size <= 0 or page_size > 65536 or page_size & (page_size - 1):
        raise ValueError(f"latent_cache: {pages} pages of {page_size} rows (a power of two up to 65536)")
    latent = torch.zeros(pages, page_size, config.kv_lora_rank, dtype=torch.uint8 if dtype == FP8 else BF16, device=device)
    k_pe = torch.zeros(pages, page_size, config.qk_rope_head_dim, dtype=BF16, device=device)
    if dtype == BF16:
        return latent, k_pe
    return latent.view(FP8), k_pe, torch.full((pages, page_size), 127, dtype=torch.uint8, device=device)


LATENT, LATENT_ROPE = 512, 64  # values of a row


def _latent_parts(cache, what: str) -> tuple:
    """(latent, k_pe, scales or None) of a checked cache."""
    if not isinstance(cache, (tuple, list)) or len(cache) not in (2, 3):
        raise ValueError(f"{what}: the cache is (latent, k_pe) or (latent, k_pe, scales)")
    latent, k_pe = cache[0], cache[1]
    scales = cache[2] if len(cache) == 3 else None
    _need(latent, "latent", BF16 if scales is None else FP8)
    dev, shape = latent.device, latent.shape
    _need(k_pe, "k_pe", BF16, dev)
    if len(shape) != 3 or shape[2] != LATENT or k_pe.shape != (shape[0], shape[1], LATENT_ROPE) or not latent.numel():
        raise ValueError(f"{what}: cache of {tuple(shape)} and {tuple(k_pe.shape)}, expected (pages, page_size, "
                         f"{LATENT}) and (pages, page_size, {LATENT_ROPE})")
    if scales is not None:
        _need(scales, "scales", torch.uint8, dev)
        if scales.shape != shape[:2]:
            raise ValueError(f"{what}: scales {tuple(scales.shape)} of a cache of {tuple(shape)}")
    return latent, k_pe, scales


def _need_i32(t, name: str, what: str, dev, shape: tuple) -> None:
    if not isinstance(t, torch.Tensor) or t.dtype != torch.int32 or t.device != dev or t.shape != shape or \
            not t.is_contiguous():
        got = f"{t.dtype} {tuple(t.shape)} on {t.device}" if isinstance(t, torch.Tensor) else type(t).__name__
        raise ValueError(f"{what}: {name} must be a contiguous int32 tensor {shape} on {dev} (got {got})")


def _need_table(t, what: str, dev) -> int:
    """Checks a block table (sequences, pages of a sequence) and returns its sequences."""
    if not isinstance(t, torch.Tensor) or t.dtype != torch.int32 or t.device != dev or t.dim() != 2 or \
            (t.stride(1) != 1 and t.shape[1] > 1) or (t.stride(0) < t.shape[1] and t.shape[0] > 1):
        raise ValueError(f"{what}: block_table must be an int32 tensor (sequences, pages) with rows of unit stride on {dev}")
    return t.shape[0]


def latent_cache_write(kv: torch.Tensor, kv_a_layernorm: torch.Tensor, rope_freqs: torch.Tensor, cache: tuple,
                       block_table: torch.Tensor, position, *, offsets: torch.Tensor | None = None,
                       eps: float = 1e-6) -> None:
    """Stores new rows of the cache: the norm of inference/ops.py:148 and the rotation of :158-159,
    done once as a row is written, where the reference stores it raw (:140-141) and repeats them.

    ``kv`` bf16, the output of kv_a_proj_with_mqa: (B, S, 576), S new rows of every sequence, or with
    ``offsets`` ((B + 1,) int32 on the device, ascending) the packed rows (T, 576), offsets[b] ..
    offsets[b + 1] - 1 of sequence b.  ``position``: as for ``mla_attention``, the first new row of each
    sequence.  ``rope_freqs``: ``precompute_rope_freqs``.  ``cache``: ``latent_cache``; row i of
    sequence b is row i % page_size of page ``block_table[b, i // page_size]`` ((B, n) int32 on the
    device).  All in fp32 with one rounding, to bf16 or to e4m3 with the smallest power of two that
    keeps the row within 448 times it (2^-32 .. 2^32); an e4m3 row with an infinity or a NaN becomes one
    of NaN (bf16: what the formula gives, zeros beside a NaN for an infinity).  Rows of no sequence, of a page outside the pool or past the rope table are not written;
    nothing of that is checked on the host.  Two rows of a call must not share a place."""
    what = "latent_cache_write"
    latent, k_pe, scales = _latent_parts(cache, what)
    dev = latent.device
    _need_cuda(kv, "kv")
    if kv.dtype != BF16 or kv.device != dev:
        raise TypeError(f"{what}: kv must be bfloat16 on {dev} (got {kv.dtype} on {kv.device})")
    if kv.dim() != (3 if offsets is None else 2) or kv.shape[-1] != LATENT + LATENT_ROPE:
        raise ValueError(f"{what}: kv of shape {tuple(kv.shape)}, expected (B, S, 576), or (T, 576) with offsets")
    _need(kv_a_layernorm, "kv_a_layernorm", BF16, dev)
    if kv_a_layernorm.shape != (LATENT,):
        raise ValueError(f"{what}: kv_a_layernorm of shape {tuple(kv_a_layernorm.shape)}")
    if rope_freqs.dtype != torch.complex64 or rope_freqs.device != dev or not rope_freqs.is_contiguous() or \
            rope_freqs.dim() != 2 or rope_freqs.shape[1] != LATENT_ROPE // 2:
        raise TypeError(f"{what}: rope_freqs must be a contiguous complex64 tensor (positions, {LATENT_ROPE // 2}) on {dev}")
    B = _need_table(block_table, what, dev)
    if offsets is None:
        if kv.shape[0] != B:
            raise ValueError(f"{what}: kv of {kv.shape[0]} sequences, block_table of {B}")
        kv = kv.reshape(-1, LATENT + LATENT_ROPE)
    else:
        _need_i32(offsets, "offsets", what, dev, (B + 1,))
    pos = _positions(position, B, 1, dev, None)[0] if B else torch.empty(0, dtype=torch.int32, device=dev)
    _need_i32(pos, "position", what, dev, (B,))
    rope_freqs = rope_freqs.resolve_conj()  # (conj() leaves the values as they are and sets a flag)
    torch_ops.call_latent("latent_cache_write", kv, kv_a_layernorm, rope_freqs, latent, k_pe, scales, block_table, pos,
                          offsets, float(eps))


def latent_cache_read(cache: tuple, block_table: torch.Tensor, offsets: torch.Tensor, rows: int, *,
                      position: torch.Tensor | None = None, out: tuple | None = None) -> tuple:
    """Rows of the cache as (latent (rows, 512), k_pe (rows, 64)) bf16, packed: rows offsets[b] ..
    offsets[b + 1] - 1 ((B + 1,) int32 on the device, ascending) are rows position[b] .. of sequence b
    ((B,) int32 on the device; None: from row 0).  The values are the cache's own, exactly.  What kv_b
    takes for a prompt that continues a cached one (inference/ops.py:144-151).

    Rows of no sequence or of no page are zeros, and with ``out`` ((latent, k_pe) to write to) stay as
    they were."""
    what = "latent_cache_read"
    latent, k_pe, scales = _latent_parts(cache, what)
    dev = latent.device
    B = _need_table(block_table, what, dev)
    _need_i32(offsets, "offsets", what, dev, (B + 1,))
    if position is not None:
        _need_i32(position, "position", what, dev, (B,))
    rows = int(rows)
    if rows < 0:
        raise ValueError(f"{what}: {rows} rows")
    if out is None:
        return torch_ops.call_latent("latent_cache_read", latent, k_pe, scales, block_table, offsets, position, rows)
    for t, n in zip(out, (LATENT, LATENT_ROPE), strict=True):
        _need(t, "out", BF16, dev)
        if t.shape != (rows, n):
            raise ValueError(f"{what}: out of shape {tuple(t.shape)}, expected ({rows}, {n})")
    torch_ops.call_latent("latent_cache_read_out", latent, k_pe, scales, block_table, offsets, position, *out)
    return tuple(out)


def latent_attention(q: torch.Tensor, cache: tuple, block_table: torch.Tensor, lengths: torch.Tensor, scale: float, *,
                     return_lse: bool = False):
    """Attention of the newest tokens over the paged cache, in latent space: the scores and the weighted
    sum of ``mla_attention``'s decode (inference/ops.py:162-182, with kv_b absorbed into the query).

    ``q`` (B, S, H, 576) bf16: per head the query times W_UK (512) and the rotated rope query (64), any H,
    any strides.  ``lengths`` (B,) int32 on the device: the rows of each sequence, the S new ones
    included; token s sees rows 0 .. lengths[b] - S + s.  ``scale``: ``softmax_scale(config)``.  Returns
    (B, S, H, 512) bf16, the softmax-weighted sums of latents (times W_UV: the heads' outputs), and with
    ``return_lse`` the log of the sum of exp(scores), (B, S, H) fp32.  A token that sees no row gives
    zeros and -inf; pages outside the pool hold no rows.  A length past the table counts as its end.  A finite
    score below -2^126 log 2 counts as not seen.  The table's width, not the lengths, chooses the kernel (the
    host does not know them): a much wider one costs short sequences up to half as much time again, and the
    last bits of the result go with it."""
    what = "latent_attention"
    latent, k_pe, scales = _latent_parts(cache, what)
    dev = latent.device
    _need_cuda(q, "q")
    if q.dtype != BF16 or q.device != dev:
        raise TypeError(f"{what}: q must be bfloat16 on {dev} (got {q.dtype} on {q.device})")
    B = _need_table(block_table, what, dev)
    if q.dim() != 4 or q.shape[0] != B or q.shape[3] != LATENT + LATENT_ROPE:
        raise ValueError(f"{what}: q of shape {tuple(q.shape)}, expected ({B}, S, H, {LATENT + LATENT_ROPE})")
    _need_i32(lengths, "lengths", what, dev, (B,))
    o, lse = torch_ops.call_latent("latent_attention", q, latent, k_pe, scales, block_table, lengths, float(scale),
                                   bool(return_lse))
    return (o, lse) if return_lse else o


def packed_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, offsets: torch.Tensor, scale: float, *,
                     k_offsets: torch.Tensor | None = None, k_pe: torch.Tensor | None = None, causal: bool = True,
                     return_lse: bool = False):
    """Attention of whole prompts packed one after another (inference/ops.py:162-182 for sequences of
    different lengths): rows offsets[b] .. offsets[b + 1] - 1 of ``q`` over rows k_offsets[b] .. of ``k``
    and ``v`` (int32 (B + 1,) on the device, ascending; ``k_offsets`` None: the same).

    ``q`` (T, H, d), ``k`` (N, G, d), ``v`` (N, G, 128) bf16, H a multiple of G, each H / G heads sharing
    keys and values, d 128 or 192; or with ``k_pe`` (N, 64), a rope key shared by all heads, d = 192 and
    ``k`` (N, G, 128): kv_b's output (N, G, 256) goes in as two views.  Queries are the last tokens of
    their sequence: with ``causal`` row i of n sees key j of m where j <= i + m - n.  Returns (T, H, 128)
    bf16, with ``return_lse`` also the log of the sum of exp(scores) (T, H) fp32.  A row that sees no
    key gives zeros and -inf; scores are taken up to 2^28 in magnitude.  Offsets are not checked on the host; they are clamped to the rows, and
    the output of rows in no sequence is left unset."""
    what = "packed_attention"
    _need_cuda(q, "q")
    dev = q.device
    for t, name in ((q, "q"), (k, "k"), (v, "v")) + (((k_pe, "k_pe"),) if k_pe is not None else ()):
        _need_cuda(t, name)
        if t.dtype != BF16 or t.device != dev:
            raise TypeError(f"{what}: {name} must be bfloat16 on {dev} (got {t.dtype} on {t.device})")
    if q.dim() != 3 or k.dim() != 3 or v.dim() != 3:
        raise ValueError(f"{what}: q, k and v must be (rows, heads, values)")
    dk = k.shape[2] + (0 if k_pe is None else LATENT_ROPE)
    if dk not in (128, 192) or q.shape[2] != dk or v.shape[2] != 128:
        raise ValueError(f"{what}: heads of {q.shape[2]} query, {dk} key and {v.shape[2]} value columns (128 or 192 of the "
                         "first two, 128 of the last)")
    if v.shape[:2] != k.shape[:2] or (k_pe is not None and k_pe.shape != (k.shape[0], LATENT_ROPE)):
        raise ValueError(f"{what}: k {tuple(k.shape)}, v {tuple(v.shape)}, k_pe "
                         f"{None if k_pe is None else tuple(k_pe.shape)} do not match")
    if not k.shape[1] or q.shape[1] % k.shape[1]:
        raise ValueError(f"{what}: {q.shape[1]} heads over {k.shape[1]} key heads")
    if not 0.0 < scale < math.inf:
        raise ValueError(f"{what}: scale must be positive (got {scale})")
    if not isinstance(offsets, torch.Tensor) or offsets.dim() != 1 or not offsets.numel():
        raise ValueError(f"{what}: offsets must be an int32 tensor (sequences + 1,)")
    _need_i32(offsets, "offsets", what, dev, offsets.shape)
    if k_offsets is not None:
        _need_i32(k_offsets, "k_offsets", what, dev, offsets.shape)
    o, lse = torch_ops.call_latent("packed_attention", q, k, v, k_pe, offsets, k_offsets, float(scale), bool(causal),
                                   bool(return_lse))
    return (o, lse) if return_lse else o


# ------------------------------------------------------------------ output head

def lm_head_logits(hidden: torch.Tensor, lm_head_w: torch.Tensor) -> torch.Tensor:
    """inference/forward.py:72: ``hidden.float() @ lm_head_w.float().T`` without the fp32 copy of
    the weight: exact bf16 products summed in fp32.  Returns fp32 (*hidden.shape[:-1], vocab)."""
    _need_cuda(hidden, "hidden")
    if hidden.dtype != BF16:
        raise TypeError(f"lm_head_logits: hidden must be bfloat16 (got {hidden.dtype})")
    _need(lm_head_w, "lm_head_w", BF16, hidden.device)
    n, k = lm_head_w.shape
    if hidden.shape[-1] != k:
        raise ValueError(f"lm_head_logits: hidden has {hidden.shape[-1]} features, lm_head_w expects {k}")
    h2 = hidden.reshape(-1, k)
    if not h2.is_contiguous() or h2.data_ptr() % 16:
        h2 = h2.contiguous()
    m = h2.shape[0]
    out = torch.empty(m, n, dtype=torch.float32, device=hidden.device)
    if m:
        check(lib().amla_bf16_logits(h2.data_ptr(), m, k, lm_head_w.data_ptr(), n, out.data_ptr(), n,
                                     _stream_ptr(hidden)), "lm_head_logits")
    return out.view(*hidden.shape[:-1], n)


def final_logits(hidden: torch.Tensor, final_norm: torch.Tensor, lm_head_w: torch.Tensor, config) -> torch.Tensor:
    """inference/forward.py:67-72: final RMSNorm, then the lm_head projection in fp32."""
    return lm_head_logits(rms_norm(hidden, final_norm, config.rms_norm_eps), lm_head_w)


def sample(logits: torch.Tensor, temperature: float, top_p: float, *, seed: int | None = None) -> torch.Tensor:
    """inference/engine.py:166-186: (B, vocab) fp32 logits -> (B,) int64 token ids.

    temperature 0 is the argmax (ties to the lower index).  Otherwise nucleus
    sampling with the reference's rule (softmax(logits / T), drop a token when the
    mass strictly before it exceeds top_p, renormalise, draw one); the draw uses
    a counter-based generator keyed by ``seed`` (default: drawn from torch's CPU
    generator), so it follows the same distribution as torch.multinomial but not
    its random stream.  Each row is cut into chunks (rows x chunks workgroups); the
    result equals the one-workgroup-per-row kernels' (amla_argmax, amla_sample_top_p).
    """
    _need_cuda(logits, "logits")
    if logits.dtype != torch.float32 or logits.dim() != 2:
        raise TypeError("sample: logits must be a (B, vocab) float32 tensor")
    lg = logits if logits.stride(-1) == 1 else logits.contiguous()
    B, n = lg.shape
    out = torch.empty(B, dtype=torch.int64, device=logits.device)
    if B == 0:
        return out
    if temperature != 0 and seed is None:
        seed = int(torch.randint(0, 2 ** 62, (1,)).item())
    ws_bytes = lib().amla_sample_workspace_bytes(B, n)
    ws = workspace(logits.device, ws_bytes)
    check(lib().amla_sample(lg.data_ptr(), B, n, lg.stride(0), float(temperature), float(top_p),
                            int(seed or 0) & (2 ** 64 - 1), out.data_ptr(), ws.data_ptr(), ws_bytes,
                            _stream_ptr(logits)), "sample")
    return out
