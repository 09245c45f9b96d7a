"""The MXFP4 operators as measured cases: quantisation, linears, grouped products and experts.

MXFP4 holds a matrix row as blocks of 32 values along K: e2m1 codes (sign, 0 .. 6 in eight
steps; value 2i of a row in the low half of byte i) and one e8m0 exponent byte per block.
A serving loop for DeepSeek-R1 that keeps its weights in this form quantises a checkpoint once
(from bf16 or from the block-FP8 weights), multiplies activations quantised on the fly by
them in the linears and the dense FFN, and runs the routed experts of a MoE layer on them.
Sizes are the R1 configuration (``amla.config.DeepSeekConfig``) and generic ones around it.

``listed()`` gives the fixed cases, ``draw(rng)`` further ones of the same ranges, ``prepare``
what the program holds before the call, ``run`` one call (``own``: the package's functions, else
the plain form in fp32), ``work`` the bytes and operations the call cannot do without and
``exact`` the result in 64 bits from the definition.
"""
from __future__ import annotations

import math
import os
import sys

import torch

own = False

DEV = "cuda"
BF16, F16, F32, F64, FP8 = torch.bfloat16, torch.float16, torch.float32, torch.float64, torch.float8_e4m3fn
DTYPES = {"bf16": BF16, "fp16": F16, "fp32": F32}
BLOCK = 32

# (n, k) of the R1 linears, and generic ones: a short odd output, the smallest K, a narrow square
LINEARS = {
    "q_a": (1536, 7168), "q_b": (24576, 1536), "kv_a": (576, 7168), "kv_b": (32768, 512), "o_proj": (7168, 16384),
    "gate": (18432, 7168), "down": (7168, 18432), "expert_gate": (2048, 7168), "expert_down": (7168, 2048),
    "odd": (1001, 1152), "small": (256, 128), "square": (4096, 4096),
}
D, EI, FI, TOPK = 7168, 2048, 18432, 8
MAX_M = 4096


def _ops():
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    path = os.path.join(root, "deepseek-on-one-gpu_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    from amla import ops
    return ops


# ------------------------------------------------------------------ the cases

def _quant(rows, k, dtype):
    return {"kind": "quantize", "rows": rows, "k": k, "dtype": dtype}


def _linear(m, shape, out="bf16", held=False):
    n, k = LINEARS[shape]
    return {"kind": "linear", "m": m, "n": n, "k": k, "out": out, "held": held}


def _grouped(m, n, k, experts, out="bf16"):
    return {"kind": "grouped", "m": m, "n": n, "k": k, "experts": experts, "out": out}


def _ffn(tokens, d=D, inter=FI):
    return {"kind": "ffn", "tokens": tokens, "d": d, "inter": inter}


def _experts(tokens, experts, d=D, inter=EI, top_k=TOPK):
    return {"kind": "experts", "tokens": tokens, "experts": experts, "d": d, "inter": inter, "top_k": top_k}


def listed():
    return [
        # hidden states of a prompt quantised ahead of the linears that share them
        {"name": "quantize_1999_bf16", **_quant(1999, D, "bf16")},
        # loading: one block-FP8 o_proj of a checkpoint turned into MXFP4
        {"name": "quantize_o_proj_fp8", **_quant(7168, 16384, "fp8")},
        # one user's decode step: the o_proj of one token, where the weights' bytes and latency count
        {"name": "linear_1_o_proj", **_linear(1, "o_proj")},
        # forty sequences decoding together, q_b
        {"name": "linear_40_q_b", **_linear(40, "q_b")},
        # a prompt of some pages through q_a, fp32 out
        {"name": "linear_777_q_a_f32", **_linear(777, "q_a", "fp32")},
        # a 4k prompt through o_proj
        {"name": "linear_4096_o_proj", **_linear(4096, "o_proj")},
        # one product of an expert-parallel rank (32 of 256 experts): decode of many sequences, a prompt
        {"name": "grouped_150_gate", **_grouped(150, EI, D, 32)},
        {"name": "grouped_8111_down", **_grouped(8111, D, EI, 32)},
        # FFN of the three dense layers: a decode step of eight, and a prompt
        {"name": "ffn_8", **_ffn(8)},
        {"name": "ffn_1000", **_ffn(1000)},
        # routed experts of the 58 MoE layers, all resident: a decode step of eight, and a prompt
        {"name": "experts_8", **_experts(8, 256)},
        {"name": "experts_2000", **_experts(2000, 256)},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    what = rng.choice(["quantize", "linear", "linear", "grouped", "ffn", "experts"])
    if what == "quantize":
        dtype = rng.choice(["bf16", "fp16", "fp32", "fp8"])
        k = 128 * _log_int(rng, 1, 144) if dtype == "fp8" else 32 * _log_int(rng, 1, 576)
        return _quant(_log_int(rng, 1, 7168), k, dtype)
    if what == "linear":
        return _linear(_log_int(rng, 1, 4000), rng.choice([s for s in LINEARS if s not in ("gate", "down")]),
                       rng.choice(["bf16", "bf16", "fp32"]), rng.random() < 0.3)
    if what == "grouped":
        n, k = rng.choice([(EI, D), (D, EI), (1536, 2048), (2048, 1536), (520, 640)])
        return _grouped(_log_int(rng, 1, 8192), n, k, rng.choice([1, 5, 8, 32, 64]), rng.choice(["bf16", "bf16", "fp32"]))
    if what == "ffn":
        d, inter = rng.choice([(D, FI), (D, EI), (2048, 1536), (1152, 640)])
        return _ffn(_log_int(rng, 1, 1000), d, inter)
    d, inter, experts = rng.choice([(D, EI, 256), (D, EI, 32), (2048, 1536, 64), (1152, 640, 8)])
    return _experts(_log_int(rng, 1, 2000), experts, d, inter, rng.choice([1, 2, 6, 8]))


# ------------------------------------------------------------------ inputs

class _Draw:
    """Seeded values on the GPU."""

    def __init__(self, seed):
        self.g = torch.Generator(device=DEV)
        self.g.manual_seed(seed)

    def randn(self, *shape, std=1.0):
        return torch.randn(shape, generator=self.g, device=DEV, dtype=F32).mul_(std)

    def activations(self, m, k):
        """Hidden states: normal, each row with a scale of its own, a few large channels."""
        x = self.randn(m, k) * torch.exp(0.3 * self.randn(m, 1))
        x[:, :: max(1, k // 6)] *= 12.0
        return x.to(BF16)

    def weight(self, n, k):
        """A weight matrix as it lies in memory: (codes, exponents) of normal values, per-row scales."""
        return _plain_quantize(self.randn(n, k, std=0.02) * torch.exp(0.2 * self.randn(n, 1)))

    def stacked(self, experts, n, k):
        codes = torch.empty(experts, n, k // 2, dtype=torch.uint8, device=DEV)
        scales = torch.empty(experts, n, k // BLOCK, dtype=torch.uint8, device=DEV)
        for e in range(experts):
            codes[e], scales[e] = self.weight(n, k)
        return codes, scales


def _group_offsets(case, g):
    """Ragged group sizes (some of them empty) that add up to the rows of the case."""
    share = torch.rand(case["experts"], generator=g) ** 2
    share[torch.rand(case["experts"], generator=g) < 0.1] = 0
    if share.sum() == 0:
        share[0] = 1
    ends = torch.floor(torch.cumsum(share, 0) / share.sum() * case["m"] + 0.5).long()
    ends[-1] = case["m"]
    return [0] + ends.clamp(max=case["m"]).tolist()


def prepare(case, seed):
    d = _Draw(seed)
    host = torch.Generator()
    host.manual_seed(seed)
    st = {"case": case}
    kind = case["kind"]
    if kind == "quantize":
        rows, k = case["rows"], case["k"]
        if case["dtype"] == "fp8":
            nb, kb = -(-rows // 128), k // 128
            st["x"] = (d.randn(rows, k, std=60.0)).clamp_(-448, 448).to(FP8)
            st["scale_inv"] = torch.rand(nb, kb, generator=d.g, device=DEV) * 4e-4 + 1e-4
        else:
            x = d.activations(rows, k).float() * 0.7
            x[rows // 2, : k // 2] = 0.0  # a padded stretch: blocks of zeros
            st["x"] = x.to(DTYPES[case["dtype"]])
    elif kind == "linear":
        x = d.activations(case["m"], case["k"])
        st["x"] = _plain_quantize(x.float()) if case["held"] else x
        st["w"] = d.weight(case["n"], case["k"])
    elif kind == "grouped":
        st["x"] = d.activations(case["m"], case["k"])
        st["w"] = d.stacked(case["experts"], case["n"], case["k"])
        st["groups"] = _group_offsets(case, host)
        st["offsets"] = torch.tensor(st["groups"], dtype=torch.int32, device=DEV)
    elif kind == "ffn":
        st["x"] = d.activations(case["tokens"], case["d"])
        st["w"] = {"gate_proj": d.weight(case["inter"], case["d"]), "up_proj": d.weight(case["inter"], case["d"]),
                   "down_proj": d.weight(case["d"], case["inter"])}
    else:
        E, m = case["experts"], case["tokens"]
        st["x"] = d.activations(m, case["d"])
        # routers prefer some experts: scores with a bias per expert, the top_k of them per token
        score = torch.randn(m, E, generator=host) + 0.5 * torch.randn(1, E, generator=host)
        st["host_idx"] = torch.topk(score, case["top_k"], dim=1).indices
        st["idx"] = st["host_idx"].to(DEV)
        st["w"] = {"gate_proj": d.stacked(E, case["inter"], case["d"]), "up_proj": d.stacked(E, case["inter"], case["d"]),
                   "down_proj": d.stacked(E, case["d"], case["inter"])}
    return st


# ------------------------------------------------------------------ plain forms

def _plain_quantize(x):
    """fp32 (rows, k) -> (codes, exponents): the exponent floor(log2(max |block|)) - 2, clamped to
    e8m0, values to the nearest e2m1 (ties to even), saturating at 6."""
    rows, k = x.shape
    b = x.reshape(rows, k // BLOCK, BLOCK)
    amax = b.abs().amax(-1)
    e = (torch.frexp(amax).exponent - 3).clamp(-127, 127)
    e = torch.where(amax == 0, torch.full_like(e, -127), e)
    v = b * ((127 - e) << 23).view(F32)[..., None]  # 2^-e from its bits, exact
    a = v.abs()
    code = ((a > 0.25).to(torch.uint8) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0))
    code = (code + 8 * torch.signbit(v)).to(torch.uint8).reshape(rows, k)
    return code[:, 0::2] | (code[:, 1::2] << 4), (e + 127).to(torch.uint8)


def _plain_values(codes, scales):
    """The fp32 values of (rows, k/2) codes and (rows, k/32) exponents."""
    lut = torch.tensor([0., .5, 1., 1.5, 2., 3., 4., 6., -0., -.5, -1., -1.5, -2., -3., -4., -6.], device=codes.device)
    pair = torch.stack([codes & 15, codes >> 4], -1).reshape(codes.shape[0], -1)
    v = lut[pair.int()].reshape(codes.shape[0], -1, BLOCK)
    s = scales.int()
    unit = torch.where(s == 0, 1 << 22, s << 23).view(F32)  # 2^(s - 127) from its bits (2^-127 is subnormal)
    return (v * unit[..., None]).reshape(codes.shape[0], -1)


def _plain_round(x):
    return _plain_values(*_plain_quantize(x))


def _plain_ffn(x, gate, up, down):
    """x the fp32 values of quantised rows: silu(gate) * up, quantised, times down."""
    g = x @ _plain_values(*gate).T
    u = x @ _plain_values(*up).T
    return _plain_round(g / (1.0 + torch.exp(-g)) * u) @ _plain_values(*down).T


def _plain(st):
    c = st["case"]
    kind = c["kind"]
    if kind == "quantize":
        if c["dtype"] == "fp8":
            s = st["scale_inv"].repeat_interleave(128, 0)[: c["rows"]].repeat_interleave(128, 1)
            x = st["x"].float() * s
        else:
            x = st["x"].float()
        return _plain_round(x).to(BF16)
    if kind == "linear":
        x = _plain_values(*st["x"]) if c["held"] else _plain_round(st["x"].float())
        return (x @ _plain_values(*st["w"]).T).to(DTYPES[c["out"]])
    if kind == "grouped":
        x = _plain_round(st["x"].float())
        y = torch.empty(c["m"], c["n"], dtype=DTYPES[c["out"]], device=DEV)
        for e in range(c["experts"]):
            a, b = st["groups"][e], st["groups"][e + 1]
            if b > a:
                y[a:b] = (x[a:b] @ _plain_values(st["w"][0][e], st["w"][1][e]).T).to(y.dtype)
        return y
    if kind == "ffn":
        w = st["w"]
        return _plain_ffn(_plain_round(st["x"].float()), w["gate_proj"], w["up_proj"], w["down_proj"]).to(BF16)
    x = _plain_round(st["x"].float())
    y = torch.empty(c["tokens"] * c["top_k"], c["d"], dtype=BF16, device=DEV)
    flat = st["host_idx"].reshape(-1)
    for e in torch.unique(flat).tolist():
        slots = (flat == e).nonzero()[:, 0].to(DEV)
        w = [(st["w"][k][0][e], st["w"][k][1][e]) for k in ("gate_proj", "up_proj", "down_proj")]
        y[slots] = _plain_ffn(x[slots // c["top_k"]], *w).to(BF16)
    return y.view(c["tokens"], c["top_k"], c["d"])


def run(st):
    if not own:
        return _plain(st)
    ops = _ops()
    c = st["case"]
    kind = c["kind"]
    if kind == "quantize":
        q = ops.mxfp4_quantize_fp8(st["x"], st["scale_inv"]) if c["dtype"] == "fp8" else ops.mxfp4_quantize(st["x"])
        return ops.mxfp4_dequantize(*q)
    if kind == "linear":
        return ops.mxfp4_linear(st["x"], *st["w"], out_dtype=DTYPES[c["out"]])
    if kind == "grouped":
        return ops.mxfp4_grouped_linear(st["x"], *st["w"], st["offsets"], out_dtype=DTYPES[c["out"]])
    if kind == "ffn":
        return ops.dense_ffn(st["x"], st["w"])
    return ops.mxfp4_moe_experts(st["x"], st["idx"], st["w"])


# ------------------------------------------------------------------ work

def _weight_bytes(n, k):
    return n * k / 2 + n * k / BLOCK


def work(case):
    kind = case["kind"]
    if kind == "quantize":
        rows, k = case["rows"], case["k"]
        size = {"bf16": 2, "fp16": 2, "fp32": 4, "fp8": 1 + 4 / 16384}[case["dtype"]]
        return {"bytes": rows * k * (size + 2), "flops": 4 * rows * k}
    if kind == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        xb = _weight_bytes(m, k) if case["held"] else 2 * m * k
        return {"bytes": xb + _weight_bytes(n, k) + m * n * (4 if case["out"] == "fp32" else 2), "flops": 2 * m * n * k}
    if kind == "grouped":
        m, n, k = case["m"], case["n"], case["k"]
        used = min(case["experts"], m)
        return {"bytes": 2 * m * k + used * _weight_bytes(n, k) + m * n * (4 if case["out"] == "fp32" else 2),
                "flops": 2 * m * n * k}
    m, d, i = case["tokens"], case["d"], case["inter"]
    if kind == "ffn":
        return {"bytes": 4 * m * d + 3 * _weight_bytes(d, i), "flops": 6 * m * d * i}
    E, top_k = case["experts"], case["top_k"]
    used = E * (1.0 - (1.0 - top_k / E) ** m)  # distinct experts of an even routing
    return {"bytes": 2 * m * d + 2 * m * top_k * d + used * 3 * _weight_bytes(d, i), "flops": 6 * m * top_k * d * i}


# ------------------------------------------------------------------ 64 bits

def _pow2(e):
    """2^e in fp64 from its bits (e an integer tensor above -1023)."""
    return ((e.long() + 1023) << 52).view(F64)


def _exact_round(x):
    """fp64 (rows, k) -> the MXFP4 values of its blocks, by the spacing of e2m1 at each value."""
    b = x.reshape(x.shape[0], -1, BLOCK)
    top = b.abs().amax(-1, keepdim=True)
    floor_log2 = (top.view(torch.int64) >> 52) - 1023  # of a normal double; zero gives -1023
    unit = _pow2((floor_log2 - 2).clamp(-127, 127))
    a = (b / unit).abs()
    step = torch.where(a >= 4, 2.0, torch.where(a >= 2, 1.0, 0.5)).to(F64)
    q = (torch.round(a / step) * step).clamp(max=6.0)
    return (torch.copysign(q, b) * unit).reshape(x.shape)


def _exact_values(codes, scales):
    """A code's value from its bits: (-1)^s m / 2 at exponent field 0, else (2 + m) 2^(e - 2)."""
    rows = codes.shape[0]
    c = torch.empty(rows, codes.shape[1] * 2, dtype=torch.int32, device=codes.device)
    c[:, 0::2] = (codes % 16).int()
    c[:, 1::2] = torch.div(codes, 16, rounding_mode="floor").int()
    ef, mf = torch.div(c, 2, rounding_mode="floor") % 4, (c % 2).to(F64)
    v = torch.where(ef == 0, mf / 2, (2.0 + mf) * _pow2(ef - 2))
    v = torch.where(c >= 8, -v, v).view(rows, -1, BLOCK)
    return (v * _pow2(scales.int() - 127)[..., None]).reshape(rows, -1)


def _exact_ffn(x, gate, up, down):
    g, u = x @ _exact_values(*gate).T, x @ _exact_values(*up).T
    return _exact_round(g * torch.sigmoid(g) * u) @ _exact_values(*down).T


def exact(case, seed):
    st = prepare(case, seed)
    kind = case["kind"]
    if kind == "quantize":
        x = st["x"].to(F64)
        if case["dtype"] == "fp8":
            i = torch.arange(case["rows"], device=DEV) // 128
            j = torch.arange(case["k"], device=DEV) // 128
            # the dequantised weight is an fp32 value by its definition: one rounding of the product
            x = (x * st["scale_inv"].to(F64)[i][:, j]).to(F32).to(F64)
        return _exact_round(x)
    if kind == "linear":
        x = _exact_values(*st["x"]) if case["held"] else _exact_round(st["x"].to(F64))
        return x @ _exact_values(*st["w"]).T
    if kind == "grouped":
        x = _exact_round(st["x"].to(F64))
        y = torch.empty(case["m"], case["n"], dtype=F64, device=DEV)
        for e in range(case["experts"]):
            s = slice(st["groups"][e], st["groups"][e + 1])
            y[s] = x[s] @ _exact_values(st["w"][0][e], st["w"][1][e]).T
        return y
    w = st["w"]
    if kind == "ffn":
        return _exact_ffn(_exact_round(st["x"].to(F64)), w["gate_proj"], w["up_proj"], w["down_proj"])
    x = _exact_round(st["x"].to(F64))
    y = torch.empty(case["tokens"], case["top_k"], case["d"], dtype=F64, device=DEV)
    for e in sorted(set(st["host_idx"].reshape(-1).tolist())):
        t, j = torch.where(st["idx"] == e)
        y[t, j] = _exact_ffn(x[t], *[(w[k][0][e], w[k][1][e]) for k in ("gate_proj", "up_proj", "down_proj")])
    return y
