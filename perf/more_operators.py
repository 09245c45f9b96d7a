"""The operators of a paged latent cache as measured cases: its store and load, the attention that
reads it, and the attention of packed prompts.

A serving loop for DeepSeek-R1 keeps what attention needs of a token as one row: the latent, already
normed, and the rope key, already rotated. Rows live in pages of a pool; a sequence's block table says
which. A row is held in bf16, or its latent as e4m3 codes with one power of two per row. Prompts of
several sequences are packed one after another, with int32 offsets between them. Sizes are the R1
configuration (``amla.config.DeepSeekConfig``) with the heads of a whole layer or of a tensor-parallel
rank, and generic ones around it.

``listed()`` gives the fixed cases, ``draw(rng)`` further ones of the same ranges, ``prepare`` what the
program holds before the call, ``run`` one call (``own``: the package's functions, else the plain form
in fp32), ``work`` the bytes and operations the call cannot do without and ``exact`` the result in 64
bits from the definition.
"""
from __future__ import annotations

import math
import os
import random
import sys

import torch

own = False

DEV = "cuda"
BF16, F32, F64, FP8 = torch.bfloat16, torch.float32, torch.float64, torch.float8_e4m3fn
LORA, ROPE, VDIM = 512, 64, 128
EPS = 1e-6
SCALE = (0.1 * math.log(40.0) + 1.0) / math.sqrt(192)  # the softmax scale of the R1 configuration
MAX_POS = 40960


def _ops():
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    path = os.path.join(root, "deepseek-on-one-gpu_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    from amla import ops
    return ops


# ------------------------------------------------------------------ the cases
#
# rows / context: of all sequences / of the longest one; mix: which ragged lengths (_lengths).

def _store(seqs, rows, dtype, page, mix=1):
    return {"kind": "store", "seqs": seqs, "rows": rows, "dtype": dtype, "page": page, "mix": mix}


def _load(seqs, rows, dtype, page, mix=1):
    return {"kind": "load", "seqs": seqs, "rows": rows, "dtype": dtype, "page": page, "mix": mix}


def _decode(seqs, context, heads, dtype, page, new=1, ragged=True, mix=1):
    return {"kind": "decode", "seqs": seqs, "context": context, "heads": heads, "dtype": dtype, "page": page, "new": new,
            "ragged": ragged, "mix": mix}


def _prompt(seqs, rows, heads, kv_heads, form, past=0, causal=True, mix=1):
    return {"kind": "prompt", "seqs": seqs, "rows": rows, "heads": heads, "kv_heads": kv_heads, "form": form, "past": past,
            "causal": causal, "mix": mix}


def listed():
    return [
        # a decode step of 32 sequences: one new row each, where latency counts
        {"name": "store_32_fp8", **_store(32, 32, "fp8", 64)},
        # prompts of eleven requests, odd lengths
        {"name": "store_8111_fp8", **_store(11, 8111, "fp8", 64)},
        # cached contexts of three follow-up prompts, read back ahead of kv_b
        {"name": "load_40001_fp8", **_load(3, 40001, "fp8", 64)},
        # the same of one short bf16 cache with small pages
        {"name": "load_1501_bf16", **_load(2, 1501, "bf16", 16)},
        # one user's decode step over a short chat
        {"name": "decode_1x257_fp8", **_decode(1, 257, 128, "fp8", 64, ragged=False)},
        # eight long documents
        {"name": "decode_8x32768_fp8", **_decode(8, 32768, 128, "fp8", 64, ragged=False)},
        # a batch of forty on a tensor-parallel rank with 16 heads, ragged, one slot of the batch empty
        {"name": "decode_40_rank_bf16", **_decode(40, 16384, 16, "bf16", 64)},
        # six sequences with two proposed tokens checked beside the new one
        {"name": "decode_6x3_bf16", **_decode(6, 12345, 128, "bf16", 16, new=3)},
        # one short prompt
        {"name": "prompt_333", **_prompt(1, 333, 128, 128, "mla")},
        # prompts of five requests, packed
        {"name": "prompt_5_4099", **_prompt(5, 4099, 128, 128, "mla")},
        # a chunk of two prompts over what was cached of them
        {"name": "prompt_2_past", **_prompt(2, 1000, 128, 128, "mla", past=4000)},
        # heads that share keys and values in groups of four, packed
        {"name": "prompt_grouped", **_prompt(3, 6000, 32, 8, "plain")},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    case = _any(rng)
    while work(case)["flops"] > 6e11:  # the largest listed case's
        case = _any(rng)
    return case


def _any(rng):
    what = rng.choice(["store", "load", "decode", "decode", "decode", "prompt", "prompt"])
    dtype, page, mix = rng.choice(["fp8", "fp8", "bf16"]), rng.choice([1, 16, 32, 64, 64, 128]), rng.randrange(1 << 20)
    if what in ("store", "load"):
        rows = _log_int(rng, 1, 8111 if what == "store" else 40000)
        return (_store if what == "store" else _load)(min(rows, _log_int(rng, 1, 64)), rows, dtype, page, mix)
    if what == "decode":
        heads, new = rng.choice([8, 16, 20, 32, 64, 128, 128]), rng.choice([1, 1, 1, 2, 4])
        seqs = _log_int(rng, 1, 64)
        context = _log_int(rng, 1, min(40000, 262144 // seqs, 262144 * 128 // (seqs * heads * new)))
        return _decode(seqs, context, heads, dtype, page, new, rng.random() < 0.7, mix)
    form = rng.choice(["mla", "mla", "whole", "plain"])
    heads, kv_heads = {"mla": [(128, 128), (16, 16)], "whole": [(32, 32), (16, 4)], "plain": [(32, 8), (24, 24), (8, 1)]}[form][
        rng.randrange(2)]
    seqs = _log_int(rng, 1, 16)
    rows = max(seqs, _log_int(rng, 1, 4000))
    past = rng.choice([0, 0, _log_int(rng, 1, 4000)])
    return _prompt(seqs, rows, heads, kv_heads, form, past if rows <= 1000 else 0, rng.random() < 0.85, mix)


def _split(total, parts, mix):
    """Ragged parts, some of them short, none below 1, that add up to total."""
    r = random.Random(mix)
    share = [r.random() ** 2 + 0.02 for _ in range(parts)]
    ends, run = [0], 0.0
    for s in share:
        run += s
        ends.append(int(run / sum(share) * (total - parts) + 0.5))
    return [b - a + 1 for a, b in zip(ends, ends[1:])]


def _lengths(case):
    """(new rows of each sequence, all rows of each sequence with the new ones)."""
    kind, n, mix = case["kind"], case["seqs"], case["mix"]
    if kind == "decode":
        r = random.Random(mix)
        T = case["context"]
        lens = [max(1, int(T * (r.random() if case["ragged"] else 1.0))) for _ in range(n)]
        lens[0] = T
        if case["ragged"] and n > 4:
            lens[n // 2] = 0
        return [case["new"]] * n, lens
    new = _split(case["rows"], n, mix)
    if kind == "prompt":
        past = _split(case["past"] * n, n, mix + 7) if case["past"] else [0] * n
        return new, [a + b for a, b in zip(new, past)]
    if kind == "store":  # behind some rows that are there already
        r = random.Random(mix + 7)
        return new, [a + r.randrange(0, 700) for a in new]
    return new, new


def _offsets(lens):
    out = [0]
    for n in lens:
        out.append(out[-1] + n)
    return out


# ------------------------------------------------------------------ inputs

class _Draw:
    """Seeded values on the GPU."""

    def __init__(self, seed):
        self.g = torch.Generator(device=DEV)
        self.g.manual_seed(seed)

    def randn(self, *shape, std=1.0):
        return torch.randn(shape, generator=self.g, device=DEV, dtype=F32).mul_(std)

    def gamma(self):
        return (1.0 + 0.2 * self.randn(LORA)).to(BF16)

    def raw(self, rows):
        """kv_a's outputs: latents with some large channels, each row at a scale of its own, and rope keys."""
        x = self.randn(rows, LORA + ROPE) * torch.exp(0.4 * self.randn(rows, 1))
        x[:, 5:LORA:97] *= 6.0
        return x.to(BF16)


def _rope_table():
    inv = 1.0 / (10000.0 ** (torch.arange(0, ROPE, 2, dtype=F64) / ROPE))
    ang = torch.outer(torch.arange(MAX_POS, dtype=F64), inv)
    return torch.polar(torch.ones_like(ang), ang).to(torch.complex64).to(DEV)


def _pool(case, lens, d, host):
    """(cache, block table) with every sequence's rows held, pages in no order, the rest old rows."""
    page = case["page"]
    need = [-(-n // page) for n in lens]
    pages = sum(need) + 3
    order = torch.randperm(pages, generator=host).tolist()
    table = torch.full((len(lens), max(1, max(need))), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = torch.tensor(order[at:at + n], dtype=torch.int32)
        at += n
    rows = pages * page
    ckv = torch.empty(rows, LORA, dtype=FP8 if case["dtype"] == "fp8" else BF16, device=DEV)
    scales = torch.empty(rows, dtype=torch.uint8, device=DEV)
    for r in range(0, rows, 65536):
        n = d.randn(min(65536, rows - r), LORA) * torch.exp(0.1 * d.randn(min(65536, rows - r), 1))
        n[:, 5::97] *= 3.0
        if case["dtype"] == "fp8":
            codes, e = _plain_quantize(n)
            ckv[r:r + 65536], scales[r:r + 65536] = codes, e
        else:
            ckv[r:r + 65536] = n.to(BF16)
    kpe = d.randn(rows, ROPE).to(BF16).view(pages, page, ROPE)
    ckv = ckv.view(pages, page, LORA)
    cache = (ckv, kpe, scales.view(pages, page)) if case["dtype"] == "fp8" else (ckv, kpe)
    return cache, table.to(DEV)


def prepare(case, seed):
    d = _Draw(seed)
    host = torch.Generator()
    host.manual_seed(seed)
    new, lens = _lengths(case)
    st = {"case": case, "new": new, "lens": lens}
    dev = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)  # noqa: E731
    kind = case["kind"]
    if kind == "prompt":
        H, G, rows, keys = case["heads"], case["kv_heads"], sum(new), sum(lens)
        st["offsets"], st["k_offsets"] = dev(_offsets(new)), dev(_offsets(lens))
        if case["form"] == "mla":  # kv_b's output: per head 128 of the key, then the value; one rope key for all heads
            kvb = d.randn(keys, G, 128 + VDIM).to(BF16)
            st["q"], st["k"], st["v"] = d.randn(rows, H, 192).to(BF16), kvb[..., :128], kvb[..., 128:]
            st["k_pe"] = d.randn(keys, ROPE).to(BF16)
            st["scale"] = SCALE
        else:
            dk = 192 if case["form"] == "whole" else 128
            st["q"], st["k"], st["v"] = (d.randn(n, h, w).to(BF16) for n, h, w in ((rows, H, dk), (keys, G, dk), (keys, G, VDIM)))
            st["k_pe"], st["scale"] = None, 1.0 / math.sqrt(dk)
        return st
    st["cache"], st["table"] = _pool(case, lens, d, host)
    if kind == "decode":
        q = d.randn(case["seqs"], case["new"], case["heads"], LORA + ROPE, std=0.7)
        st["q"], st["lengths"] = q.to(BF16), dev(lens)
        return st
    st["offsets"], st["position"] = dev(_offsets(new)), dev([b - a for a, b in zip(new, lens)])
    if kind == "store":
        st["kv"], st["gamma"], st["freqs"] = d.raw(sum(new)), d.gamma(), _rope_table()
    return st


# ------------------------------------------------------------------ plain forms

def _plain_quantize(n):
    """fp32 (rows, 512) -> (e4m3 codes, exponent bytes): per row the smallest power of two 2^e with
    max |n| <= 448 2^e, -32 <= e <= 32, byte e + 127; n / 2^e to the nearest code, saturating."""
    amax = n.abs().amax(-1)
    f, e = torch.frexp(amax)
    e = torch.where(f > 0.875, e - 8, e - 9).clamp(-32, 32)
    e = torch.where(amax == 0, torch.full_like(e, -32), e)
    v = n * ((127 - e) << 23).view(F32)[:, None]
    return v.clamp(-448.0, 448.0).to(FP8), (e + 127).to(torch.uint8)


def _plain_values(cache, slots):
    """fp32 latents and rope keys of pool rows."""
    c = cache[0].view(-1, LORA)[slots].float()
    if len(cache) == 3:
        c = c * (cache[2].view(-1)[slots].int() << 23).view(F32)[..., None]
    return c, cache[1].view(-1, ROPE)[slots].float()


def _plain_rows(offsets, start, rows):
    """(sequence, position) of each packed row."""
    i = torch.arange(rows, device=DEV)
    b = (i[:, None] >= offsets[None, 1:]).sum(1)
    return b, start[b] + i - offsets[b]


def _plain_slots(table, page, b, pos):
    return table[b, pos // page].long() * page + pos % page


def _plain_load(st):
    b, pos = _plain_rows(st["offsets"].long(), st["position"].long(), sum(st["new"]))
    c, r = _plain_values(st["cache"], _plain_slots(st["table"], st["case"]["page"], b, pos))
    return c.to(BF16), r.to(BF16)


def _plain_store(st):
    b, pos = _plain_rows(st["offsets"].long(), st["position"].long(), sum(st["new"]))
    slots = _plain_slots(st["table"], st["case"]["page"], b, pos)
    x = st["kv"].float()
    c = x[:, :LORA]
    n = c * torch.rsqrt((c * c).mean(-1, keepdim=True) + EPS) * st["gamma"].float()
    f = torch.view_as_real(st["freqs"])[pos]
    a, s = x[:, LORA::2], x[:, LORA + 1::2]
    r = torch.stack([a * f[..., 0] - s * f[..., 1], a * f[..., 1] + s * f[..., 0]], -1).flatten(-2)
    cache = st["cache"]
    if len(cache) == 3:
        codes, e = _plain_quantize(n)
        cache[0].view(torch.uint8).view(-1, LORA)[slots] = codes.view(torch.uint8)
        cache[2].view(-1)[slots] = e
    else:
        cache[0].view(-1, LORA)[slots] = n.to(BF16)
    cache[1].view(-1, ROPE)[slots] = r.to(BF16)
    return _plain_load(st)


def _plain_softmax(s, seen):
    """(exp(s - max) over what is seen, its sum, log of the sum of exp): rows that see nothing give zeros and -inf."""
    s = torch.where(seen, s, float("-inf"))
    m = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(m == float("-inf"), 0.0, m))
    total = p.sum(-1, keepdim=True)
    return p, total, (m + torch.log(total))[..., 0]


def _plain_decode(st):
    c = st["case"]
    B, S, H, T = c["seqs"], c["new"], c["heads"], max(st["lens"])
    t = torch.arange(T, device=DEV)
    held = t[None] < st["lengths"][:, None]
    page = torch.where(held, st["table"].long()[:, t // c["page"]], 0)
    lat, rope = _plain_values(st["cache"], page * c["page"] + t % c["page"])
    k = torch.cat([lat, rope], -1)
    s = st["q"].float().view(B, S * H, -1) @ k.transpose(1, 2) * SCALE
    sees = st["lengths"][:, None] - (S - 1) + torch.arange(S, device=DEV)
    seen = t[None, None] < sees.repeat_interleave(H, 1)[..., None]
    p, total, lse = _plain_softmax(s, seen)
    o = (p @ lat) / torch.where(total == 0, 1.0, total)
    return o.view(B, S, H, LORA).to(BF16), lse.view(B, S, H)


def _plain_prompt(st):
    c = st["case"]
    qo, ko = st["offsets"].long(), st["k_offsets"].long()
    nq, nk = qo[1:] - qo[:-1], ko[1:] - ko[:-1]
    i, j = (torch.arange(max(v), device=DEV) for v in (st["new"], st["lens"]))
    qi = (qo[:-1, None] + i).clamp(max=sum(st["new"]) - 1)
    ki = (ko[:-1, None] + j).clamp(max=sum(st["lens"]) - 1)
    q = st["q"][qi].float().transpose(1, 2)
    k = st["k"][ki].float()
    if st["k_pe"] is not None:
        k = torch.cat([k, st["k_pe"][ki].float()[:, :, None].expand(-1, -1, c["kv_heads"], -1)], -1)
    group = c["heads"] // c["kv_heads"]
    k = k.transpose(1, 2).repeat_interleave(group, 1)
    v = st["v"][ki].float().transpose(1, 2).repeat_interleave(group, 1)
    s = q @ k.transpose(2, 3) * st["scale"]
    last = (i[None] + (nk - nq)[:, None])[..., None] if c["causal"] else (nk - 1)[:, None, None]
    seen = (j[None, None] <= last) & (j[None, None] < nk[:, None, None])
    p, total, lse = _plain_softmax(s, seen[:, None])
    o = ((p @ v) / torch.where(total == 0, 1.0, total)).transpose(1, 2)
    b, at = _plain_rows(qo, torch.zeros_like(qo), sum(st["new"]))
    return o[b, at].to(BF16), lse.transpose(1, 2)[b, at]


def run(st):
    kind = st["case"]["kind"]
    if not own:
        return {"store": _plain_store, "load": _plain_load, "decode": _plain_decode, "prompt": _plain_prompt}[kind](st)
    ops = _ops()
    if kind == "decode":
        return ops.latent_attention(st["q"], st["cache"], st["table"], st["lengths"], SCALE, return_lse=True)
    if kind == "prompt":
        return ops.packed_attention(st["q"], st["k"], st["v"], st["offsets"], st["scale"], k_offsets=st["k_offsets"], k_pe=st["k_pe"],
                                    causal=st["case"]["causal"], return_lse=True)
    if kind == "store":
        ops.latent_cache_write(st["kv"], st["gamma"], st["freqs"], st["cache"], st["table"], st["position"], offsets=st["offsets"],
                               eps=EPS)
    return ops.latent_cache_read(st["cache"], st["table"], st["offsets"], sum(st["new"]), position=st["position"])


# ------------------------------------------------------------------ work

def _row_bytes(case):
    return 2 * ROPE + (LORA + 1 if case["dtype"] == "fp8" else 2 * LORA)


def work(case):
    kind = case["kind"]
    new, lens = _lengths(case)
    if kind == "decode":
        H, S = case["heads"], case["new"]
        rows, io = sum(lens), case["seqs"] * S * H * (2 * (2 * LORA + ROPE) + 4)
        seen = sum(max(0, n - (S - 1) + s) for n in lens for s in range(S))
        return {"bytes": rows * (_row_bytes(case) + 4 / case["page"]) + io, "flops": 2 * seen * H * (2 * LORA + ROPE)}
    if kind == "prompt":
        H, G = case["heads"], case["kv_heads"]
        dk = 128 if case["form"] == "plain" else 192
        key = 2 * G * (128 + VDIM) + 2 * ROPE if case["form"] == "mla" else 2 * G * (dk + VDIM)
        pairs = sum(a * b - (a * (a - 1) // 2 if case["causal"] else 0) for a, b in zip(new, lens))
        return {"bytes": sum(new) * H * (2 * (dk + VDIM) + 4) + sum(lens) * key, "flops": 2 * pairs * H * (dk + VDIM)}
    rows, row, wide = sum(new), _row_bytes(case), 2 * (LORA + ROPE)
    if kind == "load":
        return {"bytes": rows * (row + wide + 4 / case["page"]), "flops": rows * LORA}
    return {"bytes": rows * (2 * row + 2 * wide + 4 * ROPE), "flops": rows * 8 * LORA}


# ------------------------------------------------------------------ 64 bits

def _exact_values(st, b, n, start=0):
    """fp64 (latents, rope keys) of n rows of sequence b, by its pages; a code's value from its bits."""
    page = st["case"]["page"]
    used = st["table"][b, : -(-(start + n) // page)].long()
    c = st["cache"][0][used].flatten(0, 1)[start:start + n]
    if len(st["cache"]) == 3:
        bits = c.view(torch.uint8).int()
        ef, mf = torch.div(bits, 8, rounding_mode="floor") % 16, (bits % 8).to(F64)
        c = torch.where(ef == 0, mf * 2.0 ** -9, torch.ldexp(8.0 + mf, ef - 10)) * torch.where(bits >= 128, -1.0, 1.0)
        c = torch.ldexp(c, st["cache"][2][used].flatten()[start:start + n].int()[:, None] - 127)
    return c.to(F64), st["cache"][1][used].flatten(0, 1)[start:start + n].to(F64)


def _exact_e4m3(n):
    """fp64 rows -> the values of their codes, by the spacing of e4m3 at each value."""
    unit = torch.exp2(torch.ceil(torch.log2(n.abs().amax(-1, keepdim=True) / 448.0)).clamp(-32, 32))
    a = (n / unit).abs()
    step = torch.exp2(torch.floor(torch.log2(a.clamp(min=2.0 ** -6))) - 3)
    return torch.copysign((torch.round(a / step) * step).clamp(max=448.0), n) * unit


def _exact_attention(q, k, v, scale, seen):
    """(H, n, .) queries, keys and values in fp64."""
    s = torch.matmul(q, k.transpose(-2, -1)) * scale
    s = s.masked_fill(~seen, float("-inf"))
    return torch.nan_to_num(torch.softmax(s, -1), nan=0.0) @ v, torch.logsumexp(s, -1)


def exact(case, seed):
    st = prepare(case, seed)
    kind = case["kind"]
    new, lens = st["new"], st["lens"]
    if kind == "load":
        parts = [_exact_values(st, b, n, lens[b] - n) for b, n in enumerate(new)]
        return torch.cat([p[0] for p in parts]), torch.cat([p[1] for p in parts])
    if kind == "store":
        at = _offsets(new)
        lat, rope = [], []
        for b, n in enumerate(new):
            x = st["kv"][at[b]:at[b] + n].to(F64)
            c = x[:, :LORA]
            c = c / torch.sqrt(c.square().mean(-1, keepdim=True) + EPS) * st["gamma"].to(F64)
            lat.append(_exact_e4m3(c) if case["dtype"] == "fp8" else c)
            z = torch.view_as_complex(x[:, LORA:].reshape(n, -1, 2)) * st["freqs"][lens[b] - n:lens[b]].to(torch.complex128)
            rope.append(torch.view_as_real(z).flatten(1))
        return torch.cat(lat), torch.cat(rope)
    outs, lses = [], []
    if kind == "decode":
        S, H = case["new"], case["heads"]
        for b, n in enumerate(lens):
            lat, rope = _exact_values(st, b, n)
            t = torch.arange(n, device=DEV)
            seen = (t < n - (S - 1) + torch.arange(S, device=DEV)[:, None]).repeat_interleave(H, 0)
            q = st["q"][b].to(F64).reshape(S * H, -1)
            if n == 0:
                o, lse = torch.zeros(S * H, LORA, dtype=F64, device=DEV), torch.full((S * H,), float("-inf"), dtype=F64, device=DEV)
            else:
                o, lse = _exact_attention(q, torch.cat([lat, rope], -1), lat, SCALE, seen)
            outs.append(o.view(S, H, LORA))
            lses.append(lse.view(S, H))
        return torch.stack(outs), torch.stack(lses)
    qo, ko = _offsets(new), _offsets(lens)
    group = case["heads"] // case["kv_heads"]
    for b in range(case["seqs"]):
        n, m = new[b], lens[b]
        seen = torch.ones(n, m, dtype=torch.bool, device=DEV)
        if case["causal"]:
            seen = torch.tril(seen, diagonal=m - n)
        o = torch.empty(n, case["heads"], VDIM, dtype=F64, device=DEV)
        lse = torch.empty(n, case["heads"], dtype=F64, device=DEV)
        for h in range(0, case["heads"], 8):
            hs = torch.arange(h, min(h + 8, case["heads"]), device=DEV)
            k = st["k"][ko[b]:ko[b + 1]][:, hs // group].to(F64)
            if st["k_pe"] is not None:
                k = torch.cat([k, st["k_pe"][ko[b]:ko[b + 1], None].to(F64).expand(-1, len(hs), -1)], -1)
            v = st["v"][ko[b]:ko[b + 1]][:, hs // group].to(F64)
            oh, lh = _exact_attention(st["q"][qo[b]:qo[b + 1]][:, hs].to(F64).transpose(0, 1), k.transpose(0, 1), v.transpose(0, 1),
                                      st["scale"], seen)
            o[:, hs], lse[:, hs] = oh.transpose(0, 1), lh.transpose(0, 1)
        outs.append(o)
        lses.append(lse)
    return torch.cat(outs), torch.cat(lses)
