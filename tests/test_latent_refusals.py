"""What the operators of the paged latent cache and of packed prompts refuse, and what they look like to tracers
(no GPU: nothing runs)."""
import ctypes
import os
import subprocess

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from amla import _lib, ops, torch_ops  # noqa: F401  (registers the operators)
from amla.config import DeepSeekConfig
from test_capi import ROOT

EINVAL, EWORKSPACE, EUNSUPPORTED = -1, -2, -3
P = 1 << 20  # an aligned address that nothing reads
BIG = 1 << 60
BF16, FP8 = torch.bfloat16, torch.float8_e4m3fn


@pytest.fixture(scope="module")
def L():
    return _lib.lib()


def _cache(latent=P, k_pe=P, scales=P, table=P, ld=8, cols=8, pages=100, page=64):
    return _lib.LatentCache(latent, k_pe, scales, table, ld, cols, pages, page)


def _write(L, c=None, kv=P, rows=4, ldkv=576, gamma=P, rope=P, rope_rows=10, off=None, seqs=2, pos=P):
    return L.amla_latent_cache_write(c or _cache(), kv, rows, ldkv, gamma, 1e-6, rope, rope_rows, off, seqs, pos, None)


def _read(L, c=None, rows=4, off=P, seqs=2, out=P, pe=P):
    return L.amla_latent_cache_read(c or _cache(), rows, off, seqs, None, out, pe, 1, None)


def _attend(L, c=None, q=P, seqs=2, S=1, H=16, ld=(16 * 576, 16 * 576, 576), lens=P, out=P, ws=P, need=BIG):
    return L.amla_latent_attention(c or _cache(), q, seqs, S, H, *ld, lens, 0.1, out, None, ws, need, None)


def _packed(L, **kw):
    a = dict(q=P, k=P, v=P, k_pe=None, out=P, lse=None, offsets=P, k_offsets=None, q_rows=10, k_rows=10, seqs=2, ldq=512,
             ldq_head=128, ldk=512, ldk_head=128, ldv=512, ldv_head=128, ld_pe=64, heads=4, kv_heads=4, dn=128, causal=1,
             scale=0.1, workspace=P, workspace_bytes=BIG)
    a.update(kw)
    return L.amla_packed_attention(_lib.PackedArgs(*[a[f] for f, _ in _lib.PackedArgs._fields_]), None)


@pytest.mark.parametrize("call", [_write, _read, _attend])
def test_caches(L, call):
    for bad in (dict(latent=None), dict(k_pe=None), dict(table=None), dict(pages=0), dict(cols=-1), dict(ld=7)):
        assert call(L, _cache(**bad)) == EINVAL, bad
    for bad in (dict(page=0), dict(page=48), dict(page=1 << 17), dict(pages=2 ** 25), dict(cols=2 ** 25, ld=2 ** 25),
                dict(latent=P + 8), dict(k_pe=P + 8)):
        assert call(L, _cache(**bad)) == EUNSUPPORTED, bad


def test_nothing_to_do(L):
    empty = _cache(table=None, cols=0, ld=0)
    assert _write(L, empty, rows=0, seqs=0) == 0 and _read(L, empty, rows=0, seqs=0) == 0
    assert _attend(L, empty, seqs=0) == 0 and _attend(L, S=0) == 0 and _attend(L, H=0) == 0
    assert _packed(L, q_rows=0) == 0 and _packed(L, heads=0, kv_heads=0) == 0 and _packed(L, seqs=0) == 0


def test_rows(L):
    for call in (_write, _read):
        assert call(L, rows=-1) == EINVAL and call(L, seqs=-1) == EINVAL
        assert call(L, off=None, rows=5, seqs=2) == EINVAL
        assert call(L, off=None, rows=5, seqs=0) == EINVAL
        assert call(L, seqs=65536) == EUNSUPPORTED and call(L, rows=2 ** 31) == EUNSUPPORTED
    assert _write(L, rows=2 ** 26, off=P) == EUNSUPPORTED and _read(L, rows=2 ** 28) == EUNSUPPORTED
    for bad in (dict(kv=None), dict(gamma=None), dict(rope=None), dict(pos=None), dict(rope_rows=-1)):
        assert _write(L, **bad) == EINVAL, bad
    for bad in (dict(ldkv=568), dict(ldkv=580), dict(kv=P + 8), dict(gamma=P + 8)):
        assert _write(L, **bad) == EUNSUPPORTED, bad
    assert _read(L, out=None) == EINVAL and _read(L, pe=None) == EINVAL
    assert _read(L, out=P + 8) == EUNSUPPORTED and _read(L, pe=P + 4) == EUNSUPPORTED


def test_attention(L):
    for bad in (dict(q=None), dict(lens=None), dict(out=None), dict(seqs=-1), dict(S=-1), dict(H=-1)):
        assert _attend(L, **bad) == EINVAL, bad
    for bad in (dict(q=P + 8), dict(out=P + 8), dict(ld=(9216, 9216, 577)), dict(ld=(9217, 9216, 576)), dict(seqs=65536),
                dict(H=2 ** 24), dict(S=2 ** 20, H=2 ** 12), dict(ws=P + 8)):
        assert _attend(L, **bad) == EUNSUPPORTED, bad
    need = L.amla_latent_attention_workspace_bytes(2, 1, 16, 512)
    assert need > 0 and _attend(L, need=need - 1) == EWORKSPACE and _attend(L, ws=None) == EWORKSPACE
    assert L.amla_latent_attention_workspace_bytes(0, 1, 1, 1) == 0
    assert L.amla_latent_attention_workspace_bytes(1, 1, 2 ** 40, 1) == 0


def test_packed(L):
    for bad in (dict(q=None), dict(k=None), dict(v=None), dict(out=None), dict(offsets=None), dict(q_rows=-1), dict(k_rows=-1),
                dict(kv_heads=3), dict(kv_heads=0), dict(scale=0.0), dict(scale=-1.0), dict(scale=float("inf")),
                dict(scale=float("nan"))):
        assert _packed(L, **bad) == EINVAL, bad
    for bad in (dict(dn=64), dict(dn=192, k_pe=P), dict(ldq=516), dict(ldv_head=100), dict(k_pe=P, ld_pe=60), dict(ldk=2 ** 28),
                dict(q=P + 8), dict(v=P + 8), dict(k_pe=P + 8), dict(seqs=65536), dict(k_rows=2 ** 31),
                dict(q_rows=2 ** 31 - 1, heads=4)):
        assert _packed(L, **bad) == EUNSUPPORTED, bad
    bytes_of = L.amla_packed_attention_workspace_bytes
    need = bytes_of(10, 9000, 2, 4)
    assert need > 0 and _packed(L, k_rows=9000, workspace_bytes=need - 1) == EWORKSPACE
    assert _packed(L, k_rows=9000, workspace=None) == EWORKSPACE
    assert _packed(L, k_rows=9000, workspace=P + 8) == EUNSUPPORTED
    assert bytes_of(100000, 100000, 2, 128) == bytes_of(10, 10, 2, 4) == 0  # enough blocks, or few keys: nothing is split
    assert bytes_of(0, 9000, 1, 1) == bytes_of(1, 9000, 1, 0) == bytes_of(1, -1, 1, 1) == 0


@pytest.mark.parametrize("struct,name", [(_lib.LatentCache, "amla_latent_cache"), (_lib.PackedArgs, "amla_packed_args")])
def test_struct_layouts_match_c(tmp_path, struct, name):
    fields = [f for f, _ in struct._fields_]
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    body = "\n".join(f'  printf("%zu ", offsetof({name}, {f}));' for f in fields)
    src.write_text(f'#include <stdio.h>\n#include <stddef.h>\n#include "amla.h"\nint main(void){{\n{body}\n'
                   f'  printf("%zu", sizeof({name}));\n  return 0;\n}}\n')
    subprocess.run(["gcc", "-std=c11", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)], check=True)
    got = [int(x) for x in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    assert got == [getattr(struct, f).offset for f in fields] + [ctypes.sizeof(struct)]


def test_workspaces_hold_a_split_of_every_query_row(L):
    for b, s, h, t in ((1, 1, 128, 64), (1, 1, 128, 32768), (64, 1, 128, 200), (300, 1, 8, 100), (2, 3, 16, 100000), (1, 1, 1, 0)):
        assert L.amla_latent_attention_workspace_bytes(b, s, h, t) >= b * (32 * -(-s * h // 32)) * (512 * 2 + 4)


def _fake(mode, *shape, dtype=BF16):
    with mode:
        return torch.empty(*shape, dtype=dtype, device="cuda")


def test_shapes_under_fake_tensors():
    mode = FakeTensorMode()
    f = lambda *shape, dtype=BF16: _fake(mode, *shape, dtype=dtype)  # noqa: E731
    i32 = torch.int32
    for cache in ((f(9, 16, 512), f(9, 16, 64)), (f(9, 16, 512, dtype=FP8), f(9, 16, 64), f(9, 16, dtype=torch.uint8))):
        table, off = f(3, 5, dtype=i32), f(4, dtype=i32)
        with mode:
            ops.latent_cache_write(f(3, 2, 576), f(512), f(100, 32, dtype=torch.complex64), cache, table, f(3, dtype=i32))
            lat, pe = ops.latent_cache_read(cache, table, off, 70)
            o, lse = ops.latent_attention(f(3, 2, 20, 576), cache, table, f(3, dtype=i32), 0.1, return_lse=True)
            only = ops.latent_attention(f(3, 2, 20, 576), cache, table, f(3, dtype=i32), 0.1)
        assert lat.shape == (70, 512) and pe.shape == (70, 64) and lat.dtype == pe.dtype == BF16
        assert o.shape == only.shape == (3, 2, 20, 512) and o.dtype == BF16 and lse.shape == (3, 2, 20)
        assert lse.dtype == torch.float32
    with mode:
        kvb = f(80, 8, 256)
        o, lse = ops.packed_attention(f(50, 16, 192), kvb[..., :128], kvb[..., 128:], f(4, dtype=i32), 0.1, k_pe=f(80, 64),
                                      k_offsets=f(4, dtype=i32), return_lse=True)
    assert o.shape == (50, 16, 128) and o.dtype == BF16 and lse.shape == (50, 16) and lse.dtype == torch.float32


def test_schemas_name_what_is_written():
    def mutated(name):
        return {a.name for a in getattr(torch.ops.amla, name).default._schema.arguments
                if a.alias_info is not None and a.alias_info.is_write}
    assert mutated("latent_cache_write") == {"latent", "k_pe", "scales"}
    assert mutated("latent_cache_read_out") == {"out", "out_pe"}
    for name in ("latent_cache_read", "latent_attention", "packed_attention"):
        assert not mutated(name)


def test_python_checks():
    """Shapes, types and devices are named before anything runs."""
    mode = FakeTensorMode()
    f = lambda *shape, dtype=BF16: _fake(mode, *shape, dtype=dtype)  # noqa: E731
    i32 = torch.int32
    cache, fp8 = (f(9, 16, 512), f(9, 16, 64)), (f(9, 16, 512, dtype=FP8), f(9, 16, 64), f(9, 16, dtype=torch.uint8))
    table, lens, q = f(3, 5, dtype=i32), f(3, dtype=i32), f(3, 1, 4, 576)
    attend = lambda q=q, c=cache, t=table, n=lens: ops.latent_attention(q, c, t, n, 0.1)  # noqa: E731
    cpu = torch.zeros(3, 1, 4, 576, dtype=BF16)
    with mode:
        for bad in (dict(c=cache[:1]), dict(c=(cache[0], f(9, 16, 32))), dict(c=(f(9, 16, 256), cache[1])),
                    dict(c=fp8[:2] + (f(9, 15, dtype=torch.uint8),)), dict(c=(f(0, 16, 512), f(0, 16, 64))), dict(q=f(3, 4, 576)),
                    dict(q=f(2, 1, 4, 576)), dict(q=f(3, 1, 4, 512)), dict(t=f(3, 5)), dict(t=f(3, dtype=i32)),
                    dict(n=f(2, dtype=i32)), dict(n=f(3, dtype=torch.int64)), dict(c=(cache[0].transpose(0, 1), cache[1])),
                    dict(t=f(3, 10, dtype=i32)[:, ::2])):
            with pytest.raises(ValueError):
                attend(**bad)
        for bad in (dict(c=(fp8[0], fp8[1])), dict(c=cache + (fp8[2],)), dict(q=f(3, 1, 4, 576, dtype=torch.float32))):
            with pytest.raises(TypeError):
                attend(**bad)
    with pytest.raises(ValueError):
        ops.latent_attention(cpu, cache, table, lens, 0.1)
    with pytest.raises(ValueError):
        ops.packed_attention(cpu[0], cpu[0], cpu[0], torch.zeros(2, dtype=i32), 0.1)
    with mode:
        qp, k, v, off = f(50, 16, 192), f(80, 8, 128), f(80, 8, 128), f(4, dtype=i32)
        pe = f(80, 64)
        good = dict(q=qp, k=k, v=v, o=off, s=0.1, pe=pe)
        for bad in (dict(pe=None), dict(pe=f(79, 64)), dict(q=f(50, 12, 192)), dict(v=f(80, 8, 64)), dict(v=f(80, 4, 128)),
                    dict(k=f(80, 8, 192)), dict(o=f(4)), dict(o=f(0, dtype=i32)), dict(s=0.0), dict(s=float("nan")),
                    dict(q=f(50, 192))):
            a = {**good, **bad}
            with pytest.raises(ValueError):
                ops.packed_attention(a["q"], a["k"], a["v"], a["o"], a["s"], k_pe=a["pe"])
        with pytest.raises(ValueError):
            ops.packed_attention(qp, k, v, off, 0.1, k_pe=pe, k_offsets=f(5, dtype=i32))
        with pytest.raises(TypeError):
            ops.packed_attention(qp, k, f(80, 8, 128, dtype=torch.float16), off, 0.1, k_pe=pe)
        kv, gamma, rope, pos = f(3, 2, 576), f(512), f(100, 32, dtype=torch.complex64), f(3, dtype=i32)
        for bad in (dict(kv=f(2, 2, 576)), dict(kv=f(6, 576)), dict(kv=f(3, 2, 512)), dict(g=f(256)), dict(p=f(2, dtype=i32)),
                    dict(p=[1, 2]), dict(p=-1)):
            a = {**dict(kv=kv, g=gamma, p=pos), **bad}
            with pytest.raises(ValueError):
                ops.latent_cache_write(a["kv"], a["g"], rope, cache, table, a["p"])
        with pytest.raises(TypeError):
            ops.latent_cache_write(kv, gamma, f(100, 32), cache, table, pos)
        with pytest.raises(ValueError):
            ops.latent_cache_read(cache, table, f(3, dtype=i32), 10)
        with pytest.raises(ValueError):
            ops.latent_cache_read(cache, table, off, -1)
        with pytest.raises(ValueError):
            ops.latent_cache_read(cache, table, off, 10, out=(f(10, 512), f(9, 64)))


def test_new_caches():
    config = DeepSeekConfig()
    lat, pe = ops.latent_cache(7, 16, config, "cpu", BF16)
    assert lat.shape == (7, 16, 512) and pe.shape == (7, 16, 64) and lat.dtype == BF16
    lat, pe, scales = ops.latent_cache(7, 16, config, "cpu")
    assert lat.dtype == FP8 and scales.shape == (7, 16) and (scales == 127).all()
    for pages, page_size in ((0, 16), (7, 48), (7, 0), (7, 1 << 17)):
        with pytest.raises(ValueError):
            ops.latent_cache(pages, page_size, config, "cpu")
    with pytest.raises(ValueError):
        ops.latent_cache(7, 16, DeepSeekConfig(kv_lora_rank=256), "cpu")
    with pytest.raises(TypeError):
        ops.latent_cache(7, 16, config, "cpu", torch.float16)
