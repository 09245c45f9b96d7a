"""The register checks of the paged cache's and packed prompts' kernels along every path."""
import os

import pytest

from _asm_paths import kernels, path_hazards
from _asm_waits import device_asm
from test_asm_waits import CSRC, HIPCC, INCLUDE

M = "v_mfma_f32_32x32x16_bf16 v[0:15], v[20:23], a[0:3], v[0:15]"


@pytest.mark.skipif(not os.path.exists(HIPCC), reason="hipcc not available")
@pytest.mark.parametrize("source,least", [("latent_attn.hip", 15), ("packed_attn.hip", 5)])
def test_no_path_uses_a_register_too_early(source, least):
    ks = kernels(device_asm(os.path.join(CSRC, source), [CSRC, INCLUDE], HIPCC))
    assert len(ks) >= least and all(len(labels) > 3 for _, labels in ks.values())
    problems = [f"{name[:60]}: {p}" for name, k in ks.items() for p in path_hazards(k)[:3]]
    assert not problems, "\n".join(problems)


def _kernel(*lines):
    """Instructions and labels, all of inline asm."""
    text = "_Zkernel:\n;;#ASMSTART\n" + "\n".join(lines) + "\n;;#ASMEND\n.Lfunc_end0:\n"
    return kernels(text)["_Zkernel"]


def test_the_check_sees_loops_and_branches():
    nops = ["s_nop 7"] * 3
    # the result of a loop's last product, in its first instruction
    loop = [".L1:", "v_add_f32 v60, v3, v3", *nops, M, "s_cbranch_scc1 .L1", *nops]
    assert path_hazards(_kernel(*loop))
    assert not path_hazards(_kernel(*loop[:-2 - len(nops)], M, *nops, "s_cbranch_scc1 .L1", *nops))
    # an operand written at the end of a loop, and across a branch
    assert path_hazards(_kernel(".L1:", M, *nops, "v_mov_b32 v20, v40", "s_cbranch_scc1 .L1"))
    assert path_hazards(_kernel("v_mov_b32 a1, v40", "s_branch .L2", ".L1:", *nops, ".L2:", M, *nops))
    assert not path_hazards(_kernel("v_mov_b32 a1, v40", "s_branch .L2", M, *nops, ".L2:", "s_nop 1", M, *nops))
    # a read issued at the end of a loop, waited for behind its first instruction or before it
    read = "ds_read_b128 v[4:7], v60"
    assert path_hazards(_kernel(".L1:", "v_mov_b32 v5, v61", "s_waitcnt lgkmcnt(0)", read, "s_cbranch_scc1 .L1", "s_waitcnt lgkmcnt(0)"))
    assert not path_hazards(_kernel(".L1:", "s_waitcnt lgkmcnt(0)", "v_mov_b32 v5, v61", read, "s_cbranch_scc1 .L1"))
    assert path_hazards(_kernel(read, "ds_read_b32 v9, v60", "s_waitcnt lgkmcnt(2)", "v_mov_b32 v40, v4"))
    assert not path_hazards(_kernel(read, "ds_read_b32 v9, v60", "s_waitcnt lgkmcnt(1)", "v_mov_b32 v40, v4"))
