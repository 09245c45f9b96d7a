"""The register checks over the kernels of the paged latent cache and of packed prompts."""
import os

import pytest

from _asm_waits import device_asm, inflight_uses, kernels
from _mfma_hazards import mfma_hazards
from test_asm_waits import CSRC, HIPCC, INCLUDE


@pytest.mark.skipif(not os.path.exists(HIPCC), reason="hipcc not available")
@pytest.mark.parametrize("source,least", [("latent_attn.hip", 15), ("packed_attn.hip", 5), ("latent_cache.hip", 4)])
def test_no_kernel_uses_a_register_too_early(source, least):
    ks = kernels(device_asm(os.path.join(CSRC, source), [CSRC, INCLUDE], HIPCC))
    problems = [f"{name[:60]}: {p}" for name, instrs in ks.items() for p in inflight_uses(instrs)[:3] + mfma_hazards(instrs)[:3]]
    assert len(ks) >= least, "expected the kernels in the assembly"
    assert not problems, "\n".join(problems)


def test_the_hazard_check_sees_hazards():
    m = "v_mfma_f32_32x32x16_bf16 v[0:15], v[20:23], a[0:3], v[0:15]"
    pairs = lambda *t: [(s, True) for s in t]  # noqa: E731
    assert not mfma_hazards(pairs("v_mov_b32 v20, v1", "s_nop 1", m, "s_nop 7", "s_nop 7", "s_nop 7", "v_mov_b32 v60, v3"))
    assert mfma_hazards(pairs("v_mov_b32 v20, v31", "s_nop 0", m))
    assert mfma_hazards(pairs("v_accvgpr_write_b32 a2, v31", m))
    assert mfma_hazards(pairs(m, "s_nop 7", "s_nop 7", "v_mov_b32 v60, v3"))
    assert mfma_hazards(pairs(m, "s_nop 7", "v_mov_b32 v3, v60"))
    assert not mfma_hazards(pairs(m, m, "v_mov_b32 v60, v30"))
