"""The register-before-retired check of test_asm_waits.py over the MXFP4 kernels."""
import os

import pytest

from _asm_waits import device_asm, inflight_uses, kernels
from test_asm_waits import CSRC, HIPCC, INCLUDE


@pytest.mark.skipif(not os.path.exists(HIPCC), reason="hipcc not available")
@pytest.mark.parametrize("source,least", [("mxfp4_gemm.hip", 10), ("mxfp4_quant.hip", 6)])
def test_no_mxfp4_kernel_uses_a_register_before_its_load_retired(source, least):
    ks = kernels(device_asm(os.path.join(CSRC, source), [CSRC, INCLUDE], HIPCC))
    problems = [f"{name[:60]}: {p}" for name, instrs in ks.items() for p in inflight_uses(instrs)[:3]]
    assert len(ks) >= least, "expected the MXFP4 kernels in the assembly"
    assert not problems, "\n".join(problems)
