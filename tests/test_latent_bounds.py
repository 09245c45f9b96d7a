"""Sizes at which the 32-bit counts of the paged cache's attention end (no GPU: nothing runs)."""
import collections
import ctypes
import subprocess

import pytest

from test_asm_waits import CSRC
from test_latent_refusals import EUNSUPPORTED, EWORKSPACE, L, P, _attend, _cache, _packed  # noqa: F401  (L: a fixture)


@pytest.mark.parametrize("scales", [P, None])
@pytest.mark.parametrize("page", [1, 2, 16, 32, 64, 128, 256, 65536])
def test_rows_of_a_table_end_below_two_to_31(L, page, scales):  # noqa: F811
    """The kernels look up to three tiles of 64 rows past a sequence's last row before they stop at it."""
    for cols in {(2 ** 31 - 1) // page, (2 ** 31 - 512) // page + 1, (2 ** 31 - 512) // page}:
        if cols > (2 ** 31 - 1) // page:
            continue
        c = _cache(scales=scales, ld=cols, cols=cols, pages=1, page=page)
        last = cols * page - 1
        fits = (last // 64 + 3) * 64 + 63 < 2 ** 31 and cols * page <= 2 ** 31 - 512
        # (what is taken goes on to ask for its workspace)
        assert _attend(L, c, need=1) == (EWORKSPACE if fits else EUNSUPPORTED), (page, cols)


@pytest.fixture(scope="module")
def plan(tmp_path_factory):
    """csrc/latent_plan.h, compiled for the host."""
    d = tmp_path_factory.mktemp("plan")
    (d / "plan.cpp").write_text('''#include "latent_plan.h"
using namespace amla;
extern "C" int low(long long s) { return plan_low(s); }
extern "C" int high(long long s) { return plan_high(s); }
extern "C" long long total(int l, int h) { return plan_total(l, h); }
extern "C" void range(long long t, int most, int chunks, int seqs, int slots, int *out) {
  const PlanRange r = plan_range(t, most, chunks, seqs, slots);
  out[0] = r.lo; out[1] = r.hi;
}
''')
    subprocess.run(["g++", "-std=c++17", "-O1", "-shared", "-fPIC", f"-I{CSRC}", str(d / "plan.cpp"), "-o", str(d / "plan.so")], check=True)
    lib = ctypes.CDLL(str(d / "plan.so"))
    lib.low.argtypes = lib.high.argtypes = [ctypes.c_longlong]
    lib.total.argtypes, lib.total.restype = [ctypes.c_int, ctypes.c_int], ctypes.c_longlong
    lib.range.argtypes = [ctypes.c_longlong] + [ctypes.c_int] * 4 + [ctypes.POINTER(ctypes.c_int)]
    return lib


CASES = [  # (tiles of each sequence, chunks, slots)
    ([5], 1, 256), ([2 ** 26 - 16], 4, 256), ([1], 1, 1), ([3, 0, 7], 2, 256), ([2 ** 12 - 1, 2 ** 12, 2 ** 12 + 1] * 50, 1, 278),
    ([32768 * 2] * 65535, 1, 65535 + 128),         # 2^32 tiles: sequences of 2 million rows
    ([2 ** 26 - 16] * 65535, 1, 65535 + 128),      # the longest tables of as many sequences as a call takes
    ([2 ** 26 - 16] * 65535, 200, 65535 * 200 + 128), ([2 ** 26 - 16] + [0] * 65534, 7, 65535 * 7 + 128), ([1] * 65535, 3, 65535 * 3 + 128),
]


@pytest.mark.parametrize("tiles,chunks,slots", CASES, ids=range(len(CASES)))
def test_sums_of_tiles_past_two_to_31(plan, tiles, chunks, slots):
    """What a wave forms of its 64 lanes' sums in 32 bits is the number of all tiles, and the smallest length whose splits fit
    the slots lies in the range."""
    assert slots >= chunks * len(tiles)
    lanes = [sum(tiles[i::64]) for i in range(64)]
    low, high = sum(plan.low(s) for s in lanes), sum(plan.high(s) for s in lanes)
    assert 0 <= low < 2 ** 31 and 0 <= high < 2 ** 31
    total = plan.total(low, high)
    assert total == sum(tiles)
    out = (ctypes.c_int * 2)()
    plan.range(total, max(tiles), chunks, len(tiles), slots, out)
    lo, hi = out
    kinds = collections.Counter(tiles)
    used = lambda n: chunks * sum(-(-t // n) * k for t, k in kinds.items())  # noqa: E731
    assert 1 <= lo <= hi and used(hi) <= slots and (lo == 1 or used(lo - 1) > slots)
    assert all(used(n) < 2 ** 31 for n in (lo, hi, (lo + hi) // 2))  # (counted in 32 bits)


def test_rows_of_packed_prompts_end_below_two_to_31(L):  # noqa: F811
    """Keys of one row for all (a stride of 0) can be that many; blocks of 256 queries and tiles of 64 keys are counted past the
    last of them."""
    for rows in (2 ** 31 - 512, 2 ** 31 - 511, 2 ** 31 - 256, 2 ** 31 - 63, 2 ** 31 - 1):
        fits = rows + 256 + 64 < 2 ** 31 and rows <= 2 ** 31 - 512
        # (what is taken goes on to ask for its workspace, or finds too many blocks)
        assert _packed(L, k_rows=rows, ldk=0, ldv=0, workspace=None) == (EWORKSPACE if fits else EUNSUPPORTED), rows
        assert _packed(L, q_rows=rows, heads=4) == EUNSUPPORTED
