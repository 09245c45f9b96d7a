"""Sizes at which the 32-bit counts of the paged cache's attention end (no GPU: nothing runs)."""
import pytest

from test_latent_refusals import EUNSUPPORTED, EWORKSPACE, L, P, _attend, _cache  # noqa: F401  (L: a fixture)


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
