"""Which kernels the sizes of the GPU tests reach (CPU-only)."""
import pytest

import decoder_plain as R
from ppocr_native_amd import decoder as D
from test_gpu_decoder import PRODUCT_SIZES
from test_gpu_decoder_edges import TILES


@pytest.mark.parametrize("x_type", [D.F32, D.BF16, D.F16, D.E4M3, D.I8])
def test_product_sizes_reach_every_number_of_tiles(x_type):
    got = {}
    for m, n, k, group in TILES:
        got.setdefault(D.q4_product_tiles(m, n, k, x_type), set()).add(group)
    wanted = {2, 4, 8} if x_type == D.F32 else {2, 4}
    assert wanted <= set(got)
    assert got[max(wanted)] == {32, 64, 128}  # the most tiles, with groups of every size
    assert {D.q4_product_tiles(m, n, k, x_type) for m, n, k in PRODUCT_SIZES} >= {1}
    most = [(m, n, k) for m, n, k, _ in TILES if D.q4_product_tiles(m, n, k, x_type) == max(wanted)]
    rows = [(k + 1) // 2 for _, _, k in most]
    assert {16 if r % 16 == 0 else 4 if r % 4 == 0 else 1 for r in rows} == {16, 4, 1}
    assert any(m > 16 for m, _, _ in most) and all(n % (16 * max(wanted)) for _, n, _ in most)


def test_tiles_of_sizes_that_are_refused():
    for m, n, k, t in ((0, 16, 32, D.F32), (1, 0, 32, D.F32), (1, 16, 0, D.F32), (1, 16, 1 << 25, D.F32),
                       (1, 16, 32, 5), (1, 16, 32, -1), (1 << 21, 16, 32, D.F16), (1 << 20, 1 << 20, 32, D.F16)):
        assert D.q4_product_tiles(m, n, k, t) == 0
    assert D.q4_product_tiles(1, 16, 32, D.I8) == 1
