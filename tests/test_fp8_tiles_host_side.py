"""tests/test_gpu_fp8_tiles.py holds the 256 x 256 kernel of the 8-bit products to what it computes: all its cases have to
reach it, by the library's own choice."""
from tests import fp8_tiles as T
from tests import test_gpu_fp8_tiles as cases


def test_the_cases_take_the_256_tiles(tmp_path):
    calls = [(trans, block, ct, sizes, m, k, 0 if len(sizes) == 1 else cases.EXTRA) for sizes, m, k, _, trans, block, ct, *_ in cases.CALLS]
    for case, kinds in zip(cases.CALLS, T.of(calls, tmp_path)):
        assert kinds[0] == "256" and ("fold" in kinds) == case[3], (case, kinds)


def test_the_captured_product_has_sums_in_the_workspace(tmp_path):
    sizes, m, k, cut = cases.CAPTURED
    assert cut
    for kinds in T.of([(trans, block, "bf16", sizes, m, k) for trans, block in ((1, 128), (1, 1), (0, 128))], tmp_path):
        assert "fold" in kinds, kinds
