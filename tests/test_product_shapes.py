"""The rule that gives a product its kernel, on the host."""
import test_gpu_weights
from _shapes import product_places, product_shapes

PRODUCT = {(16, 16, 8), (16, 32, 8), (16, 64, 8), (32, 32, 4), (32, 32, 8), (32, 64, 4), (32, 128, 1), (32, 256, 1),
           (64, 128, 2), (64, 256, 1)}
GATED = {(16, 32, 8), (32, 32, 8), (32, 32, 4), (32, 64, 2), (32, 128, 1), (64, 64, 2), (64, 128, 1)}


def test_the_gpu_tests_meet_every_kernel():
    got = product_shapes([(False, *c[:3]) for c in test_gpu_weights.SHAPES])
    assert got == [c[3] for c in test_gpu_weights.SHAPES] and set(got) == PRODUCT
    got = product_shapes([(True, *c[:3]) for c in test_gpu_weights.GATED_SHAPES])
    assert got == [c[3] for c in test_gpu_weights.GATED_SHAPES] and set(got) == GATED


def test_launches_stay_within_their_limits():
    """At most 65535 workgroups along the rows, up to 2^20 rows."""
    calls = [(g, m, n, k) for g in (False, True) for m in (2, 17, 1000, 65537, (1 << 20) - 1, 1 << 20)
             for n in (1, 32, 4096, 1 << 20) for k in (32, 4096, 1 << 24)]
    for (_, m, n, _), (rows, outs, waves) in zip(calls, product_shapes(calls)):
        assert -(-m // rows) <= 65535 and -(-n // outs) < 1 << 31 and 64 * waves <= 1024


def test_few_rows_take_small_pieces_and_many_large_ones():
    assert product_shapes([(False, 2, 4096, 4096), (False, 4096, 12288, 4096)]) == [(16, 16, 8), (64, 256, 1)]
    assert product_shapes([(True, 2, 5632, 4096), (True, 4096, 5632, 4096)]) == [(16, 32, 8), (64, 128, 1)]


def test_an_xcd_works_on_whole_columns():
    """Every place once; columns that XCDs share only where they are no multiple of 8."""
    grids = [(c, r) for c in (*range(1, 34), 49, 88, 126, 501) for r in (1, 2, 3, 7, 8, 9, 31, 64)]
    for (c, r), (once, shared) in zip(grids, product_places(grids)):
        assert once, (c, r)
        assert shared <= (c if c < 8 else c % 8) or r == 1, (c, r, shared)
