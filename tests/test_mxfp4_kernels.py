"""The sizes of mxfp4_kernels.py reach every kernel of inner_prod_mxfp4."""
from mxfp4_kernels import ALL, FLOATING, KEPT, kernel_of, stages_of, up


def test_every_kernel_has_sizes():
    for floating, sizes in ((False, ALL), (True, FLOATING)):
        for size, without, *rest in sizes:
            assert kernel_of(*size, floating=floating) == without, size
            assert kernel_of(*size, residual=True, floating=floating) == (rest[0] if rest else without), size
    reached = {want for _, want, *_ in ALL + FLOATING}
    assert reached >= {("few", tokens, ctas, False) for tokens in (16, 32, 64) for ctas in (1, 2, 4)} | {("few", 16, ctas, True) for ctas in (1, 2, 4)}
    assert reached >= {("tiles", bn, 1, several, False) for bn in (64, 128, 256) for several in (False, True)} | {("tiles", bn, 1, True, True) for bn in (64, 128)}
    assert reached >= {("tiles", 64, 2, False, False), ("tiles", 128, 4, False, False)}


def test_kept_weights_divide_the_ring_and_do_not():
    """Blocks of K as many as stages, some that divide them and some that leave stages over; one, two, three and more tiles of channels beside each other."""
    rings = [(up(up(k, 32) * 16, 128), stages_of(bn, False, 1, False)) for (_, _, k), (_, bn, *_), *_ in KEPT]
    assert any(b == s for b, s in rings) and any(1 < b < s and s % b == 0 for b, s in rings) and any(s % b for b, s in rings)
    assert {up(n, bn) for (_, n, _), (_, bn, *_), *_ in KEPT} == {1, 2, 3}
