"""That the inputs of decoder_precision.py show a lost part: the kernels' arithmetic in numpy is within the bounds as it is and outside with a
third part, or one of the six products, left out."""
import numpy as np
import pytest

from decoder_precision import WINDOWS, by_parts, expected, keys, queries, values


def run(what, elem, d, **broken):
    rng = np.random.default_rng(d)
    n = 120
    q, k, v = queries(rng, what, n, d), keys(rng, what, (n, d), elem), values(rng, what, (n, d), elem)
    at = np.arange(n)
    seen = (at <= at[:, None]) & (at > at[:, None] - WINDOWS[what])
    want, bound = expected(what, q, k, v, seen)
    return np.abs(by_parts(q, k, v, seen, elem, **broken) - want) <= bound


@pytest.mark.parametrize("what", sorted(WINDOWS))
@pytest.mark.parametrize("elem", ["f32", "bf16"])
@pytest.mark.parametrize("d", [64, 96, 128, 256])
def test_three_parts_are_within_the_bounds(what, elem, d):
    assert run(what, elem, d).all()


@pytest.mark.parametrize("what,elem,broken", [
    ("scores", "f32", dict(keep=(2, 3, 3, 3))), ("scores", "f32", dict(keep=(3, 2, 3, 3))), ("weights", "f32", dict(keep=(3, 3, 2, 3))), ("values", "f32", dict(keep=(3, 3, 3, 2))),
    ("scores", "bf16", dict(keep=(2, 3, 3, 3))), ("weights", "bf16", dict(keep=(3, 3, 2, 3))),
    ("scores", "f32", dict(without=[(1, 1)])), ("scores", "f32", dict(without=[(0, 2)])), ("scores", "f32", dict(without=[(2, 0)]))])
@pytest.mark.parametrize("d", [64, 96, 128, 256])
def test_a_part_or_product_left_out_shows(what, elem, broken, d):
    assert not run(what, elem, d, **broken).all()
