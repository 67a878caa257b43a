"""The inputs of paged_planes, on a model of the arithmetic in which parts and products can be left out."""
import numpy as np
import pytest

import paged_planes as P


def error(name, hd, turn=0, **left):
    K, V, q, scale, bar = P.case(name, hd, 100, 40, turn)
    p = P.softmax(scale * (q @ K.T))
    return np.max(np.abs(P.model(K, V, q, scale, **left) - p @ V) / np.maximum(bar(p, V, len(K)), 1e-300))


@pytest.mark.parametrize("name", P.CASES)
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("turn", [0, 1])
def test_six_products_are_within_the_bars(name, hd, turn):
    assert error(name, hd, turn) < 0.5


@pytest.mark.parametrize("which", ["scores", "sums"])
@pytest.mark.parametrize("lost", P.SIX)
def test_each_product_is_missed(which, lost):
    left = {which: [x for x in P.SIX if x != lost]}
    assert max(error(name, 128, **left) for name in P.CASES) > 2


def test_parts_sum_to_the_number():
    x = np.float32(np.random.default_rng(0).standard_normal(10000)).astype(np.float64)
    assert np.array_equal(sum(P.parts(x)), x)
