"""Sampling at the ends of its arguments' ranges, against tests/paged_ref.py in 64 bits with the bars of test_gpu_sampling."""
import numpy as np
import pytest

from test_gpu_sampling import check

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


def far_apart(rng, n, high, low):
    """-inf but for `high` logits next to 3e38 and `low` next to -3e38, whose distance f32 cannot hold."""
    x = np.full(n, -np.inf, np.float32)
    at = rng.permutation(n)[:high + low]
    x[at[:high]] = np.float32(3e38) * (1 - rng.integers(0, 3, high) / 64)
    x[at[high:]] = np.float32(-3e38) * (1 - rng.integers(0, 5, low) / 64)
    return x


def test_top_k_of_logits_further_apart_than_f32(gpu):
    x = np.full((1, 2048), -3e38, np.float32)
    x[0, :100] = 3e38
    check(x, [1e38], np.float32([0.9999]), [200])


@pytest.mark.parametrize("n", [500, 2048, 9000, 32768, 40000, 262144])
def test_filters_of_logits_further_apart_than_f32(gpu, n):
    rng = np.random.default_rng(n)
    high, low, k, p, m = zip(*[(100, 150, 200, 1.0, 0.0), (3, 200, 30, 1.0, 0.0), (100, 390, 101, 0.99, 0.0), (1, 400, 300, 1.0, 0.002),
                               (100, 150, 0, 0.995, 0.0), (100, 150, 0, 1.0, 0.0026), (5, 9, 14, 1.0, 0.0), (200, 290, 450, 0.9999, 1e-4)])
    x = np.stack([far_apart(rng, n, *c) for c in zip(high, low)])
    for t in (1e38, 3e38):
        for r in (0.9999, 0.999, 0.5):
            check(x, [t] * len(x), np.full(len(x), r, np.float32), k, p, m)


@pytest.mark.parametrize("n", [6000, 50000])
def test_top_k_of_many_logits_further_apart_than_f32(gpu, n):
    rng = np.random.default_rng(n)
    x = np.stack([far_apart(rng, n, 1500, 4000), far_apart(rng, n, 400, 4000), far_apart(rng, n, 40, 2000)])
    check(x, [1e38] * 3, np.float32([0.99995, 0.998, 0.9]), [5000, 1024, 900])


@pytest.mark.parametrize("n", [2, 4000, 32768, 70001])
@pytest.mark.parametrize("m", [1e-20, 1e-25, 1e-40])
def test_min_p_below_the_weights_that_sums_hold(gpu, n, m):
    """A draw of exactly 0 takes the first token of any weight: of those not below min_p, however small that is."""
    x = np.full((6, n), -np.inf, np.float32)
    x[:, n - 1] = 0
    x[0, 0] = -60  # (a weight of 9e-27)
    x[1, 0] = -46  # 1e-20: 1.05e-20
    x[2, 0] = -100  # 4e-44, between the smallest numbers of f32
    x[3, 0], x[3, n // 2] = -120, -40
    x[4, 0] = -92.2  # 9e-41, just below 1e-40
    x[5, 0] = -45.9
    zero = np.zeros(6, np.float32)
    check(x, [1.0] * 6, zero, None, None, [m] * 6)
    check(x, [0.5] * 6, zero, None, None, [m] * 6)
    check(x, [1.0] * 6, zero, [2] * 6, [0.9] * 6, [m] * 6)


@pytest.mark.parametrize("l,t,r", [(-0.005526490043848753, 1.0212681293487549, 0.501352846622467), (-0.005455499980598688, 1.0065972805023193, 0.5013549327850342),
                                   (-0.005429748445749283, 1.0016255378723145, 0.5013552308082581)])
def test_weights_are_within_two_to_the_minus_44(gpu, l, t, r):
    """Draws that are 1.07 to 1.14 times 2^-44 of the larger weight away from the border of two tokens, of 2^19: a sum that is
    2^-44 off finds the same token as the definition. (In 64 bits the border is off by 2^-52.)"""
    x = np.full((1, 2 ** 19), -np.inf, np.float32)
    x[0, :2] = 0, l
    check(x, [t], np.float32([r]))
