"""Sampling from rows of which more tokens lie next to each other than a list holds: such a row is picked from value by value."""
import numpy as np
import pytest

from tests.test_gpu_sample import BF16, F32, compare

pytestmark = pytest.mark.gpu
LAST = 1.0 - 2.0 ** -24  # the largest fp32 number below 1


@pytest.mark.parametrize("n", [4090, 32000, 32003, 64000, 128256, 256000])
@pytest.mark.parametrize("rows", [4, 12])  # long rows by several workgroups each, and by one
def test_the_last_of_equal_tokens_are_drawn(n, rows):
    """a row of one value, as long as a vocabulary is: random numbers close to 1 take its last tokens"""
    x = np.full((rows, n), 0.25)
    u = np.resize([0.9985, LAST, 0.9999, 0.98, 0.99995, 0.5], rows)
    compare(F32, x, u)
    compare(BF16, x, u, t=[0.7] * rows, k=[n] * rows)


@pytest.mark.parametrize("n", [50, 1500, 70000])
@pytest.mark.parametrize("rows", [3, 12])
def test_min_p_of_one_among_logits_that_weigh_the_same(n, rows):
    """logits that differ by less than a 64-bit weight can show: all of them weigh 1, and a min-p of 1 keeps them"""
    rng = np.random.default_rng(n)
    x = np.where(rng.random((rows, n)) < 0.5, 1e-40, 3e-40)
    for t in (1.0, 0.01):
        compare(F32, x, rng.random(rows), t=[t] * rows, m=[1.0] * rows)
        compare(F32, x, rng.random(rows), t=[t] * rows, m=[1.0] * rows, k=[n // 2] * rows, p=[0.7] * rows)
    compare(F32, x, rng.random(rows), t=[1.0] * rows, m=[1.0 - 2.0 ** -24] * rows)
