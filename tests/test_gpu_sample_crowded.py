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
