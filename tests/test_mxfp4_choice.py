"""Which kernel a 4-bit product takes, by the estimates between them (no GPU): every one of them has sizes of its own, and sizes far
apart in time take the kernel that measured fastest."""
import random

import pytest

from gemm_amd import qlinear

F32, BF16 = 0, 30


def choice(rows, cols, tok, pair=False, y=F32):
    return qlinear.load().qlin_probe_mxfp4_kernel(int(pair), y, rows, cols, tok)


@pytest.mark.parametrize("rows,cols,tok,pair,want", [
    (14336, 4096, 1, False, 0), (151936, 4096, 4, False, 0), (4096, 14336, 24, False, 0), (4096, 14336, 64, False, 0), (1342, 9344, 17, True, 0),
    (23207, 576, 64, False, 11), (1136, 1792, 811, False, 11), (2433, 4128, 880, True, 22), (14336, 4096, 256, False, 22), (14336, 4096, 2048, False, 44),
    (4096, 4096, 4096, False, 44), (14336, 4096, 512, True, 44), (6002, 832, 687, True, 21), (4096, 4096, 512, False, 21),
])
def test_choice(rows, cols, tok, pair, want):
    assert choice(rows, cols, tok, pair) == want


def test_every_kernel_has_its_sizes():
    rng = random.Random(1)
    seen = set()
    for _ in range(3000):
        rows, cols, tok = (int(lo * (hi / lo) ** rng.random()) for lo, hi in ((64, 28672), (64, 14336), (1, 4096)))
        for pair in (False, True):
            k = choice(rows, cols, tok, pair, rng.choice([F32, BF16]))
            assert k in ((0, 21, 22, 44) if pair else (0, 11, 21, 22, 44))
            seen.add((pair, k))
    assert len(seen) == 9


def test_refuses_what_is_no_product():
    for args in ((0, 5, 64, 64, 4), (0, F32, 0, 64, 4), (0, F32, 64, 0, 4), (0, F32, 64, 64, 0), (0, F32, 64, 1 << 24, 4)):
        assert qlinear.load().qlin_probe_mxfp4_kernel(*args) == qlinear.ERR_ARG
