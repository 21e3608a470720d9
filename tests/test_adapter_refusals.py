"""What routing by scores and the adapters' calls refuse, before anything reaches the GPU (these calls return without one), and what
the workspace's size says."""
import ctypes as C

import numpy as np
import pytest

from gemm_amd import qlinear

F32, F16, BF16, MXFP4, Q4K = 0, 1, 30, 39, 12
P = 0x10000  # an aligned address that no refused call reads
ARG, TYPE = qlinear.ERR_ARG, qlinear.ERR_TYPE


@pytest.fixture(scope="module")
def lib():
    return qlinear.load()


ROUTE = dict(score=0, type=F32, logits=P, n_tok=4, n_expert=64, ld=64, bias=P, n_group=8, used=4, top=2, k=8, renorm=1, scale=1.0, idx=P, w=P)


@pytest.mark.parametrize("code,change", [
    (TYPE, dict(type=Q4K)), (TYPE, dict(type=99)), (ARG, dict(score=2)), (ARG, dict(score=-1)), (ARG, dict(n_tok=-1)), (ARG, dict(n_expert=0)), (ARG, dict(n_expert=-8)),
    (ARG, dict(n_expert=4104, ld=4104)), (ARG, dict(ld=63)), (ARG, dict(n_group=0)), (ARG, dict(n_group=7)), (ARG, dict(n_group=-8)), (ARG, dict(n_expert=512, ld=512, n_group=512)),
    (ARG, dict(used=0)), (ARG, dict(used=9)), (ARG, dict(top=0)), (ARG, dict(top=3)), (ARG, dict(k=0)), (ARG, dict(k=33)), (ARG, dict(logits=None)), (ARG, dict(logits=P + 2)),
    (ARG, dict(type=BF16, logits=P + 1)), (ARG, dict(bias=P + 2)), (ARG, dict(idx=None)), (ARG, dict(idx=P + 2)), (ARG, dict(w=None)), (ARG, dict(w=P + 1)), (ARG, dict(n_tok=1 << 26)),
])
def test_routing_refuses(lib, code, change):
    a = dict(ROUTE, **change)
    assert lib.qlin_moe_route_scores_dev(*[a[n] for n in ROUTE], None) == code
    assert lib.qlin_last_error()


def test_routing_of_no_tokens(lib):
    a = dict(ROUTE, n_tok=0, logits=None, idx=None, w=None)
    assert lib.qlin_moe_route_scores_dev(*[a[n] for n in ROUTE], None) == qlinear.OK


ADD = dict(n_mat=1, lora=BF16, n_adapter=4, max_rank=16, ids=P, x_type=BF16, X=P, y_type=F32, out_type=F32, n_cols=64, n_tok=4, ldx=64, ws=P, ws_bytes=1 << 30)
TENSOR = dict(adapters=P, Y=P, out=P, n_rows=64, ldy=64, ldo=64)
BOTH = [(TYPE, dict(lora=Q4K)), (TYPE, dict(lora=MXFP4)), (TYPE, dict(x_type=MXFP4)), (TYPE, dict(y_type=Q4K)), (TYPE, dict(out_type=39)), (ARG, dict(n_adapter=-1)),
        (ARG, dict(max_rank=0)), (ARG, dict(max_rank=257)), (ARG, dict(max_rank=-16)), (ARG, dict(ids=None)), (ARG, dict(ids=P + 2)), (ARG, dict(X=None)), (ARG, dict(X=P + 1)),
        (ARG, dict(x_type=F32, X=P + 2)), (ARG, dict(n_cols=0)), (ARG, dict(n_cols=-64)), (ARG, dict(n_cols=1 << 24, ldx=1 << 24)), (ARG, dict(n_tok=-1)), (ARG, dict(ldx=63)),
        (ARG, dict(ws=None)), (ARG, dict(ws=P + 8)), (ARG, dict(ws_bytes=255))]


def add(lib, change, tensor):
    a, t = dict(ADD, **change), dict(TENSOR, **tensor)
    tensors = (qlinear.LoraTensor * 3)(*[qlinear.LoraTensor(*[t[n] for n in TENSOR], 0)] * 3)
    return lib.qlin_lora_add_dev(a["n_mat"], C.addressof(tensors), *[a[n] for n in list(ADD)[1:]], None)


def silu_mul(lib, change, tensor):
    a, t = dict(ADD, **change), dict(dict(TENSOR, up_adapters=P, up=P), **tensor)
    return lib.qlin_lora_silu_mul_dev(t["adapters"], t["up_adapters"], a["lora"], a["n_adapter"], a["max_rank"], a["ids"], a["x_type"], a["X"], a["y_type"], t["Y"], t["up"],
                                      a["out_type"], t["out"], t["n_rows"], a["n_cols"], a["n_tok"], a["ldx"], t["ldy"], t["ldo"], a["ws"], a["ws_bytes"], None)


@pytest.mark.parametrize("call", [add, silu_mul])
@pytest.mark.parametrize("code,change", BOTH)
def test_adapters_refuse(lib, call, code, change):
    assert call(lib, change, {}) == code
    assert lib.qlin_last_error()


@pytest.mark.parametrize("call", [add, silu_mul])
@pytest.mark.parametrize("change,tensor", [
    ({}, dict(adapters=None)), ({}, dict(adapters=P + 4)), ({}, dict(Y=None)), ({}, dict(Y=P + 2)), ({}, dict(out=None)), ({}, dict(out=P + 2)), (dict(out_type=BF16), dict(out=P + 1)),
    ({}, dict(n_rows=-1)), ({}, dict(ldy=63)), ({}, dict(ldo=63)), (dict(n_tok=1 << 28, ws_bytes=1 << 60), dict(n_rows=1 << 28, ldy=1 << 28, ldo=1 << 28)),
    (dict(n_tok=1, ws_bytes=1 << 60), dict(n_rows=2 ** 31 - 1, ldy=2 ** 31 - 1, ldo=2 ** 31 - 1)), ({}, dict(n_rows=2 ** 30 + 1, ldy=2 ** 30 + 1, ldo=2 ** 30 + 1)),
    (dict(n_tok=2 ** 31 - 1, ws_bytes=1 << 60), dict(n_rows=1 << 14, ldy=1 << 14, ldo=1 << 14)),
])
def test_a_tensor_is_refused(lib, call, change, tensor):
    assert call(lib, change, tensor) == ARG
    assert lib.qlin_last_error()


def test_up_is_refused(lib):
    for t in (dict(up=None), dict(up=P + 2), dict(up_adapters=None), dict(up_adapters=P + 4)):
        assert silu_mul(lib, {}, t) == ARG


def test_number_of_tensors(lib):
    for n in (0, 4, -1):
        assert add(lib, dict(n_mat=n), {}) == ARG
    assert lib.qlin_lora_add_dev(1, None, BF16, 4, 16, P, BF16, P, F32, F32, 64, 4, 64, P, 1 << 30, None) == ARG


@pytest.mark.parametrize("call", [add, silu_mul])
def test_nothing_to_do(lib, call):
    assert call(lib, dict(n_tok=0, X=None, ids=None, ws=None, ws_bytes=0), {}) == qlinear.OK
    assert call(lib, dict(ids=None, ws=None, ws_bytes=0), dict(n_rows=0, Y=None, out=None, adapters=None)) == qlinear.OK


def test_workspace(lib):
    size = lib.qlin_lora_workspace_bytes
    for bad in ((0, 16, 64, 4), (1, 0, 64, 4), (1, 16, 0, 4), (1, 16, 64, 0), (-1, -1, -1, -1)):
        assert size(*bad) == 0
    assert size(1, 16, 64, 4) >= 4 * 16 * 4
    for n_mat in (1, 2, 3):
        for rank in (1, 16, 17, 100, 256):
            for n_tok in (1, 64, 65, 5000):
                assert size(n_mat, rank, 4096, n_tok) >= n_mat * n_tok * rank * 4
    assert size(3, 256, 14336, 1 << 20) <= 3 * 256 * 6 + 160 << 20  # many tokens: the columns are not cut into parts


def test_structures():
    assert qlinear.LORA_DTYPE.itemsize == 24 and C.sizeof(qlinear.LoraTensor) == 40


def test_a_workspace_holds_what_smaller_calls_need(lib):
    rng = np.random.default_rng(3)
    for _ in range(3000):
        large = [int(rng.integers(1, n + 1)) for n in (3, 256, 20000, rng.choice([64, 600, 5000]))]
        small = [int(rng.integers(1, n + 1)) for n in large]
        assert lib.qlin_lora_workspace_bytes(*small) <= lib.qlin_lora_workspace_bytes(*large), (small, large)
