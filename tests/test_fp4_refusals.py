"""What the 4-bit products and the sampler refuse, before anything reaches the GPU (these calls return without one), and what their
size functions say."""
import pytest

from gemm_amd import qlinear

F32, F16, BF16, MXFP4, Q4K = 0, 1, 30, 39, 12
P = 0x10000  # an aligned address that no refused call reads
ARG, TYPE = qlinear.ERR_ARG, qlinear.ERR_TYPE


@pytest.fixture(scope="module")
def lib():
    return qlinear.load()


def test_operand_bytes(lib):
    one = 1024 + 256
    assert lib.qlin_mxfp4_operand_bytes(1, 1) == one == lib.qlin_mxfp4_operand_bytes(16, 128)
    assert lib.qlin_mxfp4_operand_bytes(17, 128) == 2 * one
    assert lib.qlin_mxfp4_operand_bytes(16, 129) == 2 * 1024 + 256
    assert lib.qlin_mxfp4_operand_bytes(16, 513) == 5 * 1024 + 2 * 256
    assert lib.qlin_mxfp4_operand_bytes(14336, 4096) == 14336 * 4096 // 32 * 17
    assert lib.qlin_mxfp4_operand_bytes(2 ** 31 - 1, 2 ** 20) == 2 ** 31 * 2 ** 15 * 17
    for r, c in ((0, 5), (5, 0), (-1, 5), (5, -1)):
        assert lib.qlin_mxfp4_operand_bytes(r, c) == 0 == lib.qlin_mxfp4_gemm_workspace_bytes(c, r)
    assert lib.qlin_mxfp4_gemm_workspace_bytes(4096, 33) == lib.qlin_mxfp4_operand_bytes(33, 4096)
    assert lib.qlin_sample_workspace_bytes(0, 100) == 0 == lib.qlin_sample_workspace_bytes(4, 0) == lib.qlin_sample_workspace_bytes(-1, -1)


@pytest.mark.parametrize("code,args", [
    (TYPE, (MXFP4, P, P, 4, 64, 64)), (TYPE, (Q4K, P, P, 4, 64, 64)), (TYPE, (99, P, P, 4, 64, 64)),
    (ARG, (F32, P, P, 4, 65, 65)), (ARG, (F32, P, P, 4, 64, 63)), (ARG, (F32, P, P, -1, 64, 64)), (ARG, (F32, P, P, 4, -32, 64)),
    (ARG, (F32, None, P, 4, 64, 64)), (ARG, (F32, P, None, 4, 64, 64)), (ARG, (F32, P + 2, P, 4, 64, 64)), (ARG, (BF16, P + 1, P, 4, 64, 64)),
])
def test_quantize_refuses(lib, code, args):
    assert lib.qlin_quantize_mxfp4_dev(*args, None) == code
    assert lib.qlin_last_error()


@pytest.mark.parametrize("code,args", [
    (TYPE, (Q4K, P, P, 4, 256, 256)), (ARG, (MXFP4, P, P, 4, 65, 65)), (ARG, (MXFP4, P, P, 4, 64, 96)), (ARG, (MXFP4, None, P, 4, 64, 64)), (ARG, (F32, P, P, 4, 64, 60)),
    (ARG, (F32, P, P + 8, 4, 64, 64)), (ARG, (F32, P, None, 4, 64, 64)), (ARG, (F16, P + 1, P, 4, 64, 64)), (ARG, (F32, P, P, -4, 64, 64)), (ARG, (MXFP4, P, P, -4, 64, 64)),
    (ARG, (F32, P, P, 4, 1 << 24, 1 << 24)), (ARG, (F32, P, P, 2 ** 31 - 1, 1 << 20, 1 << 20)),
])
def test_operand_refuses(lib, code, args):
    assert lib.qlin_mxfp4_operand_dev(*args, None) == code
    assert lib.qlin_last_error()


GOOD = dict(W=P, up=P, x_type=BF16, X=P, y_type=F32, Y=P, n_rows=64, n_cols=128, n_tok=4, ldx=128, ldy=64, ws=P, ws_bytes=1 << 20)


@pytest.mark.parametrize("pair", [False, True])
@pytest.mark.parametrize("code,change", [
    (TYPE, dict(x_type=Q4K)), (TYPE, dict(y_type=F16)), (TYPE, dict(y_type=MXFP4)), (ARG, dict(n_rows=-1)), (ARG, dict(n_cols=0)), (ARG, dict(n_cols=-128)), (ARG, dict(n_tok=-1)),
    (ARG, dict(ldy=63)), (ARG, dict(ldx=127)), (ARG, dict(W=None)), (ARG, dict(W=P + 8)), (ARG, dict(X=None)), (ARG, dict(X=P + 1)), (ARG, dict(x_type=MXFP4, X=P + 4)),
    (ARG, dict(Y=None)), (ARG, dict(Y=P + 2)), (ARG, dict(y_type=BF16, Y=P + 1)), (ARG, dict(ws=None)), (ARG, dict(ws=P + 8)), (ARG, dict(ws_bytes=1279)),
    (ARG, dict(n_cols=1 << 24, ldx=1 << 24)), (ARG, dict(n_rows=2 ** 31 - 1, n_tok=2 ** 31 - 1, ldy=2 ** 31 - 1)),
])
def test_products_refuse(lib, pair, code, change):
    a = dict(GOOD, **change)
    call = lib.qlin_mxfp4_gemm_silu_mul_dev if pair else lib.qlin_mxfp4_gemm_dev
    rc = call(*([a["W"], a["up"]] if pair else [a["W"]]), a["x_type"], a["X"], a["y_type"], a["Y"], a["n_rows"], a["n_cols"], a["n_tok"], a["ldx"], a["ldy"], a["ws"], a["ws_bytes"], None)
    assert rc == code
    assert lib.qlin_last_error()


def test_gate_and_up_refuse_a_missing_operand(lib):
    for up in (None, P + 4):
        assert lib.qlin_mxfp4_gemm_silu_mul_dev(P, up, BF16, P, F32, P, 64, 128, 4, 128, 64, P, 1 << 20, None) == ARG


@pytest.mark.parametrize("code,change", [
    (TYPE, dict(type=Q4K)), (ARG, dict(n_seq=-1)), (ARG, dict(n_vocab=-1)), (ARG, dict(n_vocab=0)), (ARG, dict(n_vocab=(1 << 30) + 1, ld=(1 << 31) - 1)), (ARG, dict(ld=99)), (ARG, dict(logits=None)), (ARG, dict(logits=P + 2)),
    (ARG, dict(u=None)), (ARG, dict(ids=None)), (ARG, dict(u=P + 2)), (ARG, dict(ids=P + 1)), (ARG, dict(probs=P + 2)), (ARG, dict(t=P + 2)), (ARG, dict(k=P + 2)), (ARG, dict(p=P + 2)),
    (ARG, dict(m=P + 2)), (ARG, dict(n_vocab=100000, ld=100000, ws=None)), (ARG, dict(n_vocab=100000, ld=100000, ws=P + 128)), (ARG, dict(n_vocab=100000, ld=100000, ws_bytes=1000)),
])
def test_sample_refuses(lib, code, change):
    a = dict(dict(type=F32, logits=P, n_seq=4, n_vocab=100, ld=100, t=P, k=P, p=P, m=P, u=P, ids=P, probs=P, ws=P, ws_bytes=1 << 30), **change)
    assert lib.qlin_sample_dev(*[a[n] for n in ("type", "logits", "n_seq", "n_vocab", "ld", "t", "k", "p", "m", "u", "ids", "probs", "ws", "ws_bytes")], None) == code
    assert lib.qlin_last_error()


@pytest.mark.parametrize("args", [(F32, P, P, 1 << 28, 128, 128), (F32, P, P, 2 ** 31 - 1, 1, 1), (MXFP4, P, P, 1 << 28, 32, 32), (BF16, P, P, 1 << 20, 1 << 19, 1 << 19)])
def test_operands_of_more_workgroups_than_a_launch_takes(lib, args):
    """a launch has less than 2^32 threads, 256 for each 16 rows of 512 columns"""
    assert lib.qlin_mxfp4_operand_dev(*args, None) == ARG


@pytest.mark.parametrize("pair", [False, True])
@pytest.mark.parametrize("change", [dict(n_rows=2 ** 31 - 1, n_cols=1, n_tok=1, ldy=2 ** 31 - 1), dict(n_rows=1 << 27, n_tok=1, ldy=1 << 27), dict(n_rows=1 << 27, n_tok=16, ldy=1 << 27),
                                    dict(n_rows=17, n_tok=2 ** 31 - 1, x_type=MXFP4), dict(n_rows=1 << 26, n_tok=1 << 26, ldy=1 << 26, x_type=MXFP4)])
def test_products_of_more_workgroups_than_a_launch_takes(lib, pair, change):
    a = dict(GOOD, ws_bytes=1 << 60, **change)
    call = lib.qlin_mxfp4_gemm_silu_mul_dev if pair else lib.qlin_mxfp4_gemm_dev
    rc = call(*([a["W"], a["up"]] if pair else [a["W"]]), a["x_type"], a["X"], a["y_type"], a["Y"], a["n_rows"], a["n_cols"], a["n_tok"], a["ldx"], a["ldy"], a["ws"], a["ws_bytes"], None)
    assert rc == ARG


@pytest.mark.parametrize("n_seq", [1 << 22, 2 ** 31 - 1])
def test_more_sequences_than_a_launch_takes(lib, n_seq):
    """1024 threads for each"""
    assert lib.qlin_sample_dev(F32, P, n_seq, 100, 100, None, None, None, None, P, P, None, None, 0, None) == ARG


def test_blocks_of_more_workgroups_than_a_launch_takes(lib):
    """256 blocks for each"""
    assert lib.qlin_quantize_mxfp4_dev(BF16, P, P, 1 << 17, 1 << 20, 1 << 20, None) == ARG
