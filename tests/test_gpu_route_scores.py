"""qlin_moe_route_scores_dev against its definition in 64 bits: every score, group and type, rows of which nothing or too little is there,
equal and nearly equal values, one expert to 4096, one token to thousands."""
import numpy as np
import pytest

from gemm_amd import qlinear
from tests import adapter_formulas as f

pytestmark = pytest.mark.gpu
F32, F16, BF16 = f.F32, f.F16, f.BF16
NAN, INF = np.nan, np.inf


def call(x, t, sigmoid, bias, n_group, used, group_top, k, renorm, scale, pad=0, stream=None):
    """x: float rows -> (indices, weights, the logits' values)"""
    n_tok, n = x.shape
    wide = np.full((n_tok, n + pad), 1e4, np.float32)
    wide[:, :n] = x
    raw, v = f.as_type(wide, t)
    dx, db = qlinear.DevBuf.from_numpy(raw), qlinear.DevBuf.from_numpy(np.asarray(bias, np.float32)) if bias is not None else None
    guard = 64
    didx = qlinear.DevBuf.from_numpy(np.full(n_tok * k + guard, 77, np.int32))
    dw = qlinear.DevBuf.from_numpy(np.full(n_tok * k + guard, 77, np.float32))
    qlinear.moe_route_scores_dev(int(sigmoid), t, dx, n_tok, n, n + pad, db, n_group, used, group_top, k, renorm, scale, didx, dw, stream)
    qlinear.sync(stream)
    idx, w = didx.to_numpy(np.int32, (n_tok * k + guard,)), dw.to_numpy(np.float32, (n_tok * k + guard,))
    assert (idx[n_tok * k:] == 77).all() and (w[n_tok * k:] == 77).all()
    return idx[:n_tok * k].reshape(n_tok, k), w[:n_tok * k].reshape(n_tok, k), v[:, :n]


def check(x, t, sigmoid, bias, n_group, used, group_top, k, renorm, scale, pad=0):
    idx, w, v = call(x, t, sigmoid, bias, n_group, used, group_top, k, renorm, scale, pad)
    b = None if bias is None else np.asarray(bias, np.float32).astype(np.float64)
    for row in range(len(x)):
        want_idx, want_w = f.route(v[row], sigmoid, b, n_group, used, group_top, k, renorm, float(np.float32(scale)))
        assert idx[row].tolist() == want_idx.tolist(), row
        assert (np.abs(w[row] - want_w) <= f.route_bound(v[row], sigmoid, want_idx, want_w)).all(), (row, w[row], want_w)
    return idx, w


def rows(seed, n_tok, n, spread=1.5):
    return spread * np.random.default_rng(seed).standard_normal((n_tok, n))


def small_bias(seed, n):
    return 0.05 * np.random.default_rng(seed).standard_normal(n)


@pytest.mark.parametrize("sigmoid", [False, True])
@pytest.mark.parametrize("biased", [False, True])
@pytest.mark.parametrize("t", [F32, F16, BF16])
@pytest.mark.parametrize("n_tok,n,n_group,used,group_top,k,pad", [
    (1, 128, 1, 1, 1, 8, 0), (3, 256, 8, 4, 2, 8, 0), (5, 60, 1, 1, 1, 4, 4), (4, 160, 8, 3, 1, 6, 3), (70, 64, 4, 2, 2, 6, 0), (2, 1, 1, 1, 1, 1, 0), (7, 2, 2, 1, 1, 1, 1),
    (2, 17, 1, 1, 1, 17, 0), (3, 512, 16, 5, 2, 10, 0), (2, 513, 27, 11, 2, 9, 2), (9, 96, 32, 7, 2, 5, 0), (2, 384, 1, 1, 1, 22, 5), (3, 72, 72, 9, 2, 9, 0)])
def test_routes(sigmoid, biased, t, n_tok, n, n_group, used, group_top, k, pad):
    x = rows(n_tok * n + k, n_tok, n)
    check(x, t, sigmoid, small_bias(n, n) if biased else None, n_group, used, group_top, k, biased != sigmoid, 2.5 if sigmoid else 1.0, pad)


@pytest.mark.parametrize("n,n_group,k", [(1024, 1, 64), (1000, 8, 65), (4096, 256, 100), (4096, 1, 4096), (300, 1, 300)])
def test_many_experts_and_places(n, n_group, k):
    check(rows(n, 2, n), F32, True, small_bias(1, n), n_group, max(1, n_group // 2), 2, min(k, n // n_group * max(1, n_group // 2)), True, 1.0)
    check(rows(n, 2, n), BF16, False, None, n_group, n_group, 1, k, False, 1.0)


@pytest.mark.parametrize("n_tok", [64, 65, 1000, 4097])
def test_many_tokens(n_tok):
    check(rows(n_tok, n_tok, 64), F32, True, small_bias(2, 64), 8, 4, 2, 6, True, 2.5)


@pytest.mark.parametrize("sigmoid", [False, True])
@pytest.mark.parametrize("biased", [False, True])
@pytest.mark.parametrize("n,n_group", [(64, 1), (64, 8), (200, 4)])
def test_what_is_not_there(sigmoid, biased, n, n_group):
    """nothing, one expert, fewer than top_k, one group, the type's lowest value, infinities and NaN"""
    x = rows(3, 12, n)
    x[0] = -INF
    x[1] = NAN
    x[2] = -INF
    x[2, n // 2 + 1] = -3.0
    x[3, 3:] = -INF
    x[4, n // n_group:] = NAN
    x[5] = np.finfo(np.float32).min
    x[6, :] = np.finfo(np.float32).min
    x[6, 5:9] = [1.0, 2.0, 0.5, 0.25]
    x[7, [4, 9, 30]] = INF
    x[8, ::2] = NAN
    x[9] = 0.0
    x[10, :n - 1] = -INF
    x[11, 7] = INF
    bias = small_bias(4, n) if biased else None
    if biased:
        bias[[8, 40]] = [-INF, NAN]
    for k in (1, 5, 8):
        for renorm in (False, True):
            check(x, F32, sigmoid, bias, n_group, max(1, n_group // 2), 2, k, renorm, 1.0)
    check(np.where(x < -1e38, -INF, x), BF16, sigmoid, bias, n_group, max(1, n_group // 2), 1, 6, True, 1.0)


@pytest.mark.parametrize("sigmoid", [False, True])
@pytest.mark.parametrize("low", [np.finfo(np.float32).min, -3.4e38, -1e38])
@pytest.mark.parametrize("n,n_group,free,k", [(8, 1, 1, 4), (8, 1, 2, 8), (17, 1, 1, 9), (60, 1, 3, 4), (60, 4, 3, 12), (64, 1, 0, 8), (64, 8, 1, 8), (96, 1, 2, 6), (96, 8, 5, 12),
                                              (160, 1, 4, 8), (160, 8, 9, 16), (160, 16, 2, 16), (256, 8, 6, 8), (256, 1, 1, 17), (257, 1, 1, 12), (512, 16, 3, 10)])
def test_a_bias_of_the_lowest_value(sigmoid, low, n, n_group, free, k):
    """the usual mask, a finite one: its experts come behind all others, by index, and none that is not there comes with them"""
    x = rows(n + k, 6, n)
    order = np.random.default_rng(n).permutation(n)
    bias = small_bias(n, n)
    bias[order[free:]] = low
    x[1, ::3] = -INF
    x[2, order[free:free + n // 2]] = NAN
    x[3] = -INF
    x[4, :n - 1] = -INF
    x[5, order[:free]] = -INF
    used = max(1, n_group // 2)
    for group_top in (1, 2):
        check(x, F32, sigmoid, bias, n_group, used, group_top, k, group_top == 1, 1.0)
    check(x, BF16, sigmoid, bias, n_group, n_group, 1, k, True, 2.5)


@pytest.mark.parametrize("t", [F32, BF16])
@pytest.mark.parametrize("biased", [False, True])
def test_equal_values_go_by_index(t, biased):
    rng = np.random.default_rng(5)
    x = rng.integers(-2, 3, (40, 128)).astype(np.float32)
    bias = rng.integers(0, 2, 128) * 0.25 if biased else None
    for sigmoid in (False, True):
        for group_top in (1, 2):
            check(x, t, sigmoid, bias, 8, 3, group_top, 12, True, 1.0)
            check(x, t, sigmoid, bias, 1, 1, group_top, 12, True, 1.0)


@pytest.mark.parametrize("sigmoid", [False, True])
@pytest.mark.parametrize("n,n_group,k", [(256, 8, 8), (128, 1, 8), (60, 1, 4)])
def test_neighbours(sigmoid, n, n_group, k):
    """values an fp32 step or less apart: the choice is the one of 64 bits"""
    rng = np.random.default_rng(n)
    x = np.float32(0.7) + rng.integers(-3, 4, (64, n)) * np.float32(2.0 ** -24)
    bias = (np.float32(0.3) + rng.integers(-3, 4, n) * np.float32(2.0 ** -25)).astype(np.float32)
    check(x, F32, sigmoid, None, n_group, max(1, n_group // 2), 2, k, True, 1.0)
    check(x, F32, sigmoid, bias, n_group, max(1, n_group // 2), 2, k, True, 1.0)
    check(x, F32, sigmoid, bias, n_group, max(1, n_group // 2), 1, k, False, 1.0)


def test_saturated_sigmoid():
    """scores of 1 in 64 bits stay in the order of their logits without a bias, and go by index with one"""
    x = np.tile(np.linspace(38, 60, 64, dtype=np.float32), (2, 1))
    idx, w = check(x, F32, True, None, 1, 1, 1, 5, False, 1.0)
    assert idx[0].tolist() == [63, 62, 61, 60, 59]
    idx, w = check(x, F32, True, np.zeros(64), 1, 1, 1, 5, False, 1.0)
    assert idx[0].tolist() == [0, 1, 2, 3, 4]
    x = np.tile(np.linspace(-120, -60, 64, dtype=np.float32), (2, 1))
    check(x, F32, True, np.zeros(64), 1, 1, 1, 5, True, 1.0)
    check(x, F32, False, np.zeros(64), 1, 1, 1, 5, True, 1.0)


def shares(x, sigmoid, idx):
    """the weights of the chosen experts, renormalised to 1, from the logarithms of their scores (up to what all have in common): right however small
    the scores are; and how far fp32 may be off: the exponential's argument is the distance to the largest, rounded, besides as in route_bound"""
    there = idx >= 0
    v = np.where(there, x[np.maximum(idx, 0)], 0.0)
    log = np.where(there, (np.minimum(v, 0.0) - np.log1p(np.exp(-np.abs(v)))) if sigmoid else v, -np.inf)
    far = np.where(there, log.max() - log, 0.0)
    w = np.where(there, np.exp(-far), 0.0)
    w = w / w.sum()
    return w, 2.0 ** -23 * (far + far.max() + 24.0) * w + 2.0 ** -126


@pytest.mark.parametrize("k", [1, 5, 16, 17, 64])  # 16 lanes to a token, a wave
@pytest.mark.parametrize("t", [F32, BF16])
def test_renormalised_scores_below_fp32(k, t):
    """all chosen scores denormal in fp32 or 0 there: the weights are those of the definition all the same; 0 where the scores are 0 in 64 bits too"""
    rng = np.random.default_rng(k)
    n, n_tok = 96, 9
    x = rng.uniform(-104, -86, (n_tok, n))
    x[1] = rng.uniform(-300, -90, n)
    x[2] = rng.uniform(-130, -110, n)
    x[3] = rng.uniform(-2000, -800, n)
    x[4, :90] = -INF
    x[5] = rng.uniform(-20, 3, n)
    x[6] = rng.uniform(-100.0, -99.0, n)
    x[7, 0] = 1.0
    x[8] = -90.0
    far = rng.standard_normal((n_tok, n))
    far[:, 17] = np.linspace(60.0, 2000.0, n_tok)
    far[8, 17] = INF
    dominant = rng.permutation(n) / 8.0 + 1.0  # decides alone, in 64 bits too
    without = dominant.copy()
    without[17] = -INF
    for x, sigmoid, bias in ((x, True, None), (x, True, dominant), (far, False, without)):
        idx, w, v = call(x, t, sigmoid, bias, 1, 1, 1, k, True, 2.5)
        for row in range(n_tok):
            want_idx, _ = f.route(v[row], sigmoid, bias, 1, 1, 1, k, True, 2.5)
            assert idx[row].tolist() == want_idx.tolist()
            want, bound = shares(v[row], sigmoid, want_idx)
            if not f.scores(v[row], sigmoid)[want_idx[want_idx >= 0]].any():
                want = bound = 0.0 * want
            assert (np.abs(w[row] - 2.5 * want) <= 2.5 * bound).all(), (row, w[row], 2.5 * want)


def test_agrees_with_the_plain_router():
    """softmax over all, top_k, renormalised is what qlin_moe_route_dev does, but for its order among equal ones"""
    x = rows(8, 33, 128).astype(np.float32)
    idx, w, _ = call(x, F32, False, None, 1, 1, 1, 8, True, 1.0)
    d = [qlinear.DevBuf.from_numpy(x), qlinear.DevBuf(33 * 8 * 4), qlinear.DevBuf(33 * 8 * 4)]
    qlinear.moe_route_dev(d[0], 33, 128, 8, d[1], d[2])
    qlinear.sync()
    assert np.array_equal(d[1].to_numpy(np.int32, (33, 8)), idx)
    assert np.abs(d[2].to_numpy(np.float32, (33, 8)) - w).max() <= 2.0 ** -19  # both in fp32, logits of at most 8: 2^-23 (8 + 8 + 24) and less than half


def test_same_bits_again():
    x = rows(9, 500, 256)
    a = call(x, F32, True, small_bias(1, 256), 8, 4, 2, 8, True, 2.5)
    b = call(x, F32, True, small_bias(1, 256), 8, 4, 2, 8, True, 2.5)
    assert np.array_equal(a[0], b[0]) and np.array_equal(a[1], b[1])
    for n in (1, 3, 64):  # and a token's result does not depend on the others
        c = call(x[:n], F32, True, small_bias(1, 256), 8, 4, 2, 8, True, 2.5)
        assert np.array_equal(a[0][:n], c[0]) and np.array_equal(a[1][:n], c[1])


@pytest.mark.parametrize("biased", [False, True])
@pytest.mark.parametrize("n,n_group,k", [(256, 1, 16), (250, 1, 16), (512, 1, 16), (256, 8, 12), (256, 16, 16), (100, 1, 12)])
def test_all_picks_among_neighbouring_experts(biased, n, n_group, k):
    """the largest values stand next to each other, a step of 64 bits apart, equal and far ones among them"""
    rng = np.random.default_rng(n + k)
    x = rng.standard_normal((24, n)) * 0.1
    for row in range(24):
        at = rng.integers(0, n - 20)
        x[row, at:at + 20] = 2.0 + rng.integers(0, 3, 20) * [2.0 ** -24, 2.0 ** -20, 0.01, 0.0][row % 4]
    bias = np.where(rng.random(n) < 0.5, 0.25, 0.25 + 2.0 ** -25) if biased else None
    for sigmoid in (False, True):
        check(x, F32, sigmoid, bias, n_group, max(1, n_group // 2), 2, k, True, 1.0)
        check(x, F16, sigmoid, bias, n_group, n_group, 1, k, True, 1.0)


@pytest.mark.parametrize("n,k", [(60, 4), (60, 17)])  # 16 lanes to a token, a wave
def test_rows_far_apart(n, k):
    """rows 2^27 elements apart: offsets that 32 bits do not hold"""
    n_tok, pitch = 20, 1 << 27
    x = rows(5, n_tok, n).astype(np.float32)
    want = call(x, F32, False, None, 1, 1, 1, k, True, 1.0)
    far = qlinear.DevBuf(((n_tok - 1) * pitch + n) * 4)
    for t in range(n_tok):
        qlinear.check(qlinear.load().qlin_dev_upload(far.ptr + t * pitch * 4, x[t].ctypes.data, n * 4))
    idx, w = qlinear.DevBuf(n_tok * k * 4), qlinear.DevBuf(n_tok * k * 4)
    qlinear.moe_route_scores_dev(qlinear.ROUTE_SOFTMAX, F32, far, n_tok, n, pitch, None, 1, 1, 1, k, True, 1.0, idx, w)
    qlinear.sync()
    assert np.array_equal(idx.to_numpy(np.int32, (n_tok, k)), want[0]) and np.array_equal(w.to_numpy(np.float32, (n_tok, k)), want[1])


@pytest.mark.parametrize("n,n_group,k", [(256, 8, 8), (60, 1, 17)])
def test_in_a_graph(n, n_group, k):
    """captured once, replayed on other logits, with eager calls between"""
    import ctypes as C
    hip = C.CDLL("libamdhip64.so")
    n_tok, used = 33, max(1, n_group // 2)
    bias = small_bias(3, n).astype(np.float32)
    dx, db = qlinear.DevBuf(n_tok * n * 4), qlinear.DevBuf.from_numpy(bias)
    idx, w = qlinear.DevBuf(n_tok * k * 4), qlinear.DevBuf(n_tok * k * 4)
    stream, graph, gexec = C.c_void_p(), C.c_void_p(), C.c_void_p()
    qlinear.check(qlinear.load().qlin_init(0))
    assert hip.hipStreamCreate(C.byref(stream)) == 0
    assert hip.hipStreamBeginCapture(stream, 0) == 0
    qlinear.moe_route_scores_dev(qlinear.ROUTE_SIGMOID, F32, dx, n_tok, n, n, db, n_group, used, 2, k, True, 2.5, idx, w, stream)
    assert hip.hipStreamEndCapture(stream, C.byref(graph)) == 0
    assert hip.hipGraphInstantiate(C.byref(gexec), graph, None, None, C.c_size_t(0)) == 0
    for replay in range(4):
        x = np.ascontiguousarray(rows(replay, n_tok, n), np.float32)
        qlinear.check(qlinear.load().qlin_dev_upload(dx.ptr, x.ctypes.data, x.nbytes))
        assert hip.hipGraphLaunch(gexec, stream) == 0 and hip.hipStreamSynchronize(stream) == 0
        want = call(x, F32, True, bias, n_group, used, 2, k, True, 2.5)
        assert np.array_equal(idx.to_numpy(np.int32, (n_tok, k)), want[0]) and np.array_equal(w.to_numpy(np.float32, (n_tok, k)), want[1])
    assert hip.hipGraphExecDestroy(gexec) == 0 and hip.hipGraphDestroy(graph) == 0 and hip.hipStreamDestroy(stream) == 0
