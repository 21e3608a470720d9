"""Sampling on the GPU through the C ABI against a sorted list in 64 bits. The pick is compared as it is: a random number within 2^-40
of a border between two tokens (relative to the sum; integer weights of 2^-44 and their sums are off by less) is moved off it
before the call."""
import numpy as np
import pytest

from gemm_amd import qlinear
import synth
from tests import fp4_formulas as f

pytestmark = pytest.mark.gpu
F32, F16, BF16 = 0, 1, 30


def typed(x, type_id):
    a = np.asarray(x, np.float32)
    if type_id == F16:
        with np.errstate(over="ignore"):
            a = a.astype(np.float16)
        return a, a.astype(np.float64)
    if type_id == BF16:
        a = synth.to_bf16_bits(a)
        return a, synth.bf16_bits_to_f32(a).astype(np.float64)
    return a, a.astype(np.float64)


def device(a, dtype):
    return None if a is None else qlinear.DevBuf.from_numpy(np.asarray(a, dtype))


def draw(type_id, a, u, t=None, k=None, p=None, m=None, probs=True):
    """-> ids, probs"""
    n_seq, ld = a.shape
    n = draw.vocab or ld
    ids, pr = qlinear.DevBuf.from_numpy(np.full(n_seq + 4, -77, np.int32)), qlinear.DevBuf.from_numpy(np.full(n_seq + 4, 7.5, np.float32))
    need = qlinear.sample_workspace_bytes(n_seq, n)
    ws = qlinear.DevBuf.from_numpy(np.full(need + 256, 0xA5, np.uint8))
    dl = qlinear.DevBuf.from_numpy(a)
    opts = [device(t, np.float32), device(k, np.int32), device(p, np.float32), device(m, np.float32), device(u, np.float32)]
    qlinear.sample_dev(type_id, dl, n_seq, n, ld, *opts, ids, pr if probs else None, ws)
    qlinear.sync()
    assert (ws.to_numpy(np.uint8, (need + 256,))[need:] == 0xA5).all()
    got, got_p = ids.to_numpy(np.int32, (n_seq + 4,)), pr.to_numpy(np.float32, (n_seq + 4,))
    assert (got[n_seq:] == -77).all() and (got_p[n_seq if probs else 0:] == 7.5).all()
    return got[:n_seq], got_p[:n_seq]


draw.vocab = None


def compare(type_id, logits, u, t=None, k=None, p=None, m=None, vocab=None):
    a, x = typed(logits, type_id)
    n = vocab or a.shape[1]
    u = np.array(u, np.float32)
    want = []
    for s in range(len(a)):
        row = dict(t=1.0 if t is None else np.float32(t[s]), k=0 if k is None else k[s], p=1.0 if p is None else np.float32(p[s]), m=0.0 if m is None else np.float32(m[s]))
        for _ in range(20):  # a random number on a border goes to the middle between its neighbours
            one = f.sample(x[s, :n], u=u[s], **row)
            if one[2] > 2.0 ** -40 or u[s] <= 0 or u[s] >= 1:
                break
            u[s] = np.float32(u[s] * np.float32(0.999))
        want.append(one)
    draw.vocab = n
    ids, probs = draw(type_id, a, u, t, k, p, m)
    draw.vocab = None
    assert ids.tolist() == [w[0] for w in want]
    # the weight and the sum are off by 2^-40 at most, the quotient is rounded once to fp32
    want_p = np.array([w[1] for w in want])
    assert (np.abs(probs - want_p) <= 2.0 ** -23 * want_p + 2.0 ** -40).all(), (probs, want_p)


def random_logits(rng, n_seq, n, sigma=2.0, peaks=8):
    x = rng.standard_normal((n_seq, n)) * sigma
    for s in range(n_seq):
        x[s, rng.integers(0, n, min(peaks, n))] += 6.0
    return x


def random_settings(rng, n_seq):
    return dict(t=rng.choice([0.0, 0.2, 0.7, 1.0, 1.0, 1.7], n_seq), k=rng.choice([0, 0, 1, 2, 20, 50, 1000], n_seq), p=rng.choice([1.0, 0.0, 0.3, 0.9, 0.95, 0.999], n_seq),
                m=rng.choice([0.0, 0.0, 0.02, 0.1, 0.5, 1.0], n_seq))


@pytest.mark.parametrize("type_id", [F32, F16, BF16])
@pytest.mark.parametrize("n_seq,n,pad", [(1, 1, 0), (3, 2, 1), (5, 7, 0), (9, 63, 0), (4, 64, 3), (7, 65, 0), (40, 1000, 0), (12, 1025, 7), (33, 4097, 0), (300, 500, 0), (2, 32003, 0),
                                         (3, 32768, 64), (1, 151936, 0), (5, 128256, 8),
                                         (8, 65536, 0), (9, 65536, 3), (20, 16383, 0), (66, 70000, 0), (8, 65541, 1)])
def test_picks(type_id, n_seq, n, pad):
    rng = np.random.default_rng(n_seq * 1000 + n)
    x = np.pad(random_logits(rng, n_seq, n), ((0, 0), (0, pad)), constant_values=99.0)  # what lies behind a row is larger than all of it
    compare(type_id, x, rng.random(n_seq), vocab=n)
    for _ in range(2):
        compare(type_id, x, rng.random(n_seq), **random_settings(rng, n_seq), vocab=n)


@pytest.mark.parametrize("name,value", [("k", 5), ("k", 40), ("k", 128), ("k", 129), ("k", 512), ("k", 600), ("k", 1024), ("k", 1025), ("k", 5000), ("p", 0.9), ("p", 0.5), ("p", 0.0), ("p", -1.0), ("m", 0.05), ("m", 1.0), ("m", 2.0), ("t", 0.0), ("t", -1.0),
                                        ("t", 100.0), ("t", 1e-3), ("t", np.inf), ("t", np.nan), ("p", np.nan), ("m", np.nan), ("k", -3)])
@pytest.mark.parametrize("n_seq,n", [(16, 5000), (8, 66000), (70, 20000)])  # by one workgroup per sequence, by several, and by one
def test_one_setting(n_seq, n, name, value):
    rng = np.random.default_rng(11)
    compare(F32, random_logits(rng, n_seq, n), rng.random(n_seq), **{name: [value] * n_seq})


@pytest.mark.parametrize("rows,n", [(24, 50), (24, 3000), (24, 40000), (8, 66000)])
def test_equal_logits(rows, n):
    """equal tokens: the lower index first, wherever a cut falls between them"""
    rng = np.random.default_rng(n)
    few = rng.integers(0, 4, (rows, n)).astype(np.float64)  # four values
    flat = np.full((rows, n), -3.25)
    zeros = np.where(rng.random((rows, n)) < 0.5, 0.0, -0.0)
    for x in (few, flat, zeros):
        for type_id in (F32, BF16):
            u = rng.random(rows)
            compare(type_id, x, u)
            compare(type_id, x, u, **random_settings(rng, rows))
            compare(type_id, x, u, k=rng.integers(2, n + 5, rows))


@pytest.mark.parametrize("n", [3001, 66001])
def test_masks(n):
    """tokens that are ruled out by -infinity or NaN, or pushed down to the type's lowest value; rows of which nothing is left"""
    rng = np.random.default_rng(5)
    x = random_logits(rng, 14, n)
    x[0] = -np.inf
    x[1] = np.nan
    x[2, 1:] = -np.inf
    x[3, :-1] = np.nan
    x[4, ::2] = -np.inf
    x[5, 1::2] = np.nan
    x[6, 10:] = np.finfo(np.float32).min
    x[7] = np.finfo(np.float32).min
    x[8, 100] = np.inf
    x[9, [5, 900, 2000]] = np.inf
    x[10, :] = -np.inf
    x[10, 17] = np.finfo(np.float32).min
    x[11, 3:] = -1e30
    x[12] = np.where(rng.random(n) < 0.5, np.finfo(np.float32).max, np.finfo(np.float32).min)
    x[13, :] = 1e-40  # subnormal logits
    x[13, 7] = 2e-40
    for rows in (slice(0, 14), slice(0, 7), slice(7, 14)):  # the halves by several workgroups per row where rows are long
        m = len(x[rows])
        compare(F32, x[rows], rng.random(m))
        for _ in range(4):
            compare(F32, x[rows], rng.random(m), **random_settings(rng, m))
    lowest = random_logits(rng, 4, n)
    lowest[:, 20:] = -65504.0
    compare(F16, lowest, rng.random(4), p=[0.9] * 4)
    lowest[:, 20:] = -3.3895314e38
    compare(BF16, lowest, rng.random(4), k=[50] * 4)


def test_random_numbers_at_the_ends():
    rng = np.random.default_rng(6)
    x = random_logits(rng, 8, 2000)
    u = [0.0, 1.0 - 2.0 ** -24, 1.0, 5.0, -1.0, np.nan, np.inf, 1e-38]
    compare(F32, x, u)
    compare(F32, x, u, k=[30] * 8, p=[0.9] * 8, m=[0.01] * 8)


def test_frequencies_follow_the_weights():
    """20000 draws of one row: every token's share within five standard deviations of its probability"""
    rng = np.random.default_rng(12)
    n, draws = 40, 20000
    row = rng.standard_normal(n)
    u = (np.arange(draws) + 0.5) / draws
    a = np.tile(row.astype(np.float32), (draws, 1))
    ids, _ = draw(F32, a, u, t=[0.8] * draws)
    w = np.exp((row - row.max()) / np.float32(0.8))
    p = w / w.sum()
    share = np.bincount(ids, minlength=n) / draws
    assert (np.abs(share - p) <= 5 * np.sqrt(p / draws)).all()


def test_no_probabilities_and_no_settings():
    rng = np.random.default_rng(2)
    x = random_logits(rng, 5, 700).astype(np.float32)
    u = rng.random(5).astype(np.float32)
    ids, _ = draw(F32, x, u, probs=False)
    assert ids.tolist() == [f.sample(x[s], u=u[s])[0] for s in range(5)]


def test_greedy_is_the_greedy_pick():
    """temperature 0 takes the token that qlin_gemv_argmax_dev takes"""
    K, V = 512, 6000
    W = synth.make_weights(synth.GGML_Q4_K, V, K, seed=1)
    dW, dx = qlinear.DevBuf.from_numpy(W), qlinear.DevBuf.from_numpy(synth.make_activation(K, seed=2))
    dl, dr = qlinear.DevBuf(V * 4), qlinear.DevBuf(qlinear.ARGMAX_RESULT_BYTES)
    qlinear.gemv_argmax_dev(synth.GGML_Q4_K, dW, dx, dl, dr, V, K)
    qlinear.sync()
    ids, probs = draw(F32, dl.to_numpy(np.float32, (1, V)), [0.7], t=[0.0])
    assert ids[0] == dr.to_numpy(np.int32, (2,))[0] and probs[0] == 1.0


@pytest.mark.parametrize("n_seq", [1, 70])
def test_same_token_every_time(n_seq):
    rng = np.random.default_rng(3)
    x = random_logits(rng, n_seq, 20000).astype(np.float32)
    u = rng.random(n_seq)
    s = random_settings(rng, n_seq)
    first = draw(F32, x, u, **s)
    for _ in range(3):
        again = draw(F32, x, u, **s)
        assert np.array_equal(again[0], first[0]) and np.array_equal(again[1], first[1])


@pytest.mark.parametrize("type_id,n", [(F32, 40960), (BF16, 81920), (F16, 20483)])
def test_top_k_where_few_threads_hold_tokens(type_id, n):
    """one workgroup's thread reads 16 bytes in every 16 KB: rows whose tokens, or whose large ones, are a few threads'; rows that fall off so
    fast that the 64th token weighs nothing; the largest tokens at the very ends"""
    rng = np.random.default_rng(n)
    per = 4 if type_id == F32 else 8
    thread = np.arange(n) // per % 1024
    x = random_logits(rng, 18, n)
    for s, mine in enumerate(([0], [5], [1023], [0, 512], list(range(40)), list(range(63)))):
        x[s, ~np.isin(thread, mine)] = -np.inf
        x[6 + s, np.isin(thread, mine)] += 15.0
    x[12] = -np.arange(n) * 0.5
    x[13] = np.arange(n) * 0.5
    x[14, :3] = x[14, -3:] = 40.0
    x[15, :] = -np.inf
    x[15, -1] = 3.0
    x[16] = np.where(thread == 7, x[16], -50.0)
    x[17] = 8.0 - 4.0 * (thread == 1)
    for k in (2, 40, 64, 512):
        for t in (1.0, 0.05, 30.0):
            u = rng.random(18)
            compare(type_id, x, u, t=[t] * 18, k=[k] * 18)
            compare(type_id, x, u, t=[t] * 18, k=[k] * 18, p=[0.9] * 18, m=[0.02] * 18)
