"""The 4-bit products and the sampler together, as an engine runs them: activations to an operand, gate and up with their
activation, the down projection, the output projection, the sampled tokens and their embeddings - eager, captured in a graph that is
replayed between other work, and on two streams from two threads at once. Every step is compared with its own definition in 64 bits on
what the step before really gave."""
import ctypes as C
import threading

import numpy as np
import pytest

from gemm_amd import qlinear
import synth
from tests import fp4_formulas as f
from tests.test_gpu_mxfp4 import activations, as_type, gated

pytestmark = pytest.mark.gpu
F32, BF16, MXFP4 = 0, 30, synth.GGML_MXFP4
HIDDEN, FFN, VOCAB = 512, 1056, 2080


class Model:
    def __init__(self, seed=1):
        shapes = {"gate": (FFN, HIDDEN), "up": (FFN, HIDDEN), "down": (HIDDEN, FFN), "head": (VOCAB, HIDDEN)}
        self.blocks = {n: synth.make_weights(MXFP4, *s, seed=seed + i) for i, (n, s) in enumerate(shapes.items())}
        self.raw = {n: qlinear.DevBuf.from_numpy(b) for n, b in self.blocks.items()}
        self.op = {}
        for n, (rows, cols) in shapes.items():
            self.op[n] = qlinear.DevBuf(qlinear.mxfp4_operand_bytes(rows, cols))
            qlinear.mxfp4_operand_dev(MXFP4, self.raw[n], self.op[n], rows, cols, cols)
        qlinear.sync()


class Step:
    """the buffers of one sequence batch and the calls on them"""

    def __init__(self, model, tokens, seed):
        self.m, self.n = model, tokens
        rng = np.random.default_rng(seed)
        self.x_host = as_type(activations(tokens, HIDDEN, seed) * 0.1, BF16)[0]
        self.settings = [rng.choice([0.0, 0.7, 1.0, 1.4], tokens).astype(np.float32), rng.choice([0, 1, 20, 300], tokens).astype(np.int32),
                         rng.choice([1.0, 0.9, 0.5], tokens).astype(np.float32), rng.choice([0.0, 0.05], tokens).astype(np.float32), rng.random(tokens).astype(np.float32)]
        self.x = qlinear.DevBuf.from_numpy(self.x_host)
        self.set = [qlinear.DevBuf.from_numpy(a) for a in self.settings]
        self.x_op = qlinear.DevBuf(qlinear.mxfp4_operand_bytes(tokens, HIDDEN))
        self.h, self.y, self.logits = qlinear.DevBuf(tokens * FFN * 2), qlinear.DevBuf(tokens * HIDDEN * 4), qlinear.DevBuf(tokens * VOCAB * 4)
        self.ids, self.probs, self.next = qlinear.DevBuf(tokens * 4), qlinear.DevBuf(tokens * 4), qlinear.DevBuf(tokens * HIDDEN * 4)
        self.ws = qlinear.DevBuf(max(qlinear.mxfp4_gemm_workspace_bytes(FFN, tokens), qlinear.sample_workspace_bytes(tokens, VOCAB), 256))

    def enqueue(self, stream):
        m, n = self.m, self.n
        qlinear.mxfp4_operand_dev(BF16, self.x, self.x_op, n, HIDDEN, HIDDEN, stream)
        qlinear.mxfp4_gemm_silu_mul_dev(m.op["gate"], m.op["up"], MXFP4, self.x_op, BF16, self.h, FFN, HIDDEN, n, 0, FFN, None, stream)
        qlinear.mxfp4_gemm_dev(m.op["down"], BF16, self.h, F32, self.y, HIDDEN, FFN, n, FFN, HIDDEN, self.ws, stream)
        qlinear.mxfp4_gemm_dev(m.op["head"], F32, self.y, F32, self.logits, VOCAB, HIDDEN, n, HIDDEN, VOCAB, self.ws, stream)
        qlinear.sample_dev(F32, self.logits, n, VOCAB, VOCAB, *self.set, self.ids, self.probs, self.ws, stream)
        qlinear.embed_rows_dev(MXFP4, m.raw["head"], VOCAB, self.ids, n, self.next, HIDDEN, stream)

    def results(self):
        n = self.n
        return [self.h.to_numpy(np.uint16, (n, FFN)), self.y.to_numpy(np.float32, (n, HIDDEN)), self.logits.to_numpy(np.float32, (n, VOCAB)), self.ids.to_numpy(np.int32, (n,)),
                self.probs.to_numpy(np.float32, (n,)), self.next.to_numpy(np.float32, (n, HIDDEN))]

    def wipe(self):
        for b in (self.x_op, self.h, self.y, self.logits, self.ids, self.probs, self.next, self.ws):
            fill = np.full(b.nbytes, 0xFF, np.uint8)
            assert qlinear.load().qlin_dev_upload(b.ptr, fill.ctypes.data, fill.nbytes) == 0

    def check(self):
        h, y, logits, ids, probs, nxt = self.results()
        w = {n: f.values_of(b) for n, b in self.m.blocks.items()}
        xq = f.values_of(f.quantized(synth.bf16_bits_to_f32(self.x_host).astype(np.float64)))
        want, bound = gated(xq, w["gate"], w["up"])
        h64 = synth.bf16_bits_to_f32(h).astype(np.float64)
        assert (np.abs(h64 - want) <= bound * (1 + 2.0 ** -8) + 2.0 ** -8 * np.abs(want)).all()
        hq = f.values_of(f.quantized(h64))
        assert (np.abs(y - hq @ w["down"].T) <= f.product_bound(hq, w["down"])).all()
        yq = f.values_of(f.quantized(y.astype(np.float64)))
        assert (np.abs(logits - yq @ w["head"].T) <= f.product_bound(yq, w["head"])).all()
        t, k, p, m, u = self.settings
        for s in range(self.n):
            one = f.sample(logits[s], t[s], k[s], p[s], m[s], u[s])
            assert one[2] <= 2.0 ** -40 or ids[s] == one[0]  # (a random number on a border between two tokens may take either)
            assert ids[s] != one[0] or abs(probs[s] - one[1]) <= 2.0 ** -23 * one[1] + 2.0 ** -40
        assert np.array_equal(nxt, qlinear.dequant_rows(MXFP4, self.m.blocks["head"][ids], self.n, HIDDEN))


@pytest.fixture(scope="module")
def model():
    return Model()


@pytest.mark.parametrize("tokens", [1, 3, 16, 70, 200])
def test_a_step(model, tokens):
    s = Step(model, tokens, seed=tokens)
    s.wipe()
    s.enqueue(None)
    qlinear.sync()
    s.check()


def stream_of(hip):
    stream = C.c_void_p()
    assert hip.hipStreamCreate(C.byref(stream)) == 0
    return stream


@pytest.mark.parametrize("tokens", [1, 70])
def test_a_step_in_a_graph(model, tokens):
    hip = C.CDLL("libamdhip64.so")
    s, other = Step(model, tokens, seed=5), Step(model, tokens + 1, seed=6)
    s.enqueue(None)
    qlinear.sync()
    want = s.results()
    stream, graph, gexec = stream_of(hip), C.c_void_p(), C.c_void_p()
    assert hip.hipStreamBeginCapture(stream, 0) == 0
    s.enqueue(stream)
    assert hip.hipStreamEndCapture(stream, C.byref(graph)) == 0
    assert hip.hipGraphInstantiate(C.byref(gexec), graph, None, None, C.c_size_t(0)) == 0
    for replay in range(4):
        s.wipe()
        assert hip.hipGraphLaunch(gexec, stream) == 0
        assert hip.hipStreamSynchronize(stream) == 0
        for a, b in zip(s.results(), want):
            assert np.array_equal(a, b), replay
        other.enqueue(None)  # eager work of the program between replays
        qlinear.sync()
    assert hip.hipGraphExecDestroy(gexec) == 0 and hip.hipGraphDestroy(graph) == 0 and hip.hipStreamDestroy(stream) == 0


@pytest.mark.parametrize("vocab", [2080, 70000])
def test_sampling_in_a_graph(vocab):
    """the sampler alone, by one and by several workgroups per sequence, on new random numbers at every replay"""
    hip = C.CDLL("libamdhip64.so")
    n = 5
    rng = np.random.default_rng(vocab)
    logits = (rng.standard_normal((n, vocab)) * 2).astype(np.float32)
    d = [qlinear.DevBuf.from_numpy(a) for a in (logits, np.array([1.0, 0.7, 0.0, 1.2, 1.0], np.float32), np.array([0, 40, 0, 700, 0], np.int32), np.array([1.0, 0.9, 1.0, 1.0, 0.95], np.float32))]
    u, ids = qlinear.DevBuf(n * 4), qlinear.DevBuf(n * 4)
    ws = qlinear.DevBuf(max(256, qlinear.sample_workspace_bytes(n, vocab)))

    def enqueue(stream):
        qlinear.sample_dev(F32, d[0], n, vocab, vocab, d[1], d[2], d[3], None, u, ids, None, ws, stream)

    enqueue(None)
    qlinear.sync()
    stream, graph, gexec = stream_of(hip), C.c_void_p(), C.c_void_p()
    assert hip.hipStreamBeginCapture(stream, 0) == 0
    enqueue(stream)
    assert hip.hipStreamEndCapture(stream, C.byref(graph)) == 0
    assert hip.hipGraphInstantiate(C.byref(gexec), graph, None, None, C.c_size_t(0)) == 0
    seen = set()
    for _ in range(6):
        draw = rng.random(n).astype(np.float32)
        assert qlinear.load().qlin_dev_upload(u.ptr, draw.ctypes.data, draw.nbytes) == 0
        assert hip.hipGraphLaunch(gexec, stream) == 0
        assert hip.hipStreamSynchronize(stream) == 0
        replayed = ids.to_numpy(np.int32, (n,)).tolist()
        enqueue(None)
        qlinear.sync()
        assert ids.to_numpy(np.int32, (n,)).tolist() == replayed
        seen.add(tuple(replayed))
    assert len(seen) > 1
    assert hip.hipGraphExecDestroy(gexec) == 0 and hip.hipGraphDestroy(graph) == 0 and hip.hipStreamDestroy(stream) == 0


def test_two_threads_on_streams_of_their_own(model):
    hip = C.CDLL("libamdhip64.so")
    steps = [Step(model, 33, seed=8), Step(model, 90, seed=9)]
    want = []
    for s in steps:
        s.enqueue(None)
        qlinear.sync()
        want.append(s.results())
        s.wipe()
    streams = [stream_of(hip) for _ in steps]
    errors = []

    def work(s, stream):
        try:
            for _ in range(20):
                s.enqueue(stream)
            qlinear.sync(stream)
        except Exception as e:  # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=work, args=a) for a in zip(steps, streams)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors
    for s, w in zip(steps, want):
        for a, b in zip(s.results(), w):
            assert np.array_equal(a, b)
    for stream in streams:
        assert hip.hipStreamDestroy(stream) == 0


@pytest.mark.parametrize("tokens", [1, 3, 40])
def test_a_sequence_that_is_lost(model, tokens):
    """a sequence whose activations hold a NaN has no token left: id -1, probability 0 and an embedding of zeros, and the others' step is
    what it was"""
    step = Step(model, tokens, 7)
    step.enqueue(None)
    qlinear.sync()
    before = step.results()
    bad = step.x_host.copy()
    bad[tokens - 1, 300] = 0x7FC0
    assert qlinear.load().qlin_dev_upload(step.x.ptr, bad.ctypes.data, bad.nbytes) == 0
    step.enqueue(None)
    qlinear.sync()
    for a, b in zip(step.results(), before):
        assert np.array_equal(a[:tokens - 1], b[:tokens - 1])
    assert step.ids.to_numpy(np.int32, (tokens,))[-1] == -1 and step.probs.to_numpy(np.float32, (tokens,))[-1] == 0
    assert not step.next.to_numpy(np.float32, (tokens, HIDDEN))[-1].any()
    assert (before[3] >= 0).all()
