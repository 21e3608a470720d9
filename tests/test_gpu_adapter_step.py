"""Adapters and routing by scores as an engine runs them beside the operators that were there: Q, K and V with the adapters of many requests,
gate and up with their adapters and activation, the down projection with its own, and from that a router's logits, its choice and the experts -
eager, in a graph that is replayed between other work and on other adapters, on two streams from two threads at once, in a batch padded with
rows of NaN. Every step is compared with its own definition in 64 bits on what the step before really gave."""
import ctypes as C
import threading

import numpy as np
import pytest

from gemm_amd import qlinear
import synth
from tests import adapter_formulas as f
from tests.adapter_formulas import BF16, F32
from tests.conftest import rel_l2
from tests.test_gpu_lora import table_of

pytestmark = pytest.mark.gpu
Q4K = synth.GGML_Q4_K
HIDDEN, KV, FFN, EXPERT_FFN, EXPERTS, TOP_K = 512, 256, 768, 256, 32, 4
RANKS = [8, 0, 16, 5]  # of an adapter; 0: the table's entry is none
GROUPS, USED = 8, 3


class Model:
    def __init__(self):
        shapes = {"q": (HIDDEN, HIDDEN), "k": (KV, HIDDEN), "v": (KV, HIDDEN), "gate": (FFN, HIDDEN), "up": (FFN, HIDDEN), "down": (HIDDEN, FFN),
                  "gates": (EXPERTS * EXPERT_FFN, HIDDEN), "ups": (EXPERTS * EXPERT_FFN, HIDDEN), "downs": (EXPERTS * HIDDEN, EXPERT_FFN)}
        blocks = {n: synth.make_weights(Q4K, *s, seed=40 + i) for i, (n, s) in enumerate(shapes.items())}
        self.w = {n: qlinear.DevBuf.from_numpy(b) for n, b in blocks.items()}
        self.experts = [qlinear.dequant_rows(Q4K, blocks[n], *shapes[n]).astype(np.float64) for n in ("gates", "ups", "downs")]
        rng = np.random.default_rng(50)
        self.bias = (0.05 * rng.standard_normal(EXPERTS)).astype(np.float32)
        self.router = qlinear.DevBuf.from_numpy((0.02 * rng.standard_normal((EXPERTS, HIDDEN))).astype(np.float32).view(np.uint8))
        self.dbias = qlinear.DevBuf.from_numpy(self.bias)
        self.shapes = shapes


def adapters(seed, n_rows, n_cols):
    rng = np.random.default_rng(seed)
    return [f.Adapter(rng, r, n_rows, n_cols, BF16, 0.5 + i) if r else None for i, r in enumerate(RANKS)]


class Step:
    """the buffers of one batch and the calls on them; a batch of one takes the calls for one token, with activations in fp32"""

    def __init__(self, model, n, seed, padded=0):
        self.m, self.n, self.real, self.one = model, n, n - padded, n == 1
        rng = np.random.default_rng(seed)
        x = synth.make_activation(HIDDEN, seed=seed, tokens=n).reshape(n, HIDDEN)
        self.ids_host = rng.integers(-1, len(RANKS), n).astype(np.int32)
        x[self.real:], self.ids_host[self.real:] = np.nan, -1
        self.x16_host, self.xv = f.as_type(x, BF16)
        self.x16 = qlinear.DevBuf.from_numpy(self.x16_host)
        self.x32 = qlinear.DevBuf.from_numpy(self.xv.astype(np.float32))
        self.ids = qlinear.DevBuf.from_numpy(self.ids_host)
        self.tables, self.held, self.ad = {}, {}, {}
        for name in ("q", "k", "v", "gate", "up", "down"):
            self.tables[name] = qlinear.DevBuf(len(RANKS) * qlinear.LORA_DTYPE.itemsize)
        self.adopt(seed)
        f32 = lambda cols: qlinear.DevBuf(n * cols * 4)  # noqa: E731
        self.y = {name: f32(model.shapes[name][0]) for name in ("q", "k", "v", "gate", "up")}
        self.out = {name: f32(model.shapes[name][0]) for name in ("q", "k", "v", "down")}
        self.h = qlinear.DevBuf(n * FFN * (4 if self.one else 2))
        self.logits, self.idx, self.weight, self.moe = f32(EXPERTS), f32(TOP_K), f32(TOP_K), f32(HIDDEN)
        self.ws = qlinear.DevBuf(max(qlinear.lora_workspace_bytes(3, max(RANKS), HIDDEN, n), qlinear.lora_workspace_bytes(1, max(RANKS), FFN, n),
                                     qlinear.gemm_bf16_any_workspace_bytes(max(HIDDEN, FFN), max(HIDDEN, FFN)), qlinear.moe_workspace_bytes(n, TOP_K, HIDDEN, EXPERT_FFN, EXPERTS)))
        self.qkv = qlinear.lora_tensors([(self.tables[t], self.y[t], self.out[t], model.shapes[t][0], model.shapes[t][0], model.shapes[t][0]) for t in ("q", "k", "v")])
        self.down = qlinear.lora_tensors([(self.tables["down"], self.out["down"], self.out["down"], HIDDEN, HIDDEN, HIDDEN)])

    def adopt(self, seed):
        """other adapters in the same tables"""
        for i, (name, table) in enumerate(self.tables.items()):
            n_rows, n_cols = self.m.shapes[name]
            self.ad[name] = adapters(100 * seed + i, n_rows, n_cols)
            fresh, self.held[name] = table_of(self.ad[name])
            raw = fresh.to_numpy(np.uint8, (table.nbytes,))
            assert qlinear.load().qlin_dev_upload(table.ptr, raw.ctypes.data, raw.nbytes) == 0

    def base_down(self, out, stream):
        if self.one:
            qlinear.gemv_dev(Q4K, self.m.w["down"], self.h, out, HIDDEN, FFN, stream)
        else:
            qlinear.gemm_bf16_any_dev(Q4K, self.m.w["down"], self.h, out, HIDDEN, FFN, self.n, FFN, HIDDEN, self.ws, stream)

    def enqueue(self, stream):
        m, n = self.m, self.n
        x, x_type, h_type = (self.x32, F32, F32) if self.one else (self.x16, BF16, BF16)
        for names in (("q", "k", "v"), ("gate", "up")):
            rows = [m.shapes[t][0] for t in names]
            if self.one:
                qlinear.gemv_multi_dev(Q4K, [m.w[t] for t in names], [self.y[t] for t in names], rows, x, HIDDEN, stream)
            else:
                qlinear.gemm_bf16_multi_dev(Q4K, [m.w[t] for t in names], x, [self.y[t] for t in names], rows, HIDDEN, n, HIDDEN, rows, self.ws, stream)
        qlinear.lora_add_dev(self.qkv, BF16, len(RANKS), max(RANKS), self.ids, x_type, x, F32, F32, HIDDEN, n, HIDDEN, self.ws, stream)
        qlinear.lora_silu_mul_dev(self.tables["gate"], self.tables["up"], BF16, len(RANKS), max(RANKS), self.ids, x_type, x, F32, self.y["gate"], self.y["up"], h_type, self.h,
                                  FFN, HIDDEN, n, HIDDEN, FFN, FFN, self.ws, stream)
        self.base_down(self.out["down"], stream)
        qlinear.lora_add_dev(self.down, BF16, len(RANKS), max(RANKS), self.ids, h_type, self.h, F32, F32, FFN, n, FFN, self.ws, stream)
        qlinear.gemm_f32_dev(0, m.router, self.out["down"], self.logits, EXPERTS, HIDDEN, n, HIDDEN, EXPERTS, stream)
        qlinear.moe_route_scores_dev(qlinear.ROUTE_SIGMOID, F32, self.logits, n, EXPERTS, EXPERTS, m.dbias, GROUPS, USED, 2, TOP_K, True, 2.5, self.idx, self.weight, stream)
        qlinear.moe_ffn_dev(Q4K, m.w["gates"], m.w["ups"], m.w["downs"], self.x16, self.idx, self.weight, self.moe, n, TOP_K, HIDDEN, EXPERT_FFN, EXPERTS, self.ws, stream)

    def wipe(self):
        for b in [*self.y.values(), *self.out.values(), self.h, self.logits, self.idx, self.weight, self.moe, self.ws]:
            fill = np.full(b.nbytes, 0xFF, np.uint8)
            assert qlinear.load().qlin_dev_upload(b.ptr, fill.ctypes.data, fill.nbytes) == 0

    def check(self):
        n, real = self.n, slice(0, self.real)
        ids, native = self.ids_host[real], not self.one
        h_type = F32 if self.one else BF16
        read = lambda b, cols: b.to_numpy(np.float32, (n, cols)).astype(np.float64)[real]  # noqa: E731
        x = self.xv[real]
        for t in ("q", "k", "v"):
            rows = self.m.shapes[t][0]
            y, got = read(self.y[t], rows), read(self.out[t], rows)
            delta, off = f.added(x, self.ad[t], ids, rows, native)
            assert (np.abs(got - (y + delta)) <= f.add_bound(y, delta, off, F32)).all(), t
            assert np.array_equal(got[ids < 0], y[ids < 0])
        (g, dg, og), (u, du, ou) = [(read(self.y[t], FFN), *f.added(x, self.ad[t], ids, FFN, native)) for t in ("gate", "up")]
        og, ou = og + 2.0 ** -23 * (np.abs(g) + np.abs(dg)), ou + 2.0 ** -23 * (np.abs(u) + np.abs(du))
        h = f.values(self.h.to_numpy(f.NUMPY[h_type], (n, FFN)), h_type)[real]
        want = f.silu(g + dg) * (u + du)
        assert (np.abs(h - want) <= f.silu_mul_bound(g + dg, og, u + du, ou, h_type)).all()
        base = qlinear.DevBuf(n * HIDDEN * 4)
        self.base_down(base, None)
        qlinear.sync()
        y, got = read(base, HIDDEN), read(self.out["down"], HIDDEN)
        delta, off = f.added(h, self.ad["down"], ids, HIDDEN, native)
        assert (np.abs(got - (y + delta)) <= f.add_bound(y, delta, off, F32)).all()
        logits = read(self.logits, EXPERTS)
        idx, w = self.idx.to_numpy(np.int32, (n, TOP_K)), self.weight.to_numpy(np.float32, (n, TOP_K))
        for t in range(self.real):
            want_idx, want_w = f.route(logits[t], True, self.m.bias.astype(np.float64), GROUPS, USED, 2, TOP_K, True, 2.5)
            assert idx[t].tolist() == want_idx.tolist()
            assert (np.abs(w[t] - want_w) <= f.route_bound(logits[t], True, want_idx, want_w)).all()
        gates, ups, downs = self.m.experts
        moe = self.moe.to_numpy(np.float32, (n, HIDDEN))
        for t in range(self.real):
            want = np.zeros(HIDDEN)
            for e, we in zip(idx[t], w[t]):
                mine = slice(e * EXPERT_FFN, (e + 1) * EXPERT_FFN)
                want += float(we) * (downs[e * HIDDEN:(e + 1) * HIDDEN] @ (f.silu(gates[mine] @ x[t]) * (ups[mine] @ x[t])))
            assert rel_l2(moe[t], want) <= 2e-4  # what that operator is held to for a token
        assert (idx[self.real:] == -1).all() and (w[self.real:] == 0).all()
        return got, idx


@pytest.fixture(scope="module")
def model():
    return Model()


@pytest.mark.parametrize("tokens", [1, 2, 9, 70, 300])
def test_a_step(model, tokens):
    s = Step(model, tokens, seed=tokens)
    s.wipe()
    s.enqueue(None)
    qlinear.sync()
    s.check()


@pytest.mark.parametrize("tokens,padded", [(8, 3), (100, 37)])
def test_a_padded_batch(model, tokens, padded):
    """rows of NaN behind the last token: no adapter, no expert, and nothing of theirs in the others' results"""
    s = Step(model, tokens, seed=7, padded=padded)
    s.wipe()
    s.enqueue(None)
    qlinear.sync()
    s.check()


def stream_of(hip):
    stream = C.c_void_p()
    assert hip.hipStreamCreate(C.byref(stream)) == 0
    return stream


@pytest.mark.parametrize("tokens", [1, 33, 130])
def test_a_step_in_a_graph(model, tokens):
    """replayed on the adapters that the tables hold then, with eager work of another batch between"""
    hip = C.CDLL("libamdhip64.so")
    s, other = Step(model, tokens, seed=5), Step(model, tokens + 1, seed=6)
    s.enqueue(None)
    qlinear.sync()
    stream, graph, gexec = stream_of(hip), C.c_void_p(), C.c_void_p()
    assert hip.hipStreamBeginCapture(stream, 0) == 0
    s.enqueue(stream)
    assert hip.hipStreamEndCapture(stream, C.byref(graph)) == 0
    assert hip.hipGraphInstantiate(C.byref(gexec), graph, None, None, C.c_size_t(0)) == 0
    for replay in range(4):
        s.adopt(20 + replay)
        s.wipe()
        assert hip.hipGraphLaunch(gexec, stream) == 0
        assert hip.hipStreamSynchronize(stream) == 0
        s.check()
        replayed = s.out["q"].to_numpy(np.uint32, (tokens, HIDDEN))
        s.wipe()
        s.enqueue(None)
        qlinear.sync()
        assert np.array_equal(s.out["q"].to_numpy(np.uint32, (tokens, HIDDEN)), replayed)
        other.enqueue(None)
        qlinear.sync()
    assert hip.hipGraphExecDestroy(gexec) == 0 and hip.hipGraphDestroy(graph) == 0 and hip.hipStreamDestroy(stream) == 0


def test_two_threads_on_streams_of_their_own(model):
    hip = C.CDLL("libamdhip64.so")
    steps = [Step(model, 33, seed=8), Step(model, 300, seed=9)]
    for s in steps:
        s.enqueue(None)
        qlinear.sync()
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
    for s in steps:
        s.check()
    for stream in streams:
        assert hip.hipStreamDestroy(stream) == 0
