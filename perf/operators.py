"""The 4-bit operators and the sampler as cases that can be timed and compared.

A case is one call, or one group of calls that only make sense together, as an engine that keeps its activations on the GPU
makes it. Kinds:

  quantize  float rows to MXFP4 blocks (a key or value, an expert's input, a tensor quantised at load time), and the blocks
            decoded to bf16 again: what the 4 bits stand for
  linear    activations times a weight tensor in MXFP4, both in 4 bits: the activations, which are floats, are quantised in
            the call
  gate_up   silu(x . gate) * (x . up) on the same operands: the first half of a gated feed-forward block
  sample    the next token of each sequence from its logits: temperature, top-k, top-p, min-p, and a random number per
            sequence that the caller has drawn

Weights are MXFP4 blocks (17 bytes per 32 elements: a power of two and 32 e2m1 codes) with random codes and powers of two of
about the size that a trained model's blocks have; an engine lays them out as an operand once, when the model is loaded.
Activations are N(0, 1) with a few channels ten times as large. Logits are N(0, 2) with a few likely tokens, and tokens that
the caller has ruled out hold -infinity.
"""
import math

import numpy as np
import torch

own = False  # False: elementary torch operations; True: the calls of gemm_amd.qlinear

MXFP4 = 39
TYPES = {"f32": (0, torch.float32), "f16": (1, torch.float16), "bf16": (30, torch.bfloat16)}
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def listed():
    return [
        # activations of a batch of decoding sequences
        {"name": "quantize_64x4096_bf16", "kind": "quantize", "rows": 64, "cols": 4096, "x": "bf16", "pad": 0},
        # a short prompt of no round length, rows out of a wider buffer
        {"name": "quantize_77x11008_f16", "kind": "quantize", "rows": 77, "cols": 11008, "x": "f16", "pad": 24},
        # a feed-forward tensor at load time
        {"name": "quantize_4096x14336_f32", "kind": "quantize", "rows": 4096, "cols": 14336, "x": "f32", "pad": 0},
        # one user, one token: the up projection of an 8B model
        {"name": "linear_1_14336x4096", "kind": "linear", "tokens": 1, "rows": 14336, "cols": 4096, "x": "f32", "y": "f32", "pad": 0},
        # sequences decoding together, the down projection (long rows)
        {"name": "linear_24_4096x14336", "kind": "linear", "tokens": 24, "rows": 4096, "cols": 14336, "x": "bf16", "y": "f32", "pad": 0},
        # a few sequences at the output projection, the largest tensor of a model
        {"name": "linear_4_151936x4096", "kind": "linear", "tokens": 4, "rows": 151936, "cols": 4096, "x": "bf16", "y": "f32", "pad": 0},
        # a short prompt on a narrow model, nothing a multiple of a tile
        {"name": "linear_77_1000x2080", "kind": "linear", "tokens": 77, "rows": 1000, "cols": 2080, "x": "f16", "y": "f32", "pad": 8},
        # a long prompt, the largest product
        {"name": "linear_2048_14336x4096", "kind": "linear", "tokens": 2048, "rows": 14336, "cols": 4096, "x": "bf16", "y": "bf16", "pad": 0},
        # one token through gate and up
        {"name": "gate_up_1_14336x4096", "kind": "gate_up", "tokens": 1, "rows": 14336, "cols": 4096, "x": "f32", "y": "f32", "pad": 0},
        # a prefill chunk through gate and up
        {"name": "gate_up_512_14336x4096", "kind": "gate_up", "tokens": 512, "rows": 14336, "cols": 4096, "x": "bf16", "y": "bf16", "pad": 0},
        # one user with the usual settings
        {"name": "sample_1x151936_f32", "kind": "sample", "seqs": 1, "vocab": 151936, "x": "f32", "pad": 0, "filters": "usual"},
        # a large batch, every sequence with settings of its own, logits in 16 bits out of a padded buffer
        {"name": "sample_256x128256_bf16", "kind": "sample", "seqs": 256, "vocab": 128256, "x": "bf16", "pad": 64, "filters": "mixed"},
    ]


def _spread(rng, lo, hi, step=1):
    """A multiple of `step` between lo and hi, even over the logarithm."""
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random() / step)) * step))


def draw(rng):
    """Another case of the same ranges: any size of the blocks' 32 columns, any row and token counts."""
    kind = rng.choice(["quantize", "linear", "linear", "linear", "gate_up", "gate_up", "sample", "sample"])
    pad = rng.choice([0, 0, 8, 40])
    x = rng.choice(["bf16", "bf16", "f32", "f16"])
    if kind == "quantize":
        return {"kind": kind, "rows": _spread(rng, 1, 4096), "cols": _spread(rng, 1024, 14336, 32), "x": x, "pad": pad}
    if kind == "sample":
        return {"kind": kind, "seqs": _spread(rng, 1, 256), "vocab": _spread(rng, 2000, 128256), "x": x, "pad": pad,
                "filters": rng.choice(["usual", "mixed", "none"])}
    tokens = rng.choice([1, _spread(rng, 2, 64), _spread(rng, 65, 2048), _spread(rng, 1, 2048)])
    if kind == "linear" and tokens <= 64 and rng.random() < 0.2:  # an output projection
        rows, cols = _spread(rng, 32000, 151936), _spread(rng, 1024, 4096, 32)
    else:
        rows, cols = _spread(rng, 256, 14336), _spread(rng, 256, 14336, 32)
    most = 2048 * 14336 * 4096 // (2 if kind == "gate_up" else 1)
    tokens = max(1, min(tokens, most // (rows * cols)))
    return {"kind": kind, "tokens": tokens, "rows": rows, "cols": cols, "x": x, "y": rng.choice(["f32", "bf16"]), "pad": pad}


# ------------------------------------------------------------------ inputs

def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _activations(g, rows, cols, dtype, pad):
    """[rows, cols] out of rows of cols + pad elements"""
    x = torch.randn(rows, cols + pad, device="cuda", generator=g)
    loud = torch.randint(0, cols, (max(1, cols // 256),), device="cuda", generator=g)
    x[:, loud] *= 10.0
    return x.to(dtype)[:, :cols]


def _weights(g, rows, cols):
    """MXFP4 blocks, [rows, cols / 32, 17] bytes"""
    n = rows * (cols // 32)
    words = torch.randint(-(1 << 63), (1 << 63) - 1, ((n * 17 + 7) // 8,), dtype=torch.int64, device="cuda", generator=g)
    blocks = words.view(torch.uint8)[: n * 17].view(rows, cols // 32, 17)
    blocks[:, :, 0] = torch.randint(117, 122, (rows, cols // 32), dtype=torch.uint8, device="cuda", generator=g)
    return blocks


def _logits(g, seqs, vocab, dtype, pad, filters):
    x = 2.0 * torch.randn(seqs, vocab + pad, device="cuda", generator=g)
    likely = torch.randint(0, vocab, (seqs, 12), device="cuda", generator=g)
    x.scatter_add_(1, likely, 6.0 + 2.0 * torch.randn(seqs, 12, device="cuda", generator=g))
    if filters != "none":  # tokens outside the tokenizer's vocabulary, and a few that the caller rules out
        x[:, vocab - vocab // 500:] = -math.inf
        x[:, torch.randint(0, vocab, (16,), device="cuda", generator=g)] = -math.inf
    if filters == "mixed" and seqs >= 8:  # a grammar that allows a handful of tokens; one that allows none
        allowed = x[3, :40].clone()
        x[3] = torch.finfo(dtype).min
        x[3, :40] = allowed
        x[7] = -math.inf
    return x.to(dtype)[:, :vocab]


def _settings(g, seqs, filters):
    """temperature, top_k, top_p, min_p and a random number of [0, 1) per sequence"""
    def pick(values, dtype):
        at = torch.randint(0, len(values), (seqs,), device="cuda", generator=g)
        return torch.tensor(values, dtype=dtype, device="cuda")[at]
    if filters == "usual":
        out = [pick([0.8], torch.float32), pick([40], torch.int32), pick([0.95], torch.float32), pick([0.05], torch.float32)]
    elif filters == "none":
        out = [pick([1.0], torch.float32), pick([0], torch.int32), pick([1.0], torch.float32), pick([0.0], torch.float32)]
    else:
        out = [pick([0.0, 0.3, 0.7, 1.0, 1.0, 1.4], torch.float32), pick([0, 0, 1, 20, 50, 1000], torch.int32),
               pick([1.0, 0.5, 0.9, 0.95, 0.99], torch.float32), pick([0.0, 0.0, 0.02, 0.1], torch.float32)]
    return out + [torch.rand(seqs, device="cuda", generator=g)]


class Buf:
    """A torch tensor as the binding takes device buffers."""

    def __init__(self, t):
        self.t, self.ptr, self.nbytes = t, t.data_ptr(), t.numel() * t.element_size()


def _bytes(n):
    return Buf(torch.empty(max(1, n), dtype=torch.uint8, device="cuda"))


def prepare(case, seed):
    g = _generator(seed)
    kind, (type_x, dtype_x) = case["kind"], TYPES[case["x"]]
    s = {"case": case}
    if kind == "sample":
        s["x"] = _logits(g, case["seqs"], case["vocab"], dtype_x, case["pad"], case["filters"])
        s["settings"] = _settings(g, case["seqs"], case["filters"])
    else:
        s["x"] = _activations(g, case.get("tokens", case["rows"]), case["cols"], dtype_x, case["pad"])
    if kind in ("linear", "gate_up"):
        s["w"] = [_weights(g, case["rows"], case["cols"]) for _ in range(2 if kind == "gate_up" else 1)]
    if own:
        from gemm_amd import qlinear
        if kind == "sample":
            s["ids"] = torch.empty(case["seqs"], dtype=torch.int32, device="cuda")
            s["probs"] = torch.empty(case["seqs"], dtype=torch.float32, device="cuda")
            s["ws"] = _bytes(qlinear.sample_workspace_bytes(case["seqs"], case["vocab"]))
        elif kind == "quantize":
            s["blocks"] = _bytes(case["rows"] * (case["cols"] // 32) * 17)
            s["out"] = torch.empty(case["rows"], case["cols"], dtype=torch.bfloat16, device="cuda")
        else:
            s["ops"] = []
            for w in s.pop("w"):  # the operand replaces the blocks, as it does in an engine
                op = _bytes(qlinear.mxfp4_operand_bytes(case["rows"], case["cols"]))
                qlinear.mxfp4_operand_dev(MXFP4, Buf(w), op, case["rows"], case["cols"], case["cols"], _stream())
                s["ops"].append(op)
            s["ws"] = _bytes(qlinear.mxfp4_gemm_workspace_bytes(case["cols"], case["tokens"]))
            s["out"] = torch.empty(case["tokens"], case["rows"], dtype=TYPES[case["y"]][1], device="cuda")
    return s


def _stream():
    return torch.cuda.current_stream().cuda_stream


# ------------------------------------------------------------------ a pass

def run(s):
    case = s["case"]
    if own:
        return _run_own(s, case)
    if case["kind"] == "quantize":
        return _quantized(s["x"].float()).to(torch.bfloat16)
    if case["kind"] == "sample":
        return _sampled(s["x"], *s["settings"])
    x = _quantized(s["x"].float())
    y = x @ _decoded(s["w"][0]).t()
    if case["kind"] == "gate_up":
        y = y / (1.0 + torch.exp(-y)) * (x @ _decoded(s["w"][1]).t())
    return y.to(TYPES[case["y"]][1])


def _run_own(s, case):
    from gemm_amd import qlinear
    x, type_x = s["x"], TYPES[case["x"]][0]
    if case["kind"] == "sample":
        t, k, p, m, u = (Buf(v) for v in s["settings"])
        qlinear.sample_dev(type_x, Buf(x), case["seqs"], case["vocab"], x.stride(0), t, k, p, m, u, Buf(s["ids"]), Buf(s["probs"]),
                           s["ws"], _stream())
        return s["ids"], s["probs"]
    if case["kind"] == "quantize":
        qlinear.quantize_mxfp4_dev(type_x, Buf(x), s["blocks"], case["rows"], case["cols"], x.stride(0), _stream())
        qlinear.dequant_bf16_dev(MXFP4, s["blocks"], Buf(s["out"]), case["rows"], case["cols"], _stream())
        return s["out"]
    sizes = (case["rows"], case["cols"], case["tokens"], x.stride(0), case["rows"])
    type_y = TYPES[case["y"]][0]
    if case["kind"] == "linear":
        qlinear.mxfp4_gemm_dev(s["ops"][0], type_x, Buf(x), type_y, Buf(s["out"]), *sizes, s["ws"], _stream())
    else:
        qlinear.mxfp4_gemm_silu_mul_dev(s["ops"][0], s["ops"][1], type_x, Buf(x), type_y, Buf(s["out"]), *sizes, s["ws"], _stream())
    return s["out"]


# ------------------------------------------------------------------ the plain forms

def _quantized(x):
    """fp32 rows to the values of their 4-bit codes. A block's power of two puts its largest magnitude into [4, 8); a code is the
    nearest e2m1 number, on a tie the one with the even code, and 6 beyond 6."""
    b = x.reshape(x.shape[0], -1, 32)
    exponent = torch.frexp(b.abs().amax(dim=2, keepdim=True))[1] - 1
    power = torch.clamp(exponent - 2, min=-127)
    v = torch.ldexp(b.abs(), -power)
    code = (v > 0.25).int() + (v >= 0.75) + (v > 1.25) + (v >= 1.75) + (v > 2.5) + (v >= 3.5) + (v > 5.0)
    size = torch.tensor(E2M1, device=x.device)[code]
    return torch.where(b < 0, -torch.ldexp(size, power), torch.ldexp(size, power)).reshape(x.shape)


def _decoded(blocks):
    """MXFP4 blocks to fp32: byte j of a block's sixteen holds elements j (low) and j + 16 (high)"""
    table = torch.tensor(E2M1 + tuple(-v for v in E2M1), device=blocks.device)
    codes = torch.cat([blocks[:, :, 1:] & 15, blocks[:, :, 1:] >> 4], dim=2)
    scale = torch.exp2(blocks[:, :, :1].float() - 127.0)
    return (table[codes.int()] * scale).reshape(blocks.shape[0], -1)


def _sampled(logits, temperature, top_k, top_p, min_p, u):
    """The token order is by logit, equal ones by index; weights and their sums in 64 bits, since a border between two tokens may
    lie close to the random number."""
    x = torch.where(torch.isnan(logits), -math.inf, logits.float())
    n = x.shape[1]
    order_x, order = torch.sort(x, dim=1, descending=True, stable=True)
    there = order_x > -math.inf
    t = temperature.double()[:, None]
    d = order_x.double() - order_x[:, :1].double()
    w = torch.where(there, torch.exp(d / torch.where(t > 0, t, 1.0)), 0.0)
    place = torch.arange(n, device=x.device)[None, :]
    k = torch.where(top_k > 0, top_k, n)[:, None]
    w = torch.where((place < k) & ((t > 0) | (place < 1)), w, 0.0)
    sums = torch.cumsum(w, dim=1)
    p = top_p.double()[:, None]
    before = torch.cat([torch.zeros_like(sums[:, :1]), sums[:, :-1]], dim=1)
    w = torch.where((p >= 1) | (before < p * sums[:, -1:]) | (place < 1), w, 0.0)
    w = torch.where((w >= min_p.double()[:, None]) | (place < 1), w, 0.0)
    sums = torch.cumsum(w, dim=1)
    total = sums[:, -1:]
    past = (sums > u.double()[:, None] * total).int().argmax(dim=1, keepdim=True)
    weight = w.gather(1, past)
    some = there[:, :1]
    ids = torch.where(some, order.gather(1, past), -1)[:, 0].int()
    return ids, torch.where(some, weight / total, 0.0)[:, 0].float()


# ------------------------------------------------------------------ the definition in 64 bits

def exact(case, seed):
    s = prepare_plain(case, seed)
    if case["kind"] == "sample":
        return _sampled_exactly(s["x"], [v.cpu().numpy() for v in s["settings"]])
    x = _nearest_exactly(s["x"].double())
    if case["kind"] == "quantize":
        return x
    y = x @ _decoded_exactly(s["w"][0]).t()
    if case["kind"] == "gate_up":
        y = y * torch.sigmoid(y) * (x @ _decoded_exactly(s["w"][1]).t())
    return y


def prepare_plain(case, seed):
    """the inputs of prepare(case, seed), whichever side is being run"""
    global own
    was, own = own, False
    try:
        return prepare(case, seed)
    finally:
        own = was


def _nearest_exactly(x):
    b = x.reshape(x.shape[0], -1, 32)
    largest = b.abs().amax(dim=2, keepdim=True)
    power = torch.floor(torch.log2(torch.where(largest > 0, largest, 1.0))) - 2
    power = torch.clamp(torch.where(largest > 0, power, -127.0), min=-127)
    v = (b / torch.exp2(power)).abs()
    step = torch.where(v < 2, 0.5, torch.where(v < 4, 1.0, 2.0))  # between neighbouring e2m1 numbers; round() takes ties to even
    q = torch.clamp(torch.round(v / step) * step, max=6.0)
    return (torch.sign(b) * q * torch.exp2(power)).reshape(x.shape)


def _decoded_exactly(blocks):
    rows, per_row, _ = blocks.shape
    qs = blocks[:, :, 1:].to(torch.int32)
    out = torch.empty(rows, per_row, 32, dtype=torch.float64, device=blocks.device)
    for half in (0, 1):
        c = (qs >> (4 * half)) & 15
        e, m = (c >> 1) & 3, (c & 1).double()
        size = torch.where(e == 0, 0.5 * m, (1.0 + 0.5 * m) * torch.exp2(e.double() - 1.0))
        out[:, :, 16 * half:16 * half + 16] = torch.where(c >= 8, -size, size)
    out *= torch.exp2(blocks[:, :, :1].double() - 127.0)
    return out.reshape(rows, -1)


def _sampled_exactly(logits, settings):
    x = logits.float().cpu().numpy().astype(np.float64)
    ids, probs = np.full(len(x), -1, np.int32), np.zeros(len(x))
    for row, (v, t, k, p, m, u) in enumerate(zip(x, *settings)):
        at = np.flatnonzero(v > -np.inf)  # false for NaN
        if len(at) == 0:
            continue
        if t <= 0 or k == 1:
            ids[row], probs[row] = at[np.argmax(v[at])], 1.0
            continue
        if 0 < k < len(at):  # the k largest, and of those equal to the last of them the first
            least = np.partition(v[at], len(at) - k)[len(at) - k]
            above, equal = at[v[at] > least], at[v[at] == least]
            at = np.concatenate([above, equal[:k - len(above)]])
        at = at[np.lexsort((at, -v[at]))]
        w = np.exp((v[at] - v[at[0]]) / np.float64(t))
        if p < 1:
            keep = 1 + np.searchsorted(np.cumsum(w), np.float64(p) * w.sum(), side="left")
            at, w = at[:keep], w[:keep]
        keep = max(1, np.count_nonzero(w >= np.float64(m)))
        at, w = at[:keep], w[:keep]
        sums = np.cumsum(w)
        j = min(int(np.searchsorted(sums, np.float64(u) * sums[-1], side="right")), len(at) - 1)
        ids[row], probs[row] = at[j], w[j] / sums[-1]
    return torch.from_numpy(ids), torch.from_numpy(probs)


# ------------------------------------------------------------------ what a pass cannot do without

def work(case):
    size = {"f32": 4, "f16": 2, "bf16": 2}
    if case["kind"] == "sample":
        n = case["seqs"] * case["vocab"]
        return {"bytes": n * size[case["x"]] + case["seqs"] * 28, "flops": 2 * n}
    if case["kind"] == "quantize":  # the values that the codes stand for are written in bf16
        n = case["rows"] * case["cols"]
        return {"bytes": n * (size[case["x"]] + 2) + n // 32 * 17, "flops": 2 * n}
    t, r, c = case["tokens"], case["rows"], case["cols"]
    n = 2 if case["kind"] == "gate_up" else 1
    return {"bytes": n * r * (c // 32) * 17 + t * c * size[case["x"]] + t * r * size[case["y"]], "flops": 2 * n * t * r * c}
