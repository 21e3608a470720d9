"""Routing to experts and low-rank adapters as cases that can be timed and compared.

A case is one call, as an engine that keeps its activations on the GPU makes it. Kinds:

  route    the experts of each token and their weights from the router's logits: softmax or sigmoid scores, a bias that balances the
           choice, groups of experts, top-k, weights renormalised or not
  add      one to three projections of the same activations (Q, K and V; one down projection) plus, for each token, the low-rank
           product of the adapter that its request came with
  gate_up  silu(gate) * up of two projections, each with the token's adapter added before the activation

Logits are N(0, 1.5) with experts of different popularity; the balancing bias is small beside the scores. "holes": a few experts are
out of service (-infinity), and the last tokens of the batch are padding (nothing but -infinity). Adapters are A ~ N(0, 1/columns)
and B of about the size that the added product reaches a third of the projection; every other one has half the largest rank.
Tokens and adapters: "one" adapter for all, "mixed" (decoding sequences, each with its own, one in eight with none), "runs"
(the prompts of several requests one after the other, one of them without an adapter).
"""
import math
import random
import struct

import numpy as np
import torch

own = False  # False: elementary torch operations; True: the calls of gemm_amd.qlinear

TYPES = {"f32": (0, torch.float32), "f16": (1, torch.float16), "bf16": (30, torch.bfloat16)}
SCORES = {"softmax": 0, "sigmoid": 1}


def listed():
    return [
        # one token, 128 experts: what a decoding user waits for in every layer
        {"name": "route_1x128_softmax", "kind": "route", "tokens": 1, "experts": 128, "x": "f32", "pad": 0, "score": "softmax", "bias": False,
         "groups": 1, "used": 1, "group_top": 1, "k": 8, "renorm": True, "scale": 1.0, "holes": False},
        # decoding sequences, a balanced router with groups
        {"name": "route_48x256_sigmoid_groups", "kind": "route", "tokens": 48, "experts": 256, "x": "f32", "pad": 0, "score": "sigmoid", "bias": True,
         "groups": 8, "used": 4, "group_top": 2, "k": 8, "renorm": True, "scale": 2.5, "holes": False},
        # a short prompt of no round length, logits in 16 bits out of a wider buffer, experts out of service and padding
        {"name": "route_333x60_softmax_bf16", "kind": "route", "tokens": 333, "experts": 60, "x": "bf16", "pad": 4, "score": "softmax", "bias": False,
         "groups": 1, "used": 1, "group_top": 1, "k": 4, "renorm": False, "scale": 1.0, "holes": True},
        # the prompts of many requests at once
        {"name": "route_16384x256_sigmoid_groups", "kind": "route", "tokens": 16384, "experts": 256, "x": "f32", "pad": 0, "score": "sigmoid", "bias": True,
         "groups": 8, "used": 4, "group_top": 2, "k": 8, "renorm": True, "scale": 2.5, "holes": True},
        # one user, one token: Q, K and V of an 8B model
        {"name": "add_1_qkv_4096", "kind": "add", "tokens": 1, "rows": "4096 1024 1024", "cols": 4096, "rank": 16, "adapters": 4, "ids": "one",
         "w": "bf16", "x": "f32", "y": "f32", "out": "f32", "pad": 0},
        # sequences decoding together, most with an adapter of their own
        {"name": "add_48_qkv_4096", "kind": "add", "tokens": 48, "rows": "4096 1024 1024", "cols": 4096, "rank": 16, "adapters": 24, "ids": "mixed",
         "w": "bf16", "x": "bf16", "y": "f32", "out": "f32", "pad": 0},
        # a short prompt on a narrow model, nothing a multiple of a tile
        {"name": "add_77_1000x2080_f16", "kind": "add", "tokens": 77, "rows": "1000", "cols": 2080, "rank": 12, "adapters": 3, "ids": "runs",
         "w": "f16", "x": "f16", "y": "f32", "out": "f32", "pad": 8},
        # a large decoding batch at the down projection (long rows)
        {"name": "add_200_4096x14336", "kind": "add", "tokens": 200, "rows": "4096", "cols": 14336, "rank": 32, "adapters": 32, "ids": "mixed",
         "w": "bf16", "x": "bf16", "y": "f32", "out": "f32", "pad": 0},
        # the prompts of several requests, Q, K and V
        {"name": "add_2048_qkv_4096_r64", "kind": "add", "tokens": 2048, "rows": "4096 1024 1024", "cols": 4096, "rank": 64, "adapters": 6, "ids": "runs",
         "w": "bf16", "x": "bf16", "y": "f32", "out": "f32", "pad": 0},
        # one token through gate and up
        {"name": "gate_up_1_14336x4096", "kind": "gate_up", "tokens": 1, "rows": "14336", "cols": 4096, "rank": 16, "adapters": 4, "ids": "one",
         "w": "bf16", "x": "f32", "y": "f32", "out": "f32", "pad": 0},
        # sequences decoding together, adapters in fp16
        {"name": "gate_up_24_14336x4096_f16", "kind": "gate_up", "tokens": 24, "rows": "14336", "cols": 4096, "rank": 32, "adapters": 8, "ids": "mixed",
         "w": "f16", "x": "f16", "y": "f32", "out": "f16", "pad": 0},
        # a prefill chunk, the activation rounded for the next product: the largest
        {"name": "gate_up_2048_14336x4096", "kind": "gate_up", "tokens": 2048, "rows": "14336", "cols": 4096, "rank": 32, "adapters": 6, "ids": "runs",
         "w": "bf16", "x": "bf16", "y": "f32", "out": "bf16", "pad": 0},
    ]


def _spread(rng, lo, hi, step=1):
    """A multiple of `step` between lo and hi, even over the logarithm."""
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random() / step)) * step))


def draw(rng):
    """Another case of the same ranges: any token count, expert count, rank and alignment, every type."""
    kind = rng.choice(["route", "route", "add", "add", "add", "gate_up", "gate_up"])
    pad = rng.choice([0, 0, 8, 3])
    if kind == "route":
        groups = rng.choice([1, 1, 2, 4, 8])
        experts = groups * max(2, _spread(rng, 8, 512) // groups)
        used = rng.randint(1, groups)
        k = min(rng.choice([1, 2, 4, 6, 8, 8, 10, 16]), used * (experts // groups))
        return {"kind": kind, "tokens": rng.choice([1, _spread(rng, 2, 64), _spread(rng, 65, 8192)]), "experts": experts, "x": rng.choice(["f32", "f32", "bf16", "f16"]),
                "pad": pad, "score": rng.choice(["softmax", "sigmoid"]), "bias": rng.choice([False, True]), "groups": groups, "used": used,
                "group_top": rng.choice([1, 2]), "k": k, "renorm": rng.choice([False, True]), "scale": rng.choice([1.0, 2.5]), "holes": rng.choice([False, True])}
    tokens = rng.choice([1, _spread(rng, 2, 64), _spread(rng, 65, 2048), _spread(rng, 1, 2048)])
    cols, step = _spread(rng, 256, 14336, rng.choice([32, 8, 1])), rng.choice([32, 8, 1])
    rows = [_spread(rng, 256, 14336, step)]
    if kind == "add" and rng.random() < 0.5:
        kv = _spread(rng, 128, 1024, step)
        rows = [_spread(rng, 256, 8192, step), kv, kv]
    rank, adapters = rng.choice([4, 8, 8, 16, 16, 32, 64, 128, 5, 12, 24]), _spread(rng, 1, 64)
    adapters = max(1, min(adapters, (1024 if tokens <= 256 else 256) // rank))
    ids = rng.choice(["one", "mixed"]) if tokens <= 256 else "runs"
    case = {"kind": kind, "tokens": tokens, "rows": " ".join(map(str, rows)), "cols": cols, "rank": rank, "adapters": adapters, "ids": ids,
            "w": rng.choice(["bf16", "bf16", "f16", "f32"]), "x": rng.choice(["bf16", "bf16", "f32", "f16"]), "y": rng.choice(["f32", "f32", "bf16"]),
            "out": rng.choice(["f32", "bf16", "f16"]), "pad": pad}
    w, most = work(case), work(listed()[-1])  # no more than the largest listed one
    case["tokens"] = max(1, int(tokens * min(1.0, most["bytes"] / w["bytes"], most["flops"] / w["flops"])))
    return case


# ------------------------------------------------------------------ inputs

def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _normal(g, rows, cols, dtype, pad, size=1.0):
    """[rows, cols] out of rows of cols + pad elements"""
    return (size * torch.randn(rows, cols + pad, device="cuda", generator=g)).to(dtype)[:, :cols]


def _logits(g, case):
    t, n = case["tokens"], case["experts"]
    x = 1.5 * torch.randn(t, n + case["pad"], device="cuda", generator=g)
    x += 0.5 * torch.randn(n + case["pad"], device="cuda", generator=g)
    if case["holes"]:
        x[:, torch.randint(0, n, (max(1, n // 32),), device="cuda", generator=g)] = -math.inf
        x[t - t // 20:] = -math.inf
    return x.to(TYPES[case["x"]][1])[:, :n]


def _adapter_ids(case, seed):
    t, n, rng = case["tokens"], case["adapters"], random.Random(seed)
    if case["ids"] == "one":
        return [rng.randrange(n)] * t
    if case["ids"] == "mixed":
        return [-1 if rng.random() < 0.125 else rng.randrange(n) for _ in range(t)]
    cuts = sorted(rng.randrange(t + 1) for _ in range(5))
    out, bare = [], rng.randrange(6)
    for i, (a, b) in enumerate(zip([0] + cuts, cuts + [t])):
        out += [-1 if i == bare else rng.randrange(n)] * (b - a)
    return out


def _ranks(case):
    return [case["rank"] if a % 2 == 0 else max(1, case["rank"] // 2) for a in range(case["adapters"])]


def _rows(case):
    return [int(r) for r in case["rows"].split()] * (2 if case["kind"] == "gate_up" else 1)


def _adapters(g, case, n_rows):
    """A [adapters, rank, cols] and B [adapters, n_rows, rank], zero behind an adapter's own rank"""
    n, r, dtype = case["adapters"], case["rank"], TYPES[case["w"]][1]
    a = (torch.randn(n, r, case["cols"], device="cuda", generator=g) / math.sqrt(case["cols"])).to(dtype)
    b = (torch.randn(n, n_rows, r, device="cuda", generator=g) / (3.0 * math.sqrt(r))).to(dtype)
    for i, own_rank in enumerate(_ranks(case)):
        a[i, own_rank:] = 0
        b[i, :, own_rank:] = 0
    return a, b


class Buf:
    """A torch tensor as the binding takes device buffers."""

    def __init__(self, t):
        self.t, self.ptr, self.nbytes = t, t.data_ptr(), t.numel() * t.element_size()


def _empty(rows, cols, dtype):
    return torch.empty(rows, cols, dtype=dtype, device="cuda")


def prepare(case, seed):
    g = _generator(seed)
    s = {"case": case}
    if case["kind"] == "route":
        s["x"] = _logits(g, case)
        s["bias"] = 0.05 * torch.randn(case["experts"], device="cuda", generator=g) if case["bias"] else None
        if own:
            s["ids"] = torch.empty(case["tokens"], case["k"], dtype=torch.int32, device="cuda")
            s["weights"] = _empty(case["tokens"], case["k"], torch.float32)
        return s
    t, out = case["tokens"], TYPES[case["out"]][1]
    s["x"] = _normal(g, t, case["cols"], TYPES[case["x"]][1], case["pad"])
    s["y"] = [_normal(g, t, r, TYPES[case["y"]][1], case["pad"]) for r in _rows(case)]
    s["scale"] = 0.5 + 1.5 * torch.rand(case["adapters"], device="cuda", generator=g)
    s["lora"] = [_adapters(g, case, r) for r in _rows(case)]
    s["ids"] = torch.tensor(_adapter_ids(case, seed), dtype=torch.int32, device="cuda")
    if own:
        _lay_out(s, case, t, out)
    return s


def _lay_out(s, case, t, out):
    """Each adapter's two tensors by themselves, as they are loaded, and the table of them that an engine keeps for every projection."""
    from gemm_amd import qlinear
    s["held"], s["tables"] = [], []
    scales = s["scale"].tolist()
    for a, b in s.pop("lora"):
        words = []
        for i, r in enumerate(_ranks(case)):
            pair = a[i, :r].clone(), b[i, :, :r].contiguous()
            s["held"].append(pair)
            words += [pair[0].data_ptr(), pair[1].data_ptr(), struct.unpack("<q", struct.pack("<if", r, scales[i]))[0]]
        s["tables"].append(Buf(torch.tensor(words, dtype=torch.int64, device="cuda")))
    s["out"] = [_empty(t, r, out) for r in _rows(case)[:1 if case["kind"] == "gate_up" else 3]]
    s["ws"] = Buf(torch.empty(max(1, qlinear.lora_workspace_bytes(len(s["tables"]), case["rank"], case["cols"], t)), dtype=torch.uint8, device="cuda"))
    if case["kind"] == "add":
        s["tensors"] = qlinear.lora_tensors([(table, Buf(y), Buf(o), r, y.stride(0), r) for table, y, o, r in zip(s["tables"], s["y"], s["out"], _rows(case))])


def _stream():
    return torch.cuda.current_stream().cuda_stream


# ------------------------------------------------------------------ a pass

def run(s):
    case = s["case"]
    if own:
        return _run_own(s, case)
    if case["kind"] == "route":
        return _routed(s["x"], s["bias"], case)
    out = TYPES[case["out"]][1]
    y = [_with_adapter(s["x"], y, a, b, s["scale"], s["ids"]) for y, (a, b) in zip(s["y"], s["lora"])]
    if case["kind"] == "gate_up":
        return (y[0] / (1.0 + torch.exp(-y[0])) * y[1]).to(out)
    return [v.to(out) for v in y]


def _run_own(s, case):
    from gemm_amd import qlinear
    x, type_x = s["x"], TYPES[case["x"]][0]
    if case["kind"] == "route":
        qlinear.moe_route_scores_dev(SCORES[case["score"]], type_x, Buf(x), case["tokens"], case["experts"], x.stride(0),
                                     Buf(s["bias"]) if case["bias"] else None, case["groups"], case["used"], case["group_top"], case["k"],
                                     case["renorm"], case["scale"], Buf(s["ids"]), Buf(s["weights"]), _stream())
        return s["ids"], s["weights"]
    type_w, type_y, type_out = (TYPES[case[n]][0] for n in ("w", "y", "out"))
    if case["kind"] == "add":
        qlinear.lora_add_dev(s["tensors"], type_w, case["adapters"], case["rank"], Buf(s["ids"]), type_x, Buf(x), type_y, type_out,
                             case["cols"], case["tokens"], x.stride(0), s["ws"], _stream())
        return s["out"]
    gate, up, out = s["y"][0], s["y"][1], s["out"][0]
    qlinear.lora_silu_mul_dev(s["tables"][0], s["tables"][1], type_w, case["adapters"], case["rank"], Buf(s["ids"]), type_x, Buf(x), type_y,
                              Buf(gate), Buf(up), type_out, Buf(out), out.shape[1], case["cols"], case["tokens"], x.stride(0), gate.stride(0),
                              out.stride(0), s["ws"], _stream())
    return out


# ------------------------------------------------------------------ the plain forms

def _with_adapter(x, y, a, b, scale, ids):
    """y + scale (x A^T) B^T with each token's own A, B and scale: the products with every adapter, of which a token keeps its own"""
    n, r = a.shape[:2]
    h = (x.float() @ a.reshape(n * r, -1).float().t()).reshape(-1, n, r)
    mine = ids[:, None] == torch.arange(n, device=x.device, dtype=torch.int32)
    h = torch.where(mine[:, :, None], h * scale[None, :, None], 0.0)
    return y.float() + h.reshape(-1, n * r) @ b.permute(0, 2, 1).reshape(n * r, -1).float()


def _routed(logits, bias, case):
    """The choice is by 64-bit values, since the last place may lie between neighbours; equal ones by index."""
    x = logits.double()
    there = x > -math.inf  # false for NaN
    x = torch.where(there, x, -math.inf)
    if case["score"] == "sigmoid":
        score = 1.0 / (1.0 + torch.exp(-x))
    else:
        e = torch.exp(x - torch.where(there.any(1, keepdim=True), x.amax(1, keepdim=True), 0.0))
        score = e / torch.where(there.any(1, keepdim=True), e.sum(1, keepdim=True), 1.0)
    value = torch.where(there, score + bias.double() if bias is not None else score, -math.inf)
    order = value if bias is not None else x
    t, n, groups = x.shape[0], x.shape[1], case["groups"]
    if groups > 1:
        best = torch.sort((value if case["group_top"] > 1 else order).reshape(t, groups, -1), dim=2, descending=True)[0][:, :, :case["group_top"]]
        some = best > -math.inf
        of_group = torch.where(some[:, :, 0], torch.where(some, best, 0.0).sum(2), -math.inf)
        kept = torch.sort(of_group, dim=1, descending=True, stable=True)[1][:, :case["used"]]
        in_kept = torch.zeros(t, groups, dtype=torch.bool, device=x.device).scatter_(1, kept, True)
        order = torch.where(in_kept.repeat_interleave(n // groups, dim=1), order, -math.inf)
    top, ids = torch.sort(order, dim=1, descending=True, stable=True)
    top, ids = top[:, :case["k"]], ids[:, :case["k"]]
    w = torch.where(top > -math.inf, score.gather(1, ids), 0.0)
    if case["renorm"]:
        total = w.sum(1, keepdim=True)
        w = w / torch.where(total > 0, total, 1.0)
    return torch.where(top > -math.inf, ids, -1).int(), (w * case["scale"]).float()


# ------------------------------------------------------------------ the definition in 64 bits

def exact(case, seed):
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    if case["kind"] == "route":
        return _routed_exactly(s, case)
    out = []
    for y, (a, b) in zip(s["y"], s["lora"]):
        z, ids = y.double(), s["ids"].tolist()
        for i, r in enumerate(_ranks(case)):  # adapter by adapter, the tokens that came with it
            at = torch.tensor([t for t, j in enumerate(ids) if j == i], dtype=torch.int64, device=y.device)
            h = s["x"][at].double() @ a[i, :r].double().t()
            z[at] += s["scale"][i].double() * (h @ b[i, :, :r].double().t())
        out.append(z)
    if case["kind"] == "gate_up":
        return out[0] * torch.sigmoid(out[0]) * out[1]
    return out


def _routed_exactly(s, case):
    x = s["x"].double().cpu().numpy()
    bias = s["bias"].double().cpu().numpy() if case["bias"] else None
    t, n, k, per = x.shape[0], x.shape[1], case["k"], case["experts"] // case["groups"]
    ids, weights = np.full((t, k), -1, np.int32), np.zeros((t, k))
    for row in range(t):
        at = np.flatnonzero(x[row] > -np.inf)
        if len(at) == 0:
            continue
        v = x[row, at]
        if case["score"] == "sigmoid":
            score = np.where(v >= 0, 1.0 / (1.0 + np.exp(-np.abs(v))), np.exp(-np.abs(v)) / (1.0 + np.exp(-np.abs(v))))
        else:
            score = np.exp(v - v.max())
            score /= score.sum()
        choose = v if bias is None else score + bias[at]
        if case["groups"] > 1:
            by = choose if bias is not None or case["group_top"] == 1 else score
            best = {g: np.sort(by[at // per == g])[::-1][:case["group_top"]].sum() for g in set((at // per).tolist())}
            used = sorted(best, key=lambda g: (-best[g], g))[:case["used"]]
            keep = np.isin(at // per, used)
            at, score, choose = at[keep], score[keep], choose[keep]
        first = np.lexsort((at, -choose))[:k]
        w = score[first]
        ids[row, :len(first)] = at[first]
        weights[row, :len(first)] = case["scale"] * (w / w.sum() if case["renorm"] else w)
    return torch.from_numpy(ids), torch.from_numpy(weights)


# ------------------------------------------------------------------ what a pass cannot do without

def work(case):
    size = {"f32": 4, "f16": 2, "bf16": 2}
    t = case["tokens"]
    if case["kind"] == "route":
        n = t * case["experts"]
        return {"bytes": n * size[case["x"]] + t * case["k"] * 8, "flops": 8 * n}
    rows, cols, r = _rows(case), case["cols"], case["rank"]
    used = {"one": 1, "mixed": min(t, case["adapters"]), "runs": min(t, case["adapters"], 5)}[case["ids"]]
    results = rows[0] if case["kind"] == "gate_up" else sum(rows)
    moved = used * r * (len(rows) * cols + sum(rows)) * size[case["w"]]
    moved += t * (cols * size[case["x"]] + sum(rows) * size[case["y"]] + results * size[case["out"]])
    return {"bytes": moved, "flops": 2 * t * r * (len(rows) * cols + sum(rows))}
