"""Routing by scores and low-rank adapters by their definitions, in 64 bits, and how far a kernel's results may be off."""
import numpy as np

import synth

F32, F16, BF16 = 0, 1, 30
HALF_STEP = {F32: 2.0 ** -24, F16: 2.0 ** -11, BF16: 2.0 ** -8}  # a rounding, relative
SMALLEST = {F32: 0.0, F16: 2.0 ** -25, BF16: 0.0}  # half of fp16's smallest step


def as_type(a, t):
    """-> (what the GPU holds, its values in 64 bits)"""
    a = np.asarray(a, np.float32)
    if t == F32:
        return a, a.astype(np.float64)
    if t == F16:
        h = a.astype(np.float16)
        return h, h.astype(np.float64)
    b = synth.to_bf16_bits(a).reshape(a.shape)
    return b, synth.bf16_bits_to_f32(b).astype(np.float64).reshape(a.shape)


NUMPY = {F32: np.float32, F16: np.float16, BF16: np.uint16}
BYTES = {F32: 4, F16: 2, BF16: 2}


def values(raw, t):
    return synth.bf16_bits_to_f32(raw).astype(np.float64).reshape(raw.shape) if t == BF16 else raw.astype(np.float64)


# ------------------------------------------------------------------ routing

def scores(x, sigmoid):
    """of a row; 0 for those that are not there"""
    there = x > -np.inf
    with np.errstate(invalid="ignore", over="ignore"):
        if sigmoid:
            e = np.exp(-np.abs(x))
            s = np.where(x >= 0, 1.0, e) / (1.0 + e)
        else:
            top = x[there].max() if there.any() else 0.0
            e = np.where(x == top, 1.0, np.exp(x - top))
            s = e / max(e[there].sum(), 1e-300)
    return np.where(there, s, 0.0)


def route(x, sigmoid, bias, n_group, used, group_top, k, renorm, scale):
    """one token -> (experts, weights)"""
    x = np.where(np.isnan(x), -np.inf, x)
    s = scores(x, sigmoid)
    v = x.copy()
    if bias is not None:
        v = np.where(x > -np.inf, s + bias, -np.inf)
        v = np.where(np.isnan(v), -np.inf, v)
    n = len(x)
    per = n // n_group
    if used < n_group:
        worth = []
        for g in range(n_group):
            at = [e for e in range(g * per, (g + 1) * per) if v[e] > -np.inf]
            at.sort(key=lambda e: -v[e])
            if not at:
                worth.append(-np.inf)
            elif group_top == 1:
                worth.append(v[at[0]])
            else:
                worth.append(sum(s[e] if bias is None else v[e] for e in at[:2]))
        keep = sorted((g for g in range(n_group) if worth[g] > -np.inf), key=lambda g: (-worth[g], g))[:used]
        v = np.where(np.isin(np.arange(n) // per, keep), v, -np.inf)
    first = sorted((e for e in range(n) if v[e] > -np.inf), key=lambda e: (-v[e], e))[:k]
    idx, w = np.full(k, -1, np.int32), np.zeros(k)
    idx[:len(first)] = first
    w[:len(first)] = s[first]
    if renorm and w.sum() > 0:
        w /= w.sum()
    return idx, w * scale


def route_bound(x, sigmoid, idx, w):
    """Scores in fp32: the exponential's argument is rounded (2^-24 of it and of the difference), the rest is a handful of roundings,
    and a sum of at most 2^12 positive terms in tree order a dozen more; w is what comes out. Below the smallest normal number the
    step is absolute."""
    x = np.where(np.isnan(x), -np.inf, x)
    top = x.max()
    with np.errstate(invalid="ignore"):  # (infinities share)
        far = np.where(idx >= 0, np.abs(x[np.maximum(idx, 0)] - (0.0 if sigmoid else top)), 0.0)
    far = np.where(np.isfinite(far), far, 0.0)
    spread = far.max() if len(far) else 0.0  # (renormalised weights take part of the other chosen scores' errors)
    return 2.0 ** -23 * (far + spread + 24.0) * np.abs(w) + 2.0 ** -126


# ------------------------------------------------------------------ adapters

class Adapter:
    def __init__(self, rng, rank, n_rows, n_cols, t, scale, size=1.0):
        self.rank, self.scale = rank, np.float32(scale)
        self.a_raw, self.a = as_type(size * rng.standard_normal((rank, n_cols)) / np.sqrt(n_cols), t)
        self.b_raw, self.b = as_type(rng.standard_normal((n_rows, rank)) / np.sqrt(rank), t)


def added(x, adapters, ids, n_rows, native):
    """-> (what the adapters add [tokens, n_rows], how far it may be off). A matrix instruction is taken to add its products to its
    sum within 2^-22 of their magnitudes: 32 columns each where both factors are of one 16-bit type (native), 4 otherwise; ranks go by
    4; a few roundings for parts, waves and the scale."""
    out, off = np.zeros((len(x), n_rows)), np.zeros((len(x), n_rows))
    n_cols = x.shape[1]
    chain = (n_cols + 31) // 32 * (1 if native else 8) + 80
    for t, i in enumerate(ids):
        if not 0 <= i < len(adapters) or adapters[i] is None:
            continue
        ad = adapters[i]
        h = ad.a @ x[t]
        h_off = chain * 2.0 ** -22 * (np.abs(ad.a) @ np.abs(x[t]))
        scale = abs(float(ad.scale))
        out[t] = float(ad.scale) * (ad.b @ h)
        off[t] = scale * (np.abs(ad.b) @ (h_off + (ad.rank / 4 + 16) * 2.0 ** -22 * np.abs(h)))
    return out, off


def add_bound(y, delta, off, out_type):
    total = y + delta
    off = off + 2.0 ** -23 * (np.abs(y) + np.abs(delta))
    return off * (1 + HALF_STEP[out_type]) + HALF_STEP[out_type] * np.abs(total) + SMALLEST[out_type]


def silu(g):
    e = np.exp(-np.abs(g))
    return g * np.where(g >= 0, 1.0, e) / (1.0 + e)


def silu_mul_bound(g, g_off, u, u_off, out_type):
    """silu's slope is at most 1.1; the exponential errs by 2^-24 of its argument (of the gate, relative in the result) and a few steps"""
    s = silu(g)
    s_off = 1.1 * g_off + 2.0 ** -23 * (np.abs(g) + 8.0) * np.abs(s) + 1.2e-36
    off = s_off * (np.abs(u) + u_off) + np.abs(s) * u_off + 2.0 ** -23 * np.abs(s * u)
    return off * (1 + HALF_STEP[out_type]) + HALF_STEP[out_type] * np.abs(s * u) + SMALLEST[out_type]
