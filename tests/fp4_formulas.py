"""The 4-bit operators and the sampler written down plainly, in 64 bits: what the GPU results are compared with."""
import numpy as np

E2M1 = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
BORDERS = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0])  # half way between neighbours


def codes_of(x):
    """float rows [rows, multiple of 32] -> (exponent bytes [rows, blocks], codes [rows, blocks, 32])"""
    b = np.asarray(x, np.float64).reshape(len(x), -1, 32)
    bad = ~np.isfinite(b).all(axis=2)
    mag = np.abs(np.where(bad[:, :, None], 0.0, b))
    top = mag.max(axis=2)
    exponent = np.where(top > 0, np.frexp(top)[1] - 1, -1000)
    byte = np.maximum(exponent + 125, 0)
    v = np.ldexp(mag, (127 - byte)[:, :, None])
    # the nearest code; half way between codes c and c + 1 the even one of the two
    code = (v[..., None] > BORDERS).sum(axis=-1)
    code += np.where((v[..., None] == BORDERS) & (np.arange(7) % 2 == 1), 1, 0).sum(axis=-1)
    code = np.where(bad[:, :, None], 7, code) | np.where(np.signbit(b), 8, 0)
    return np.where(bad, 255, byte).astype(np.uint8), code.astype(np.uint8)


def blocks_of(byte, code):
    """GGML MXFP4 rows: [exponent][byte j = code j | code j + 16 << 4]"""
    out = np.empty(byte.shape + (17,), np.uint8)
    out[..., 0] = byte
    out[..., 1:] = code[..., :16] | code[..., 16:] << 4
    return out.reshape(len(byte), -1)


def quantized(x):
    return blocks_of(*codes_of(x))


def values_of(blocks):
    """rows of blocks -> their values; exponent byte 255 is NaN"""
    b = np.asarray(blocks).reshape(len(blocks), -1, 17)
    code = np.concatenate([b[..., 1:] & 15, b[..., 1:] >> 4], axis=2)
    v = np.where(code & 8, -1.0, 1.0) * E2M1[code & 7]
    v = np.ldexp(v, b[..., :1].astype(np.int64) - 127)
    return np.where(b[..., :1] == 255, np.nan, v).reshape(len(blocks), -1)


def padded(x):
    """columns up to a whole block, zeros"""
    return np.pad(x, ((0, 0), (0, -x.shape[1] % 32)))


def operand_of(byte, code, n_rows, n_cols):
    """the bytes of an operand: codes [row group][tile][16 g + r][16], exponents [row group][quad][16 g + r][tile % 4]"""
    groups, tiles = -(-n_rows // 16), -(-n_cols // 128)
    quads = -(-tiles // 4)
    full = np.zeros((groups * 16, quads * 16, 17), np.uint8)
    full[:byte.shape[0], :byte.shape[1]] = blocks_of(byte, code).reshape(byte.shape + (17,))
    full = full.reshape(groups, 16, quads * 4, 4, 17)  # [group, r, tile, g]
    codes = full[..., 1:].transpose(0, 2, 3, 1, 4)[:, :tiles]
    scales = full[..., 0].reshape(groups, 16, quads, 4, 4).transpose(0, 2, 4, 1, 3)
    return np.concatenate([np.ascontiguousarray(codes).ravel(), np.ascontiguousarray(scales).ravel()])


def product_bound(X, W):
    """How far an fp32 sum of the exact products may be off, whatever the order within 32 columns: those of a block's 32 products are
    joined with the sum so far, each joining cuts or rounds away at most 2^-23 of the largest partial sum, which no partial
    sum of magnitudes exceeds; 16 more for the joining of the waves."""
    return 2.0 ** -23 * (X.shape[1] / 32 + 16) * (np.abs(X) @ np.abs(W).T)


def silu_mul(g, u):
    with np.errstate(over="ignore"):
        return g / (1.0 + np.exp(-g)) * u


def sample(logits, t=1.0, k=0, p=1.0, m=0.0, u=0.0):
    """-> (id, prob, distance of u * sum from the nearest border between tokens, relative to the sum)"""
    x = np.asarray(logits, np.float64)
    order = np.argsort(np.where(np.isnan(x), np.inf, -x), kind="stable")
    order = order[x[order] > -np.inf]
    if len(order) == 0:
        return -1, 0.0, 1.0
    if not t > 0 or k == 1:
        return int(order[0]), 1.0, 1.0
    top = x[order[0]]
    with np.errstate(invalid="ignore"):
        w = np.where(x[order] == top, 1.0, np.exp((x[order] - top) / np.float64(t)) if np.isfinite(top) else 0.0)
    keep = len(order) if k <= 0 else min(k, len(order))
    if p < 1:
        sums = np.cumsum(w[:keep])
        keep = min(keep, 1 + int(np.searchsorted(sums, np.float64(p) * sums[-1], side="left")))
    if m > 0:
        keep = max(1, int((w[:keep] >= min(np.float64(m), 1.0)).sum()))
    sums = np.cumsum(w[:keep])
    target = (np.float64(u) if u > 0 else 0.0) * sums[-1]
    j = min(int(np.searchsorted(sums, target, side="right")), int(np.flatnonzero(w[:keep])[-1]))
    return int(order[j]), w[j] / sums[-1], float(np.abs(sums - target).min() / sums[-1])
