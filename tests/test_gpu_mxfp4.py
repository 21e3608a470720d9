"""4-bit operands on the GPU through the C ABI: quantisation bit for bit, operands byte for byte, products against the same
products in 64 bits within what fp32 sums allow."""
import numpy as np
import pytest

from gemm_amd import qlinear
import synth
from tests import fp4_formulas as f

pytestmark = pytest.mark.gpu
F32, F16, BF16, MXFP4 = 0, 1, 30, synth.GGML_MXFP4
FILL = 0xA5


def as_type(x, type_id):
    """-> (array to upload, its values in 64 bits)"""
    if type_id == F32:
        a = np.asarray(x, np.float32)
        return a, a.astype(np.float64)
    if type_id == F16:
        a = np.asarray(x, np.float32).astype(np.float16)
        return a, a.astype(np.float64)
    a = synth.to_bf16_bits(np.asarray(x, np.float32))
    return a, synth.bf16_bits_to_f32(a).astype(np.float64)


def upload_rows(a, pitch, offset=0):
    """rows of `pitch` elements starting `offset` elements into an allocation; -> (buffer, address holder)"""
    wide = np.zeros((len(a), pitch), a.dtype)
    wide[:, :a.shape[1]] = a
    flat = np.concatenate([np.zeros(offset, a.dtype), wide.ravel()])
    return At(qlinear.DevBuf.from_numpy(flat), offset * a.itemsize)


class At:
    """a device address inside a buffer, as the binding takes one"""

    def __init__(self, buf, offset=0):
        self.buf, self.ptr, self.nbytes = buf, buf.ptr + offset, buf.nbytes - offset


def filled(n_bytes):
    return qlinear.DevBuf.from_numpy(np.full(n_bytes, FILL, np.uint8))


def activations(rows, cols, seed, scale=1.0):
    rng = np.random.default_rng(seed)
    x = rng.standard_normal((rows, cols)) * scale
    x[:, rng.integers(0, cols, max(1, cols // 100))] *= 12.0
    return x


def operand(type_id, a, n_rows, n_cols, pitch=None, offset=0):
    n = qlinear.mxfp4_operand_bytes(n_rows, n_cols)
    buf = filled(n + 64)
    src = upload_rows(a, pitch or a.shape[1], offset)
    qlinear.mxfp4_operand_dev(type_id, src, buf, n_rows, n_cols, n_cols if type_id == MXFP4 else (pitch or n_cols))
    qlinear.sync()
    return buf, n


# ------------------------------------------------------------------ quantisation

def quantize(type_id, a, cols, pitch=None, offset=0, out_offset=0):
    n = len(a) * (cols // 32) * 17
    buf = filled(out_offset + n + 64)
    qlinear.quantize_mxfp4_dev(type_id, upload_rows(a, pitch or cols, offset), At(buf, out_offset), len(a), cols, pitch or cols)
    qlinear.sync()
    got = buf.to_numpy(np.uint8, (out_offset + n + 64,))
    assert (got[:out_offset] == FILL).all() and (got[out_offset + n:] == FILL).all()
    return got[out_offset:out_offset + n].reshape(len(a), -1)


@pytest.mark.parametrize("type_id", [F16, BF16])
def test_every_16_bit_pattern(type_id):
    """all 65536 numbers (subnormals, infinities and NaNs among them), in blocks of neighbours and in blocks that mix magnitudes"""
    bits = np.arange(65536, dtype=np.uint16)
    for order in (bits, bits.reshape(32, 2048).T.ravel(), np.random.default_rng(3).permutation(bits)):
        a = order.reshape(64, 1024).view(np.float16) if type_id == F16 else order.reshape(64, 1024)
        x = a.astype(np.float64) if type_id == F16 else synth.bf16_bits_to_f32(a).astype(np.float64)
        assert np.array_equal(quantize(type_id, a, 1024), f.quantized(x))


def test_ties_and_borders_fp32():
    """every border between two codes, and its neighbours on both sides, under a largest magnitude of 4 to 7.99 at all powers of two,
    subnormal blocks and the largest numbers included"""
    borders = np.concatenate([f.BORDERS, f.E2M1, [5.999, 7.0]]).astype(np.float32)
    near = np.concatenate([borders, np.nextafter(borders, np.float32(0)), np.nextafter(borders, np.float32(9))])[:31 * 2 - 1]
    rows = []
    for top in (4.0, 4.5, 6.0, 7.99):
        for power in (-149, -140, -130, -128, -127, -126, -125, -60, -3, 0, 5, 77, 124, 125):
            for part in np.array_split(near, 3):
                block = np.zeros(32, np.float64)
                block[:len(part)] = part
                block[31] = -top
                rows.append(np.ldexp(block, power).astype(np.float32))
    rows.append(np.zeros(32, np.float32))
    a = np.array(rows, np.float32)
    assert np.isfinite(a).all()
    assert np.array_equal(quantize(F32, a, 32), f.quantized(a))


@pytest.mark.parametrize("type_id", [F32, F16, BF16])
@pytest.mark.parametrize("rows,cols,pad,offset,out_offset", [(1, 32, 0, 0, 0), (3, 96, 0, 0, 0), (2, 64, 8, 0, 16), (77, 1056, 5, 0, 0), (9, 4096, 0, 1, 0), (64, 4096, 8, 8, 1),
                                                             (255, 160, 0, 0, 3), (5, 14336, 0, 0, 0), (600, 544, 24, 0, 0)])
def test_blocks(type_id, rows, cols, pad, offset, out_offset):
    a, x = as_type(activations(rows, cols, rows + cols), type_id)
    assert np.array_equal(quantize(type_id, a, cols, cols + pad, offset, out_offset), f.quantized(x))


def test_the_decoder_reads_what_is_written():
    a, x = as_type(activations(33, 2048, 5), F32)
    got = quantize(F32, a, 2048)
    assert np.array_equal(qlinear.dequant_rows(MXFP4, got, 33, 2048).astype(np.float64), f.values_of(f.quantized(x)))


@pytest.mark.parametrize("type_id", [F32, F16, BF16])
@pytest.mark.parametrize("rows,cols,pad,offset", [(1, 1, 0, 0), (1, 31, 0, 0), (2, 33, 0, 0), (17, 100, 3, 0), (16, 128, 0, 0), (15, 512, 8, 0), (33, 520, 0, 8), (40, 1000, 0, 1),
                                                  (1, 4096, 0, 0), (130, 2080, 0, 0)])
def test_operand_of_floats(type_id, rows, cols, pad, offset):
    a, x = as_type(activations(rows, cols, rows * 7 + cols), type_id)
    buf, n = operand(type_id, a, rows, cols, cols + pad, offset)
    want = f.operand_of(*f.codes_of(f.padded(x)), rows, cols)
    assert n == len(want)
    got = buf.to_numpy(np.uint8, (n + 64,))
    assert np.array_equal(got[:n], want) and (got[n:] == FILL).all()


@pytest.mark.parametrize("rows,cols", [(1, 32), (16, 512), (17, 96), (100, 2080), (3, 14336), (300, 160)])
def test_operand_of_blocks(rows, cols):
    W = synth.make_weights(MXFP4, rows, cols, seed=rows, wild=True)
    buf, n = operand(MXFP4, W, rows, cols)
    b = W.reshape(rows, -1, 17)
    want = f.operand_of(b[..., 0], np.concatenate([b[..., 1:] & 15, b[..., 1:] >> 4], axis=2), rows, cols)
    got = buf.to_numpy(np.uint8, (n + 64,))
    assert np.array_equal(got[:n], want) and (got[n:] == FILL).all()


# ------------------------------------------------------------------ products

def weights(rows, cols, seed):
    """(array to make the operand of, its type, its values): blocks where the row is a whole number of them, else floats"""
    if cols % 32 == 0:
        W = synth.make_weights(MXFP4, rows, cols, seed=seed)
        return W, MXFP4, f.values_of(W)
    a, x = as_type(activations(rows, cols, seed, 0.05), F32)
    return a, F32, f.values_of(f.quantized(f.padded(x)))


def multiply(ops, x_type, X, y_type, rows, cols, tok, pad=0, pitch=None, y_offset=0):
    """one product (two operands: gate and up) -> results in 64 bits; what lies around them is untouched"""
    size, ldy = (4 if y_type == F32 else 2), rows + pad
    buf = filled(y_offset * size + tok * ldy * size + 64)
    n_ws = 0 if x_type == MXFP4 else qlinear.mxfp4_gemm_workspace_bytes(cols, tok)
    ws = filled(n_ws + 64) if n_ws else None
    args = (x_type, X, y_type, At(buf, y_offset * size), rows, cols, tok, pitch or cols, ldy, At(ws) if ws else None)
    if len(ops) == 2:
        qlinear.mxfp4_gemm_silu_mul_dev(*ops, *args)
    else:
        qlinear.mxfp4_gemm_dev(*ops, *args)
    qlinear.sync()
    if ws:
        assert (ws.to_numpy(np.uint8, (n_ws + 64,))[n_ws:] == FILL).all()
    raw = buf.to_numpy(np.uint8, (buf.nbytes,))
    body = raw[y_offset * size:y_offset * size + tok * ldy * size].reshape(tok, ldy * size)
    assert (raw[:y_offset * size] == FILL).all() and (raw[-64:] == FILL).all() and (body[:, rows * size:] == FILL).all()
    y = np.ascontiguousarray(body[:, :rows * size])
    return y.view(np.float32).astype(np.float64) if y_type == F32 else synth.bf16_bits_to_f32(y.view(np.uint16)).astype(np.float64)


def check(got, want, bound, y_type):
    if y_type == BF16:
        bound = bound * (1 + 2.0 ** -8) + 2.0 ** -8 * np.abs(want)
    worst = np.max(np.abs(got - want) - bound)
    assert worst <= 0, (worst, np.max(np.abs(got - want)))


# (rows, cols, tokens): one token to several tiles of them, rows and columns that end inside a group, a tile, a block
SHAPES = [(16, 128, 1), (1, 32, 1), (1, 1, 1), (5, 100, 3), (17, 512, 15), (33, 544, 16), (100, 1000, 17), (64, 2048, 31), (48, 640, 33), (130, 2080, 48), (257, 160, 49),
          (300, 4096, 1), (1000, 2080, 77), (96, 14336, 2), (520, 768, 64), (129, 512, 65), (256, 1024, 128), (257, 640, 129), (513, 1056, 255), (640, 512, 300), (1030, 384, 520),
          (60, 11008, 200), (2050, 256, 40)]


@pytest.mark.parametrize("rows,cols,tok", SHAPES)
def test_product(rows, cols, tok):
    W, w_type, w = weights(rows, cols, rows + tok)
    op, _ = operand(w_type, W, rows, cols)
    for x_type, y_type, pad in ((F32, F32, 0), (BF16, BF16, 3), (F16, F32, 1), (BF16, F32, 8)):
        a, x = as_type(activations(tok, cols, cols + tok), x_type)
        xq = f.values_of(f.quantized(f.padded(x)))
        got = multiply([op], x_type, upload_rows(a, cols + pad), y_type, rows, cols, tok, pad, cols + pad, y_offset=pad)
        check(got, xq @ w.T, f.product_bound(xq, w), y_type)


def gated(xq, g, u):
    """results in 64 bits and how far they may be off: the slope of silu is at most 1.1; expf, the sum, the quotient and the product take
    at most 8 half steps; a quotient below fp32's normal numbers may be lost"""
    a, b = xq @ g.T, xq @ u.T
    ea, eb = f.product_bound(xq, g), f.product_bound(xq, u)
    want = f.silu_mul(a, b)
    return want, 1.1 * ea * (np.abs(b) + eb) + np.abs(f.silu_mul(a, 1.0)) * eb + 8 * 2.0 ** -24 * np.abs(want) + 2.0 ** -126 * (1 + np.abs(b))


@pytest.mark.parametrize("rows,cols,tok", SHAPES)
def test_gate_and_up(rows, cols, tok):
    (G, g_type, g), (U, _, u) = weights(rows, cols, rows + tok), weights(rows, cols, rows + tok + 1)
    ops = [operand(g_type, W, rows, cols)[0] for W in (G, U)]
    for x_type, y_type, pad in ((F32, F32, 0), (BF16, BF16, 2)):
        a, x = as_type(activations(tok, cols, cols + tok) * 0.5, x_type)
        xq = f.values_of(f.quantized(f.padded(x)))
        got = multiply(ops, x_type, upload_rows(a, cols + pad), y_type, rows, cols, tok, pad, cols + pad)
        want, bound = gated(xq, g, u)
        check(got, want, bound, y_type)


KERNELS = [0, 11, 21, 22, 44]


@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("rows,cols,tok", [(1, 1, 1), (100, 128, 70), (130, 384, 33), (65, 640, 130), (300, 1000, 129), (513, 1056, 255), (257, 2080, 257), (640, 512, 300)])
def test_every_kernel(kernel, rows, cols, tok):
    """each kernel on small shapes, whatever the choice between them: rows, tokens and columns inside a tile, over several, one to
    five column tiles past a whole quad"""
    (G, g_type, g), (U, _, u) = weights(rows, cols, rows), weights(rows, cols, rows + 1)
    ops = [operand(g_type, W, rows, cols)[0] for W in (G, U)]
    a, x = as_type(activations(tok, cols, cols), F32)
    xq = f.values_of(f.quantized(f.padded(x)))
    x_op, _ = operand(F32, a, tok, cols)
    for up in (None,) if kernel == 11 else (None, ops[1]):
        for y_type, size, pad in ((F32, 4, 3), (BF16, 2, 0)):
            ldy = rows + pad
            out = filled(tok * ldy * size + 64)
            qlinear.check(qlinear.load().qlin_probe_mxfp4_gemm(kernel, ops[0].ptr, up.ptr if up else None, x_op.ptr, y_type, out.ptr, rows, cols, tok, ldy, None))
            qlinear.sync()
            raw = out.to_numpy(np.uint8, (out.nbytes,))
            body = raw[:-64].reshape(tok, ldy * size)
            assert (raw[-64:] == FILL).all() and (body[:, rows * size:] == FILL).all()
            y = np.ascontiguousarray(body[:, :rows * size])
            got = y.view(np.float32).astype(np.float64) if y_type == F32 else synth.bf16_bits_to_f32(y.view(np.uint16)).astype(np.float64)
            want, bound = xq @ g.T, f.product_bound(xq, g)
            if up:
                want, bound = gated(xq, g, u)
            check(got, want, bound, y_type)


@pytest.mark.parametrize("tok", [1, 5, 40, 100, 300])
def test_activations_as_an_operand(tok):
    """x_type MXFP4 takes what qlin_mxfp4_operand_dev makes, and gives the bits of the call that quantises itself"""
    rows, cols = 200, 1056
    W, w_type, _ = weights(rows, cols, 1)
    op, _ = operand(w_type, W, rows, cols)
    a, _ = as_type(activations(tok, cols, 2), BF16)
    x_op, _ = operand(BF16, a, tok, cols)
    direct = multiply([op], BF16, upload_rows(a, cols), F32, rows, cols, tok)
    assert np.array_equal(multiply([op], MXFP4, x_op, F32, rows, cols, tok), direct)
    assert np.array_equal(multiply([op, op], MXFP4, x_op, F32, rows, cols, tok), multiply([op, op], BF16, upload_rows(a, cols), F32, rows, cols, tok))


@pytest.mark.parametrize("tok", [3, 20, 70, 200])
def test_what_is_not_finite_stays_where_it_is(tok):
    """a token with a NaN or an infinity, a weight row with exponent byte 255: their results are NaN, no others change"""
    rows, cols = 150, 640
    W = synth.make_weights(MXFP4, rows, cols, seed=4)
    a = activations(tok, cols, 6).astype(np.float32)
    op, _ = operand(MXFP4, W, rows, cols)
    plain = multiply([op], F32, upload_rows(a, cols), F32, rows, cols, tok)
    a[1, 37], a[tok - 1, 600] = np.nan, -np.inf
    W = W.copy()
    W[70, 17 * 3] = 255
    W[149, 0] = 255
    op, _ = operand(MXFP4, W, rows, cols)
    for ops in ([op], [op, op]):
        got = multiply(ops, F32, upload_rows(a, cols), F32, rows, cols, tok)
        nan = np.zeros((tok, rows), bool)
        nan[[1, tok - 1], :] = True
        nan[:, [70, 149]] = True
        assert np.array_equal(np.isnan(got), nan)
        if len(ops) == 1:
            assert np.array_equal(got[~nan], plain[~nan])


def test_extreme_powers_of_two():
    """blocks whose powers of two differ by 2^200 between rows, tokens and columns, without overflow of a product"""
    rows, cols, tok = 48, 256, 20
    rng = np.random.default_rng(8)
    W = synth.make_weights(MXFP4, rows, cols, seed=9).reshape(rows, -1, 17).copy()
    W[..., 0] = rng.integers(30, 200, W.shape[:2])
    W = W.reshape(rows, -1)
    w = f.values_of(W)
    x = np.ldexp(rng.standard_normal((tok, cols)), rng.integers(-90, 40, (tok, 8)).repeat(32, axis=1)).astype(np.float32)
    xq = f.values_of(f.quantized(x))
    op, _ = operand(MXFP4, W, rows, cols)
    got = multiply([op], F32, upload_rows(x, cols), F32, rows, cols, tok)
    check(got, xq @ w.T, f.product_bound(xq, w) + 2.0 ** -126, F32)


@pytest.mark.parametrize("tok", [1, 24, 100, 260])
def test_same_bits_every_time(tok):
    rows, cols = 700, 2080
    W, w_type, _ = weights(rows, cols, 1)
    op, _ = operand(w_type, W, rows, cols)
    a, _ = as_type(activations(tok, cols, 2), BF16)
    X = upload_rows(a, cols)
    first = multiply([op], BF16, X, F32, rows, cols, tok)
    for _ in range(3):
        assert np.array_equal(multiply([op], BF16, X, F32, rows, cols, tok), first)


def test_sizes_of_nothing():
    buf = filled(4096)
    ws = filled(4096)
    qlinear.quantize_mxfp4_dev(F32, buf, buf, 0, 64, 64)
    qlinear.quantize_mxfp4_dev(F32, buf, buf, 3, 0, 0)
    qlinear.mxfp4_operand_dev(F32, buf, buf, 0, 64, 64)
    qlinear.mxfp4_gemm_dev(buf, F32, buf, F32, buf, 0, 64, 2, 64, 4, ws)
    qlinear.mxfp4_gemm_dev(buf, F32, buf, F32, buf, 4, 64, 0, 64, 4, ws)
    qlinear.sync()
    assert (buf.to_numpy(np.uint8, (4096,)) == FILL).all()


@pytest.mark.parametrize("tok", [4, 5, 6, 7, 8, 9])
@pytest.mark.parametrize("rows,cols", [(1, 8), (200, 520), (48, 4104), (257, 1536), (4000, 4096)])
def test_tokens_quantised_in_the_product(rows, cols, tok):
    """some tokens are quantised by the product where rows can be read 16 bytes at a time and the sizes are small, and in a launch of their own
    else: the same bits either way, whatever lies behind a row"""
    (G, g_type, _), (U, _, _) = weights(rows, cols, rows), weights(rows, cols, rows + 1)
    ops = [operand(g_type, W, rows, cols)[0] for W in (G, U)]
    for x_type in (F32, F16, BF16):
        a, _ = as_type(activations(tok, cols, tok + cols), x_type)
        x_op, _ = operand(x_type, a, tok, cols)
        for some in (ops[:1], ops):
            for y_type in (F32, BF16):
                want = multiply(some, MXFP4, x_op, y_type, rows, cols, tok)
                for pad in (0, 8, 1):
                    assert np.array_equal(multiply(some, x_type, upload_rows(a, cols + pad), y_type, rows, cols, tok, pad, cols + pad), want)


@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("rows,cols,tok", [(130, 200, 130), (640, 256, 300), (257, 768, 70), (513, 736, 255), (70, 896, 257), (300, 850, 129), (65, 1408, 513)])
def test_every_kernel_two_and_three_tiles_past_a_quad(kernel, rows, cols, tok):
    """2, 6, 7 and 11 column tiles: what follows the last four together, which takes other waits and exponents than they do"""
    test_every_kernel(kernel, rows, cols, tok)


@pytest.mark.parametrize("tok", [1, 20, 130, 300])
@pytest.mark.parametrize("sign", [-1.0, 1.0])
def test_gates_far_from_zero(tok, sign):
    """gates of 80 to 95 on either side, exact in fp32: silu within 8 half steps and a product's, down to where its reciprocal is subnormal
    (below -87.3, where it is smaller than 1.1e-36: there it may be lost, not more)"""
    rows, cols = 144, 64
    G = np.zeros((rows, 2, 32))
    G[:, 0, :2] = 64.0, 16.0
    for r in range(rows):
        left = 0.5 * (30 * r // rows)  # 0 to 14.5 of numbers that are codes
        for j, c in enumerate((6.0, 6.0, 2.0, 1.0, 0.5)):
            if left >= c:
                G[r, 1, j] = c
                left -= c
    G[:, 1, 30:] = 4.0, -4.0  # (keep the block's power of two at 1)
    G = sign * G.reshape(rows, cols)
    U = np.zeros((rows, cols))
    U[:, 2] = np.where(np.arange(rows) % 2 == 0, 1.0, -6.0)
    x = np.ones((tok, cols))
    for m in (G, U):
        assert np.array_equal(f.values_of(f.quantized(m)), m)
    ops = [operand(F32, m.astype(np.float32), rows, cols)[0] for m in (G, U)]
    got = multiply(ops, F32, upload_rows(x.astype(np.float32), cols), F32, rows, cols, tok)
    gate, up = G.sum(axis=1), U.sum(axis=1)
    assert gate.min() * sign >= -95.0 and np.abs(gate).min() == 80.0 and np.abs(gate).max() >= 94.0
    want = f.silu_mul(gate, up)
    lost = gate < -87.3
    assert (np.abs(got - want)[:, ~lost] <= 9 * 2.0 ** -24 * np.abs(want)[~lost]).all()
    assert (np.abs(got)[:, lost] <= (1 + 9 * 2.0 ** -24) * np.abs(want)[lost] + 2.0 ** -149).all()
