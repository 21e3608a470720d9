"""qlin_lora_add_dev and qlin_lora_silu_mul_dev against their definitions in 64 bits: every type, ranks and sizes of no round number,
pitches and addresses, tokens and adapters in any order, table entries that are no adapter, infinities, what lies beside the results."""
import numpy as np
import pytest

from gemm_amd import qlinear
from tests import adapter_formulas as f
from tests.adapter_formulas import BF16, F16, F32

pytestmark = pytest.mark.gpu


class Held:
    """host arrays in device memory, `shift` elements behind an allocation's start"""

    def __init__(self, raw, shift=0):
        self.size = raw.itemsize
        self.buf = qlinear.DevBuf.from_numpy(np.concatenate([np.zeros(shift, raw.dtype), raw.ravel()]))
        self.ptr, self.nbytes = self.buf.ptr + shift * raw.itemsize, raw.nbytes


def table_of(adapters, shift=0):
    """-> (device table, what it points to)"""
    t = np.zeros(max(1, len(adapters)), qlinear.LORA_DTYPE)
    held = []
    for i, a in enumerate(adapters):
        if a is None:
            continue
        pair = Held(a.a_raw, shift), Held(a.b_raw, shift)
        held.append(pair)
        t[i] = (pair[0].ptr, pair[1].ptr, a.rank, a.scale)
    return qlinear.DevBuf.from_numpy(t.view(np.uint8)), held


def pitched(v, pad, fill):
    wide = np.full((v.shape[0], v.shape[1] + pad), fill, np.float32)
    wide[:, :v.shape[1]] = v
    return wide


class Case:
    def __init__(self, seed, n_tok, rows, n_cols, ranks, ids, w=BF16, x=BF16, y=F32, out=F32, pad=0, shift=0, max_rank=None, pair=False, in_place=False):
        rng = np.random.default_rng(seed)
        self.rows, self.n_cols, self.n_tok, self.pair, self.in_place = rows, n_cols, n_tok, pair, in_place
        self.types, self.pad = (w, x, y, out), pad
        self.ids = np.asarray(ids, np.int32)
        assert len(self.ids) == n_tok
        self.max_rank = max_rank or max(r for r in ranks if r)
        self.adapters = [[Adapter if r == 0 else f.Adapter(rng, r, n, n_cols, w, 0.5 + i % 3) for i, r in enumerate(ranks)] for n in rows]
        self.adapters = [[a if isinstance(a, f.Adapter) else None for a in one] for one in self.adapters]
        self.x_raw, xv = f.as_type(pitched(rng.standard_normal((n_tok, n_cols)), pad, 1e4), x)
        self.x = xv[:, :n_cols]
        ys = [f.as_type(pitched(rng.standard_normal((n_tok, n)), pad, 3e4), y) for n in rows]
        self.y_raw, self.y = [a for a, _ in ys], [v[:, :n] for (_, v), n in zip(ys, rows)]
        self.shift = shift
        self.place()

    def place(self):
        self.tables, self.held = zip(*[table_of(one, self.shift) for one in self.adapters])
        self.dx = Held(self.x_raw, self.shift)
        self.dids = qlinear.DevBuf.from_numpy(self.ids)
        self.ws = qlinear.DevBuf.from_numpy(np.full(qlinear.lora_workspace_bytes(len(self.rows), self.max_rank, self.n_cols, self.n_tok), 0xFF, np.uint8))
        self.fresh()

    def fresh(self):
        """results and what they start from anew: NaN everywhere, one row behind the last token"""
        out = self.types[3]
        self.dy = [Held(r, self.shift) for r in self.y_raw]
        n_out = 1 if self.pair else len(self.rows)
        self.empty = [f.as_type(np.full((self.n_tok + 1, n + self.pad), -7.0), out)[0] for n in self.rows[:n_out]]
        self.dout = self.dy[:n_out] if self.in_place else [Held(e, self.shift) for e in self.empty]

    def enqueue(self, stream=None):
        w, x, y, out = self.types
        ld = [n + self.pad for n in self.rows]
        if self.pair:
            qlinear.lora_silu_mul_dev(self.tables[0], self.tables[1], w, len(self.adapters[0]), self.max_rank, self.dids, x, self.dx, y, self.dy[0], self.dy[1], out, self.dout[0],
                                      self.rows[0], self.n_cols, self.n_tok, self.n_cols + self.pad, ld[0], ld[0], self.ws, stream)
        else:
            tensors = qlinear.lora_tensors([(t, a, b, n, p, p) for t, a, b, n, p in zip(self.tables, self.dy, self.dout, self.rows, ld)])
            qlinear.lora_add_dev(tensors, w, len(self.adapters[0]), self.max_rank, self.dids, x, self.dx, y, out, self.n_cols, self.n_tok, self.n_cols + self.pad, self.ws, stream)

    def results(self):
        out = self.types[3]
        got = []
        for d, e, n in zip(self.dout, self.empty, self.rows):
            shape = (self.n_tok, e.shape[1]) if self.in_place else e.shape
            buf = d.buf.to_numpy(f.NUMPY[out], (self.shift + int(np.prod(shape)),))[self.shift:].reshape(shape)
            if not self.in_place:
                assert np.array_equal(buf[self.n_tok:], e[self.n_tok:]) and np.array_equal(buf[:, n:], e[:, n:])  # beside the results nothing is written
            got.append(buf[:self.n_tok, :n])
        return got

    def run(self):
        self.enqueue()
        qlinear.sync()
        return self.results()

    def native(self):
        return self.types[0] == self.types[1] != F32

    def want(self):
        sums = []
        for one, y, n in zip(self.adapters, self.y, self.rows):
            usable = [a if a is not None and 0 < a.rank <= self.max_rank else None for a in one]
            delta, off = f.added(self.x, usable, self.ids, n, self.native())
            sums.append((y, delta, off))
        out = self.types[3]
        if self.pair:
            (g, dg, og), (u, du, ou) = sums
            og, ou = og + 2.0 ** -23 * (np.abs(g) + np.abs(dg)), ou + 2.0 ** -23 * (np.abs(u) + np.abs(du))
            return [f.silu(g + dg) * (u + du)], [f.silu_mul_bound(g + dg, og, u + du, ou, out)]
        return [y + d for y, d, _ in sums], [f.add_bound(y, d, o, out) for y, d, o in sums]

    def check(self):
        got = self.run()
        want, bound = self.want()
        for g, w, b in zip(got, want, bound):
            v = f.values(g, self.types[3])
            assert (np.abs(v - w) <= b).all(), (np.abs(v - w) / b).max()
            if self.types[3] == F32 and w.size > 100:  # random signs: a chain of at most 128 instructions errs by about sqrt(128 / 2) 2^-24 of its sum
                assert np.linalg.norm(v - w) <= 1e-6 * np.linalg.norm(w)
        return got


def mixed(n_tok, n_adapter, seed=0):
    return np.random.default_rng(seed).integers(-1, n_adapter, n_tok)


@pytest.mark.parametrize("pair", [False, True])
@pytest.mark.parametrize("w", [F32, F16, BF16])
@pytest.mark.parametrize("x", [F32, F16, BF16])
def test_types(pair, w, x):
    for y, out in ((F32, F32), (F32, BF16), (BF16, F16), (F16, F32), (BF16, BF16)):
        rows = [96, 96] if pair else [96, 40, 40]
        Case(w + 7 * x + y, 21, rows, 160, [16, 8, 16], mixed(21, 3), w, x, y, out, pair=pair).check()


@pytest.mark.parametrize("pair", [False, True])
@pytest.mark.parametrize("n_tok", [1, 2, 3, 15, 16, 17, 33, 63, 64, 65, 130, 300])
def test_token_counts(pair, n_tok):
    rows = [136, 136] if pair else [136]
    Case(n_tok, n_tok, rows, 256, [16, 16, 8, 4, 16], mixed(n_tok, 5), pair=pair).check()
    Case(n_tok, n_tok, rows, 256, [16, 16, 8, 4, 16], np.sort(mixed(n_tok, 5)), x=F32, pair=pair).check()


@pytest.mark.parametrize("pair", [False, True])
@pytest.mark.parametrize("ranks", [[1], [3, 1, 2], [5, 12, 24], [16], [17, 31], [33, 48, 64], [65, 1, 128], [256, 100, 7], [255]])
@pytest.mark.parametrize("n_tok", [1, 19, 80])
def test_ranks(pair, ranks, n_tok):
    rows = [72, 72] if pair else [72]
    for w, x in ((BF16, BF16), (F16, F16), (F32, BF16), (BF16, F32)):
        Case(n_tok + len(ranks), n_tok, rows, 320, ranks, mixed(n_tok, len(ranks)), w, x, pair=pair).check()


@pytest.mark.parametrize("rows,n_cols", [([1], 1), ([3, 2, 1], 7), ([64], 31), ([65, 64, 63], 33), ([129], 257), ([1000], 2080), ([1027, 130, 131], 519), ([300], 2049), ([17], 14336), ([2100], 64)])
@pytest.mark.parametrize("n_tok", [1, 5, 70])
def test_sizes(rows, n_cols, n_tok):
    Case(n_cols, n_tok, rows, n_cols, [8, 16], mixed(n_tok, 2)).check()
    Case(n_cols, n_tok, rows, n_cols, [12, 16], mixed(n_tok, 2), F16, F32, F32, F16, pad=3).check()
    Case(n_cols, n_tok, [rows[0]] * 2, n_cols, [8, 16], mixed(n_tok, 2), out=BF16, pair=True).check()


@pytest.mark.parametrize("pair", [False, True])
@pytest.mark.parametrize("pad,shift", [(1, 0), (2, 0), (4, 0), (8, 0), (0, 1), (0, 2), (0, 4), (3, 3), (8, 1), (8, 8)])
def test_pitches_and_addresses(pair, pad, shift):
    rows = [68, 68] if pair else [68, 36, 36]
    for n_tok in (4, 70):
        for w, x, y, out in ((BF16, BF16, F32, F32), (F16, F32, BF16, F16), (F32, F16, F16, BF16)):
            Case(pad + shift, n_tok, rows, 96, [16, 8], mixed(n_tok, 2), w, x, y, out, pad=pad, shift=shift, pair=pair).check()


@pytest.mark.parametrize("pair", [False, True])
@pytest.mark.parametrize("n_tok", [1, 40, 200])
def test_in_place(pair, n_tok):
    rows = [200, 200] if pair else [200, 100]
    for t in (F32, BF16, F16):
        a = Case(3, n_tok, rows, 128, [16, 8, 4], mixed(n_tok, 3), y=t, out=t, pair=pair, pad=4)
        b = Case(3, n_tok, rows, 128, [16, 8, 4], mixed(n_tok, 3), y=t, out=t, pair=pair, pad=4, in_place=True)
        for p, q in zip(a.check(), b.run()):
            assert np.array_equal(p, q)


@pytest.mark.parametrize("order", ["one", "each its own", "none", "alternating", "runs", "sorted"])
@pytest.mark.parametrize("n_tok", [48, 129])
def test_orders_of_adapters(order, n_tok):
    n = 70
    ids = {"one": [3] * n_tok, "each its own": [i % n for i in range(n_tok)], "none": [-1] * n_tok, "alternating": [i % 2 * 5 - 1 for i in range(n_tok)],
           "runs": [i // 20 for i in range(n_tok)], "sorted": sorted(i * 7 % n for i in range(n_tok))}[order]
    c = Case(1, n_tok, [80, 24], 96, [8] * n, ids)
    got = c.check()
    if order == "none":
        for g, y in zip(got, c.y_raw):
            assert np.array_equal(g, y)
    Case(2, n_tok, [80, 80], 96, [8] * n, ids, out=BF16, pair=True).check()


def test_a_token_keeps_its_results_in_any_company():
    """within the same number of tokens, order and neighbours change nothing"""
    n_tok = 60
    ids = mixed(n_tok, 6, 4)
    c = Case(5, n_tok, [130, 64], 512, [16, 8, 16, 32, 4, 16], ids)
    first = c.check()
    turn = np.random.default_rng(1).permutation(n_tok)
    c.ids, c.x_raw, c.x = c.ids[turn], c.x_raw[turn], c.x[turn]
    c.y_raw, c.y = [y[turn] for y in c.y_raw], [y[turn] for y in c.y]
    c.place()
    for a, b in zip(first, c.check()):
        assert np.array_equal(a[turn], b)


@pytest.mark.parametrize("pair", [False, True])
def test_entries_and_ids_that_are_no_adapter(pair):
    """rank 0, above max_rank, negative; null pointers; ids outside of the table: out is Y (or its silu), bit for bit what no adapter gives"""
    rows = [40, 40] if pair else [40, 20]
    ids = [0, 1, 2, 3, 4, 5, 6, -1, -5, 7, 100, 2 ** 31 - 1, -2 ** 31, 0]
    c = Case(6, len(ids), rows, 64, [16, 16, 16, 16, 16, 16, 40], ids, max_rank=32, pair=pair)
    for table, one in zip(c.tables, c.adapters):
        t = table.to_numpy(np.uint8, (len(one) * 24,)).view(qlinear.LORA_DTYPE)
        t["rank"][1], t["rank"][2], t["A"][3], t["B"][4] = 0, -16, 0, 0
        raw = t.view(np.uint8)
        assert qlinear.load().qlin_dev_upload(table.ptr, raw.ctypes.data, raw.nbytes) == 0
        one[1] = one[2] = one[3] = one[4] = None
    got = c.check()
    if not pair:
        for g, y in zip(got, c.y_raw):
            assert np.array_equal(g[1:5], y[1:5]) and np.array_equal(g[6:13], y[6:13])


def test_no_adapters_at_all():
    c = Case(7, 9, [30], 64, [16], [0] * 9)
    tensors = qlinear.lora_tensors([(type("Null", (), {"ptr": None})(), c.dy[0], c.dout[0], 30, 30, 30)])
    qlinear.lora_add_dev(tensors, BF16, 0, 16, c.dids, BF16, c.dx, F32, F32, 64, 9, 64, c.ws)
    qlinear.sync()
    assert np.array_equal(c.results()[0], c.y_raw[0])


def test_a_tensor_without_rows():
    c = Case(8, 5, [30, 30, 30], 64, [16], [0, -1, 0, 0, 0])
    null = type("Null", (), {"ptr": None})()
    tensors = qlinear.lora_tensors([(c.tables[0], c.dy[0], c.dout[0], 30, 30, 30), (null, null, null, 0, 0, 0), (c.tables[2], c.dy[2], c.dout[2], 30, 30, 30)])
    qlinear.lora_add_dev(tensors, BF16, 1, 16, c.dids, BF16, c.dx, F32, F32, 64, 5, 64, c.ws)
    qlinear.sync()
    want, bound = c.want()
    got = c.results()
    for i in (0, 2):
        assert (np.abs(got[i] - want[i]) <= bound[i]).all()
    assert (got[1] == -7).all()


def test_a_tensor_without_rows_has_no_table():
    """what a tensor without rows says of its adapters is not looked at: not a byte of the workspace depends on it"""
    n_tok = 80  # two launches
    c = Case(17, n_tok, [30, 30, 30], 64, [16, 8], mixed(n_tok, 2))
    null = type("Null", (), {"ptr": None})()
    seen = []
    for table in (null, c.tables[1]):
        c.ws = qlinear.DevBuf.from_numpy(np.full(c.ws.nbytes, 0xFF, np.uint8))
        c.fresh()
        tensors = qlinear.lora_tensors([(c.tables[0], c.dy[0], c.dout[0], 30, 30, 30), (table, null, null, 0, 0, 0), (c.tables[2], c.dy[2], c.dout[2], 30, 30, 30)])
        qlinear.lora_add_dev(tensors, BF16, 2, 16, c.dids, BF16, c.dx, F32, F32, 64, n_tok, 64, c.ws)
        qlinear.sync()
        want, bound = c.want()
        got = c.results()
        for i in (0, 2):
            assert (np.abs(got[i] - want[i]) <= bound[i]).all()
        assert (got[1] == -7).all()
        seen.append(c.ws.to_numpy(np.uint8, (c.ws.nbytes,)))
    assert np.array_equal(*seen)


@pytest.mark.parametrize("pair", [False, True])
@pytest.mark.parametrize("w,x", [(BF16, BF16), (F16, F16), (BF16, F32)])
@pytest.mark.parametrize("n_tok", [5, 80])
def test_what_is_not_finite_stays_with_its_tokens(pair, w, x, n_tok):
    rows = [70, 70] if pair else [70, 36]
    ids = np.arange(n_tok) % 4 - 1
    c = Case(9, n_tok, rows, 96, [16, 8, 16], ids, w, x, pair=pair)
    clean = c.run()
    poison = {BF16: [0x7F80, 0x7FC0], F16: np.array([np.inf, np.nan], np.float16), F32: np.array([np.inf, np.nan], np.float32)}
    c.x_raw[1, 3], c.x_raw[2, 90] = poison[x][0], poison[x][1]  # token 1: adapter 0, token 2: adapter 1
    c.adapters[0][2].a_raw[2, 5] = poison[w][1]  # the tokens of adapter 2
    c.place()
    got = c.run()
    lost = np.zeros(n_tok, bool)
    lost[[1, 2]] = True
    for i, (a, b) in enumerate(zip(clean, got)):
        mine = lost | (ids == 2) if i == 0 else lost
        assert np.array_equal(a[~mine], b[~mine])
        assert not np.isfinite(b[mine]).any()


@pytest.mark.parametrize("n_tok", [5, 80])
def test_the_largest_numbers_and_infinities(n_tok):
    """h is the activation itself and B 2^-100: an infinite h gives infinite results, the largest one results that are finite, off by the one rounding"""
    c = Case(12, n_tok, [8], 64, [1], [0] * n_tok, BF16, F32)
    a = c.adapters[0][0]
    a.a_raw[:], a.b_raw[:], a.scale = 0, 0x0D80, np.float32(1.0)
    a.a_raw[0, 5] = 0x3F80
    most = np.finfo(np.float32).max
    c.x_raw[:5, 5] = [1.0, np.inf, most, -most, -np.inf]
    c.place()
    got = c.run()[0]
    assert (got[1] == np.inf).all() and (got[4] == -np.inf).all()
    want = c.y_raw[0][2:4].astype(np.float64)[:, :8] + np.array([[1.0], [-1.0]]) * float(most) * 2.0 ** -100
    assert (np.abs(got[2:4] - want) <= 2.0 ** -24 * np.abs(want)).all()


@pytest.mark.parametrize("pair", [False, True])
@pytest.mark.parametrize("w", [BF16, F16, F32])
@pytest.mark.parametrize("n_tok,n_cols,ranks", [(5, 64, [16, 3]), (20, 64, [80, 5]), (80, 64, [16, 3]), (80, 64, [33, 20]), (80, 2304, [16, 3]), (300, 64, [16, 64])])  # every way h goes
def test_infinities_of_B(pair, w, n_tok, n_cols, ranks):
    """an infinite element of B makes its results infinite, whatever bits h has: here the few of an element of A"""
    ids = np.arange(n_tok) % 3 - 1
    c = Case(18, n_tok, [70, 70], n_cols, ranks, ids, w, w, pair=pair)
    one = f.as_type(np.ones(1), w)[0][0]
    c.x_raw[:], c.x[:] = 0, 0.0
    c.x_raw[:, 5], c.x[:, 5] = one, 1.0
    c.place()
    want, bound = c.want()
    inf = f.as_type(np.array([np.inf, -np.inf]), w)[0]
    for a in c.adapters[1]:  # (of gate and up: up)
        for row, k, which in ((3, 0, 0), (5, 1, 1), (7, 0, 0), (7, a.rank - 1, 0), (69, 2, 1)):
            a.b_raw[row, k], a.b[row, k] = inf[which], [np.inf, -np.inf][which]
    c.place()
    got = c.run()
    g = [f.values(v, F32) for v in got]
    if not pair:
        assert (np.abs(g[0] - want[0]) <= bound[0]).all()
    lost = np.zeros(want[-1].shape, bool)
    lost[np.ix_(ids >= 0, [3, 5, 7, 69])] = True
    assert (np.abs(g[-1] - want[-1])[~lost] <= bound[-1][~lost]).all()
    for t in np.flatnonzero(ids >= 0):
        a = c.adapters[1][ids[t]]
        with np.errstate(invalid="ignore"):
            expect = c.y[1][t] + float(a.scale) * (a.b @ a.a[:, 5])
            if pair:
                gate = c.adapters[0][ids[t]]
                expect = f.silu(c.y[0][t] + float(gate.scale) * (gate.b @ gate.a[:, 5])) * expect
        assert np.array_equal(g[-1][t][[3, 5, 7, 69]], expect[[3, 5, 7, 69]], equal_nan=True)


def test_an_adapter_of_one_row_and_column_copies_what_it_should():
    """A picks column 5, B puts it into row 3, scale 2: exact"""
    c = Case(10, 3, [8], 64, [1], [0, -1, 0])
    a = c.adapters[0][0]
    a.a_raw[:], a.b_raw[:] = 0, 0
    a.a_raw[0, 5], a.b_raw[3, 0], a.scale = 0x3F80, 0x3F80, np.float32(2.0)
    c.place()
    got = c.run()[0]
    want = c.y_raw[0].copy()
    want[[0, 2], 3] += (2 * c.x[[0, 2], 5]).astype(np.float32)
    assert np.array_equal(got, want)


def test_same_bits_again():
    for pair in (False, True):
        c = Case(11, 150, [300, 300], 1024, [16, 64, 32], mixed(150, 3), pair=pair)
        first = c.run()
        for _ in range(3):
            c.fresh()
            for a, b in zip(first, c.run()):
                assert np.array_equal(a, b)


@pytest.mark.parametrize("kind", ["add", "gate_up"])
def test_long_prompts(kind):
    """more tokens than a tile by far, several runs, large ranks; only some tokens are compared"""
    n_tok = 1100
    ids = np.repeat([2, -1, 0, 1, 2], [300, 1, 499, 200, 100])
    c = Case(12, n_tok, [520, 520], 768, [64, 32, 16], ids, out=BF16 if kind == "gate_up" else F32, pair=kind == "gate_up")
    c.check()


class Far:
    """rows 2^27 elements apart in device memory: offsets that 32 bits do not hold, of bytes and of elements"""
    PITCH = 1 << 27

    def __init__(self, raw):
        self.n, self.cols, self.dtype = raw.shape[0], raw.shape[1], raw.dtype
        self.buf = qlinear.DevBuf(((self.n - 1) * self.PITCH + self.cols) * raw.itemsize)
        self.ptr, self.nbytes = self.buf.ptr, self.buf.nbytes
        for t in range(self.n):
            row = np.ascontiguousarray(raw[t])
            qlinear.check(qlinear.load().qlin_dev_upload(self.at(t), row.ctypes.data, row.nbytes))

    def at(self, t):
        return self.ptr + t * self.PITCH * self.dtype.itemsize

    def rows(self):
        out = np.empty((self.n, self.cols), self.dtype)
        for t in range(self.n):
            row = np.empty(self.cols, self.dtype)
            qlinear.check(qlinear.load().qlin_dev_download(row.ctypes.data, self.at(t), row.nbytes))
            out[t] = row
        return out


@pytest.mark.parametrize("rank", [8, 80])  # one launch, two
def test_rows_far_apart(rank):
    """the bits of the same rows next to each other"""
    n_tok, n_rows, n_cols = 20, 70, 48
    c = Case(13, n_tok, [n_rows, n_rows], n_cols, [rank, 5], mixed(n_tok, 2), pair=True)
    want = c.run()[0]
    x, gate, up = Far(c.x_raw), Far(c.y_raw[0]), Far(c.y_raw[1])
    qlinear.lora_silu_mul_dev(c.tables[0], c.tables[1], BF16, 2, c.max_rank, c.dids, BF16, x, F32, gate, up, F32, gate, n_rows, n_cols, n_tok, Far.PITCH, Far.PITCH, Far.PITCH, c.ws)
    qlinear.sync()
    assert np.array_equal(gate.rows(), want) and np.array_equal(up.rows(), c.y_raw[1])


@pytest.mark.parametrize("n_tok", [1, 3])
def test_long_rows(n_tok):
    Case(14, n_tok, [5], (1 << 21) + 5, [2, 1], mixed(n_tok, 2) if n_tok > 1 else [0]).check()


def test_many_rows():
    n_rows = (1 << 22) + 3
    c = Case(15, 2, [n_rows], 16, [1, 2], [0, 1], y=BF16, out=BF16)
    c.check()


@pytest.mark.parametrize("n_tok,rows,n_cols,ranks", [(1, [70, 40, 40], 9000, [200]), (20, [300], 9000, [64, 80]), (70, [300], 4096, [16, 5, 16]), (300, [70, 40], 2100, [64, 3]), (2050, [70, 40], 64, [64, 20])])
@pytest.mark.parametrize("w", [F32, BF16])
def test_nothing_is_written_behind_the_workspace(n_tok, rows, n_cols, ranks, w):
    c = Case(16, n_tok, rows, n_cols, ranks, mixed(n_tok, len(ranks)), w=w)
    want, guard = c.run(), 4096
    need = c.ws.nbytes
    c.ws = qlinear.DevBuf.from_numpy(np.full(need + guard, 0xAB, np.uint8))
    whole, c.ws.nbytes = c.ws.nbytes, need
    c.fresh()
    for a, b in zip(want, c.run()):
        assert np.array_equal(a, b)
    c.ws.nbytes = whole
    assert (c.ws.to_numpy(np.uint8, (whole,))[need:] == 0xAB).all()
