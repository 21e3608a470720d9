"""Sampling from rows of which more tokens lie next to each other than a list holds: such a row is picked from value by value.
Running sums of the GPU are of bins whose tokens weigh a multiple of 2^-40 of the bin's weight (off by half of one, and by 2.4e-13 of a
polynomial): within 2^-40 of the sum."""
import math

import numpy as np
import pytest

from tests.test_gpu_sample import BF16, F16, F32, compare, draw, typed

pytestmark = pytest.mark.gpu
LAST = 1.0 - 2.0 ** -24  # the largest fp32 number below 1


@pytest.mark.parametrize("n", [4090, 32000, 32003, 64000, 128256, 256000])
@pytest.mark.parametrize("rows", [4, 12])  # long rows by several workgroups each, and by one
def test_the_last_of_equal_tokens_are_drawn(n, rows):
    """a row of one value, as long as a vocabulary is: random numbers close to 1 take its last tokens"""
    x = np.full((rows, n), 0.25)
    u = np.resize([0.9985, LAST, 0.9999, 0.98, 0.99995, 0.5], rows)
    compare(F32, x, u)
    compare(BF16, x, u, t=[0.7] * rows, k=[n] * rows)


# ------------------------------------------------------------------ the definition by values: equal tokens are counted, not added up one by one

class ByValue:
    """a row's values down the order, how many tokens each has, and running sums of weights in 64-bit mantissas"""

    def __init__(self, x, t):
        x = np.asarray(x, np.float64)
        self.x, there = x, x[x > -np.inf]  # (false for NaN)
        values, counts = np.unique(there, return_counts=True)
        self.values, self.counts = values[::-1], counts[::-1]
        top = self.values[0]
        with np.errstate(invalid="ignore"):
            w = np.exp((self.values - top) / np.float64(t)) if np.isfinite(top) else np.zeros(len(values))
        w[0] = 1.0
        self.w = w.astype(np.longdouble)

    def sum_of(self, kept):
        """of the first `kept` tokens"""
        upto = np.cumsum(self.counts)
        i = int(np.searchsorted(upto, kept))
        return np.sum((self.w * self.counts)[:i]) + self.w[i] * (kept - (upto[i - 1] if i else 0))

    def reaching(self, target, past):
        """-> (tokens until the running sum reaches, or is past, `target`; distance of the target from the nearest border of the value)"""
        upto = np.cumsum(self.w * self.counts)
        if past and target >= upto[-1]:
            return int(np.sum(self.counts)), 1.0
        i = min(int(np.searchsorted(upto, target, side="right" if past else "left")), len(upto) - 1)
        before = upto[i - 1] if i else np.longdouble(0)
        if self.w[i] == 0:
            return int(np.sum(self.counts[:i])), 1.0
        steps = (target - before) / self.w[i]
        c = int(np.floor(steps)) + 1 if past else max(1, int(np.ceil(steps)))
        return int(np.sum(self.counts[:i])) + min(c, int(self.counts[i])), float(abs(steps - np.round(steps)) * self.w[i])

    def pick(self, k, p, m, u):
        """-> (id, prob, distance of the nearest decision from a border, relative to the sum)"""
        kept = int(np.sum(self.counts))
        if k > 0:
            kept = min(kept, k)
        total, near = self.sum_of(kept), 1.0
        if p < 1:
            kept, near = self.reaching(np.longdouble(p) * total, False)
            near = near / float(total) if p > 0 else 1.0
            total = self.sum_of(kept)
        if m > 0:
            kept = max(1, min(kept, int(np.sum(self.counts[self.w >= m]))))
            total = self.sum_of(kept)
        at, off = self.reaching(np.longdouble(u) * total, True)
        near = min(near, off / float(total)) if u > 0 else near
        with_weight = int(np.sum(self.counts[self.w > 0]))
        at = min(at, kept, with_weight)
        i = int(np.searchsorted(np.cumsum(self.counts), at))
        nth = at - int(np.sum(self.counts[:i]))
        return int(np.flatnonzero(self.x == self.values[i])[nth - 1]), float(self.w[i] / total), near


def check(type_id, x, u, t=None, k=None, p=None, m=None):
    """picks and probabilities of rows against the definition; a decision within 2^-40 of a border is moved off it before the call"""
    a, values = typed(x, type_id)
    rows = len(a)
    u = np.array(u, np.float32)
    t = np.ones(rows, np.float32) if t is None else np.array(t, np.float32)
    p = None if p is None else np.array(p, np.float32)
    want = []
    for s in range(rows):
        row = ByValue(values[s], t[s])
        for _ in range(50):
            one = row.pick(0 if k is None else int(k[s]), 1.0 if p is None else p[s], 0.0 if m is None else np.float32(m[s]), u[s])
            if one[2] > 2.0 ** -40:
                break
            u[s] *= np.float32(0.9999)
            if p is not None and p[s] < 1:
                p[s] *= np.float32(0.9999)
        want.append(one)
    ids, probs = draw(type_id, a, u, t, k, p, m)
    assert ids.tolist() == [w[0] for w in want]
    # a weight and the sum are each off by 2^-40 of themselves at most, the quotient is rounded once to fp32
    want_p = np.array([w[1] for w in want])
    assert (np.abs(probs - want_p) <= (2.0 ** -24 + 2.0 ** -38) * want_p).all(), (probs, want_p)


def last_numbers(rows, rng, least):
    """fp32 numbers of [least, 1), the largest of them among them"""
    u = least + (LAST - least) * rng.random(rows)
    u[0] = LAST
    return np.minimum(u, LAST)


@pytest.mark.parametrize("n,down", [(66000, 11.0), (66000, 14.0), (128256, 20.7), (151936, 20.7), (262144, 16.0), (262144, 18.0), (262144, 20.7)])
@pytest.mark.parametrize("rows", [6, 20])
def test_a_flat_tail_far_below_the_largest(n, down, rows):
    """one large logit, all others equal: the tail weighs little, but its tokens are picked where the random number is close to 1"""
    rng = np.random.default_rng(n)
    x = np.full((rows, n), 3.0 - down)
    x[np.arange(rows), rng.integers(0, n, rows)] = 3.0
    w = math.exp(-down)
    least = 1.0 / (1.0 + (n - 1) * w)
    check(F32, x, last_numbers(rows, rng, least))
    check(F32, x, last_numbers(rows, rng, least), p=[1 - 0.1 * (1 - least)] * rows, m=[w / 2] * rows)
    check(F32, x, last_numbers(rows, rng, least), k=[n - 7] * rows, t=[1.0] * rows)
    check(F32, x, last_numbers(rows, rng, least), k=[n // 2] * rows, m=[2 * w] * rows)  # min-p takes the whole tail


@pytest.mark.parametrize("n", [30011, 128256])
@pytest.mark.parametrize("rows", [8, 24])
def test_tails_of_a_few_values(n, rows):
    """three values, the lower ones in crowds of their own: cuts inside a value, on its edge, between two"""
    rng = np.random.default_rng(n + rows)
    x = np.where(rng.random((rows, n)) < 0.5, -4.0, -9.5)
    x[:, rng.integers(0, n, 5)] = 1.5
    for _ in range(3):
        check(F32, x, rng.random(rows), k=rng.integers(0, n, rows))
        check(F32, x, rng.random(rows), p=rng.random(rows))
        check(F32, x, rng.random(rows), m=rng.choice([1e-6, 1e-4, 1e-3, 3e-3, 4.1e-3, 0.5], rows))
        check(BF16, x, rng.random(rows), k=rng.integers(0, n, rows), p=0.9 + 0.1 * rng.random(rows), m=rng.choice([0.0, 1e-4, 1e-3, 3e-3], rows), t=rng.choice([0.5, 1.0, 3.0], rows))


@pytest.mark.parametrize("type_id,centre,sigma,t,mask", [(BF16, -30.0, 2.0, 1.0, None), (BF16, -60.0, 2.0, 1.4, None), (BF16, 30.0, 2.0, 0.7, None), (F16, -200.0, 1.0, 1.0, None),
                                                         (F32, 0.0, 2.0, 6.0, np.finfo(np.float32).min), (F32, 0.0, 1.0, 1.0, -1e30), (F32, 5.0, 0.01, 1.0, -1e9), (F16, 0.0, 1.0, 2.0, -65504.0)])
@pytest.mark.parametrize("rows", [6, 20])
def test_crowded_bins(type_id, centre, sigma, t, mask, rows):
    """16-bit logits where their values lie far apart, and tokens pushed down by a finite number, which leave the others few bins"""
    rng = np.random.default_rng(7)
    n = 70001
    x = centre + sigma * rng.standard_normal((rows, n))
    if mask is not None:
        x[:, rng.integers(0, n, n // 500)] = mask
    check(type_id, x, rng.random(rows), t=[t] * rows)
    check(type_id, x, rng.random(rows), t=[t] * rows, p=rng.choice([0.0, 0.3, 0.9, 0.95, 0.999], rows))
    for _ in range(2):
        check(type_id, x, rng.random(rows), t=[t] * rows, k=rng.choice([0, 2, 20, 400, 1000, 1500, 30000], rows), p=rng.choice([1.0, 0.3, 0.95, 0.999], rows), m=rng.choice([0.0, 1e-3, 0.05, 0.9], rows))
    check(type_id, x, [0.0, LAST, 1.0, 2.0, 1e-30, 0.5][:rows] * (rows // 6) + [0.25] * (rows % 6), t=[t] * rows)


@pytest.mark.parametrize("n", [9001, 66001])
@pytest.mark.parametrize("many", [1, 2, 700, 5000])
def test_infinities(n, many):
    """several +infinities share the weight, whatever their number; finite tokens have none"""
    rng = np.random.default_rng(many)
    for rows in (7, 12):
        x = rng.standard_normal((rows, n))
        for s in range(rows):
            x[s, rng.choice(n, many, replace=False)] = np.inf
        x[0, 3] = np.nan
        x[1, 4] = -np.inf
        check(F32, x, rng.random(rows))
        check(F32, x, np.resize([0.0, LAST, 1.0, 7.0], rows))
        for _ in range(2):
            check(BF16, x, rng.random(rows), k=rng.choice([0, 2, 40, 600, 1000, 3000], rows), p=rng.choice([1.0, 0.0, 0.4, 0.95], rows), m=rng.choice([0.0, 0.3, 1.0], rows))


def test_the_same_token_every_time_in_a_crowd():
    rng = np.random.default_rng(3)
    for rows in (5, 30):
        x = typed(-30.0 + 2.0 * rng.standard_normal((rows, 70000)), BF16)[0]
        u = rng.random(rows)
        first = draw(BF16, x, u, p=[0.95] * rows)
        for _ in range(3):
            again = draw(BF16, x, u, p=[0.95] * rows)
            assert np.array_equal(again[0], first[0]) and np.array_equal(again[1], first[1])


@pytest.mark.parametrize("n", [50, 1500, 70000])
@pytest.mark.parametrize("rows", [3, 12])
def test_min_p_of_one_among_logits_that_weigh_the_same(n, rows):
    """logits that differ by less than a 64-bit weight can show: all of them weigh 1, and a min-p of 1 keeps them"""
    rng = np.random.default_rng(n)
    x = np.where(rng.random((rows, n)) < 0.5, 1e-40, 3e-40)
    for t in (1.0, 0.01):
        compare(F32, x, rng.random(rows), t=[t] * rows, m=[1.0] * rows)
        compare(F32, x, rng.random(rows), t=[t] * rows, m=[1.0] * rows, k=[n // 2] * rows, p=[0.7] * rows)
    compare(F32, x, rng.random(rows), t=[1.0] * rows, m=[1.0 - 2.0 ** -24] * rows)


@pytest.mark.parametrize("n", [3, 900, 5000, 66000])
@pytest.mark.parametrize("rows", [4, 12])
def test_random_numbers_of_one_and_more(n, rows):
    """nothing is past the whole sum: the last of the kept tokens, however little it weighs"""
    rng = np.random.default_rng(n)
    x = 2.0 * rng.standard_normal((rows, n)) - np.linspace(0.0, 10.0, n)
    u = np.resize([1.0, 2.0, np.inf, LAST], rows)
    check(F32, x, u)
    check(F32, x, u, t=[0.8] * rows, k=[0, 40, 700, 1500][:rows] * (rows // 4))
    check(F32, x, u, p=[0.95] * rows)
    check(F32, x, u, m=[1e-4] * rows, k=[0, 40, 700, 1500][:rows] * (rows // 4))


def test_a_border_between_bins_in_a_row_of_2_to_the_27():
    """The bins of a row so long hold weights in 2^-33, so that their sums are off by up to 2^-34. A crowd whose weights all round up, and a
    random number that falls between its sum and the bin's: the pick is the crowd's last token or the first behind it, not a token of another
    cut's bins far down the row."""
    n, unit = 1 << 27, 2.0 ** 33
    light = -20.7  # three tokens that weigh about 1e-9, which min-p keeps
    scale = 2040.0 / -float(np.float32(light))

    def in_bin(logit):
        """what a bin holds for a token"""
        at = np.round(-np.float64(logit) * scale)
        return np.round(np.exp((at / scale) + np.float64(logit)) * unit) / unit * np.exp(-at / scale)

    crowd = np.linspace(-0.31, -0.29, 20001).astype(np.float32)
    crowd = crowd[np.argmax(in_bin(crowd) / np.exp(crowd.astype(np.float64)))]
    assert in_bin(crowd) / math.exp(crowd) - 1 > 5e-11
    behind = np.float32(-0.32)
    assert np.round(-behind * scale) > np.round(-crowd * scale)
    head = 1.0 + 2000 * in_bin(crowd)
    fill, rest = [], head * (1 - 6e-11) - 1990 * in_bin(behind) - 3 * in_bin(light)  # the tail weighs 6e-11 less than the head by the bins
    while rest > 1e-9:
        fill.append(np.float32(min(math.log(rest), -0.5)))
        rest -= in_bin(fill[-1])
    head_exact, tail_exact = 1.0 + 2000 * math.exp(crowd), 1990 * math.exp(behind) + sum(math.exp(v) for v in fill) + 3 * math.exp(light)
    assert abs(head_exact / tail_exact - 1) < 1e-10
    x = np.full((1, n), -np.inf, np.float32)
    places = np.sort(np.random.default_rng(1).choice(n, 1 + 2000 + 1990 + len(fill) + 3, replace=False))
    x[0, places] = np.concatenate([[0.0], np.full(2000, crowd), np.full(1990, behind), fill, np.full(3, light)]).astype(np.float32)
    ids, _ = draw(F32, x, np.float32([0.5]), m=[1.0215e-9])  # a fifth of a bin below the three
    assert ids[0] in (places[2000], places[2001])
