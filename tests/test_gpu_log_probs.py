"""log_probs, log_probs_grad and log_probs_with_grad against their formulas in float64.

Tolerances, derived before the first run. u is half a step of what sums are held in (2^-24, for float64 tensors 2^-53), half that
of the logits' dtype, d = x - peak (rounded once: u |d|). An exponential has a relative error of (2 |d| + 4) u: the rounding of d and of
its product with log2 e, and three steps of the hardware's. A lane's sum is rescaled only where its largest element rises, by
exponentials whose |d| add up to no more than the row's range D, at most once a vector: R times. With K additions on any path
  total    relative E = (2 D + 4 (R + 2) + K) u           (D bounds |d| of the terms too)
  log_p    E + 4 u (|d| + log total)
  entropy  (1 + 2 M) E + 4 u (log total + M), M = mean |d| under p
  p        relative E + (2 |d| + 6) u
and the gradient what these make of its terms, then half."""

import numpy as np
import pytest

from helpers import decode, encode, logical, same_bits
from raven_amd import dtype as dt

pytestmark = pytest.mark.gpu

FLOATS = [dt.float32, dt.bfloat16, dt.float16, dt.float64]
HALF = {"float64": 2.0 ** -53, "float32": 2.0 ** -24, "float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}
TINY = {"float64": 2.0 ** -1022, "float32": 2.0 ** -126, "float16": 2.0 ** -25, "bfloat16": 2.0 ** -126}  # (2^-126: what the exponential flushes)


def tensor(hip, storage, d):
    return hip.reshape(hip.from_host(np.ascontiguousarray(storage), d), storage.shape)


def stats(d):
    return dt.float64 if d is dt.float64 else dt.float32


def unit(d):
    return 2.0 ** -53 if d is dt.float64 else 2.0 ** -24


def drawn(shape, d, oracle, seed, scale=2.5):
    s = encode(np.random.default_rng(seed).standard_normal(shape) * scale, d, oracle)
    return s, decode(s, d, oracle)


def lanes(n, d):
    v = 16 // d.itemsize
    return 8 if n <= 8 * v else 64 if n <= 256 * v else 256 if n <= 1024 * v else 1024


class Want:
    """The formulas, and what they may be off by."""

    def __init__(self, x, tokens, d, top=0):
        with np.errstate(all="ignore"):
            u, n, g = unit(d), x.shape[-1], lanes(x.shape[-1], d)
            v = 16 // d.itemsize
            self.peak = np.fmax.reduce(x, -1)
            self.d = x - self.peak[..., None]
            e = np.exp(self.d)
            self.total = e.sum(-1)
            self.log_total = np.log(self.total)
            self.m = np.where(e > 0, -self.d * e, 0).sum(-1) / self.total
            self.entropy = self.log_total + self.m
            self.p = e / self.total[..., None]
            real = np.clip(tokens, 0, n - 1)
            picked = np.take_along_axis(self.d, real[..., None], -1)[..., 0]
            self.log_p = np.where(tokens < 0, 0, np.where(tokens >= n, np.nan, picked - self.log_total))
            span = np.where(np.isfinite(self.d), -self.d, 0).max(-1)
            steps = -(-n // (g * v)) + 1
            self.e = (2 * span + 4 * (steps + 2) + steps * v + 24) * u
            size = lambda q: np.where(np.isfinite(q), np.abs(q), 0)  # noqa: E731
            self.log_p_err = self.e + 4 * u * (size(picked) + np.abs(self.log_total))
            self.entropy_err = (1 + 2 * self.m) * self.e + 4 * u * (np.abs(self.log_total) + self.m)
            self.u, self.size, self.tokens, self.n = u, size, tokens, n
            if top:
                self.top = np.argsort(-x, -1, kind="stable")[..., :top]
                self.top_log_p = np.take_along_axis(self.d, self.top, -1) - self.log_total[..., None]
                self.top_err = self.e[..., None] + 4 * u * (size(self.top_log_p) + 2 * np.abs(self.log_total)[..., None])

    def gradient(self, g, g_entropy=None):
        with np.errstate(all="ignore"):
            u, p, far = self.u, self.p, self.size(self.d)
            g = np.where(self.tokens < 0, 0, np.where(self.tokens >= self.n, np.nan, g))[..., None]
            one = (np.arange(self.n) == self.tokens[..., None]) * 1.0
            relative = self.e[..., None] + (2 * far + 6) * u
            d = g * (one - p)
            err = np.abs(g) * (p * (relative + 2 * u) + one * 2 * u)
            if g_entropy is not None:
                ge, lt, h = g_entropy[..., None], self.log_total[..., None], self.entropy[..., None]
                inner = np.where(p > 0, self.d - lt + h, 0)
                d = d - ge * p * inner
                err = err + np.abs(ge) * p * (np.abs(inner) * (relative + 2 * u) + self.e[..., None] * (3 + 2 * self.m[..., None])
                                              + 4 * u * (far + 2 * np.abs(lt) + np.abs(h) + self.m[..., None]))
            return d, err


def within(got, want, err, half, tiny, what):
    assert got.shape == want.shape, (what, got.shape, want.shape)
    assert np.array_equal(np.isnan(got), np.isnan(want)), f"{what}: NaNs elsewhere"
    with np.errstate(all="ignore"):
        inf = np.isinf(want)
        assert np.array_equal(got[inf], want[inf]), f"{what}: infinities differ"
        ok = ~(np.isnan(want) | inf)
        off, lim = np.abs(got - want)[ok], (err + half * (np.abs(want) + err) + tiny)[ok]
    if off.size:
        assert np.all(off <= lim), f"{what}: {np.max(off / lim)} times the bound"


def check_score(got, want, d, oracle, top=0, what=""):
    sd = stats(d)
    names = ("log_p", "entropy", "peak", "total")
    for t, name, w, err in zip(got, names, (want.log_p, want.entropy, want.peak, want.total),
                               (want.log_p_err, want.entropy_err, 0 * want.e, want.e * np.abs(want.total))):
        within(logical(t).astype(np.float64), w, err, HALF[sd.name], 0, f"{what} {name} of {d.name}")
    if top:
        assert np.array_equal(logical(got[5]), want.top), f"{what} most likely tokens of {d.name}"
        within(logical(got[4]).astype(np.float64), want.top_log_p, want.top_err, HALF[sd.name], 0, f"{what} their log probabilities")


def check_gradient(got, want, g, g_entropy, d, oracle, what=""):
    w, err = want.gradient(g, g_entropy)
    within(decode(logical(got), d, oracle), w, err, HALF[d.name], TINY[d.name], f"{what} gradient of {d.name}")


def values(hip, v, d):
    """Values of rows as a handle, and as they are held."""
    s = np.asarray(v).astype(stats(d).np_storage)
    return tensor(hip, s, stats(d)), s.astype(np.float64)


def everything(hip, oracle, d, hx, x, tokens, tops=(0,), what=""):
    rows = tokens.shape
    ht = tensor(hip, tokens.astype(np.int32), dt.int32)
    rng = np.random.default_rng(int(x.shape[-1]))
    (hg, g), (hge, ge) = values(hip, rng.standard_normal(rows), d), values(hip, rng.standard_normal(rows), d)
    for top in tops:
        want = Want(x, tokens, d, top)
        got = hip.log_probs(hx, ht, top)
        assert hip.last_path() == ("log_probs_top" if top else "log_probs")
        check_score(got, want, d, oracle, top, f"{what} top {top}")
        for a, b in zip(got, hip.log_probs(hx, ht, top)):
            if a is not None:
                same_bits(logical(a), logical(b), "equal calls")
    log_p, entropy, peak, total = got[:4]
    check_gradient(hip.log_probs_grad(hg, hx, ht, peak, total), want, g, None, d, oracle, what)
    check_gradient(hip.log_probs_grad(hg, hx, ht, peak, total, hge, entropy), want, g, ge, d, oracle, what + " entropy")
    for entropy_too in (False, True):
        lp, h, dx = hip.log_probs_with_grad(hg, hx, ht, hge if entropy_too else None)
        # (a row may have other lanes here than without the gradient, so its sums another order: the bounds above, not bits)
        check_score((lp, h, peak, total), want, d, oracle, 0, f"{what} beside the gradient")
        check_gradient(dx, want, g, ge if entropy_too else None, d, oracle, what + " at once")
        for a, b in zip((lp, h, dx), hip.log_probs_with_grad(hg, hx, ht, hge if entropy_too else None)):
            same_bits(logical(a), logical(b), "equal calls at once")


@pytest.mark.parametrize("d", FLOATS, ids=lambda d: d.name)
@pytest.mark.parametrize("n", [1, 2, 3, 7, 8, 10, 16, 31, 63, 64, 65, 100, 255, 257, 512, 1000, 1024, 2048, 2049, 4097, 8192, 8193, 10007, 50257, 140001])
def test_lengths(hip, oracle, d, n):
    rows = 3 if n > 10000 else 9 if n > 64 else 70
    xs, x = drawn((rows, n), d, oracle, n)
    tokens = np.random.default_rng(n + 1).integers(0, n, rows)
    tokens[0] = n - 1
    tokens[1] = -1
    everything(hip, oracle, d, tensor(hip, xs, d), x, tokens, sorted({0, 1, min(n, 5), min(n, 20), min(n, 64)}), f"{n}")


def test_many_rows(hip, oracle):
    """More rows than a launch has groups of lanes for, in blocks of 32 rows: they go on to further ones."""
    d, n = dt.float16, 5
    for rows in (70001, (1 << 21) * 32 // 16 + 77):
        xs, x = drawn((rows, n), d, oracle, rows)
        tokens = np.random.default_rng(rows).integers(-1, n, rows)
        everything(hip, oracle, d, tensor(hip, xs, d), x, tokens, (0,), f"{rows} rows")


@pytest.mark.parametrize("d", [dt.float32, dt.bfloat16, dt.float64], ids=lambda d: d.name)
@pytest.mark.parametrize("n", [300, 3001, 20011])
def test_orders_and_ties(hip, oracle, d, n):
    """Rows made to be hard for what finds the most likely tokens."""
    rng = np.random.default_rng(n)
    v, g = 16 // d.itemsize, max(256, lanes(n, d))
    rows = [np.zeros(n), np.full(n, -7.5), np.arange(n) / n * 8, -np.arange(n) / n * 8,  # equal, rising, falling
            np.where(np.arange(n) % 97 == 5, 3.0, -np.inf),  # a vocabulary that is banned but for some
            np.where(np.arange(n) == n - 1, 1.0, -np.inf),  # ... but for one
            np.where(np.arange(n) // v % g == 3, 5.0, 0.0) + np.arange(n) % 5 / 8,  # what is large lies in one lane
            np.where(np.arange(n) // v % g < 40, 5.0, 0.0) + np.arange(n) % 3 / 8,  # ... in forty of them
            rng.integers(0, 3, n) * 1.0, rng.integers(-1, 2, n) * 0.0,  # three values; zeros of both signs
            np.where(np.arange(n) == n // 2, 300.0, rng.standard_normal(n)),  # certain
            rng.standard_normal(n) * 1e-3]
    x = np.stack(rows)
    x[9] *= -1.0
    xs = encode(x, d, oracle)
    everything(hip, oracle, d, tensor(hip, xs, d), decode(xs, d, oracle), rng.integers(0, n, len(rows)), (1, 3, 17, 64), f"hard rows of {n}")


@pytest.mark.parametrize("d", FLOATS, ids=lambda d: d.name)
@pytest.mark.parametrize("n", [64, 65, 98, 130, 257, 511, 700, 1000, 2900, 40000])
def test_many_alternatives_that_tie(hip, oracle, d, n):
    """Rows of few values, of both signs, so that many an entry ties with the last alternative; of them some with NaNs, which come last,
    infinities, and elements that are banned."""
    rng = np.random.default_rng(n)
    x = np.stack([rng.integers(-m, m + 1, n) / 8 for m in (1, 2, 5, 12, 30, 100, 400)] * 4)
    x[7:14] = np.where(rng.random((7, n)) < 0.5, -np.inf, x[7:14])
    x[14:21] = -np.abs(x[14:21]) - 1
    x[21:28, rng.integers(0, n, n // 2)] = np.nan
    x[24:28, rng.integers(0, n, 3)] = np.inf
    xs = encode(x, d, oracle)
    x = decode(xs, d, oracle)
    hx, ht = tensor(hip, xs, d), hip.full(dt.int32, (28,), 0)
    for k in (1, 7, 9, 33, 64):
        want = np.argsort(-x, -1, kind="stable")[:, :k]
        assert np.array_equal(logical(hip.log_probs(hx, ht, k)[5]), want), k


@pytest.mark.parametrize("d", FLOATS, ids=lambda d: d.name)
@pytest.mark.parametrize("n", [6, 40, 700, 9000])
def test_values_that_are_no_numbers(hip, oracle, d, n):
    rng = np.random.default_rng(n)
    x = rng.standard_normal((9, n)) * 2
    x[0, 2] = np.nan
    x[1, 4] = np.inf
    x[2] = -np.inf
    x[3, 1:] = -np.inf
    x[4, ::2] = -np.inf
    x[5] = np.nan
    x[6, :4] = [np.inf, -np.inf, np.nan, np.inf]
    x[7] = np.finfo(d.np_storage if d is not dt.bfloat16 else np.float32).min / 2  # the far end of what is finite
    xs = encode(x, d, oracle)
    x = decode(xs, d, oracle)
    tokens = np.array([0, 1, 0, 0, 0, 3, 2, n - 1, n])  # (-inf at none but the second's neighbour; the last is past the row)
    hx, ht = tensor(hip, xs, d), tensor(hip, tokens.astype(np.int32), dt.int32)
    k = min(n, 6)
    want, got = Want(x, tokens, d, k), hip.log_probs(hx, ht, k)
    clean = [3, 4, 7, 8]
    no = [0, 1, 2, 5, 6]
    for name, t in zip(("log_p", "entropy", "total"), (got[0], got[1], got[3])):
        assert np.all(np.isnan(logical(t)[no])), name
    assert np.all(np.isnan(logical(got[4])[no])) and np.isnan(logical(got[0])[8])
    assert np.array_equal(logical(got[5]), want.top)
    # One element that is possible: its term 2^r, r = peak log2 e - a, and 2^-r have errors of 4 u each (|r| < 2^-22 here), their
    # product is no less than 1 by the clamp and so at most 8 u + u above it; the entropy is held to its bound above, from zero on.
    assert 1 <= logical(got[3])[3] <= 1 + 10 * unit(d) and 0 <= logical(got[1])[3] <= want.entropy_err[3]
    g, ge = np.full(9, -1.0), np.full(9, 0.5)
    (hg, _), (hge, _) = values(hip, g, d), values(hip, ge, d)
    dx = [hip.log_probs_grad(hg, hx, ht, got[2], got[3], hge, got[1]), hip.log_probs_with_grad(hg, hx, ht, hge)[2]]
    w, err = want.gradient(g, ge)
    for t in dx:
        v = decode(logical(t), d, oracle)
        assert np.all(np.isnan(v[no])) and np.all(np.isnan(v[8]))
        within(v[[3, 4, 7]], w[[3, 4, 7]], err[[3, 4, 7]], HALF[d.name], TINY[d.name], "gradient of the others")
        assert np.all(v[4, 2::2] == 0)  # what has no probability has no gradient
    for i in clean:
        one = Want(x[i:i + 1], np.zeros(1, int), d)
        within(logical(got[1])[i:i + 1].astype(np.float64), one.entropy, one.entropy_err, 2.0 ** -24, 0, "entropy")


@pytest.mark.parametrize("d", [dt.float32, dt.bfloat16], ids=lambda d: d.name)
@pytest.mark.parametrize("n", [37, 1000, 9003])
def test_views(hip, oracle, d, n):
    """Rows of views, tokens and values of their own layouts; what lies around results stays."""
    shape = (3, 6, n + 19)
    xs, xv = drawn(shape, d, oracle, n)
    h = tensor(hip, xs, d)
    cases = [("window", lambda t: hip.shrink(t, [(0, 2), (1, 5), (3, n + 3)]), lambda a: a[:2, 1:5, 3:n + 3]),
             ("flipped", lambda t: hip.flip(hip.shrink(t, [(0, 2), (1, 5), (0, n)]), (True, True, False)), lambda a: a[:2, 1:5, :n][::-1, ::-1]),
             ("swapped", lambda t: hip.permute(hip.shrink(t, [(0, 3), (0, 5), (1, n + 1)]), (1, 0, 2)), lambda a: a[:, :5, 1:n + 1].transpose(1, 0, 2)),
             ("broadcast", lambda t: hip.expand(hip.shrink(t, [(1, 2), (0, 5), (0, n)]), (4, 5, n)), lambda a: np.broadcast_to(a[1:2, :5, :n], (4, 5, n)))]
    rng = np.random.default_rng(n)
    for name, view, same in cases:
        x, hx = same(xv), view(h)
        rows = x.shape[:2]
        everything(hip, oracle, d, hx, x, rng.integers(0, n, rows), (0, 4), name)
        tokens = rng.integers(0, n, rows[::-1] + (2,)).astype(np.int32)
        ht = hip.permute(hip.reshape(hip.shrink(tensor(hip, tokens, dt.int32), [(0, rows[1]), (0, rows[0]), (1, 2)]), rows[::-1]), (1, 0))
        want = Want(x, tokens[..., 1].T, d, 4)
        sparse = lambda sd: tensor(hip, np.full(rows[::-1] + (3,), 7, sd.np_storage), sd)  # noqa: E731
        outs = [sparse(stats(d)) for _ in range(4)]
        inner = [hip.permute(hip.reshape(hip.shrink(o, [(0, rows[1]), (0, rows[0]), (1, 2)]), rows[::-1]), (1, 0)) for o in outs]
        tp, tt = tensor(hip, np.full(rows + (9,), 7, stats(d).np_storage), stats(d)), tensor(hip, np.full(rows + (9,), 7, np.int32), dt.int32)
        four = lambda t: hip.shrink(t, [(0, rows[0]), (0, rows[1]), (3, 7)])  # noqa: E731
        got = hip.log_probs(hx, ht, 4, out=(*inner, four(tp), four(tt)))
        check_score(got, want, d, oracle, 4, name)
        for o in outs:
            assert np.all(logical(o)[..., [0, 2]] == 7)
        for o in (tp, tt):
            assert np.all(logical(o)[..., [0, 1, 2, 7, 8]] == 7)
        hg = hip.expand(tensor(hip, np.full((1, 1), -0.25, stats(d).np_storage), stats(d)), rows)  # one value for all rows
        block = np.full(shape, encode(np.array([7.0]), d, oracle)[0])
        whole = tensor(hip, block, d)
        if name != "broadcast":
            for call in (lambda o: hip.log_probs_grad(hg, hx, ht, inner[2], inner[3], out=o),
                         lambda o: hip.log_probs_with_grad(hg, hx, ht, out=(None, None, o))[2]):
                check_gradient(call(view(whole)), want, np.full(rows, -0.25), None, d, oracle, name)
                after = logical(whole).copy()
                same(after)[...] = block.reshape(-1)[0]
                same_bits(after, block, f"around the gradient of {name}")


@pytest.mark.parametrize("n", [50, 1500, 30001])
def test_gradients_that_replace_logits(hip, oracle, n):
    d = dt.float32
    xs, x = drawn((6, n), d, oracle, n)
    tokens = np.random.default_rng(n).integers(0, n, 6).astype(np.int32)
    ht, (hg, _), (hge, _) = tensor(hip, tokens, dt.int32), values(hip, np.ones(6), d), values(hip, np.full(6, 0.5), d)
    log_p, entropy, peak, total = hip.log_probs(tensor(hip, xs, d), ht)[:4]
    want = logical(hip.log_probs_grad(hg, tensor(hip, xs, d), ht, peak, total, hge, entropy))
    a = tensor(hip, xs, d)
    same_bits(logical(hip.log_probs_grad(hg, a, ht, peak, total, hge, entropy, out=a)), want, "in place")
    want = [logical(t) for t in hip.log_probs_with_grad(hg, tensor(hip, xs, d), ht, hge)]
    a = tensor(hip, xs, d)
    for p, q in zip(hip.log_probs_with_grad(hg, a, ht, hge, out=(log_p, entropy, a)), want):
        same_bits(logical(p), q, "at once and in place")


@pytest.mark.parametrize("rows, n", [(70, 5), (7, 700), (5, 5001), (3, 30000), (66, 33000), (3, 40000)])
def test_results_that_replace_their_gradients(hip, oracle, rows, n):
    """log_p and entropy written where g and g_entropy are, every length's kernel."""
    d = dt.float32
    xs, _ = drawn((rows, n), d, oracle, n)
    rng = np.random.default_rng(n)
    hx, ht = tensor(hip, xs, d), tensor(hip, rng.integers(-1, n, rows).astype(np.int32), dt.int32)
    g, ge = rng.standard_normal(rows), rng.standard_normal(rows)
    want = [logical(t) for t in hip.log_probs_with_grad(values(hip, g, d)[0], hx, ht, values(hip, ge, d)[0])]
    for first in (0, 1):
        both = values(hip, g, d)[0], values(hip, ge, d)[0]
        out = (both[first], both[1 - first], hip.buffer(d, (rows, n)))
        for p, q in zip(hip.log_probs_with_grad(both[0], hx, ht, both[1], out=out), want):
            same_bits(logical(p), q, f"over {first}")


def test_differences(hip, oracle):
    """The gradient against differences of the forward pass in float64 (steps of 1e-6)."""
    rng = np.random.default_rng(3)
    d, rows, n = dt.float64, 3, 13
    x, tokens = rng.standard_normal((rows, n)), np.array([4, -1, 12], np.int32)
    g, ge = rng.standard_normal(rows), rng.standard_normal(rows)
    ht, hg, hge = tensor(hip, tokens, dt.int32), tensor(hip, g, d), tensor(hip, ge, d)

    def loss(x):
        log_p, entropy = hip.log_probs(tensor(hip, x, d), ht)[:2]
        return float((logical(log_p) * g + logical(entropy) * ge).sum())

    grad = logical(hip.log_probs_with_grad(hg, tensor(hip, x, d), ht, hge)[2])
    for at in np.ndindex(x.shape):
        step = np.zeros_like(x)
        step[at] = 1e-6
        assert abs((loss(x + step) - loss(x - step)) / 2e-6 - grad[at]) < 1e-7


def test_results_that_are_not_wanted(hip, oracle):
    d = dt.bfloat16
    xs, x = drawn((20, 900), d, oracle, 1)
    ht = tensor(hip, np.arange(20, dtype=np.int32), dt.int32)
    want = hip.log_probs(tensor(hip, xs, d), ht)[:4] + hip.log_probs(tensor(hip, xs, d), ht, 7)[4:]  # (the sums' order may go by `top`)
    for k in range(4):
        out = [None] * 6
        out[k] = hip.buffer(dt.float32, (20,))
        hip.log_probs(tensor(hip, xs, d), ht, 0, out=out)
        same_bits(logical(out[k]), logical(want[k]), f"result {k} alone")
    out = [None] * 4 + [hip.buffer(dt.float32, (20, 7)), hip.buffer(dt.int32, (20, 7))]
    hip.log_probs(tensor(hip, xs, d), ht, 7, out=out)
    for k in (4, 5):
        same_bits(logical(out[k]), logical(want[k]), f"result {k} alone")


def test_offsets_past_32_bits(hip, oracle):
    """Rows that begin further into a tensor than 2^32 bytes, and 2^32 elements."""
    d, n = dt.bfloat16, 50257
    rows = (1 << 32) // n + 40
    x = hip.full(d, (rows, n), 0.0)
    s, v = drawn((33, n), d, oracle, 8)
    last = hip.shrink(x, [(rows - 33, rows), (0, n)])
    hip.assign(last, tensor(hip, s, d))
    tokens = np.zeros(rows, np.int32)
    tokens[-33:] = np.random.default_rng(1).integers(0, n, 33)
    ht = tensor(hip, tokens, dt.int32)
    hg = hip.expand(hip.full(dt.float32, (1,), -1.0), (rows,))
    got = hip.log_probs(x, ht, 2)
    want = Want(v, tokens[-33:], d, 2)
    tail = [hip.copy(hip.shrink(t, [(rows - 33, rows)] + [(0, m) for m in t.shape[1:]])) for t in got]
    check_score(tail, want, d, oracle, 2)
    assert np.all(logical(got[5])[:-33] == [0, 1]) and np.all(np.abs(logical(got[1])[:-33] - np.log(n)) < 1e-5)
    grad = hip.log_probs_with_grad(hg, x, ht, out=(None, None, x))[2]
    check_gradient(hip.copy(hip.shrink(grad, [(rows - 33, rows), (0, n)])), want, np.full(33, -1.0), None, d, oracle)
    del x, last, grad
    hip.trim()


def test_replays(hip, oracle):
    """A recorded loss, replayed on new logits and tokens between other work of its context."""
    d, rows, n = dt.bfloat16, 12, 5003
    hx, ht = tensor(hip, drawn((rows, n), d, oracle, 0)[0], d), tensor(hip, np.zeros(rows, np.int32), dt.int32)
    hg = hip.expand(hip.full(dt.float32, (1,), -1 / rows), (rows,))

    def step():
        scored = hip.log_probs(hx, ht, 9)
        return (*scored, hip.log_probs_grad(hg, hx, ht, scored[2], scored[3]), *hip.log_probs_with_grad(hg, hx, ht, hg))

    step()
    hip.capture_begin()
    try:
        out = step()
    finally:
        graph = hip.capture_end()
    try:
        for k in range(4):
            hip.assign(hx, tensor(hip, drawn((rows, n), d, oracle, 20 + k)[0], d))
            hip.assign(ht, tensor(hip, np.random.default_rng(k).integers(0, n, rows).astype(np.int32), dt.int32))
            graph.launch()
            for a, b in zip(out, step()):
                same_bits(logical(a), logical(b), f"replay {k}")
    finally:
        graph.destroy()


def test_behind_deferred_work(hip, oracle):
    d = dt.float32
    a = tensor(hip, drawn((5, 300), d, oracle, 3)[0], d)
    ht = tensor(hip, np.arange(5, dtype=np.int32), dt.int32)
    x = hip.binary("mul", a, a)
    want = [logical(t) for t in hip.log_probs(x, ht, 3)]
    hg = hip.full(d, (5,), 1.0)
    want.append(logical(hip.log_probs_with_grad(hg, x, ht)[2]))
    hip.set_deferred(True)
    try:
        got = hip.log_probs(hip.binary("mul", a, a), ht, 3)
        y = hip.binary("add", got[0], got[0])
        dx = hip.log_probs_with_grad(hip.full(d, (5,), 1.0), hip.binary("mul", a, a), ht)[2]
        got = [logical(t) for t in (*got, dx)]
        same_bits(logical(y), 2 * got[0], "work recorded behind")
    finally:
        hip.set_deferred(False)
    for p, q in zip(got, want):
        same_bits(p, q, "behind deferred work")


def test_no_rows(hip):
    x, t = hip.buffer(dt.float32, (0, 9)), hip.buffer(dt.int32, (0,))
    got = hip.log_probs(x, t, 3)
    assert got[0].shape == (0,) and got[4].shape == (0, 3)
    s = hip.buffer(dt.float32, (0,))
    assert hip.log_probs_grad(s, x, t, s, s).shape == (0, 9) and hip.log_probs_with_grad(s, x, t)[2].shape == (0, 9)


def test_refusals(hip):
    B, f32, i32 = hip, dt.float32, dt.int32
    x, t, s = B.full(f32, (4, 8), 1.0), B.full(i32, (4,), 1), B.full(f32, (4,), 1.0)
    with pytest.raises(ValueError, match="log_probs: shape mismatch"):
        B.log_probs(x, B.full(i32, (5,), 1))
    with pytest.raises(ValueError, match="log_probs: shape mismatch"):
        B.log_probs(x, B.full(i32, (4, 1), 1))
    with pytest.raises(RuntimeError, match="dtype not supported"):
        B.log_probs(x, B.full(dt.int64, (4,), 1))
    with pytest.raises(RuntimeError, match="dtype not supported"):
        B.log_probs(B.full(i32, (4, 8), 1), t)
    with pytest.raises(ValueError, match="more alternatives than a row has"):
        B.log_probs(x, t, 9)
    with pytest.raises(RuntimeError, match="64 alternatives"):
        B.log_probs(B.full(f32, (4, 80), 1.0), t, 65)
    with pytest.raises(ValueError, match="another number of alternatives"):
        B.log_probs(x, t, 3, out=(s, s, s, s, None, None))
    with pytest.raises(RuntimeError, match="rows must be contiguous"):
        B.log_probs(B.permute(x, (1, 0)), B.full(i32, (8,), 1))
    with pytest.raises(ValueError, match="scalar"):
        B.log_probs(B.full(f32, (), 1.0), t)
    with pytest.raises(ValueError, match="empty axis"):
        B.log_probs(B.buffer(f32, (4, 0)), t)
    with pytest.raises(ValueError, match="broadcast"):
        B.log_probs(x, t, out=(B.expand(B.buffer(f32, (1,)), (4,)), None, None, None, None, None))
    with pytest.raises(RuntimeError, match="dtype not supported"):
        B.log_probs(x, t, out=(B.buffer(dt.float64, (4,)), None, None, None, None, None))
    with pytest.raises(RuntimeError, match="dtype not supported"):
        B.log_probs(x, t, 2, out=(None, None, None, None, B.buffer(f32, (4, 2)), B.buffer(f32, (4, 2))))
    with pytest.raises(ValueError, match="shape mismatch"):
        B.log_probs(x, t, 2, out=(None, None, None, None, B.buffer(f32, (4, 3)), B.buffer(i32, (4, 2))))
    with pytest.raises(ValueError, match="null argument"):
        B.log_probs(x, t, 2, out=(None, None, None, None, None, B.buffer(i32, (4, 2))))
    with pytest.raises(ValueError, match="null argument"):
        B.log_probs_grad(s, x, t, s, s, s)
    with pytest.raises(ValueError, match="log_probs_grad: shape mismatch"):
        B.log_probs_grad(B.full(f32, (3,), 1.0), x, t, s, s)
    with pytest.raises(RuntimeError, match="dtype not supported"):
        B.log_probs_grad(B.full(dt.float64, (4,), 1.0), x, t, s, s)
    with pytest.raises(RuntimeError, match="dtype not supported"):
        B.log_probs_grad(s, x, t, s, s, out=B.buffer(dt.bfloat16, (4, 8)))
    with pytest.raises(ValueError, match="broadcast"):
        B.log_probs_grad(s, x, t, s, s, out=B.expand(B.buffer(f32, (1, 8)), (4, 8)))
    with pytest.raises(ValueError, match="log_probs_with_grad: shape mismatch"):
        B.log_probs_with_grad(s, x, t, B.full(f32, (4, 1), 1.0))
    with pytest.raises(ValueError, match="shape mismatch"):
        B.log_probs_with_grad(s, x, t, out=(None, None, B.buffer(f32, (4, 7))))
    many = B.expand(B.reshape(x, (1, 1, 4, 8)), (1 << 20, 1 << 20, 4, 8))
    with pytest.raises(RuntimeError, match="too many rows"):
        B.log_probs(many, B.expand(B.reshape(t, (1, 1, 4)), (1 << 20, 1 << 20, 4)), out=(None,) * 6)


@pytest.mark.parametrize("d, n", [(dt.float32, 40000), (dt.bfloat16, 70001), (dt.float64, 17001), (dt.float16, 200000), (dt.float32, 80000), (dt.float64, 75001)], ids=lambda v: v.name if hasattr(v, "name") else str(v))
def test_few_long_rows(hip, oracle, d, n):
    """Rows that are cut into parts, with the rows that are hard for what finds the most likely tokens: large elements in one part, in
    one lane, ties within and across parts, parts of -inf, NaNs and infinities."""
    rng = np.random.default_rng(n)
    x = rng.standard_normal((10, n)) * 2
    x[1] = 0.0
    x[2] = np.arange(n) / n
    x[3, : n // 2] = -np.inf
    x[4] = -np.inf
    x[4, n - 1] = x[4, n // 3] = 2.0
    x[5] = np.where(np.arange(n) % 1000 == 7, 4.0, 0.0)
    x[6] = np.where(np.arange(n) // (16 // d.itemsize) % 256 == 5, 3.0, 0.0)
    x[7, n // 2] = np.nan
    x[8, 5] = np.inf
    x[9] = np.finfo(d.np_storage if d is not dt.bfloat16 else np.float32).min / 2
    xs = encode(x, d, oracle)
    x = decode(xs, d, oracle)
    tokens = rng.integers(0, n, 10)
    tokens[0], tokens[4], tokens[2] = n - 1, n - 1, -1
    hx, ht = tensor(hip, xs, d), tensor(hip, tokens.astype(np.int32), dt.int32)
    ok = [0, 1, 2, 3, 4, 5, 6, 9]
    g, ge = rng.standard_normal(10), rng.standard_normal(10)
    (hg, g), (hge, ge) = values(hip, g, d), values(hip, ge, d)
    for k in (0, 1, 20, 64):
        want, got = Want(x, tokens, d, k), hip.log_probs(hx, ht, k)
        some = Want(x[ok], tokens[ok], d, k)
        for t, w, err in zip(got, (some.log_p, some.entropy, some.peak, some.total), (some.log_p_err, some.entropy_err, 0 * some.e, some.e * some.total)):
            within(logical(t)[ok].astype(np.float64), w, err, HALF[stats(d).name], 0, f"top {k} of {d.name}")
        assert np.all(np.isnan(logical(got[0])[[7, 8]])) and np.all(np.isnan(logical(got[3])[[7, 8]]))
        if k:
            assert np.array_equal(logical(got[5]), want.top), f"top {k}"
            within(logical(got[4])[ok].astype(np.float64), some.top_log_p, some.top_err, HALF[stats(d).name], 0, f"their log probabilities, {k}")
    for e in (None, hge):
        w, err = want.gradient(g, None if e is None else ge)
        lp, h, dx = hip.log_probs_with_grad(hg, hx, ht, e)
        over = tensor(hip, xs, d)
        again = hip.log_probs_with_grad(hg, over, ht, e, out=(lp, h, over))[2]
        same_bits(logical(again), logical(dx), "in place")
        alone = hip.log_probs_grad(hg, hx, ht, got[2], got[3], e, None if e is None else got[1])
        for t in (dx, alone):
            v = decode(logical(t), d, oracle)
            within(v[ok], w[ok], err[ok], HALF[d.name], TINY[d.name], "gradient")
            assert np.all(np.isnan(v[[7, 8]]))
    view = hip.flip(hip.expand(hip.reshape(hip.shrink(hx, [(0, 1), (3, n)]), (1, 1, n - 3)), (2, 3, n - 3)), (True, False, False))
    got = hip.log_probs(view, hip.full(dt.int32, (2, 3), 4), 5)
    check_score(got, Want(np.broadcast_to(x[:1, 3:], (2, 3, n - 3)), np.full((2, 3), 4), d, 5), d, oracle, 5, "a view")
    hip.capture_begin()
    try:
        out = (*hip.log_probs(hx, ht, 20), *hip.log_probs_with_grad(hg, hx, ht, hge))
    finally:
        graph = hip.capture_end()
    try:
        for _ in range(3):
            graph.launch()
            for a, b in zip(out, (*hip.log_probs(hx, ht, 20), *hip.log_probs_with_grad(hg, hx, ht, hge))):
                same_bits(logical(a), logical(b), "replay")
    finally:
        graph.destroy()
