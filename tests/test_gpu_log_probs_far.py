"""Log probabilities of rows that lie far from zero. Up to a largest element of 2^20 in magnitude a row's exponentials are taken against a
rounded reference, past it by differences with the largest element: rows with a spread on both sides of both borders.

The bounds are those of test_gpu_log_probs, with three things counted anew. D is the range of the terms there are: one of e^-110 and less
(e^-750 in float64) is zero or makes no difference to a total of 1 and more. The sums' order is that of the fewest lanes that any of the
three calls gives a row: eight up to nine vectors, a wave up to 257, a block of 256 up to eight vectors a lane and the single elements, 512
beyond. And beside the border the reference's rounding r = peak L - A is not nothing: in float32 |r| <= 2^-4 (half a step of a product
below 2^21), which is part of every exponent and taken out of their mean again at the end, so that the entropy has 2 ln2 |r| E <= 0.09 E
more: 0.1 E is added. By differences nothing is lost: x - peak is rounded once, and its product with log2 e, as the bounds have it."""

import numpy as np
import pytest

import test_gpu_log_probs as plain
from helpers import decode, encode
from raven_amd import dtype as dt

pytestmark = pytest.mark.gpu


def fewest_lanes(n, d):
    v = 16 // d.itemsize
    return 8 if n < 9 * v else 64 if n < 257 * v else 256 if n < 2049 * v else 512


class Want(plain.Want):
    def __init__(self, x, tokens, d, top=0):
        super().__init__(x, tokens, d, top)
        u, v, n = self.u, 16 // d.itemsize, x.shape[-1]
        with np.errstate(invalid="ignore"):
            term = self.d > (-750 if d is dt.float64 else -110)
        span, steps = np.where(term, -self.d, 0).max(-1), -(-n // (fewest_lanes(n, d) * v)) + 1
        self.e = (2 * span + 4 * (steps + 2) + steps * v + 24) * u
        log_total = np.abs(self.log_total)
        picked = self.log_p + self.log_total
        self.log_p_err = np.where(tokens < 0, 0, self.e + 4 * u * (self.size(picked) + log_total))
        self.entropy_err = (1.1 + 2 * self.m) * self.e + 4 * u * (log_total + self.m)
        if top:
            self.top_err = self.e[..., None] + 4 * u * (self.size(self.top_log_p) + 2 * log_total[..., None])

    def gradient(self, g, g_entropy=None):
        """An exponential below 2^-126 is zero where sums are float32. The true one, less than that, is a factor of g and of g_entropy's
        (log p + entropy), which is some -87 there: the gradient may be off by so many times 2^-126 (the bounds have one)."""
        want, err = super().gradient(g, g_entropy)
        if g_entropy is not None:
            inner = self.size(self.d) + np.abs(self.log_total - self.entropy)[..., None]
            with np.errstate(invalid="ignore"):
                lost = np.where(self.p < 2.0 ** -125, 2.0 ** -126, 0) * np.where(self.p > 0, inner, 0)
            err = err + lost * np.abs(g_entropy)[..., None]
        return want, err + np.where(self.p < 2.0 ** -125, 2.0 ** -126, 0) * np.where(np.isfinite(g), np.abs(g), 0)[..., None]


@pytest.fixture
def bounds(monkeypatch):
    monkeypatch.setattr(plain, "Want", Want)


def rows_of(d, n, rng):
    """Rows whose largest element is at or beside the borders, and further out, of either sign."""
    edge = 2.0 ** 20
    rows = []
    if d is dt.bfloat16:  # its steps are 2^12 below the border and 2^13 above it: what is possible ties
        near = edge - rng.integers(0, 4, n) * 2.0 ** 12
        far = [edge + rng.integers(0, 4, n) * 2.0 ** 13, 2 * edge + rng.integers(0, 3, n) * 2.0 ** 14, -2 * edge - rng.integers(0, 3, n) * 2.0 ** 14]
        below = -edge - rng.integers(0, 2, n) * 2.0 ** 13
        near[n // 2], below[n // 2], far[0][n // 2] = edge, -edge, edge + 2.0 ** 13 * 3
        rows += [near, below, *far, np.where(rng.random(n) < 0.5, far[1], -np.inf)]
    else:
        fine = lambda step, most: rng.integers(0, int(most / step), n) * step  # noqa: E731
        for top, step in ((edge, 2.0 ** -3), (edge + 2.0 ** -3, 2.0 ** -3), (-edge, 2.0 ** -3), (-edge - 2.0 ** -3, 2.0 ** -3),
                          (edge - 2.0 ** -4, 2.0 ** -4), (2 * edge + 8, 0.25), (-2 * edge, 0.25), (4 * edge, 0.5), (-8 * edge, 1.0)):
            below = fine(step, 8)
            below[rng.integers(0, n)] = 0
            rows.append(top - below)
            rows.append(np.where((rng.random(n) < 0.5) & (below > 0), -np.inf, top - below))  # half of it banned
        rows.append(np.where(np.arange(n) == n // 3, 3 * edge, 3 * edge - 40 - fine(0.5, 60)))  # all but certain
        rows.append(np.where(np.arange(n) == n - 1, 2 * edge, rng.standard_normal(n)))  # one far element
        rows.append(np.where(np.arange(n) == 0, 1.0, -2 * edge - fine(0.25, 8)))  # all but one far below
        if d is dt.float64:
            rows.append(3 * edge + rng.standard_normal(n) * 2.5)
            rows.append(-3 * edge + rng.standard_normal(n) * 2.5)
    big = float(np.finfo(np.float32 if d is dt.bfloat16 else d.np_storage).max) / 4
    rows += [np.full(n, -big), np.where(np.arange(n) % 3 == 1, big, -big), np.where(np.arange(n) % 5 == 2, -big, -2 * big)]
    rows += [np.where(np.arange(n) == 0, 0.5, -np.inf), np.where(np.arange(n) % 2 == 0, -np.inf, rng.standard_normal(n) * 2)]
    return np.stack(rows)


@pytest.mark.parametrize("d", [dt.float32, dt.bfloat16, dt.float64], ids=lambda d: d.name)
@pytest.mark.parametrize("n", [6, 37, 300, 700, 1001, 5001, 9003, 20011, 80003])
def test_rows_far_from_zero(hip, oracle, bounds, d, n):
    rng = np.random.default_rng(n)
    xs = encode(rows_of(d, n, rng), d, oracle)
    x = decode(xs, d, oracle)
    assert np.all(np.isfinite(x.max(1))) and np.sum(np.abs(x.max(1)) > 2.0 ** 20) >= 6 and np.sum(np.abs(x.max(1)) == 2.0 ** 20) >= 2
    tokens = rng.integers(0, n, len(x))
    tokens[::2] = np.argmax(x[::2], 1)
    plain.everything(hip, oracle, d, plain.tensor(hip, xs, d), x, tokens, sorted({0, 1, min(n, 9), min(n, 64)}), f"far rows of {n}")


@pytest.mark.parametrize("n", [300, 20011])
def test_float16_reaches_its_ends(hip, oracle, bounds, n):
    """Its largest numbers are near: the reference holds them all."""
    rng = np.random.default_rng(n)
    d, most = dt.float16, 65504.0
    rows = np.stack([most - 32 * rng.integers(0, 3, n), -most + 32 * rng.integers(0, 3, n), np.where(rng.random(n) < 0.3, most, -most), np.full(n, -most)])
    xs = encode(rows, d, oracle)
    plain.everything(hip, oracle, d, plain.tensor(hip, xs, d), decode(xs, d, oracle), rng.integers(0, n, 4), (0, 1, 64), f"ends, {n}")
