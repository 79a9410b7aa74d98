"""The training layer norm (layer_norm, layer_norm_grad) against its formulas in float64.

Tolerances, derived before the first run. u is half a step of what sums are held in (2^-24, for float64 tensors 2^-53), half
the half step of the result's dtype. A row's sum has at most K = 64 roundings on any path (32 elements of a lane, or 40 of a
long row's, six steps between lanes, 15 between waves, a division).
  mean    K u mean|x|
  rstd    relative K u A + (K/2 + 5) u with A = mean|x| rstd: half of the variance's, which the mean's error (2 K u A) and its own
          sum (K u and two roundings of each term) make
  y       |gamma| (|h| (K u A + (K/2 + 5) u) + K u A) + 2 u |y|, then half |y|
  dx      rstd u (4 |w| + (K + 4) mean|w| + (K + 10) |h| mean|w h|), then half |dx|
  dgamma  128 u sum|g h|, dbeta 128 u sum|g|: a group's rows (some ten here), six steps, waves, 16 partial sums, 32 lanes; then half"""

import numpy as np
import pytest

from helpers import decode, encode, logical, same_bits
from raven_amd import dtype as dt

pytestmark = pytest.mark.gpu

FLOATS = [dt.float32, dt.bfloat16, dt.float16, dt.float64]
HALF = {"float64": 2.0 ** -53, "float32": 2.0 ** -24, "float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}
TINY = {"float64": 0.0, "float32": 2.0 ** -149, "float16": 2.0 ** -25, "bfloat16": 2.0 ** -133}  # below the normal range
EPS = 1e-5
K = 64


def tensor(hip, storage, d):
    return hip.reshape(hip.from_host(np.ascontiguousarray(storage), d), storage.shape)


def stats(d):
    return dt.float64 if d is dt.float64 else dt.float32


def unit(d):
    return 2.0 ** -53 if d is dt.float64 else 2.0 ** -24


def drawn(shape, d, oracle, seed, scale=1.0, shift=0.0):
    x = np.random.default_rng(seed).standard_normal(shape) * scale + shift
    s = encode(x, d, oracle)
    return s, decode(s, d, oracle)


def within(got, want, err, d, what):
    assert got.shape == want.shape, (what, got.shape, want.shape)
    lim = err + HALF[d.name] * (np.abs(want) + err) + TINY[d.name]
    off = np.abs(got - want)
    assert np.all(off <= lim), f"{what}: {np.nanmax(off / lim)} times the bound at {np.unravel_index(np.nanargmax(off / lim), off.shape)}"


def forward(x, gamma, beta, d, eps=EPS):
    """(y, mean, rstd) and how far each may be off."""
    u, n = unit(d), x.shape[-1]
    mean = x.mean(-1, keepdims=True)
    rstd = 1 / np.sqrt(((x - mean) ** 2).mean(-1, keepdims=True) + eps)
    h = (x - mean) * rstd
    g = np.ones(n) if gamma is None else gamma
    y = h * g + (0 if beta is None else beta)
    size = np.abs(x).mean(-1, keepdims=True)
    a = size * rstd
    r_err = K * u * a + (K / 2 + 5) * u
    return (y, mean[..., 0], rstd[..., 0]), (np.abs(g) * (np.abs(h) * r_err + K * u * a) + 2 * u * np.abs(y), (K * u * size)[..., 0],
                                              (rstd * r_err)[..., 0])


def backward(g, x, mean, rstd, gamma, d):
    u = unit(d)
    mean, rstd = mean[..., None], rstd[..., None]
    h = (x - mean) * rstd
    w = g if gamma is None else g * gamma
    m = lambda v: v.mean(-1, keepdims=True)  # noqa: E731
    dx = rstd * (w - m(w) - h * m(w * h))
    dx_err = rstd * u * (4 * np.abs(w) + (K + 4) * m(np.abs(w)) + (K + 10) * np.abs(h) * m(np.abs(w * h)))
    rows = tuple(range(x.ndim - 1))
    return (dx, (g * h).sum(rows), g.sum(rows)), (dx_err, 128 * u * np.abs(g * h).sum(rows), 128 * u * np.abs(g).sum(rows))


def check_forward(hip, oracle, d, x, gamma=None, beta=None, out=None, eps=EPS):
    """x, gamma, beta: (handle, values)."""
    got = hip.layer_norm(x[0], gamma and gamma[0], beta and beta[0], eps, out=out)
    want, err = forward(x[1], gamma and gamma[1], beta and beta[1], d, eps)
    for t, w, e, td, name in zip(got, want, err, (d, stats(d), stats(d)), ("y", "mean", "rstd")):
        within(decode(logical(t), td, oracle), w, e, td, f"{name} of {d.name} {x[1].shape}")
    return got


def check_backward(hip, oracle, d, g, x, mean, rstd, gamma=None, out=None):
    got = hip.layer_norm_grad(g[0], x[0], mean[0], rstd[0], gamma and gamma[0], out=out)
    want, err = backward(g[1], x[1], mean[1], rstd[1], gamma and gamma[1], d)
    for t, w, e, name in zip(got, want, err, ("dx", "dgamma", "dbeta")):
        within(decode(logical(t), d, oracle), w, e, d, f"{name} of {d.name} {x[1].shape}")
    return got


def of_rows(values, d):
    """Statistics as the operator holds them, and their values."""
    s = values.astype(stats(d).np_storage)
    return s, s.astype(np.float64)


# every way of holding a row: 1 to 64 lanes, three vectors to half a wave, whole blocks, rows that are walked; whole and ragged
LENGTHS = {2: [1, 2, 7, 8, 9, 16, 29, 64, 65, 128, 129, 250, 512, 513, 768, 770, 1024, 1535, 2000, 2048, 2049, 4096, 6001, 8192,
               8193, 16384, 20000, 32768, 32769, 40008],
           4: [1, 3, 4, 5, 8, 31, 64, 127, 256, 384, 385, 512, 700, 1001, 1024, 2047, 3000, 4096, 4097, 8192, 16384, 16387],
           8: [1, 2, 3, 16, 33, 64, 128, 192, 255, 384, 512, 1001, 1500, 2048, 2049, 8192, 8195]}


@pytest.mark.parametrize("d, n", [(d, n) for d in FLOATS for n in LENGTHS[d.itemsize]], ids=lambda v: v.name if hasattr(v, "name") else str(v))
def test_lengths(hip, oracle, d, n):
    rows = 5 if n > 4096 else 37 if n > 64 else 1030
    x, g = (drawn((rows, n), d, oracle, n + k, 1.5, 0.4) for k in (0, 1))
    gamma, beta = drawn((n,), d, oracle, n + 2, 0.3, 1.0), drawn((n,), d, oracle, n + 3, 0.2)
    hx, hg, hgamma, hbeta = (tensor(hip, v[0], d) for v in (x, g, gamma, beta))
    longest = 4096 * 16 // d.itemsize
    y, mean, rstd = check_forward(hip, oracle, d, (hx, x[1]), (hgamma, gamma[1]), (hbeta, beta[1]))
    assert hip.last_path() == ("layer_norm_long" if n > longest else "layer_norm")
    m, r = ((t, decode(logical(t), stats(d), oracle)) for t in (mean, rstd))
    got = check_backward(hip, oracle, d, (hg, g[1]), (hx, x[1]), m, r, (hgamma, gamma[1]))
    assert hip.last_path() == ("layer_norm_grad_long" if n > (longest // 2 if d.itemsize == 2 else longest) else "layer_norm_grad")
    for a, b in zip(got, hip.layer_norm_grad(hg, hx, mean, rstd, hgamma)):
        same_bits(logical(a), logical(b), "equal calls")
    check_forward(hip, oracle, d, (hx, x[1]))
    check_forward(hip, oracle, d, (hx, x[1]), beta=(hbeta, beta[1]))
    check_forward(hip, oracle, d, (hx, x[1]), (hgamma, gamma[1]))
    check_backward(hip, oracle, d, (hg, g[1]), (hx, x[1]), m, r)


@pytest.mark.parametrize("d", FLOATS, ids=lambda d: d.name)
@pytest.mark.parametrize("rows, n", [(1, 768), (2, 8), (700, 768), (5000, 96), (9001, 33), (40000, 8)], ids=lambda v: str(v))
def test_numbers_of_rows(hip, oracle, d, rows, n):
    """One row, fewer than a block's groups, several to a group (those of the last turn fewer)."""
    x, g = (drawn((rows, n), d, oracle, rows + k, 2.0, -1.0) for k in (0, 1))
    gamma = drawn((n,), d, oracle, n, 0.3, 1.0)
    hx, hg, hgamma = (tensor(hip, v[0], d) for v in (x, g, gamma))
    _, mean, rstd = check_forward(hip, oracle, d, (hx, x[1]), (hgamma, gamma[1]))
    m, r = ((t, decode(logical(t), stats(d), oracle)) for t in (mean, rstd))
    check_backward(hip, oracle, d, (hg, g[1]), (hx, x[1]), m, r, (hgamma, gamma[1]))


@pytest.mark.parametrize("d, n", [(dt.float32, 9001), (dt.float32, 12300), (dt.float32, 16384), (dt.float64, 5003), (dt.float64, 8191), (dt.bfloat16, 5001),
                                  (dt.bfloat16, 16381), (dt.float16, 20001)], ids=lambda v: v.name if hasattr(v, "name") else str(v))
def test_many_wide_rows(hip, oracle, d, n):
    """Several rows to a block, some blocks one fewer."""
    x, g = (drawn((523, n), d, oracle, n + k, 1.5, 0.4) for k in (0, 1))
    gamma = drawn((n,), d, oracle, n, 0.3, 1.0)
    hx, hg, hgamma = (tensor(hip, v[0], d) for v in (x, g, gamma))
    _, mean, rstd = check_forward(hip, oracle, d, (hx, x[1]), (hgamma, gamma[1]))
    m, r = ((t, decode(logical(t), stats(d), oracle)) for t in (mean, rstd))
    got = check_backward(hip, oracle, d, (hg, g[1]), (hx, x[1]), m, r, (hgamma, gamma[1]))
    over = hip.layer_norm_grad(hg, hx, mean, rstd, hgamma, out=(hx, got[1], got[2]))
    same_bits(logical(over[0]), logical(got[0]), "in place")


def views(B, n):
    """Views with rows of n elements of a [4, 7, 2 n + 3] tensor: name, the view of a handle, the same of an array."""
    return [("pitched", lambda t: B.shrink(t, [(0, 3), (0, 5), (0, n)]), lambda a: a[:3, :5, :n]),
            ("odd start", lambda t: B.shrink(t, [(1, 4), (2, 7), (1, n + 1)]), lambda a: a[1:4, 2:7, 1:n + 1]),
            ("flipped rows", lambda t: B.flip(B.shrink(t, [(0, 3), (0, 5), (3, n + 3)]), (True, True, False)),
             lambda a: a[:3, :5, 3:n + 3][::-1, ::-1]),
            ("swapped", lambda t: B.permute(B.shrink(t, [(0, 4), (0, 3), (2, n + 2)]), (1, 0, 2)),
             lambda a: a[:4, :3, 2:n + 2].transpose(1, 0, 2)),
            ("broadcast", lambda t: B.expand(B.shrink(t, [(0, 1), (0, 5), (0, n)]), (3, 5, n)),
             lambda a: np.broadcast_to(a[:1, :5, :n], (3, 5, n)))]


@pytest.mark.parametrize("d", [dt.float32, dt.bfloat16], ids=lambda d: d.name)
@pytest.mark.parametrize("n", [24, 101, 768, 33001])
def test_views(hip, oracle, d, n):
    """Rows of views, whose results go to views of their own: what lies around them stays."""
    shape = (4, 7, 2 * n + 3)
    xs, xv = drawn(shape, d, oracle, n)
    gs, gv = drawn(shape, d, oracle, n + 1)
    ws, wv = drawn((n + 1,), d, oracle, n + 2, 0.3, 1.0)
    gamma = (hip.shrink(hip.from_host(ws, d), [(1, n + 1)]), wv[1:])
    for name, view, same in views(hip, n):
        x, g = (view(tensor(hip, xs, d)), same(xv)), (view(tensor(hip, gs, d)), same(gv))
        got = check_forward(hip, oracle, d, x, gamma, gamma)
        m, r = ((t, decode(logical(t), stats(d), oracle)) for t in got[1:])
        check_backward(hip, oracle, d, g, x, m, r, gamma)
        if name == "broadcast":
            continue
        # results in views: the layout of x in a block of sevens, every second value of larger statistics
        block = np.full(shape, encode(np.array([7.0]), d, oracle)[0])
        oy, odx = tensor(hip, block, d), tensor(hip, block, d)
        lead = x[1].shape[:2]
        sparse = np.full((lead[0], lead[1], 2), 7, stats(d).np_storage)
        om, orr = tensor(hip, sparse, stats(d)), tensor(hip, sparse, stats(d))
        odg = hip.from_host(np.repeat(block.reshape(-1)[:1], 2 * n), d)
        half = lambda t: hip.reshape(hip.shrink(t, [(0, lead[0]), (0, lead[1]), (1, 2)]), lead)  # noqa: E731
        column = hip.reshape(hip.shrink(hip.reshape(odg, (n, 2)), [(0, n), (0, 1)]), (n,))
        check_forward(hip, oracle, d, x, gamma, gamma, out=(view(oy), half(om), half(orr)))
        same_bits(logical(half(om)), logical(got[1]), "statistics in a view")
        check_backward(hip, oracle, d, g, x, (half(om), m[1]), (half(orr), r[1]), gamma, out=(view(odx), column, hip.buffer(d, (n,))))
        for t, what in ((oy, "y"), (odx, "dx")):
            whole = logical(t).copy()
            same(whole)[...] = block.reshape(-1)[0]
            same_bits(whole, block, f"around {what} of {name}")
        assert np.all(logical(om)[..., 0] == 7) and np.all(logical(orr)[..., 0] == 7)
        same_bits(logical(odg)[1::2], block.reshape(-1)[:n], "between dgamma's values")


@pytest.mark.parametrize("n", [3, 96, 101, 1030, 5001, 20000, 20003])
def test_results_that_replace_inputs(hip, oracle, n):
    d = dt.float32
    x, g = (drawn((9, n), d, oracle, k) for k in (1, 2))
    fresh = lambda v: tensor(hip, v[0], d)  # noqa: E731
    hx, hg = fresh(x), fresh(g)
    y, mean, rstd = hip.layer_norm(hx)
    over = fresh(x)
    hip.layer_norm(over, out=(over, None, None))
    same_bits(logical(over), logical(y), "y over x")
    want = hip.layer_norm_grad(hg, hx, mean, rstd)
    for k in (0, 1):
        a, b = fresh(g), fresh(x)
        got = hip.layer_norm_grad(a, b, mean, rstd, out=((a, b)[k], hip.buffer(d, (n,)), hip.buffer(d, (n,))))
        for p, q in zip(got, want):
            same_bits(logical(p), logical(q), "dx over " + "gx"[k])


def test_gradients_that_are_not_wanted(hip, oracle):
    d = dt.bfloat16
    x, g, gamma = (drawn(s, d, oracle, k, 1.0, 0.5) for k, s in enumerate(((50, 200), (50, 200), (200,))))
    hx, hg, hw = (tensor(hip, v[0], d) for v in (x, g, gamma))
    _, mean, rstd = hip.layer_norm(hx, hw)
    want = hip.layer_norm_grad(hg, hx, mean, rstd, hw)
    for k in range(3):
        out = [None] * 3
        out[k] = hip.buffer(d, want[k].shape)
        hip.layer_norm_grad(hg, hx, mean, rstd, hw, out=out)
        same_bits(logical(out[k]), logical(want[k]), f"gradient {k} alone")


def test_differences(hip, oracle):
    """The gradient against differences of the forward pass in float64: loss = sum(c y), steps of 1e-6 (error of the
    difference about 1e-9 of values near one)."""
    rng = np.random.default_rng(5)
    d, n = dt.float64, 11
    x, c, gamma, beta = rng.standard_normal((3, n)), rng.standard_normal((3, n)), rng.standard_normal(n), rng.standard_normal(n)

    def loss(x, gamma, beta):
        return float((logical(hip.layer_norm(tensor(hip, x, d), tensor(hip, gamma, d), tensor(hip, beta, d))[0]) * c).sum())

    _, mean, rstd = hip.layer_norm(tensor(hip, x, d), tensor(hip, gamma, d), tensor(hip, beta, d))
    grads = [logical(t) for t in hip.layer_norm_grad(tensor(hip, c, d), tensor(hip, x, d), mean, rstd, tensor(hip, gamma, d))]
    args = [x, gamma, beta]
    for k, grad in enumerate(grads):
        for at in np.ndindex(grad.shape):
            step = np.zeros_like(args[k])
            step[at] = 1e-6
            up, down = (loss(*[a + s * step if i == k else a for i, a in enumerate(args)]) for s in (1, -1))
            assert abs((up - down) / 2e-6 - grad[at]) < 1e-7


def test_rows_with_no_spread_and_rows_that_are_no_numbers(hip, oracle):
    d = dt.float32
    x = np.ones((6, 40), np.float32)
    x[1] = 3e4
    x[2, 7] = np.nan
    x[3, 0] = np.inf
    x[4] = np.arange(40)
    y, mean, rstd = (logical(t) for t in hip.layer_norm(tensor(hip, x, d)))
    assert np.all(y[[0, 1, 5]] == 0) and np.all(rstd[[0, 1, 5]] == np.float32(1) / np.sqrt(np.float32(1e-5)))
    assert np.all(np.isnan(y[2])) and np.isnan(mean[2]) and np.all(np.isnan(y[3])) and mean[3] == np.inf
    within(y[4].astype(np.float64), forward(x[4].astype(np.float64), None, None, d)[0][0], forward(x[4].astype(np.float64), None, None, d)[1][0], d, "the row between")
    y, _, rstd = (logical(t) for t in hip.layer_norm(tensor(hip, x[:1], d), eps=0.0))
    assert np.all(np.isnan(y)) and np.isinf(rstd[0])  # no spread and no eps: 0 / 0
    # a row that is no number spoils its own dx and the columns' sums, nothing else
    g = np.ones((6, 40), np.float32)
    _, m, r = hip.layer_norm(tensor(hip, x, d))
    dx, dgamma, dbeta = (logical(t) for t in hip.layer_norm_grad(tensor(hip, g, d), tensor(hip, x, d), m, r))
    assert np.all(np.isfinite(dx[[0, 1, 4, 5]])) and np.all(np.isnan(dx[2])) and np.all(np.isnan(dgamma)) and np.all(dbeta == 6)


def test_no_rows(hip):
    d = dt.float16
    x = hip.buffer(d, (0, 5))
    y, mean, rstd = hip.layer_norm(x, hip.full(d, (5,), 1.0))
    assert y.shape == (0, 5) and mean.shape == (0,)
    dx, dgamma, dbeta = hip.layer_norm_grad(x, x, mean, rstd)
    assert dx.shape == (0, 5) and np.all(logical(dgamma) == 0) and np.all(logical(dbeta) == 0)


def test_replays(hip, oracle):
    """A recorded step, forward and backward, replayed on new inputs between other work of its context."""
    d = dt.bfloat16
    n = 768
    hx, hg = tensor(hip, drawn((100, n), d, oracle, 0)[0], d), tensor(hip, drawn((100, n), d, oracle, 1)[0], d)
    hw = tensor(hip, drawn((n,), d, oracle, 2, 0.2, 1.0)[0], d)

    def step():
        y, mean, rstd = hip.layer_norm(hx, hw, hw)
        return (y, mean, rstd, *hip.layer_norm_grad(hg, hx, mean, rstd, hw))

    step()
    graphs = []
    for _ in range(2):  # two graphs, whose partial sums are storage of their own
        hip.capture_begin()
        try:
            out = step()
        finally:
            graphs.append((hip.capture_end(), out))
    try:
        for k in range(4):
            hip.assign(hx, tensor(hip, drawn((100, n), d, oracle, 10 + k, 1.0 + k)[0], d))
            for graph, _ in graphs:
                graph.launch()
            eager = step()
            for _, out in graphs:
                for a, b in zip(out, eager):
                    same_bits(logical(a), logical(b), f"replay {k}")
    finally:
        for graph, _ in graphs:
            graph.destroy()


def test_behind_deferred_work(hip, oracle):
    d = dt.float32
    a = tensor(hip, drawn((33, 70), d, oracle, 3)[0], d)
    want = hip.layer_norm(hip.binary("mul", a, a))
    want = [logical(t) for t in (*want, *hip.layer_norm_grad(a, hip.binary("mul", a, a), *want[1:]))]
    hip.set_deferred(True)
    try:
        x = hip.binary("mul", a, a)
        y, mean, rstd = hip.layer_norm(x)
        z = hip.binary("add", y, y)  # recorded behind the call it reads
        grads = hip.layer_norm_grad(a, x, mean, rstd)
        got = [logical(t) for t in (y, mean, rstd, *grads)]
        same_bits(logical(z), 2 * got[0], "work recorded behind")
    finally:
        hip.set_deferred(False)
    for p, q in zip(got, want):
        same_bits(p, q, "behind deferred work")


@pytest.mark.parametrize("n", [5, 1001, 6001, 20003])
def test_one_row_whose_results_replace_what_has_its_shape(hip, oracle, n):
    """With no outer axis the weights, their gradients and the row are of one shape: each result in the place of each of them."""
    d = dt.float32
    held = {k: drawn((n,), d, oracle, n + i)[0] for i, k in enumerate(("x", "gamma", "beta", "g"))}

    def fresh():
        return {k: tensor(hip, v, d) for k, v in held.items()}

    t = fresh()
    y, mean, rstd = hip.layer_norm(t["x"], t["gamma"], t["beta"], EPS)
    want = [logical(v) for v in hip.layer_norm_grad(t["g"], t["x"], mean, rstd, t["gamma"])]
    for name in ("x", "gamma", "beta"):
        t = fresh()
        same_bits(logical(hip.layer_norm(t["x"], t["gamma"], t["beta"], EPS, out=(t[name], None, None))[0]), logical(y), f"over {name}")
    for names in (("x", "gamma", "g"), ("g", "x", "gamma"), ("gamma", "g", "x")):
        t = fresh()
        got = hip.layer_norm_grad(t["g"], t["x"], mean, rstd, t["gamma"], out=tuple(t[k] for k in names))
        for a, b in zip(got, want):
            same_bits(logical(a), b, f"gradients over {names}")


def test_refusals(hip):
    B, f32 = hip, dt.float32
    x, v, s = B.full(f32, (4, 8), 1.0), B.full(f32, (8,), 1.0), B.full(f32, (4,), 1.0)
    fresh = lambda: (B.buffer(f32, (4, 8)), B.buffer(f32, (4,)), B.buffer(f32, (4,)))  # noqa: E731
    with pytest.raises(ValueError, match="layer_norm: shape mismatch"):
        B.layer_norm(x, B.full(f32, (7,), 1.0))
    with pytest.raises(ValueError, match="eps"):
        B.layer_norm(x, eps=-1.0)
    with pytest.raises(ValueError, match="eps"):
        B.layer_norm(x, eps=float("nan"))
    with pytest.raises(RuntimeError, match="dtype not supported"):
        B.layer_norm(B.full(dt.int32, (4, 8), 1))
    with pytest.raises(RuntimeError, match="dtype not supported"):
        B.layer_norm(x, B.full(dt.float64, (8,), 1.0))
    with pytest.raises(RuntimeError, match="rows must be contiguous"):
        B.layer_norm(B.permute(x, (1, 0)))
    with pytest.raises(RuntimeError, match="rows must be contiguous"):
        B.layer_norm(x, B.expand(B.full(f32, (1,), 1.0), (8,)))
    with pytest.raises(ValueError, match="scalar"):
        B.layer_norm(B.full(f32, (), 1.0))
    with pytest.raises(ValueError, match="empty axis"):
        B.layer_norm(B.buffer(f32, (4, 0)))
    with pytest.raises(ValueError, match="broadcast"):
        B.layer_norm(x, out=(B.expand(B.buffer(f32, (1, 8)), (4, 8)), None, None))
    with pytest.raises(RuntimeError, match="dtype not supported"):
        y, m, _ = fresh()
        B.layer_norm(x, out=(y, m, B.buffer(dt.float64, (4,))))
    with pytest.raises(ValueError, match="shape mismatch"):
        y, m, _ = fresh()
        B.layer_norm(x, out=(y, m, B.buffer(f32, (5,))))
    with pytest.raises(RuntimeError, match="2\\^24"):
        B.layer_norm(B.expand(B.full(f32, (1,), 1.0), ((1 << 24) + 1,)), out=(B.expand(B.full(f32, (1,), 1.0), ((1 << 24) + 1,)), None, None))
    many = B.expand(B.reshape(x, (1, 1, 4, 8)), (1 << 20, 1 << 20, 4, 8))
    with pytest.raises(RuntimeError, match="too many rows"):
        B.layer_norm(many, out=(many, None, None))
    with pytest.raises(ValueError, match="layer_norm_grad: shape mismatch"):
        B.layer_norm_grad(B.full(f32, (4, 9), 1.0), x, s, s)
    with pytest.raises(ValueError, match="shape mismatch"):
        B.layer_norm_grad(x, x, s, B.full(f32, (5,), 1.0))
    with pytest.raises(RuntimeError, match="dtype not supported"):
        B.layer_norm_grad(x, x, s, B.full(dt.bfloat16, (4,), 1.0))
    with pytest.raises(RuntimeError, match="dtype not supported"):
        B.layer_norm_grad(B.full(dt.bfloat16, (4, 8), 1.0), x, s, s)
    with pytest.raises(ValueError, match="shape mismatch"):
        B.layer_norm_grad(x, x, s, s, out=(None, B.buffer(f32, (9,)), None))
    with pytest.raises(ValueError, match="null argument"):
        B.layer_norm_grad(x, x, s, s, out=(None, None, None))
    with pytest.raises(RuntimeError, match="rows must be contiguous"):
        B.layer_norm_grad(B.expand(B.full(f32, (1, 1), 1.0), (4, 8)), x, s, s, v)
    with pytest.raises(ValueError, match="broadcast"):
        B.layer_norm_grad(x, x, s, s, out=(None, B.expand(B.buffer(f32, (1,)), (8,)), None))
