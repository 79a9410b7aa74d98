"""attention_train and attention_grad against their formulas in float64; the bounds are derived in attention_oracle.py."""

import numpy as np
import pytest

import attention_oracle as ao
from helpers import decode, encode, logical, same_bits
from raven_amd import dtype as dt

pytestmark = pytest.mark.gpu

BF16, F16, F32 = dt.bfloat16, dt.float16, dt.float32


def tensor(hip, storage, d):
    return hip.reshape(hip.from_host(np.ascontiguousarray(storage), d), storage.shape)


def bhsd(hip, storage, d):
    """[batch, heads, length, dim] as it lies after a projection: the heads of a token side by side."""
    return hip.permute(tensor(hip, storage.transpose(0, 2, 1, 3), d), (0, 2, 1, 3))


def drawn(shape, d, oracle, rng, scale=1.0):
    s = encode(rng.standard_normal(shape) * scale, d, oracle)
    return s, decode(s, d, oracle)


def within(got, want, err, d, what):
    assert got.shape == want.shape, (what, got.shape, want.shape)
    none = np.isinf(want)
    assert np.array_equal(got[none], want[none]), what
    lim = err + ao.HALF[d] * (np.abs(want) + err) + ao.TINY[d]
    with np.errstate(invalid="ignore"):
        off = np.where(none, 0.0, np.abs(got - want))
    assert np.all(off <= lim), f"{what}: {np.nanmax(off / lim)} times the bound at {np.unravel_index(np.nanargmax(np.where(np.isnan(off), np.inf, off / lim)), off.shape)}"


def run(hip, oracle, d, b, h, hk, sq, sk, dim, causal=False, lengths=None, mask=None, seed=0, scale=None, spread=1.0, view=bhsd, pads=()):
    """Forward and backward of one case, both checked. ``mask``: share of pairs that it leaves."""
    rng = np.random.default_rng(seed)
    scale = dim ** -0.5 if scale is None else scale
    (q_s, q), (g_s, g) = drawn((b, h, sq, dim), d, oracle, rng, spread), drawn((b, h, sq, dim), d, oracle, rng)
    (k_s, k), (v_s, v) = drawn((b, hk, sk, dim), d, oracle, rng), drawn((b, hk, sk, dim), d, oracle, rng)
    m = None
    if mask is not None:
        m = rng.random((b, 1, sq, sk)) < mask
    keep = ao.seen(b, h, sq, sk, causal, lengths, m)
    tq, tk, tv, tg = view(hip, q_s, d), view(hip, k_s, d), view(hip, v_s, d), view(hip, g_s, d)
    tl = tensor(hip, np.array(lengths, np.int32), dt.int32) if lengths is not None else None
    tm = hip.expand(tensor(hip, m.astype(np.uint8), dt.bool_), (b, h, sq, sk)) if m is not None else None
    y, lse = hip.attention_train(tq, tk, tv, scale, causal, tl, tm)
    (want_y, want_lse), (y_err, lse_err) = ao.forward(q, k, v, scale, keep, d.name)
    y_s, got_lse = logical(y), logical(lse).astype(np.float64)
    within(got_lse, want_lse, lse_err, "float32", "lse")
    within(decode(y_s, d, oracle), want_y, y_err, d.name, "out")
    grads = hip.attention_grad(tg, tq, tk, tv, y, lse, scale, causal, tl, tm)
    want, err = ao.backward(g, q, k, v, decode(y_s, d, oracle), got_lse, scale, keep, d.name)
    for name, t, w, e in zip(("dv", "dk", "dq"), reversed(grads), reversed(want), reversed(err)):
        within(decode(logical(t), d, oracle), w, e, d.name, name)
    return y, lse, grads


@pytest.mark.parametrize("d", [F32, BF16, F16])
@pytest.mark.parametrize("sq, sk, causal", [(1, 1, True), (1, 70, False), (33, 33, True), (64, 64, False), (130, 130, True), (200, 129, False)])
def test_lengths_and_types(hip, oracle, d, sq, sk, causal):
    run(hip, oracle, d, 2, 3, 3, sq, sk, 64, causal)


@pytest.mark.parametrize("d", [F32, BF16, F16])
@pytest.mark.parametrize("dim", [1, 3, 8, 20, 32, 40, 65, 96, 100, 128])
def test_head_dimensions(hip, oracle, d, dim):
    run(hip, oracle, d, 1, 2, 2, 70, 101, dim, seed=dim)


@pytest.mark.parametrize("d", [F32, BF16])
@pytest.mark.parametrize("h, hk", [(4, 1), (6, 2), (5, 5), (8, 2)])
def test_shared_heads(hip, oracle, d, h, hk):
    run(hip, oracle, d, 2, h, hk, 150, 150, 32, True, seed=h)


@pytest.mark.parametrize("d", [F32, F16])
@pytest.mark.parametrize("sq, sk", [(100, 40), (40, 100), (129, 1), (300, 31), (31, 300)])
def test_causal_of_other_lengths(hip, oracle, d, sq, sk):
    """More queries than keys: the first see none, and are zeros with lse -inf."""
    run(hip, oracle, d, 1, 2, 1, sq, sk, 64, True, seed=sq)


@pytest.mark.parametrize("d", [F32, BF16, F16])
@pytest.mark.parametrize("causal", [False, True])
def test_padded_batches(hip, oracle, d, causal):
    run(hip, oracle, d, 5, 2, 2, 140, 140, 64, causal, lengths=[140, 0, 1, 77, 1000], seed=3)


@pytest.mark.parametrize("d", [F32, BF16])
@pytest.mark.parametrize("share", [0.0, 0.02, 0.5, 1.0])
def test_masks(hip, oracle, d, share):
    run(hip, oracle, d, 2, 2, 1, 90, 75, 40, mask=share, seed=int(share * 100))


@pytest.mark.parametrize("d", [F32, F16])
def test_mask_with_causal_and_lengths(hip, oracle, d):
    run(hip, oracle, d, 2, 2, 2, 160, 160, 64, True, lengths=[100, 160], mask=0.3)


@pytest.mark.parametrize("d", [F32, BF16, F16])
@pytest.mark.parametrize("spread, scale", [(30.0, None), (1.0, 1e-6), (0.01, 40.0)])
def test_sizes_of_scores(hip, oracle, d, spread, scale):
    run(hip, oracle, d, 1, 2, 2, 128, 200, 64, spread=spread, scale=scale)


@pytest.mark.parametrize("d", [BF16, F32])
def test_a_long_walk_in_parts(hip, oracle, d):
    """One head of keys and many queries that see them: their tiles are divided among blocks."""
    run(hip, oracle, d, 1, 4, 1, 700, 130, 64, seed=7)
    run(hip, oracle, d, 1, 2, 1, 520, 520, 128, True, seed=8)


@pytest.mark.parametrize("d", [BF16, F32])
def test_many_blocks(hip, oracle, d):
    run(hip, oracle, d, 3, 50, 50, 130, 140, 32, True, seed=9)


@pytest.mark.parametrize("d", [F32, BF16, F16])
@pytest.mark.parametrize("dim", [6, 12, 65, 127])
def test_sums_of_parts(hip, oracle, d, dim):
    run(hip, oracle, d, 1, 4, 1, 300, 130, dim, seed=14)


@pytest.mark.parametrize("d, dim", [(BF16, 64), (BF16, 128), (BF16, 63), (F16, 32), (F16, 96), (F32, 32), (F32, 64), (F32, 90), (F32, 128)])
@pytest.mark.parametrize("mask", [None, 0.4])
def test_more_blocks_than_units(hip, oracle, d, dim, mask):
    """Heads enough for the widest blocks of queries, and for gradients of keys without parts."""
    run(hip, oracle, d, 4, 64, 32, 260, 140, dim, mask is None, [140, 0, 77, 1], mask, seed=15)


@pytest.mark.parametrize("d", [F32, BF16])
def test_more_blocks_than_units_in_a_projection(hip, oracle, d):
    run(hip, oracle, d, 2, 128, 128, 270, 100, 40, True, seed=16, view=packed)


@pytest.mark.parametrize("d, dim", [(BF16, 64), (F16, 32), (BF16, 41)])
@pytest.mark.parametrize("mask", [None, 0.4])
def test_more_blocks_of_keys_than_units(hip, oracle, d, dim, mask):
    run(hip, oracle, d, 4, 128, 128, 100, 140, dim, mask is None, [140, 0, 77, 1], mask, seed=17)


# ── layouts ─────────────────────────────────────────────────────────────────────────────────────

def packed(hip, storage, d):
    """A third of rows that hold queries, keys and values of a token, one element off any alignment."""
    b, h, n, dim = storage.shape
    wide = np.zeros((b, n, 3 * h * dim + 1), storage.dtype)
    wide[:, :, 1 + h * dim:1 + 2 * h * dim] = storage.transpose(0, 2, 1, 3).reshape(b, n, h * dim)
    t = hip.shrink(tensor(hip, wide, d), [(0, b), (0, n), (1 + h * dim, 1 + 2 * h * dim)])
    return hip.permute(hip.reshape(t, (b, n, h, dim)), (0, 2, 1, 3))


def backwards(hip, storage, d):
    """Batches and heads in reverse order in memory."""
    return hip.flip(tensor(hip, storage[::-1, ::-1], d), (True, True, False, False))


@pytest.mark.parametrize("d", [F32, BF16])
@pytest.mark.parametrize("view", [tensor, packed, backwards])
def test_layouts(hip, oracle, d, view):
    run(hip, oracle, d, 2, 3, 3, 75, 75, 24, True, view=view)


def test_results_in_views_leave_their_surroundings(hip, oracle):
    b, h, n, dim, d = 2, 2, 70, 40, BF16
    rng = np.random.default_rng(1)
    (q_s, q), (g_s, g) = drawn((b, h, n, dim), d, oracle, rng), drawn((b, h, n, dim), d, oracle, rng)
    whole = {}

    def inside(name, shape, kind):
        """A view in the middle of memory full of a pattern."""
        whole[name] = tensor(hip, np.full([s + 4 for s in shape], 0x3c, kind.np_storage), kind)
        return hip.shrink(whole[name], [(2, s + 2) for s in shape])

    q, g = tensor(hip, q_s, d), tensor(hip, g_s, d)
    out = inside("y", (b, h, n, dim), d), inside("lse", (b, h, n), F32)
    hip.attention_train(q, q, q, 0.2, True, out=out)
    grads = tuple(inside(name, (b, h, n, dim), d) for name in ("dq", "dk", "dv"))
    hip.attention_grad(g, q, q, q, *out, 0.2, True, out=grads)
    plain = hip.attention_train(q, q, q, 0.2, True)
    for got, want in zip(out + grads, plain + hip.attention_grad(g, q, q, q, *plain, 0.2, True)):
        same_bits(logical(got), logical(want))
    for name, t in whole.items():
        s = logical(t).copy()
        s[tuple(slice(2, -2) for _ in s.shape)] = 0x3c
        assert np.all(s == 0x3c), name


def test_broadcast_inputs(hip, oracle):
    """One head of keys under all batches (stride 0): each gets a gradient of its own."""
    rng = np.random.default_rng(2)
    (q_s, _), (k_s, _) = drawn((3, 2, 40, 32), F32, oracle, rng), drawn((1, 1, 50, 32), F32, oracle, rng)
    q, wide = tensor(hip, q_s, F32), hip.expand(tensor(hip, k_s, F32), (3, 2, 50, 32))
    same = tensor(hip, np.broadcast_to(k_s, (3, 2, 50, 32)), F32)
    one, two = hip.attention_train(q, wide, wide, 0.3), hip.attention_train(q, same, same, 0.3)
    for x, y in zip(one + hip.attention_grad(q, q, wide, wide, *one, 0.3), two + hip.attention_grad(q, q, same, same, *two, 0.3)):
        same_bits(logical(x), logical(y))


def test_far_strides(hip, oracle):
    """Heads more than 2^32 bytes apart."""
    far = (1 << 31) + 4096
    block = hip.buffer(BF16, (far + 4096,))
    rng = np.random.default_rng(3)
    k_s, _ = drawn((1, 2, 64, 32), BF16, oracle, rng)
    heads = [hip.shrink(block, [(at, at + 2048)]) for at in (0, far)]
    for t, s in zip(heads, k_s[0]):
        hip.assign(t, tensor(hip, s.reshape(-1), BF16))
    from raven_amd.view import View

    k = hip.with_view(block, View.create((1, 2, 64, 32), (0, far, 32, 1)))
    near = tensor(hip, k_s, BF16)
    one, two = hip.attention_train(k, k, k, 0.3, True), hip.attention_train(near, near, near, 0.3, True)
    for x, y in zip(one + hip.attention_grad(near, k, k, k, *one, 0.3, True), two + hip.attention_grad(near, near, near, near, *two, 0.3, True)):
        same_bits(logical(x), logical(y))


# ── values that are no numbers ──────────────────────────────────────────────────────────────────

@pytest.mark.parametrize("d", [F32, BF16, F16])
def test_rows_past_a_length_are_not_read(hip, oracle, d):
    b, h, n, dim = 2, 2, 150, 64
    rng = np.random.default_rng(4)
    lengths = tensor(hip, np.array([70, 128], np.int32), dt.int32)
    results = []
    for fill in (0.0, np.nan, np.inf):
        rng = np.random.default_rng(4)
        x = rng.standard_normal((4, b, h, n, dim))
        x[1, 0, :, 70:] = x[2, 0, :, 70:] = x[1, 1, :, 128:] = x[2, 1, :, 128:] = fill
        q, k, v, g = (tensor(hip, encode(t, d, oracle), d) for t in x)
        y, lse = hip.attention_train(q, k, v, 0.1, False, lengths)
        results.append([logical(t) for t in (y, lse) + hip.attention_grad(g, q, k, v, y, lse, 0.1, False, lengths)])
    for other in results[1:]:
        for x, y in zip(results[0], other):
            same_bits(x, y)
    dk = decode(results[0][3], d, oracle)
    assert np.all(dk[0, :, 70:] == 0) and np.all(dk[1, :, 128:] == 0) and np.any(dk[0, :, 69] != 0)


@pytest.mark.parametrize("d", [F32, BF16])
def test_scores_that_are_no_numbers(hip, oracle, d):
    """A NaN or an infinity in a query makes its own row NaN and no other; in a key that nobody sees it does nothing to the scores."""
    x = np.random.default_rng(5).standard_normal((1, 1, 40, 32))
    bad = x.copy()
    bad[0, 0, 7, 3], bad[0, 0, 20, 0] = np.nan, np.inf
    k = tensor(hip, encode(x, d, oracle), d)
    y, lse = hip.attention_train(tensor(hip, encode(bad, d, oracle), d), k, k, 0.2)
    want, _ = hip.attention_train(k, k, k, 0.2)
    y, want, lse = decode(logical(y), d, oracle), decode(logical(want), d, oracle), logical(lse)
    assert np.isnan(y[0, 0, [7, 20]]).all() and np.isnan(lse[0, 0, [7, 20]]).all()
    rest = [i for i in range(40) if i not in (7, 20)]
    assert np.array_equal(y[0, 0, rest], want[0, 0, rest])


# ── calls ───────────────────────────────────────────────────────────────────────────────────────

def test_equal_calls_give_equal_bits(hip, oracle):
    for d in (BF16, F32):
        one = run(hip, oracle, d, 1, 4, 2, 500, 300, 64, seed=11)
        two = run(hip, oracle, d, 1, 4, 2, 500, 300, 64, seed=11)
        for x, y in zip(one[:2] + one[2], two[:2] + two[2]):
            same_bits(logical(x), logical(y))


def test_recorded_and_replayed(hip, oracle):
    """Two graphs that live together, replayed in turn with eager work between, on inputs that change."""
    rng = np.random.default_rng(12)
    made = []
    for n, d in ((130, BF16), (300, F32)):
        x = [tensor(hip, drawn((1, 2, n, 64), d, oracle, rng)[0], d) for _ in range(4)]

        def step(x=x):
            y, lse = hip.attention_train(x[0], x[1], x[2], 0.125, True)
            return (y, lse) + hip.attention_grad(x[3], x[0], x[1], x[2], y, lse, 0.125, True)

        step()
        hip.synchronize()
        hip.capture_begin()
        out = step()
        made.append((x, step, out, hip.capture_end(), d, n))
    for turn in range(3):
        for x, step, out, graph, d, n in made:
            for t in x:
                hip.assign(t, tensor(hip, drawn((1, 2, n, 64), d, oracle, rng)[0], d))
            graph.launch()
            want = step()
            hip.synchronize()
            for a, b in zip(out, want):
                same_bits(logical(a), logical(b), f"turn {turn}")
    for *_, graph, _, _ in made:
        graph.destroy()


def test_deferred_operands(hip, oracle):
    """Operands that are still recorded when the call comes."""
    rng = np.random.default_rng(13)
    x = tensor(hip, drawn((1, 2, 40, 32), F32, oracle, rng)[0], F32)
    two = hip.binary("add", x, x)
    want = hip.attention_train(two, two, two, 0.2)
    want += hip.attention_grad(two, two, two, two, *want, 0.2)
    hip.set_deferred(True)
    try:
        t = hip.binary("add", x, x)
        got = hip.attention_train(t, t, t, 0.2)
        got += hip.attention_grad(t, t, t, t, *got, 0.2)
        for a, b in zip(got, want):
            same_bits(logical(a), logical(b))
    finally:
        hip.set_deferred(False)


def test_empty(hip):
    e = lambda *s: hip.buffer(F32, s)  # noqa: E731
    y, lse = hip.attention_train(e(2, 2, 5, 8), e(2, 2, 0, 8), e(2, 2, 0, 8), 1.0)
    assert np.all(logical(y) == 0) and np.all(logical(lse) == -np.inf)
    dq, dk, dv = hip.attention_grad(e(2, 2, 5, 8), e(2, 2, 5, 8), e(2, 2, 0, 8), e(2, 2, 0, 8), y, lse, 1.0)
    assert np.all(logical(dq) == 0) and dk.shape == (2, 2, 0, 8)
    y, lse = hip.attention_train(e(2, 2, 0, 8), e(2, 2, 5, 8), e(2, 2, 5, 8), 1.0)
    dq, dk, dv = hip.attention_grad(e(2, 2, 0, 8), e(2, 2, 0, 8), e(2, 2, 5, 8), e(2, 2, 5, 8), y, lse, 1.0)
    assert np.all(logical(dk) == 0) and np.all(logical(dv) == 0)
    hip.attention_train(e(0, 2, 5, 8), e(0, 2, 5, 8), e(0, 2, 5, 8), 1.0)


def test_refusals(hip):
    t = lambda *s, d=F32: hip.buffer(d, s)  # noqa: E731
    q, k = t(2, 4, 6, 8), t(2, 2, 5, 8)
    lse = t(2, 4, 6)
    ok = (q, k, k, 1.0)
    y = hip.attention_train(*ok)
    with pytest.raises(ValueError, match="shape"):
        hip.attention_train(q, k, t(2, 2, 6, 8), 1.0)
    with pytest.raises(ValueError, match="multiple"):
        hip.attention_train(q, t(2, 3, 5, 8), t(2, 3, 5, 8), 1.0)
    with pytest.raises(ValueError, match="batch, heads"):
        hip.attention_train(t(4, 6, 8), t(4, 5, 8), t(4, 5, 8), 1.0)
    for scale in (0.0, -1.0, 1e-31, 1e31, float("nan"), float("inf")):
        with pytest.raises(ValueError, match="scale"):
            hip.attention_train(q, k, k, scale)
    with pytest.raises(ValueError, match="shape"):
        hip.attention_train(*ok, lengths=t(3, d=dt.int32))
    with pytest.raises(RuntimeError, match="dtype"):
        hip.attention_train(*ok, lengths=t(2, d=dt.int64))
    with pytest.raises(ValueError, match="shape"):
        hip.attention_train(*ok, mask=t(2, 4, 6, 6, d=dt.bool_))
    with pytest.raises(RuntimeError, match="dtype"):
        hip.attention_train(*ok, mask=t(2, 4, 6, 5, d=dt.uint8))
    with pytest.raises(RuntimeError, match="at most 128"):
        hip.attention_train(t(1, 1, 2, 129), t(1, 1, 2, 129), t(1, 1, 2, 129), 1.0)
    with pytest.raises(ValueError, match="must not be 0"):
        hip.attention_train(t(1, 1, 2, 0), t(1, 1, 2, 0), t(1, 1, 2, 0), 1.0)
    with pytest.raises(RuntimeError, match="dtype"):
        hip.attention_train(*(t(1, 1, 2, 8, d=dt.float64) for _ in range(3)), 1.0)
    with pytest.raises(RuntimeError, match="dtype"):
        hip.attention_train(q, k, t(2, 2, 5, 8, d=BF16), 1.0)
    with pytest.raises(RuntimeError, match="contiguous"):
        hip.attention_train(hip.permute(t(2, 4, 8, 6), (0, 1, 3, 2)), k, k, 1.0)
    with pytest.raises(RuntimeError, match="follow"):
        hip.attention_train(hip.flip(q, (False, False, True, False)), k, k, 1.0)
    with pytest.raises(ValueError, match="broadcast"):
        hip.attention_train(*ok, out=(hip.expand(t(1, 4, 6, 8), (2, 4, 6, 8)), lse))
    with pytest.raises(ValueError, match="broadcast"):
        hip.attention_train(*ok, out=(t(2, 4, 6, 8), hip.expand(t(1, 4, 6), (2, 4, 6))))
    with pytest.raises(ValueError, match="replace"):
        hip.attention_train(*ok, out=(q, lse))
    with pytest.raises(ValueError, match="replace"):
        hip.attention_grad(q, q, k, k, *y, 1.0, out=(t(2, 4, 6, 8), k, t(2, 2, 5, 8)))
    with pytest.raises(ValueError, match="shape"):
        hip.attention_grad(q, q, k, k, *y, 1.0, out=(t(2, 4, 6, 8), t(2, 2, 5, 8), t(2, 4, 5, 8)))
    with pytest.raises(ValueError, match="shape"):
        hip.attention_grad(k, q, k, k, *y, 1.0)
    with pytest.raises(RuntimeError, match="dtype"):
        hip.attention_grad(q, q, k, k, y[0], t(2, 4, 6, d=BF16), 1.0)


def test_results_in_one_place(hip):
    t = lambda *s: hip.buffer(F32, s)  # noqa: E731
    q, k = t(2, 2, 6, 8), t(2, 2, 6, 8)
    y = hip.attention_train(q, k, k, 1.0)
    one = t(2, 2, 6, 8)
    for out in ((one, one, t(2, 2, 6, 8)), (one, t(2, 2, 6, 8), one), (t(2, 2, 6, 8), one, one)):
        with pytest.raises(ValueError, match="one place"):
            hip.attention_grad(q, q, k, k, *y, 1.0, out=out)
    flat = t(2 * 2 * 6 * 8)
    lse = hip.reshape(hip.shrink(flat, [(0, 24)]), (2, 2, 6))
    with pytest.raises(ValueError, match="one place"):
        hip.attention_train(q, k, k, 1.0, out=(hip.reshape(flat, (2, 2, 6, 8)), lse))
    with pytest.raises(ValueError, match="replace"):
        hip.attention_train(q, hip.reshape(flat, (2, 2, 6, 8)), k, 1.0, out=(one, lse))
    with pytest.raises(ValueError, match="replace"):
        hip.attention_grad(q, q, k, k, y[0], lse, 1.0, out=(hip.reshape(flat, (2, 2, 6, 8)), one, t(2, 2, 6, 8)))
