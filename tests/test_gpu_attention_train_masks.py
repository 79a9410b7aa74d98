"""attention_train and attention_grad with masks that differ from head to head, of any strides, and with lengths of any stride; against their
formulas in float64, with the bounds of attention_oracle.py."""

import numpy as np
import pytest

import attention_oracle as ao
from helpers import decode, encode, logical, same_bits
from raven_amd import dtype as dt
from raven_amd.view import View
from test_gpu_attention_train import bhsd, drawn, tensor, within

pytestmark = pytest.mark.gpu

BF16, F16, F32 = dt.bfloat16, dt.float16, dt.float32


def check(hip, oracle, d, b, h, hk, sq, sk, dim, m, tm, causal=False, lengths=None, tl=None, seed=0):
    """Forward and backward under the mask ``m`` (``tm`` on the device), both checked."""
    rng = np.random.default_rng(seed)
    scale = dim ** -0.5
    (q_s, q), (g_s, g) = drawn((b, h, sq, dim), d, oracle, rng), drawn((b, h, sq, dim), d, oracle, rng)
    (k_s, k), (v_s, v) = drawn((b, hk, sk, dim), d, oracle, rng), drawn((b, hk, sk, dim), d, oracle, rng)
    keep = ao.seen(b, h, sq, sk, causal, lengths, m)
    if lengths is not None and tl is None:
        tl = tensor(hip, np.array(lengths, np.int32), dt.int32)
    tq, tk, tv, tg = (bhsd(hip, s, d) for s in (q_s, k_s, v_s, g_s))
    y, lse = hip.attention_train(tq, tk, tv, scale, causal, tl, tm)
    (want_y, want_lse), (y_err, lse_err) = ao.forward(q, k, v, scale, keep, d.name)
    y_s, got_lse = logical(y), logical(lse).astype(np.float64)
    within(got_lse, want_lse, lse_err, "float32", "lse")
    within(decode(y_s, d, oracle), want_y, y_err, d.name, "out")
    grads = hip.attention_grad(tg, tq, tk, tv, y, lse, scale, causal, tl, tm)
    want, err = ao.backward(g, q, k, v, decode(y_s, d, oracle), got_lse, scale, keep, d.name)
    for name, t, w, e in zip(("dv", "dk", "dq"), reversed(grads), reversed(want), reversed(err)):
        within(decode(logical(t), d, oracle), w, e, d.name, name)


def device(hip, m):
    return tensor(hip, m.astype(np.uint8), dt.bool_)


# ── masks of each head's own ─────────────────────────────────────────────────

@pytest.mark.parametrize("d", [F32, BF16, F16])
@pytest.mark.parametrize("dim", [20, 64, 80, 128])
@pytest.mark.parametrize("h, hk", [(3, 3), (6, 2)])
def test_heads(hip, oracle, d, dim, h, hk):
    m = np.random.default_rng(dim).random((2, h, 90, 75)) < 0.5
    check(hip, oracle, d, 2, h, hk, 90, 75, dim, m, device(hip, m), seed=1)


@pytest.mark.parametrize("d", [F32, BF16, F16])
@pytest.mark.parametrize("h, hk, sq, sk, dim, causal", [(8, 1, 700, 130, 64, False), (4, 1, 520, 520, 128, True), (6, 2, 333, 200, 96, False), (8, 2, 300, 310, 32, True)])
def test_heads_that_share_a_walk_in_parts(hip, oracle, d, h, hk, sq, sk, dim, causal):
    """Few keys that many queries see: a block's part of the walk begins in one head and ends in another."""
    m = np.random.default_rng(sq).random((1, h, sq, sk)) < 0.4
    check(hip, oracle, d, 1, h, hk, sq, sk, dim, m, device(hip, m), causal, seed=2)


@pytest.mark.parametrize("d, dim", [(BF16, 64), (F16, 128), (F32, 40), (F32, 96)])
def test_heads_of_more_blocks_than_units(hip, oracle, d, dim):
    b, h, hk, sq, sk = 2, 128, 64, 260, 140
    m = np.random.default_rng(dim).random((b, h, sq, sk)) < 0.6
    check(hip, oracle, d, b, h, hk, sq, sk, dim, m, device(hip, m), False, [140, 77], seed=3)


# ── masks of other strides ─────────────────────────────────────────────────

def by_keys(hip, m):
    """Queries side by side."""
    return hip.permute(device(hip, np.ascontiguousarray(m.swapaxes(2, 3))), (0, 1, 3, 2))


def every_third(hip, m):
    wide = np.repeat(~m, 3, 3)
    wide[..., 1::3] = m
    b, h, sq, sk = m.shape
    return hip.with_view(device(hip, wide), View.create(m.shape, (3 * h * sq * sk, 3 * sq * sk, 3 * sk, 3), 1))


def backwards(hip, m):
    return hip.flip(device(hip, m[:, ::-1, ::-1, ::-1]), (False, True, True, True))


def off_by_one(hip, m):
    """Rows one byte longer than their keys: of any alignment."""
    b, h, sq, sk = m.shape
    wide = np.concatenate([m, np.ones((b, h, sq, 1), bool)], 3)
    return hip.shrink(device(hip, wide), [(0, b), (0, h), (0, sq), (0, sk)])


@pytest.mark.parametrize("d", [F32, BF16])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("view", [by_keys, every_third, backwards, off_by_one])
def test_strides(hip, oracle, d, dim, view):
    m = np.random.default_rng(4).random((2, 4, 100, 150)) < 0.5
    check(hip, oracle, d, 2, 4, 2, 100, 150, dim, m, view(hip, m), seed=4)


@pytest.mark.parametrize("d", [F32, F16])
@pytest.mark.parametrize("dim", [32, 96])
@pytest.mark.parametrize("shape", [(2, 1, 1, 130), (2, 1, 70, 1), (1, 4, 1, 1), (1, 1, 70, 130), (1, 4, 1, 130), (1, 1, 1, 1)])
def test_broadcast_masks(hip, oracle, d, dim, shape):
    """Keys of a padded batch, queries that see nothing, whole heads: dimensions of stride 0."""
    m = np.random.default_rng(sum(shape)).random(shape) < 0.6
    whole = (2, 4, 70, 130)
    check(hip, oracle, d, 2, 4, 2, 70, 130, dim, np.broadcast_to(m, whole), hip.expand(device(hip, m), whole), seed=5)


@pytest.mark.parametrize("step", [2, -1, 0])
def test_strides_of_lengths(hip, oracle, step):
    b, n = 3, 100
    memory = np.array([100, 17, 50, 1000, 0, 64, 33], np.int32)
    first = 2 if step < 0 else 0
    lengths = [int(memory[first + step * i]) for i in range(b)]
    tl = hip.with_view(tensor(hip, memory, dt.int32), View.create((b,), (step,), first))
    m = np.ones((b, 2, n, n), bool)
    check(hip, oracle, BF16, b, 2, 2, n, n, 64, m, None, True, lengths, tl, seed=6)


# ── float16's range ───────────────────────────────────────────────────────

@pytest.mark.parametrize("dim", [32, 128])
def test_scores_gradients_up_to_the_range_of_float16(hip, oracle, dim):
    """One query, two keys of equal scores whose values point apart: p (g . v - g . out) is +- g . v / 2. Up to 2047 it is in range and right;
    past that no result pretends to be a number."""
    q, k, v = np.zeros((1, 1, 1, dim)), np.zeros((1, 1, 2, dim)), np.zeros((1, 1, 2, dim))
    q[..., 0], k[..., 1], v[0, 0, 0, 0], v[0, 0, 1, 0] = 0.5, 0.25, 2.0, -2.0
    keep = ao.seen(1, 1, 1, 2)
    for size, inside in ((2040.0, True), (2100.0, False)):
        g = np.zeros((1, 1, 1, dim))
        g[..., 0] = size
        tq, tk, tv, tg = (tensor(hip, encode(x, F16, oracle), F16) for x in (q, k, v, g))
        y, lse = hip.attention_train(tq, tk, tv, 1.0)
        dq, dk, dv = (decode(logical(t), F16, oracle) for t in hip.attention_grad(tg, tq, tk, tv, y, lse, 1.0))
        if inside:
            want, err = ao.backward(g, q, k, v, decode(logical(y), F16, oracle), logical(lse).astype(np.float64), 1.0, keep, "float16")
            for name, t, w, e in zip(("dq", "dk", "dv"), (dq, dk, dv), want, err):
                within(t, w, e, "float16", name)
        else:
            assert not np.isfinite(dk[..., 0]).any()
