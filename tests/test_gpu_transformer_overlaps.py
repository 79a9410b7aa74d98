"""Results of a transformer's training operators that begin where an operand of another dtype does."""

import numpy as np
import pytest

from helpers import logical
from raven_amd import dtype as dt
from raven_amd.nx_backend import Tensor
from raven_amd.view import View, c_contiguous_strides

pytestmark = pytest.mark.gpu

F32, I32, BOOL = dt.float32, dt.int32, dt.bool_


def at_start(hip, t, d, shape):
    """A tensor of another dtype in the memory of ``t``, from its first byte on."""
    return Tensor(t.buffer, View.create(shape, c_contiguous_strides(shape)), d, hip)


def memory(hip, n=4096):
    return hip.reshape(hip.from_host(np.zeros(n, np.float32), F32), (n,))


@pytest.mark.parametrize("name, d, shape", [("lengths", I32, (2,)), ("mask", BOOL, (2, 2, 6, 5))])
def test_attention_over_its_lengths_or_mask(hip, name, d, shape):
    new = lambda *s: hip.buffer(F32, s)  # noqa: E731
    q, k, lse = new(2, 2, 6, 8), new(2, 2, 5, 8), new(2, 2, 6)
    room = memory(hip)
    kw = {name: at_start(hip, room, d, shape)}
    with pytest.raises(ValueError, match="replace"):
        hip.attention_train(q, k, k, 1.0, out=(at_start(hip, room, F32, (2, 2, 6, 8)), lse), **kw)
    with pytest.raises(ValueError, match="replace"):
        hip.attention_train(q, k, k, 1.0, out=(new(2, 2, 6, 8), at_start(hip, room, F32, (2, 2, 6))), **kw)
    y, lse = hip.attention_train(q, k, k, 1.0, **kw)
    for which in range(3):
        out = [new(2, 2, 6, 8), new(2, 2, 5, 8), new(2, 2, 5, 8)]
        out[which] = at_start(hip, room, F32, out[which].shape)
        with pytest.raises(ValueError, match="replace"):
            hip.attention_grad(q, q, k, k, y, lse, 1.0, out=tuple(out), **kw)


def test_a_step_over_its_own_settings(hip):
    """Rate, step, factor and key inside what the step writes; beside it they may lie."""
    room, n = memory(hip), 300
    tensors = {"params": hip.shrink(room, [(100, 100 + n)])}
    new = lambda: hip.buffer(F32, (n,))  # noqa: E731
    inside = lambda d, at, size=1: Tensor(room.buffer, View.create((size,), (1,), at), d, hip)  # noqa: E731
    rate, step = (hip.reshape(hip.from_host(x, d), (1,)) for x, d in ((np.array([0.1], np.float32), F32), (np.array([1], np.int32), I32)))

    def call(rate=rate, step=step, **kw):
        hip.adamw([tensors["params"]], [new()], [new()], [new()], rate, step, **kw)

    call(inside(F32, 99), inside(I32, 100 + n), factor=inside(F32, 98))
    for at in (100, 250, 99 + n):
        for kw in ({"rate": inside(F32, at)}, {"step": inside(I32, at)}, {"factor": inside(F32, at)}):
            with pytest.raises(ValueError, match="twice"):
                call(**kw)


@pytest.mark.parametrize("at, stride, refused", [(99, 1, True), (100, -1, True), (98, 1, False), (98, 400, True), (400, 1, False), (402, -1, False), (402, -302, True)])
def test_a_step_over_its_key(hip, at, stride, refused):
    room, n = memory(hip), 300
    key = Tensor(room.buffer, View.create((2,), (stride,), at), I32, hip)
    new = lambda d, size=n: hip.buffer(d, (size,))  # noqa: E731
    rate, step = (hip.reshape(hip.from_host(x, d), (1,)) for x, d in ((np.array([0.1], np.float32), F32), (np.array([1], np.int32), I32)))
    args = ([hip.shrink(room, [(100, 100 + n)])], [new(F32)], [new(dt.float8_e4m3)], [new(dt.float8_e4m3)], rate, step)
    kw = {"m_scales": [new(F32, 2)], "v_scales": [new(F32, 2)], "key": key}
    if refused:
        with pytest.raises(ValueError, match="twice"):
            hip.adamw(*args, **kw)
    else:
        hip.adamw(*args, **kw)


@pytest.mark.parametrize("bits", [32, 8])
def test_an_infinite_gradient(hip, bits):
    """Its element is not finite from this step on; in 8 bits its block's scale is infinite, and the block from the next step on."""
    n, bad = 600, 261
    g = np.full(n, 1e-3, np.float32)
    g[bad] = np.inf
    host = lambda x, d: hip.reshape(hip.from_host(x, d), x.shape)  # noqa: E731
    p = host(np.ones(n, np.float32), F32)
    if bits == 32:
        m, v, kw = host(np.zeros(n, np.float32), F32), host(np.zeros(n, np.float32), F32), {}
    else:
        m, v = (host(np.zeros(n, np.uint8), dt.float8_e4m3) for _ in range(2))
        kw = {"m_scales": [memory(hip, 3)], "v_scales": [memory(hip, 3)], "key": host(np.array([3, 4], np.int32), I32)}
    rate, step = host(np.array([0.1], np.float32), F32), host(np.array([1], np.int32), I32)
    for turn in range(2):
        hip.adamw([p], [host(g, F32)], [m], [v], rate, step, **kw)
        finite = np.isfinite(logical(p))
        block = slice(256, 512) if bits == 8 and turn else slice(bad, bad + 1)
        assert not finite[block].any() and finite.sum() == n - (block.stop - block.start)
