"""What the deferred window knows of a block ends with a step of adamw that writes it."""

import numpy as np
import pytest

from helpers import encode, logical
from raven_amd import dtype as dt
from raven_amd.nx_frontend import Nx

pytestmark = pytest.mark.gpu

F32, BF16 = dt.float32, dt.bfloat16


def tensor(hip, a, d=F32):
    return hip.reshape(hip.from_host(np.ascontiguousarray(a), d), np.shape(a))


@pytest.mark.parametrize("written", ["params", "m", "v", "masters"])
def test_a_scalar_that_a_step_writes(hip, oracle, written):
    """A learned temperature: made as a fill, which the window takes for a constant, then stepped. A softmax behind the step has the new value."""
    nx = Nx(hip)
    rng = np.random.default_rng(1)
    x = tensor(hip, rng.standard_normal((20, 70)).astype(np.float32))
    rate, step = tensor(hip, np.array([0.25], np.float32)), tensor(hip, np.array([1], np.int32), dt.int32)
    hip.set_deferred(True)
    try:
        scale = hip.full(F32, (), 0.5)
        before = logical(nx.softmax(nx.mul(x, scale))).astype(np.float64)
        logical(nx.add(scale, scale))  # (the fill has been made)
        one = lambda v, d=F32: tensor(hip, encode(np.array([v], np.float32), d, oracle), d)  # noqa: E731
        d = BF16 if written == "masters" else F32
        lists = {"params": one(0.5, d), "grads": one(1.0, d), "m": one(0.0), "v": one(0.0)}
        if written == "masters":
            lists["masters"] = one(0.5)
        lists[written] = hip.reshape(scale, (1,))
        hip.adamw(*([lists[k]] for k in ("params", "grads", "m", "v")), rate, step, masters=[lists["masters"]] if "masters" in lists else None)
        got = logical(nx.softmax(nx.mul(x, scale))).astype(np.float64)
        now = float(logical(scale))
    finally:
        hip.set_deferred(False)
    # the step's results are those of the formula to float32's rounding: 0.5 - 0.25; 0.9 0.5 + 0.1; 0.999 0.5 + 0.001
    assert abs(now - {"params": 0.25, "m": 0.55, "v": 0.5005, "masters": 0.25}[written]) <= 2e-7
    s = logical(x).astype(np.float64) * now
    e = np.exp(s - s.max(1, keepdims=True))
    want = e / e.sum(1, keepdims=True)
    # products of a rounded scale, differences and powers, a sum of 70: (4 |s| + 80) half steps of a probability
    assert np.all(np.abs(got - want) <= 2.0 ** -24 * (4 * np.abs(s).max() + 80) * want)
    s = s / now * 0.5
    e = np.exp(s - s.max(1, keepdims=True))
    assert np.all(np.abs(before - e / e.sum(1, keepdims=True)) <= 2.0 ** -24 * (4 * np.abs(s).max() + 80))
