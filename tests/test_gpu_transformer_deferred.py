"""The transformer block's steps of test_gpu_transformer_step.py in deferred mode beside the same steps call by call: their losses' elements and
gradients, and the weights where the gradients say which way they go.

Both are float32's results of one formula, each off by at most 1e-3 of a gradient's root mean square (derived there), so they are 2e-3 apart at
most; weights after three steps, where all gradients are above 1e-2 of it, by 2 x 0.3 rates."""

import numpy as np
import pytest

from helpers import logical
from raven_amd import dtype as dt
from test_gpu_transformer_step import NAMES, RATE, SHAPES, Block, problem, tensor

pytestmark = pytest.mark.gpu


def steps_of(hip, seed):
    """What each step leaves: the loss's elements, gradients; and the weights at the end."""
    weights, batches, f, lengths = problem(seed)
    block, made = Block(hip, weights, f, lengths), []
    for step, (x, positions, target) in enumerate(batches, 1):
        hip.assign(block.step, tensor(hip, np.array([step], np.int32), dt.int32))
        off, grads = block.train(tensor(hip, x), tensor(hip, positions, dt.int32), tensor(hip, target))
        made.append((logical(off).copy(), {n: logical(grads[n]).copy() for n in NAMES}))
    return made, {n: logical(block.w[n]).copy() for n in NAMES}


def size(x):
    return np.sqrt((x.astype(np.float64) ** 2).mean())


@pytest.mark.parametrize("seed", [3, 6])
def test_gradients_and_weights(hip, seed):
    want, weights = steps_of(hip, seed)
    hip.set_deferred(True)
    try:
        got, deferred = steps_of(hip, seed)
    finally:
        hip.set_deferred(False)
    off, grads = want[0]
    assert np.max(np.abs(got[0][0] - off)) <= 2e-3 * size(off)
    for n in NAMES:
        assert np.max(np.abs(got[0][1][n] - grads[n])) <= 2e-3 * size(grads[n]), n
        sure = np.ones(SHAPES[n], bool)
        for _, g in want:
            sure &= np.abs(g[n]) > 1e-2 * size(g[n])
        apart = np.abs(deferred[n] - weights[n])
        assert sure.mean() > 0.9 and np.max(apart[sure]) <= 2 * 0.3 * RATE, n


def test_gradients_tell_steps_apart(hip):
    """What the bounds above are worth: another batch's gradients are as far off as they are large."""
    a, b = (steps_of(hip, s)[0][0][1] for s in (3, 6))
    for n in NAMES:
        assert np.max(np.abs(a[n] - b[n])) > size(a[n])
