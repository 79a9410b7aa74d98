"""The formulas that attention's gradient is tested against, against differences of the forward formula."""

import numpy as np
import pytest

import attention_oracle as ao


@pytest.mark.parametrize("causal, lengths, masked", [(False, None, False), (True, None, False), (False, [3, 5], False), (True, [4, 0], True)])
def test_gradient_is_the_forwards_slope(causal, lengths, masked):
    rng = np.random.default_rng(5)
    b, h, hk, sq, sk, d, scale = 2, 4, 2, 4, 5, 6, 0.37
    q, g = rng.standard_normal((2, b, h, sq, d))
    k, v = rng.standard_normal((2, b, hk, sk, d))
    mask = rng.random((b, h, sq, sk)) < 0.6 if masked else None
    keep = ao.seen(b, h, sq, sk, causal, lengths, mask)
    (out, lse), _ = ao.forward(q, k, v, scale, keep)
    grads, _ = ao.backward(g, q, k, v, out, lse, scale, keep)
    step = 1e-5
    for name, x, dx in zip("qkv", (q, k, v), grads):
        for _ in range(12):
            at = tuple(rng.integers(0, n) for n in x.shape)
            old, side = x[at], []
            for delta in (step, -step):
                x[at] = old + delta
                side.append((ao.forward(q, k, v, scale, keep)[0][0] * g).sum())
            x[at] = old
            # the difference's own error: step^2 times a third derivative of some tens, and 1e-16 of sums of some ten over the step
            assert abs((side[0] - side[1]) / (2 * step) - dx[at]) <= 1e-8, (name, at)


def test_a_row_without_keys_is_zero():
    keep = ao.seen(1, 1, 3, 2, causal=True)  # the first query lies before all keys
    assert not keep[0, 0, 0].any()
    x = np.random.default_rng(6).standard_normal((3, 1, 1, 3, 4))
    (out, lse), _ = ao.forward(x[0], x[1][:, :, :2], x[2][:, :, :2], 1.0, keep)
    assert np.all(out[0, 0, 0] == 0) and lse[0, 0, 0] == -np.inf
    (dq, dk, dv), _ = ao.backward(x[1], x[0], x[1][:, :, :2], x[2][:, :, :2], out, lse, 1.0, keep)
    assert np.all(dq[0, 0, 0] == 0) and np.isfinite(dk).all() and np.isfinite(dv).all()
