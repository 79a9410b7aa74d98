"""Training steps of one transformer block by the backend's calls: projections, rotary positions, attention, loss, their gradients, and AdamW;
against the same steps in float64 with automatic differentiation.

How far weights may be off, derived before the first run. With every tensor float32, u = 2^-24, the longest chain from a weight to its
gradient has seven matrix products, the deepest over n = 96 terms, and a softmax: each is off by at most 4 n u relative to the sum of its
terms' sizes, and a gradient here is a sum of 2 x 48 x 2 such terms whose sizes add up to less than 200 times the gradients' own root mean
square: 7 x 4 x 96 x 200 u = 0.03 of that, at the very worst; rounding errors have random signs, so their square root counts, 1e-3 of it.
AdamW's first step divides a gradient by its own size (m / sqrt v = sign): its elements below 1e-2 of the root mean square may move by anything
up to the rate, those above by 1e-3 / 1e-2 of it, a tenth. So weights are compared after three steps where all three gradients are above
that: within 3 x 0.1 rates; and no weight is off by more than 6 rates."""

import threading

import numpy as np
import pytest
import torch

from helpers import logical, same_bits
from raven_amd import dtype as dt
from raven_amd.nx_backend import Backend

pytestmark = pytest.mark.gpu

B, S, H, HK, D, N = 2, 48, 4, 2, 16, 64  # batch, tokens, heads, shared heads, their size, features
RATE, DECAY = 1e-2, 0.1
NAMES = ("wq", "wk", "wv", "wo")
SHAPES = {"wq": (N, H * D), "wk": (N, HK * D), "wv": (N, HK * D), "wo": (H * D, N)}


def tensor(hip, x, d=dt.float32):
    return hip.reshape(hip.from_host(np.ascontiguousarray(x), d), np.shape(x))


class Block:
    def __init__(self, hip, weights, frequencies, lengths):
        self.hip = hip
        self.w = {n: tensor(hip, w) for n, w in weights.items()}
        self.m, self.v = ([tensor(hip, np.zeros(SHAPES[n], np.float32)) for n in NAMES] for _ in range(2))
        self.f, self.lengths = tensor(hip, frequencies, dt.float64), tensor(hip, lengths, dt.int32)
        self.rate, self.step = tensor(hip, np.array([RATE], np.float32)), tensor(hip, np.array([1], np.int32), dt.int32)

    def split(self, x, heads):
        return self.hip.permute(self.hip.reshape(x, (B, S, heads, D)), (0, 2, 1, 3))

    def merge(self, x):
        """Back to rows of all heads."""
        return self.hip.reshape(self.hip.contiguous(self.hip.permute(x, (0, 2, 1, 3))), (B * S, x.shape[1] * D))

    def train(self, x, positions, target):
        """One step; the loss's elements and the weights' gradients."""
        hip, w, scale = self.hip, self.w, D ** -0.5
        t = lambda y: hip.permute(y, (1, 0))  # noqa: E731
        q, k, v = (self.split(hip.matmul(x, w[n]), h) for n, h in (("wq", H), ("wk", HK), ("wv", HK)))
        qr, kr = hip.rotary(q, k, positions, self.f)
        y, lse = hip.attention_train(qr, kr, v, scale, True, self.lengths)
        rows = self.merge(y)
        off = hip.binary("sub", hip.matmul(rows, w["wo"]), target)  # loss: half the sum of its squares
        grads = {"wo": hip.matmul(t(rows), off)}
        dy = self.split(hip.matmul(off, t(w["wo"])), H)
        dqr, dkr, dv = hip.attention_grad(dy, qr, kr, v, y, lse, scale, True, self.lengths)
        dq, dk = hip.rotary(dqr, dkr, positions, self.f, inverse=True)
        for n, d in (("wq", dq), ("wk", dk), ("wv", dv)):
            grads[n] = hip.matmul(t(x), self.merge(d))
        hip.adamw([w[n] for n in NAMES], [grads[n] for n in NAMES], self.m, self.v, self.rate, self.step, decay=DECAY)
        return off, grads


def plain(weights, x, positions, target, frequencies, lengths):
    """The gradients in float64."""
    w = {n: torch.tensor(a, dtype=torch.float64, requires_grad=True) for n, a in weights.items()}
    x, target = torch.tensor(x, dtype=torch.float64), torch.tensor(target, dtype=torch.float64)
    turn = torch.tensor(positions, dtype=torch.float64)[:, None, :, None] * torch.tensor(frequencies)

    def split(y, heads):
        return y.reshape(B, S, heads, D).transpose(1, 2)

    def turned(y):
        a, b = y[..., :D // 2], y[..., D // 2:]
        return torch.cat((a * turn.cos() - b * turn.sin(), a * turn.sin() + b * turn.cos()), 3)

    q, k, v = (split(x @ w[n], h) for n, h in (("wq", H), ("wk", HK), ("wv", HK)))
    q, k, v = turned(q), turned(k).repeat_interleave(H // HK, 1), v.repeat_interleave(H // HK, 1)
    j = torch.arange(S)
    seen = (j[None, :] <= j[:, None])[None, None] & (j[None, :] < torch.tensor(lengths)[:, None])[:, None, None, :]
    p = torch.softmax((q @ k.transpose(2, 3) * D ** -0.5).masked_fill(~seen, -np.inf), 3)
    off = (p @ v).transpose(1, 2).reshape(B * S, H * D) @ w["wo"] - target
    (off * off).sum().div(2).backward()
    return {n: a.grad.numpy() for n, a in w.items()}


def problem(seed):
    rng = np.random.default_rng(seed)
    weights = {n: (rng.standard_normal(s) / np.sqrt(s[0])).astype(np.float32) for n, s in SHAPES.items()}
    batches = [(rng.standard_normal((B * S, N)).astype(np.float32), (rng.integers(0, 100000, (B, 1)) + np.arange(S)).astype(np.int32),
                rng.standard_normal((B * S, N)).astype(np.float32)) for _ in range(3)]
    return weights, batches, Backend.rotary_frequencies(D // 2), np.array([S, S - 19], np.int32)


def test_three_steps(hip):
    weights, batches, f, lengths = problem(1)
    block = Block(hip, weights, f, lengths)
    w = {n: a.astype(np.float64) for n, a in weights.items()}
    m, v = ({n: np.zeros(s) for n, s in SHAPES.items()} for _ in range(2))
    sure = {n: np.ones(s, bool) for n, s in SHAPES.items()}
    for step, (x, positions, target) in enumerate(batches, 1):
        hip.assign(block.step, tensor(hip, np.array([step], np.int32), dt.int32))
        _, grads = block.train(tensor(hip, x), tensor(hip, positions, dt.int32), tensor(hip, target))
        for n, g in plain(w, x, positions, target, f, lengths).items():
            size = np.sqrt((g * g).mean())
            if step == 1:  # (later ones are of weights that are off by now)
                assert np.max(np.abs(logical(grads[n]) - g)) <= 1e-3 * size, n
            sure[n] &= np.abs(g) > 1e-2 * size
            m[n], v[n] = 0.9 * m[n] + 0.1 * g, 0.999 * v[n] + 0.001 * g * g
            w[n] = w[n] * (1 - RATE * DECAY) - RATE * (m[n] / (1 - 0.9 ** step)) / (np.sqrt(v[n] / (1 - 0.999 ** step)) + 1e-8)
    for n in NAMES:
        off = np.abs(logical(block.w[n]) - w[n])
        assert sure[n].mean() > 0.9 and np.max(off[sure[n]]) <= 0.3 * RATE and np.max(off) <= 6 * RATE, n


def test_recorded_step(hip):
    """A step as a graph, replayed over batches that change, beside the same steps made call by call."""
    weights, batches, f, lengths = problem(2)
    eager, recorded = Block(hip, weights, f, lengths), Block(hip, weights, f, lengths)
    x, positions, target = (tensor(hip, a, a.dtype.type is np.int32 and dt.int32 or dt.float32) for a in batches[0])
    warm = Block(hip, weights, f, lengths)
    warm.train(x, positions, target)
    hip.synchronize()
    hip.capture_begin()
    off, grads = recorded.train(x, positions, target)
    graph = hip.capture_end()
    for step, batch in enumerate(batches, 1):
        for t, a in zip((x, positions, target), batch):
            hip.assign(t, tensor(hip, a, t.dtype))
        for block in (eager, recorded):
            hip.assign(block.step, tensor(hip, np.array([step], np.int32), dt.int32))
        graph.launch()
        off_e, grads_e = eager.train(x, positions, target)
        hip.synchronize()
        same_bits(logical(off), logical(off_e))
        for n in NAMES:
            same_bits(logical(grads[n]), logical(grads_e[n]), n)
            same_bits(logical(recorded.w[n]).copy(), logical(eager.w[n]).copy(), n)
    graph.destroy()


def steps_of(hip, seed):
    """The weights after a problem's steps."""
    weights, batches, f, lengths = problem(seed)
    block = Block(hip, weights, f, lengths)
    for step, (x, positions, target) in enumerate(batches, 1):
        hip.assign(block.step, tensor(hip, np.array([step], np.int32), dt.int32))
        block.train(tensor(hip, x), tensor(hip, positions, dt.int32), tensor(hip, target))
    return {n: logical(block.w[n]).copy() for n in NAMES}


def test_deferred_steps(hip):
    want = steps_of(hip, 3)
    hip.set_deferred(True)
    try:
        got = steps_of(hip, 3)
    finally:
        hip.set_deferred(False)
    for n in NAMES:
        np.testing.assert_allclose(got[n], want[n], rtol=0, atol=2 * 3 * RATE)  # (fused sums may turn a sign: two rates a step)


def test_steps_of_two_threads(hip):
    """On one context, and on two of the one GPU: the bits that the steps alone get."""
    want = [steps_of(hip, s) for s in (4, 5)]
    other = Backend()
    try:
        for contexts in ((hip, hip), (hip, other)):
            errors = []

            def body(i, contexts=contexts, errors=errors):
                try:
                    for _ in range(4):
                        got = steps_of(contexts[i], i + 4)
                        for n in NAMES:
                            same_bits(got[n], want[i][n], f"{n} of thread {i}")
                except BaseException as exc:  # noqa: BLE001 - reported below
                    errors.append((i, repr(exc)))

            threads = [threading.Thread(target=body, args=(i,)) for i in range(2)]
            for t in threads:
                t.start()
            for t in threads:
                t.join()
            assert not errors, errors
    finally:
        other.close()
