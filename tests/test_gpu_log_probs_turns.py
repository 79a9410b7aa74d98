"""More rows than a launch has groups of lanes: groups go on to further rows, with the other half of the shared memory of their sums and
a list of candidates that has to be free again. A launch has at most 2^31 lanes, so that takes logits that are one small tensor, broadcast
over the rows: the k-th row of it comes again and again, and has to give the same bits in every turn."""

import numpy as np
import pytest

from helpers import encode, logical, same_bits
from raven_amd import dtype as dt

pytestmark = pytest.mark.gpu

KINDS = 5  # rows that differ
LANES = 1 << 31


def broadcast(hip, oracle, d, n, rows):
    """[rows / KINDS, KINDS, n] logits and their tokens, and the KINDS rows themselves."""
    rng = np.random.default_rng(n)
    x = rng.standard_normal((KINDS, n)) * 2
    x[1, n // 2], x[2], x[3, : n // 2] = 30.0, 1.5, -np.inf  # certain, equal, half banned
    x[4] -= 2.0 ** 21 if d is not dt.float16 else 0
    small = hip.reshape(hip.from_host(encode(x, d, oracle), d), (KINDS, n))
    tokens = hip.from_host(np.array([0, n // 2, n - 1, n - 1, 1 % n], np.int32), dt.int32)
    turns = rows // KINDS + 2
    wide = hip.expand(hip.reshape(small, (1, KINDS, n)), (turns, KINDS, n))
    return small, tokens, wide, hip.expand(hip.reshape(tokens, (1, KINDS)), (turns, KINDS)), turns


def repeats(hip, whole, want, turns, what):
    """Every turn of `whole` has the bits of the small call."""
    same_bits(logical(hip.copy(hip.shrink(whole, [(turns - 3, turns)] + [(0, m) for m in whole.shape[1:]]))), np.broadcast_to(want, (3, *want.shape)), f"{what}: the last")
    got = logical(whole)
    view = got.view(np.uint64 if got.itemsize == 8 else np.uint32)
    assert np.all(view == want.view(view.dtype)[None]), what


# (lanes of a row, lanes of a block, length): a group of eight, a wave, blocks of four and of eight waves
@pytest.mark.parametrize("d, group, block, n", [(dt.float16, 8, 256, 9), (dt.float32, 64, 256, 40), (dt.float32, 256, 256, 1030), (dt.bfloat16, 512, 512, 16400)],
                         ids=lambda v: v.name if hasattr(v, "name") else str(v))
def test_scores(hip, oracle, d, group, block, n):
    small, tokens, wide, wide_tokens, turns = broadcast(hip, oracle, d, n, LANES // group)
    assert turns * KINDS > LANES // block * (block // group)
    want = [logical(t) for t in hip.log_probs(small, tokens)[:2]]
    out = [hip.buffer(dt.float32, (turns, KINDS)), None, None, None, None, None]
    hip.log_probs(wide, wide_tokens, out=out)
    repeats(hip, out[0], want[0], turns, "log_p")
    if group > 64:
        out[:2] = None, out[0]
        hip.log_probs(wide, wide_tokens, out=out)
        repeats(hip, out[1], want[1], turns, "entropy")
    del out
    hip.trim()


@pytest.mark.parametrize("d, block, n, top", [(dt.float16, 64, 70, 3), (dt.float32, 64, 90, 1), (dt.float32, 256, 1030, 3), (dt.float64, 256, 700, 2),
                                              (dt.bfloat16, 512, 16400, 20)], ids=lambda v: v.name if hasattr(v, "name") else str(v))
def test_alternatives(hip, oracle, d, block, n, top):
    small, tokens, wide, wide_tokens, turns = broadcast(hip, oracle, d, n, LANES // block)
    assert turns * KINDS > LANES // block
    want = [logical(t) for t in hip.log_probs(small, tokens, top)[4:]]
    stats = dt.float64 if d is dt.float64 else dt.float32
    out = [None] * 4 + [hip.buffer(stats, (turns, KINDS, top)), hip.buffer(dt.int32, (turns, KINDS, top))]
    hip.log_probs(wide, wide_tokens, top, out=out)
    for t, w, what in zip(out[4:], want, ("top_log_p", "top_tokens")):
        repeats(hip, t, w, turns, what)
    del out
    hip.trim()


def test_statistics_and_gradients_of_rows_that_are_read_again(hip, oracle):
    """float64 rows that registers do not hold: a block of sixteen waves each."""
    d, n = dt.float64, 515
    small, tokens, wide, wide_tokens, turns = broadcast(hip, oracle, d, n, LANES // 1024)
    hg = hip.full(d, (1,), -1.0)
    want = [logical(t) for t in hip.log_probs_with_grad(hip.expand(hg, (KINDS,)), small, tokens)]
    out = hip.buffer(d, (turns, KINDS)), hip.buffer(d, (turns, KINDS)), hip.buffer(d, (turns, KINDS, n))
    hip.log_probs_with_grad(hip.expand(hip.reshape(hg, (1, 1)), (turns, KINDS)), wide, wide_tokens, out=out)
    for t, w, what in zip(out, want, ("log_p", "entropy")):
        repeats(hip, t, w, turns, what)
    for at in (0, turns // 2, turns - 4):
        got = logical(hip.copy(hip.shrink(out[2], [(at, at + 4), (0, KINDS), (0, n)])))
        same_bits(got, np.broadcast_to(want[2], got.shape), f"gradients from turn {at} on")
    del out
    hip.trim()
