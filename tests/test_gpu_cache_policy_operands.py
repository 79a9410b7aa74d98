"""What the memory-side cache policy learns from an entry point with many operands: each of them counts as read."""

import numpy as np
import pytest

from raven_amd import dtype as dt

pytestmark = pytest.mark.gpu

N = 4096  # queries and keys; a mask of 16 MiB, where 8 are followed


def tensor(hip, storage, d):
    return hip.reshape(hip.from_host(np.ascontiguousarray(storage), d), storage.shape)


def test_the_last_operand_of_a_gradient_is_read(hip):
    """A mask that is written again after each gradient that reads it. What reads it soon keeps it in the cache; if that read went
    unseen, a block written twice without a reader would be written past the cache."""
    like = lambda: tensor(hip, np.zeros((1, 1, N, 64), np.float16), dt.float16)  # noqa: E731
    q, g, dq, dk, dv = (like() for _ in range(5))
    mask, other = (tensor(hip, np.ones((1, 1, N, N), np.uint8), dt.bool_) for _ in range(2))
    lengths = tensor(hip, np.array([N - 5], np.int32), dt.int32)
    y, lse = hip.attention_train(q, q, q, 0.125, True, lengths, mask)
    wide = [tensor(hip, np.zeros((12, 1 << 20), np.float64), dt.float64) for _ in range(3)]  # 288 MiB: more than the cache holds
    hip.synchronize()
    hip.set_cache_policy(3)
    try:
        for turn in range(6):
            before = hip.cache_policy_stats()["streaming_out"]
            hip.assign(mask, other)
            after = hip.cache_policy_stats()["streaming_out"]
            assert after == before, turn
            hip.attention_grad(g, q, q, q, y, lse, 0.125, True, lengths, mask, out=(dq, dk, dv))
            for i in range(3):
                hip.assign(wide[i], wide[i - 1])
    finally:
        hip.set_cache_policy(3)


def test_a_block_without_a_reader_is_written_past_the_cache(hip):
    """The same without the gradient: what the test above would see of a read that goes unseen."""
    mask, other = (tensor(hip, np.ones((1, 1, N, N), np.uint8), dt.bool_) for _ in range(2))
    wide = [tensor(hip, np.zeros((12, 1 << 20), np.float64), dt.float64) for _ in range(3)]
    hip.synchronize()
    hip.set_cache_policy(3)
    past = 0
    for _ in range(6):
        before = hip.cache_policy_stats()["streaming_out"]
        hip.assign(mask, other)
        past += hip.cache_policy_stats()["streaming_out"] - before
        for i in range(3):
            hip.assign(wide[i], wide[i - 1])
    assert past >= 2
