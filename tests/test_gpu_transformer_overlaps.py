"""Results of a transformer's training operators that begin where an operand of another dtype does."""

import numpy as np
import pytest

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
