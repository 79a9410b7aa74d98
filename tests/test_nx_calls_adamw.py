"""The optimiser's step of the host path in C (raven_amd/host_c/nx_calls.c) between its descriptors and its return, with a stand-in for the
library, whose entry points the module holds for the whole process."""

import pytest

from test_nx_calls_handles import in_a_process

CALL = """
import ctypes as C, gc, weakref
from raven_amd import _ffi, dtype as dt
from raven_amd.nx_backend import View
from raven_amd._nxcalls import Calls, DeviceBuffer, Tensor, bind
places = iter(range(4096, 1 << 20, 4096))
def alloc(ctx, n, p):
    C.cast(p, C.POINTER(C.c_void_p))[0] = next(places)
    return 0
def free(ctx, p):
    freed.append(p)
    return 0
def adamw(*a):
    during(a)
    return 0
freed, seen = [], []
alloc = C.CFUNCTYPE(C.c_int, C.c_void_p, C.c_size_t, C.c_void_p)(alloc)
free = C.CFUNCTYPE(C.c_int, C.c_void_p, C.c_void_p)(free)
adamw = C.CFUNCTYPE(C.c_int, C.c_void_p, C.c_int, *[C.POINTER(C.c_void_p)] * 7, *[C.c_void_p] * 4, *[C.c_double] * 4)(adamw)
bind({name: C.cast({"nxh_free": free, "nxh_adamw": adamw}.get(name, alloc), C.c_void_p).value for name in _ffi.SIGNATURES})
class Context(Calls):
    pass
c = Context()
c._h = 77
def tensor():
    return Tensor(DeviceBuffer(c, 64), View.create((16,)), dt.float32, c)
one = tensor()
"""


@pytest.mark.parametrize("change", ["l.clear()", "l[:] = [tensor(), tensor()]", "l.pop()"])
def test_a_step_holds_its_tensors(change):
    """Entries that another thread takes out of the lists while the library has the call: their storage is still the step's. (The
    library's stand-in runs where such a thread would, with the interpreter's lock let go.)"""
    out = in_a_process(CALL + f"""
lists = [[tensor(), tensor()] for _ in range(7)]
def during(a):
    for l in lists:
        {change}
    gc.collect()
    seen.append(len(freed))
c.adamw(*lists[:4], one, one, masters=lists[4], m_scales=lists[5], v_scales=lists[6], key=one)
gc.collect()
print(seen, len(freed) > 0)
""")
    assert out == ["[0]", "True"]


def test_what_a_step_gets():
    """Lists, tuples and iterators; those left out are null."""
    out = in_a_process(CALL + """
p, g, m, v = ([tensor(), tensor(), tensor()] for _ in range(4))
def during(a):  # (a descriptor begins with its data's address)
    data = lambda x: C.cast(x, C.POINTER(C.c_void_p))[0]
    seen.append([a[1]] + [[data(l[i]) for i in range(a[1])] if l else None for l in a[2:9]] + [data(x) if x else None for x in a[9:13]])
c.adamw(p, tuple(g), iter(m), v, one, one)
at = one.buffer.ptr
print(seen[0] == [3] + [[t.buffer.ptr for t in l] for l in (p, g, m, v)] + [None] * 3 + [at, at, None, None])
c.adamw([], [], (), iter([]), one, one)
print(seen[1][0])
try:
    c.adamw(p, g, m, v[:2], one, one)
except ValueError as e:
    print("lengths" in str(e), len(seen))
""")
    assert out == ["True", "0", "True", "2"]
