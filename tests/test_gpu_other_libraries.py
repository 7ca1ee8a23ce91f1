"""Arrays that pass between this library and other users of the device, which work in streams of their own: who waits for
whom, and how long memory stays.  The other user here calls the HIP runtime directly."""
import ctypes
import gc
import weakref

import numpy as np
import pytest

import theano_amd as th
from theano_amd import hip, tensor as T
from theano_amd.compile import Out
from theano_amd.hip.runtime import HipArray
from theano_amd.tensor import inplace

pytestmark = pytest.mark.gpu

N = 1 << 16
TO_DEVICE, TO_HOST, ON_DEVICE = 1, 2, 3


class Runtime(object):
    """The HIP runtime that the library itself has loaded."""

    def __init__(self):
        self.lib = ctypes.CDLL("libamdhip64.so.7")
        self.held = []
        self.big = [self.malloc(1 << 30) for _ in range(2)]

    def call(self, name, *args):
        assert getattr(self.lib, name)(*args) == 0, name

    def malloc(self, nbytes):
        p = ctypes.c_void_p()
        self.call("hipMalloc", ctypes.byref(p), ctypes.c_size_t(nbytes))
        self.held.append(p)
        return p.value

    def stream(self):
        s = ctypes.c_void_p()
        self.call("hipStreamCreateWithFlags", ctypes.byref(s), 1)     # waits for no other stream
        return s.value

    def sync(self):
        self.call("hipDeviceSynchronize")

    def copy(self, to, source, nbytes, kind, stream):
        self.call("hipMemcpyAsync", ctypes.c_void_p(to), ctypes.c_void_p(source), ctypes.c_size_t(nbytes), kind, ctypes.c_void_p(stream))

    def busy(self, stream):
        """Some 50 ms of work: 100 copies of 1 GiB."""
        for _ in range(100):
            self.copy(self.big[0], self.big[1], 1 << 30, ON_DEVICE, stream)

    def fill(self, array, value, stream):
        bits = int(np.float32(value).view("int32"))
        self.call("hipMemsetD32Async", ctypes.c_void_p(array.ptr), bits, ctypes.c_size_t(array.n), ctypes.c_void_p(stream))

    def read(self, array):
        out = np.empty(array.n, "float32")
        self.sync()
        self.copy(out.ctypes.data, array.ptr, out.nbytes, TO_HOST, 0)
        self.sync()
        return out


@pytest.fixture(scope="module")
def rt():
    hip.sync()
    r = Runtime()
    yield r
    hip.sync()
    r.sync()
    for p in r.held:
        r.call("hipFree", p)


class Array(object):
    """``n`` floats, as another library shows them; ``stream`` None: without the entry that names the stream."""

    def __init__(self, rt, n=N, stream=None, value=0.0, read_only=False, ptr=None):
        self.n, self.ptr = n, rt.malloc(4 * n) if ptr is None else ptr
        if ptr is None:
            rt.fill(self, value, 0)
            rt.sync()
        self.__cuda_array_interface__ = {"shape": (n,), "typestr": "<f4", "data": (self.ptr, read_only), "version": 3}
        if stream is not None:
            self.__cuda_array_interface__["stream"] = stream


@pytest.fixture(scope="module")
def plus_one():
    x = T.fvector()
    f = th.function([x], Out(x + 1, device=True))
    f(HipArray.from_numpy(np.zeros(N, "float32")))            # compiled and loaded
    hip.sync()
    return f


@pytest.mark.parametrize("default", [False, True])
def test_the_stream_that_an_array_names_is_waited_for(rt, plus_one, default):
    s = 0 if default else rt.stream()
    x = Array(rt, stream=1 if default else s)
    rt.busy(s)
    rt.fill(x, 7, s)
    assert (plus_one(HipArray.from_cuda_array_interface(x)).to_numpy() == 8).all()


def test_streams_ordered_by_the_caller(rt, plus_one):
    """For arrays that name no stream: arguments, results, and the memory of results that are let go."""
    s = rt.stream()
    x, z, late = [Array(rt) for _ in range(3)]
    rt.busy(s)
    rt.fill(x, 7, s)
    hip.wait_for_stream(s)
    rt.busy(hip.stream())
    y = plus_one(HipArray.from_cuda_array_interface(x))
    hip.let_stream_wait(s)
    rt.copy(z.ptr, y.ptr, 4 * N, ON_DEVICE, s)
    rt.busy(s)
    rt.copy(late.ptr, y.ptr, 4 * N, ON_DEVICE, s)
    at = y.ptr
    del y
    hip.wait_for_stream(s)
    zeros = [HipArray.from_numpy(np.zeros(N, "float32")) for _ in range(4)]
    assert at in [a.ptr for a in zeros + [plus_one(a) for a in zeros]]      # used again, behind what read it
    assert (rt.read(z) == 8).all() and (rt.read(late) == 8).all()
    hip.wait_for_stream(hip.stream())                         # nothing to wait for


def test_memory_stays_until_queued_work_has_ended(rt, plus_one):
    hip.sync()
    for n in (100, 300 << 20):                                # one of many that share a mark, and one with its own
        owner = Array(rt, n)
        there = weakref.ref(owner)
        rt.busy(hip.stream())
        plus_one(HipArray.from_cuda_array_interface(owner))
        del owner
        gc.collect()
        assert there() is not None
        hip.sync()
        assert there() is None
    refs = []
    for _ in range(200):
        owner = Array(rt, 10)
        refs.append(weakref.ref(owner))
        plus_one(HipArray.from_cuda_array_interface(owner))
        rt.sync()
    del owner
    assert sum(r() is not None for r in refs) <= 130          # let go on the way
    hip.sync()
    assert not any(r() is not None for r in refs)


def test_recordings_and_other_libraries_arrays(rt, plus_one):
    """A recording keeps what it reads, and takes no array that has to be waited for."""
    owner = Array(rt, 1000)
    mine = Array(rt, 1000, ptr=owner.ptr)                     # the same memory
    there = weakref.ref(owner)
    plus_one(HipArray.from_cuda_array_interface(owner))
    with hip.capture() as c:
        r = plus_one(HipArray.from_cuda_array_interface(owner))
    del owner
    hip.sync()
    gc.collect()
    assert there() is not None
    for k in range(3):
        rt.fill(mine, k, 0)
        rt.sync()
        c.graph.launch()
        assert (r.to_numpy() == k + 1).all()
    del c
    gc.collect()
    hip.sync()
    assert there() is None
    with pytest.raises(ValueError, match="recording"):
        with hip.capture():
            HipArray.from_cuda_array_interface(Array(rt, 1000, stream=rt.stream(), ptr=mine.ptr))
    with hip.capture() as c:                                  # the library's own stream needs no order
        r = plus_one(HipArray.from_cuda_array_interface(Array(rt, 1000, stream=hip.stream(), ptr=mine.ptr)))
    c.graph.launch()
    assert (r.to_numpy() == 3).all()


def test_arrays_that_a_function_overwrites(rt):
    x, y = T.fvector(), T.fvector()
    f = th.function([x, y], inplace.add_inplace(x, y), accept_inplace=True)
    t = Array(rt, 10)
    u, fixed = Array(rt, 10, value=1, read_only=True), Array(rt, 10, ptr=t.ptr, read_only=True)
    with pytest.raises(ValueError, match="read-only"):
        f(HipArray.from_cuda_array_interface(fixed), HipArray.from_cuda_array_interface(u))
    f(HipArray.from_cuda_array_interface(t), HipArray.from_cuda_array_interface(u))
    hip.sync()
    assert (rt.read(t) == 1).all() and (rt.read(u) == 1).all()
