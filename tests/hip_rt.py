"""Streams and graphs of the HIP runtime that the library is linked with."""
import contextlib
import ctypes as C

import numpy as np


def _rt(name):
    from yallma3_mini_inference_amd import lib
    fn = getattr(lib(), name)      # (looked up in the library's dependencies)
    fn.restype = C.c_int
    return fn


def _ok(status):
    assert status == 0, f"HIP error {status}"


class Stream:
    def __init__(self):
        h = C.c_void_p()
        _ok(_rt("hipStreamCreate")(C.byref(h)))
        self.handle = h.value

    def synchronize(self):
        _ok(_rt("hipStreamSynchronize")(C.c_void_p(self.handle)))

    def __del__(self):
        with contextlib.suppress(Exception):
            _rt("hipStreamDestroy")(C.c_void_p(self.handle))


class Graph:
    """What `enqueue(stream handle)` enqueues, captured on a stream of its own."""

    def __init__(self, enqueue):
        self.stream = Stream()
        s, graph, self.exec = C.c_void_p(self.stream.handle), C.c_void_p(), C.c_void_p()
        _ok(_rt("hipStreamBeginCapture")(s, 0))
        try:
            enqueue(self.stream.handle)
        finally:
            status = _rt("hipStreamEndCapture")(s, C.byref(graph))
        _ok(status)
        _ok(_rt("hipGraphInstantiate")(C.byref(self.exec), graph, None, None, C.c_size_t(0)))
        _ok(_rt("hipGraphDestroy")(graph))

    def replay(self):
        _ok(_rt("hipGraphLaunch")(self.exec, C.c_void_p(self.stream.handle)))
        self.stream.synchronize()

    def __del__(self):
        with contextlib.suppress(Exception):
            _rt("hipGraphExecDestroy")(self.exec)


def buffer(x):
    from yallma3_mini_inference_amd import DeviceBuffer
    return DeviceBuffer.from_numpy(np.ascontiguousarray(x))


def filled(shape, value, dtype=np.float32):
    return buffer(np.full(shape, value, dtype))


def bytes_of(n, value):
    """n bytes of one value (at least one)."""
    from yallma3_mini_inference_amd import DeviceBuffer, check, lib
    b = DeviceBuffer(max(1, n))
    check(lib().yl_memset_d(b.ptr, value, max(1, n)))
    return b
