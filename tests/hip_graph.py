"""HIP streams and graphs for tests, through the HIP runtime that the library
itself is linked to."""
from __future__ import annotations

import ctypes as C

from midge_amd import _lib

_hip = None


def hip_call(name, *args):
    global _hip
    if _hip is None:
        _lib.load()
        with open("/proc/self/maps") as f:      # the runtime that is loaded, by its own path
            path = next(line.split()[-1] for line in f if "libamdhip64" in line)
        _hip = C.CDLL(path)
    rc = getattr(_hip, name)(*args)
    assert rc == 0, (name, rc)


class Stream:
    def __init__(self):
        self.h = C.c_void_p()
        hip_call("hipStreamCreateWithFlags", C.byref(self.h), 1)       # non-blocking

    def sync(self):
        hip_call("hipStreamSynchronize", self.h)

    def __enter__(self):
        _lib.call("mh_set_stream", self.h)
        return self

    def __exit__(self, *exc):
        _lib.call("mh_set_stream", None)
        return False

    def free(self):
        hip_call("hipStreamDestroy", self.h)


class Graph:
    """What fn() launches on the library's stream, captured on `stream`."""

    def __init__(self, stream: Stream, fn):
        g = C.c_void_p()
        with stream:
            hip_call("hipStreamBeginCapture", stream.h, 0)             # global: nothing in the process may allocate
            try:
                fn()
            finally:
                hip_call("hipStreamEndCapture", stream.h, C.byref(g))
        self.h = C.c_void_p()
        hip_call("hipGraphInstantiate", C.byref(self.h), g, None, None, C.c_size_t(0))
        hip_call("hipGraphDestroy", g)

    def launch(self, stream: Stream):
        hip_call("hipGraphLaunch", self.h, stream.h)

    def free(self):
        hip_call("hipGraphExecDestroy", self.h)
