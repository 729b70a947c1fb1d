"""Device memory, streams and graphs of the HIP runtime that libdraco_hip.so
links (/opt/rocm libamdhip64, through ctypes), for tests of its device-pointer
entry points: torch bundles a HIP runtime of its own, and two runtimes in one
process are not relied on."""
import ctypes as ct
import os

import numpy as np


class Hip:
    def __init__(self):
        self.rt = ct.CDLL(os.path.join(os.environ.get("ROCM_PATH", "/opt/rocm"), "lib", "libamdhip64.so"))
        v, s = ct.c_void_p, ct.c_size_t
        for name, args in {
            "hipMalloc": [ct.POINTER(v), s], "hipFree": [v], "hipMemcpy": [v, v, s, ct.c_int],
            "hipMemcpyAsync": [v, v, s, ct.c_int, v], "hipDeviceSynchronize": [],
            "hipStreamCreateWithFlags": [ct.POINTER(v), ct.c_uint], "hipStreamDestroy": [v], "hipStreamSynchronize": [v],
            "hipStreamBeginCapture": [v, ct.c_int], "hipStreamEndCapture": [v, ct.POINTER(v)],
            "hipGraphInstantiate": [ct.POINTER(v), v, v, v, s], "hipGraphLaunch": [v, v], "hipGraphExecDestroy": [v],
            "hipGraphDestroy": [v],
        }.items():
            getattr(self.rt, name).argtypes = args
        self.live, self.streams, self.graphs = [], [], []

    def ok(self, name, *args):
        rc = getattr(self.rt, name)(*args)
        assert rc == 0, f"{name} rc={rc}"

    def empty(self, nbytes):
        p = ct.c_void_p()
        self.ok("hipMalloc", ct.byref(p), max(int(nbytes), 16))
        self.live.append(p.value)
        return p.value

    def up(self, a, at=None):
        a = np.ascontiguousarray(a)
        p = at or self.empty(a.nbytes)
        if a.nbytes:
            self.ok("hipMemcpy", p, a.ctypes.data, a.nbytes, 1)
        return p

    def down(self, p, shape, dtype):
        a = np.empty(shape, dtype)
        self.ok("hipDeviceSynchronize")
        if a.nbytes:
            self.ok("hipMemcpy", a.ctypes.data, p, a.nbytes, 2)
        return a

    def stream(self):
        p = ct.c_void_p()
        self.ok("hipStreamCreateWithFlags", ct.byref(p), 1)  # non-blocking
        self.streams.append(p.value)
        return p.value

    def sync(self, stream):
        self.ok("hipStreamSynchronize", stream)

    def capture(self, stream, fn):
        """fn's work on `stream` as an instantiated graph."""
        g, e = ct.c_void_p(), ct.c_void_p()
        self.ok("hipStreamBeginCapture", stream, 2)  # relaxed
        fn()
        self.ok("hipStreamEndCapture", stream, ct.byref(g))
        self.ok("hipGraphInstantiate", ct.byref(e), g, None, None, 0)
        self.graphs.append((g.value, e.value))
        return e.value

    def replay(self, graph, stream):
        self.ok("hipGraphLaunch", graph, stream)

    def free(self):
        self.rt.hipDeviceSynchronize()
        for g, e in self.graphs:
            self.rt.hipGraphExecDestroy(e)
            self.rt.hipGraphDestroy(g)
        for s in self.streams:
            self.rt.hipStreamDestroy(s)
        for p in self.live:
            self.rt.hipFree(p)
        self.live, self.streams, self.graphs = [], [], []
