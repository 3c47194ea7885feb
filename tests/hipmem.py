"""Device buffers and stream capture for the GPU tests, through the HIP
runtime that the library itself links (a second runtime in the process, such
as torch's bundled one, cannot initialise once this one has)."""
import ctypes

import numpy as np

_vp = ctypes.c_void_p


class Hip:
    def __init__(self):
        self.rt = ctypes.CDLL("libamdhip64.so.7")
        self.bufs = []
        self._ok("hipSetDevice", 0)

    def _ok(self, name, *args):
        rc = getattr(self.rt, name)(*args)
        assert rc == 0, (name, rc)

    def alloc(self, nbytes):
        p = _vp()
        self._ok("hipMalloc", ctypes.byref(p), ctypes.c_size_t(max(nbytes, 16)))
        self.bufs.append(p)
        return p.value

    def put(self, a, to=None):
        """`a` copied to device memory (a new buffer, or the address `to`)."""
        a = np.ascontiguousarray(a)
        p = self.alloc(a.nbytes) if to is None else to
        if a.nbytes:
            self._ok("hipMemcpy", _vp(p), a.ctypes.data_as(_vp), ctypes.c_size_t(a.nbytes), 1)
        return p

    def get(self, p, shape, dtype):
        out = np.zeros(shape, dtype)
        if out.nbytes:
            self._ok("hipMemcpy", out.ctypes.data_as(_vp), _vp(p), ctypes.c_size_t(out.nbytes), 2)
        return out

    def sync(self):
        self._ok("hipDeviceSynchronize")

    def capture(self, stream, work):
        """`work()` captured on `stream`; the instantiated graph."""
        graph, ex = _vp(), _vp()
        self._ok("hipStreamBeginCapture", _vp(stream), 0)
        try:
            work()
        finally:
            rc = self.rt.hipStreamEndCapture(_vp(stream), ctypes.byref(graph))
        assert rc == 0, ("hipStreamEndCapture", rc)
        self._ok("hipGraphInstantiate", ctypes.byref(ex), graph, None, None, ctypes.c_size_t(0))
        return ex

    def replay(self, ex, stream):
        self._ok("hipGraphLaunch", ex, _vp(stream))

    def free(self):
        for p in self.bufs:
            self.rt.hipFree(p)
        self.bufs = []

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        self.sync()
        self.free()
