"""Calls of the 8-bit products and the experts that meet a capture they cannot join: HIP's
own error, not one of memory."""
import ctypes as C

import numpy as np
import pytest

import fp8_ref as ref
from test_gpu_experts import build, random_experts
from test_gpu_fp8 import host16, run

pytestmark = pytest.mark.gpu

EHIP = -3
GLOBAL, RELAXED = 0, 2  # capture modes


@pytest.fixture(scope="module")
def hip(smg):
    import torch
    torch.cuda.init()
    path = next(line.split()[-1] for line in open("/proc/self/maps") if "libamdhip64" in line)
    L = C.CDLL(path)
    for name, args in (("hipStreamCreate", [C.POINTER(C.c_void_p)]), ("hipStreamDestroy", [C.c_void_p]),
                       ("hipStreamBeginCapture", [C.c_void_p, C.c_int]),
                       ("hipStreamEndCapture", [C.c_void_p, C.POINTER(C.c_void_p)]), ("hipGraphDestroy", [C.c_void_p]),
                       ("hipMalloc", [C.POINTER(C.c_void_p), C.c_size_t]), ("hipFree", [C.c_void_p])):
        getattr(L, name).argtypes = args
    return L


class Capture:
    """A capture on a new blocking stream."""

    def __init__(self, hip, mode):
        self.hip, self.mode, self.stream, self.graph = hip, mode, C.c_void_p(), C.c_void_p()

    def __enter__(self):
        assert self.hip.hipStreamCreate(C.byref(self.stream)) == 0
        assert self.hip.hipStreamBeginCapture(self.stream, self.mode) == 0
        return self.stream

    def __exit__(self, *_):
        self.hip.hipStreamEndCapture(self.stream, C.byref(self.graph))
        if self.graph.value:
            self.hip.hipGraphDestroy(self.graph)
        self.hip.hipGetLastError()
        self.hip.hipStreamDestroy(self.stream)


@pytest.mark.parametrize("case", ["null stream", "invalidated"])
def test_hip_errors_keep_their_own_code(smg, hip, case):
    import torch
    rng = np.random.default_rng(2)
    n, k, m = 256, 256, 300
    w = smg.Fp8Weights(*ref.random_weights(rng, n, k), n, k)
    e = build(smg, random_experts(rng, 2, 64, 64), 2, 64, 64)
    a = torch.randn(m, k, device="cuda").half()
    x = torch.randn(m, 64, device="cuda").half()
    ids, wt = torch.zeros(m, 2, dtype=torch.int32, device="cuda"), torch.ones(m, 2, device="cuda")
    c = torch.full((m, n), 7.0, device="cuda").half()
    out = torch.full((m, 64), 7.0, device="cuda").half()
    torch.cuda.synchronize()
    L = smg.lib()
    with Capture(hip, RELAXED if case == "null stream" else GLOBAL) as s:
        if case == "invalidated":
            p = C.c_void_p()
            assert hip.hipMalloc(C.byref(p), 4096) != 0  # (not allowed while a global capture goes on)
        at = None if case == "null stream" else s
        got = []
        for rc in (lambda: L.smg_fp8_matmul_dev(m, w._h, c.data_ptr(), a.data_ptr(), None, 0, at),
                   lambda: L.smg_experts_forward_dev(e._h, x.data_ptr(), 0, ids.data_ptr(), wt.data_ptr(), m, 2, out.data_ptr(),
                                                     at)):
            got.append((rc(), smg.last_error()))
    assert all(rc == EHIP and "scratch" not in text for rc, text in got), got
    torch.cuda.synchronize()
    assert bool((c == 7).all()) and bool((out == 7).all())
    assert np.isfinite(host16(c).view(np.float16)).all() and run(smg, a, w, m, False).any()
