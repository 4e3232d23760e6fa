"""Refusals of 8-bit weights whose products would need launches of 2^32 threads. No GPU."""
import ctypes as C

import numpy as np


def test_too_many_columns_are_refused():
    import smegemm
    L = smegemm.lib()
    c, s, h = np.zeros(16, np.uint8), np.zeros(1, np.float32), C.c_void_p()
    for n in (1 << 27, 1 << 29, (1 << 30) - 1):
        assert L.smg_fp8_create(c.ctypes.data, s.ctypes.data, n, 1, C.byref(h)) == -1
        assert L.smg_fp8_create_dev(c.ctypes.data, s.ctypes.data, n, 1, None, C.byref(h)) == -1
    assert not h.value
