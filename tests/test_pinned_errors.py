"""Calls on page-locked memory that the runtime refuses leave no HIP error behind: the runtime keeps the last error per
thread, and the library's next launch check would report it as its own."""
import ctypes as C

import numpy as np
import pytest

import jxlt_testlib as T


@pytest.mark.gpu
def test_undoing_a_registration_that_is_not_there_does_not_fail_the_next_frame(built):
    """What a caller does whose jxlt_pinned_register was refused and who cleans up all the same."""
    hip = built.hip_lib()
    hip.jxlt_pinned_unregister.argtypes = [C.c_void_p]
    hip.jxlt_pinned_unregister.restype = None
    planes = T.to_planes(T.synthetic_image(200, 137))
    enc = built.Encoder(0)
    enc.upload(planes)
    want = enc.encode_resident(1.0)
    hip.hipPeekAtLastError.restype = C.c_int
    never_registered = np.zeros(1 << 16, np.uint8)
    hip.jxlt_pinned_unregister(never_registered.ctypes.data)
    assert hip.hipPeekAtLastError() == 0
    assert enc.encode_resident(1.0) == want
    enc.close()
