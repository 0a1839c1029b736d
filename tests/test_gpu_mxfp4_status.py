"""What salt_b200_mxfp4_status answers."""
import ctypes as C

import pytest

from test_gpu_mxfp4 import Held, check_matmul

pytestmark = pytest.mark.gpu


def error_word(held):
    """Device address of a handle's error word: behind eight ints and the tiles' address (Mxfp4Weights in csrc/mxfp4.h)."""
    return C.cast(held.handle.handle, C.POINTER(C.c_uint64))[5]


def test_an_error_is_answered_once_and_cleared():
    """A word that a wait leaves when it runs out (8) reads as failed, as every other; the handle is usable afterwards."""
    import torch
    held = Held(4, 1, 130, 320, "silu")
    cu = C.CDLL("libcuda.so.1")
    for word in (8, 1, 1 << 30):
        assert held.handle.status() == 0
        torch.cuda.synchronize()
        assert cu.cuMemsetD32_v2(C.c_uint64(error_word(held)), C.c_uint(word), C.c_size_t(1)) == 0
        torch.cuda.synchronize()
        assert held.handle.status() == -1
        assert held.handle.status() == 0
    check_matmul(held, 7, 130, 320)
    assert held.handle.lib.salt_b200_mxfp4_status(None, None) == -1
