"""HIP streams of a test's own.  torch.cuda.Stream() deals out 32 pooled handles
in turn, so a test that takes some decides which of the later ones come round
to a handle whose workspace an earlier test left; these are outside that pool."""
import ctypes

import torch

from compiler_amd import runtime as rt

_streams = {}


def own_stream(i=0):
    """The i-th stream (created once, default priority, never destroyed)."""
    if i not in _streams:
        torch.cuda.current_stream().synchronize()  # the device is set up
        create = ctypes.CDLL(str(rt.LIB_PATH)).hipStreamCreateWithFlags  # the HIP runtime the library uses
        handle = ctypes.c_void_p()
        assert create(ctypes.byref(handle), ctypes.c_uint(1)) == 0  # hipStreamNonBlocking
        _streams[i] = torch.cuda.ExternalStream(handle.value)
    return _streams[i]
