"""The dense layers around a forest, as far as no GPU is needed: workspaces that the entries refuse."""
import ctypes

import pytest

from hingetreefortorch_b200 import _cabi
from test_dense_host import DenseProblem


@pytest.mark.parametrize("dtype", [0, 1, 2])
def test_a_workspace_starts_on_256_bytes(dtype):
    """Gradients are stored 32 bytes at a time in it, at offsets that are multiples of 256."""
    lib = _cabi.library()
    size, null = ctypes.c_size_t, None
    p = DenseProblem(dtype, 0, 300, 16, 32, 16, 0)
    host = (ctypes.c_char * 8192)()
    at = (ctypes.addressof(host) + 255) // 256 * 256
    ptr, room = ctypes.c_void_p(at), size(1 << 30)
    for offset in (16, 32, 128):
        ws = ctypes.c_void_p(at + offset)
        g = ctypes.byref(p)
        assert lib.ht_gated_linear_forward(g, ptr, ptr, ptr, null, null, ptr, null, ws, room, null, null) == -4
        assert lib.ht_gated_linear_backward(g, ptr, ptr, ptr, null, null, ptr, null, ptr, ptr, ptr, null, null, ws, room, null, null) == -4
        assert lib.ht_linear_class_loss_forward(g, ptr, ptr, null, ptr, ctypes.c_int64(-100), 1, ptr, null, null, ws, room, null, null) == -4
        assert lib.ht_linear_class_loss_backward(g, ptr, ptr, null, ptr, ctypes.c_int64(-100), 1, ptr, ptr, null, ptr, ptr, null, ws, room, null, null) == -4
