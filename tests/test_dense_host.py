"""The dense layers around a forest, as far as no GPU is needed: what is refused, and with which exception; modules; workspaces."""
import ctypes

import pytest
import torch

from hingetreefortorch_b200 import HingeTree as F, RandomHingeForest as R, _cabi


class DenseProblem(ctypes.Structure):
    _fields_ = [("dtype", ctypes.c_int32), ("activation", ctypes.c_int32), ("rows", ctypes.c_int64), ("features", ctypes.c_int64),
                ("outputs", ctypes.c_int64), ("x_stride", ctypes.c_int64), ("scratch_limit", ctypes.c_int64)]


def test_class_loss_refuses():
    x, w, b, t = torch.randn(4, 5), torch.randn(7, 5), torch.randn(7), torch.randint(0, 7, (4,))
    for bad in [dict(x=x.double(), w=w.double(), b=None), dict(w=w.bfloat16()), dict(b=b.half()), dict(w=torch.randn(7, 6)), dict(b=b[:6]),
                dict(t=t.int()), dict(t=t[:3]), dict(w=torch.randn(0, 5), b=None), dict(x=torch.randn(4, 0), w=torch.randn(7, 0)),
                dict(w=torch.randn(5))]:
        a = {"x": x, "w": w, "b": b, "t": t, **bad}
        with pytest.raises(ValueError, match="Error: "):
            F.linear_class_loss(a["x"], a["w"], a["b"], a["t"])
    with pytest.raises(ValueError, match="reduction"):
        F.linear_class_loss(x, w, b, t, reduction="median")
    with pytest.raises(RuntimeError, match="CUDA devices only"):
        F.linear_class_loss(x, w, b, t)


def test_gated_linear_refuses():
    x, w, b = torch.randn(4, 5), torch.randn(7, 5), torch.randn(7)
    for args in [(x.double(), w.double(), w.double()), (x, w.half(), w), (x, w, w[:6]), (x, w, w, b[:3]), (x, w, w, b, b.bfloat16()),
                 (x, torch.randn(7, 4), torch.randn(7, 4)), (x.int(), w.int(), w.int())]:
        with pytest.raises(ValueError, match="Error: "):
            F.gated_linear(*args)
    with pytest.raises(ValueError, match="activation"):
        F.gated_linear(x, w, w, activation="tanh")
    with pytest.raises(RuntimeError, match="CUDA devices only"):
        F.gated_linear(x, w, w, b, b)


def test_modules():
    gated = R.GatedLinear(5, 7)
    assert [k for k, _ in gated.named_parameters()] == ["gate_weight", "gate_bias", "value_weight", "value_bias"]
    assert R.GatedLinear(5, 7, bias=False).gate_bias is None and gated.gate_weight.shape == (7, 5) and "silu" in repr(gated)
    with pytest.raises(ValueError):
        R.GatedLinear(5, 7, activation="tanh")
    loss = R.LinearClassLoss(5, 3)
    assert loss.weight.shape == (3, 5) and loss.bias.shape == (3,)
    linear = torch.nn.Linear(5, 3)
    loss.load_state_dict(linear.state_dict())
    x = torch.randn(2, 5)
    assert torch.equal(loss.scores(x), linear(x))
    with pytest.raises(ValueError):
        R.LinearClassLoss(5, 3, reduction="median")
    with pytest.raises(RuntimeError, match="extra_outputs"):
        R.RandomHingeForestFusedLinear(5, 6, 3, 2, extra_outputs=2).class_loss(x, torch.zeros(2, dtype=torch.long))


def test_entries_screen_before_they_touch_a_device():
    lib = _cabi.library()
    lib.ht_gated_linear_workspace_bytes.restype = lib.ht_linear_class_loss_workspace_bytes.restype = ctypes.c_size_t
    null, size = None, ctypes.c_size_t
    good = DenseProblem(1, 0, 8, 16, 32, 16, 0)
    for change in [("dtype", 3), ("dtype", -1), ("rows", -1), ("features", 0), ("outputs", 0), ("x_stride", 15)]:
        p = DenseProblem(1, 0, 8, 16, 32, 16, 0)
        setattr(p, *change)
        for backward in (0, 1):
            assert lib.ht_gated_linear_workspace_bytes(ctypes.byref(p), backward) == 0
            assert lib.ht_linear_class_loss_workspace_bytes(ctypes.byref(p), backward) == 0
        assert lib.ht_gated_linear_forward(ctypes.byref(p), null, null, null, null, null, null, null, null, size(0), null, null) == -1
        assert lib.ht_linear_class_loss_forward(ctypes.byref(p), null, null, null, null, ctypes.c_int64(-100), 1, null, null, null, null, size(0), null, null) == -1
    p = DenseProblem(1, 4, 8, 16, 32, 16, 0)
    assert lib.ht_gated_linear_forward(ctypes.byref(p), null, null, null, null, null, null, null, null, size(0), null, null) == -1
    host = (ctypes.c_char * 4096)()
    at = (ctypes.addressof(host) + 255) // 256 * 256
    ptr, odd = ctypes.c_void_p(at), ctypes.c_void_p(at + 2)
    g = ctypes.byref(good)
    # a pointer that does not start on 16 bytes; no room for a workspace; a reduction that there is not; nothing to write to
    assert lib.ht_gated_linear_forward(g, odd, ptr, ptr, null, null, ptr, null, ptr, size(1 << 20), null, null) == -5
    assert lib.ht_gated_linear_backward(g, ptr, ptr, ptr, null, null, ptr, null, ptr, ptr, ptr, null, null, ptr, size(16), null, null) == -4
    assert lib.ht_linear_class_loss_forward(g, ptr, ptr, null, ptr, ctypes.c_int64(-100), 3, ptr, null, null, ptr, size(1 << 20), null, null) == -1
    assert lib.ht_linear_class_loss_forward(g, ptr, ptr, null, ptr, ctypes.c_int64(-100), 1, null, null, null, ptr, size(1 << 20), null, null) == -1
    assert lib.ht_linear_class_loss_forward(g, ptr, ptr, null, ptr, ctypes.c_int64(-100), 1, ptr, null, null, null, size(0), null, null) == -4
    assert lib.ht_linear_class_loss_backward(g, ptr, ptr, null, ptr, ctypes.c_int64(-100), 1, ptr, null, null, ptr, ptr, null, ptr, size(1 << 20), null, null) == -1


@pytest.mark.parametrize("dtype,planes", [(0, 3), (1, 1), (2, 1)])
def test_a_backward_holds_pieces_within_the_limit(dtype, planes):
    """What a smaller limit saves is the gradient of the scores: all of it is held where it fits, 256 outputs at the least."""
    lib = _cabi.library()
    lib.ht_gated_linear_workspace_bytes.restype = lib.ht_linear_class_loss_workspace_bytes.restype = ctypes.c_size_t
    rows, outputs = 4096, 50000
    for entry, matrices in [(lib.ht_linear_class_loss_workspace_bytes, 1), (lib.ht_gated_linear_workspace_bytes, 2)]:
        sizes = []
        for limit in (0, 1 << 28, 1 << 24, 1):
            p = DenseProblem(dtype, 0, rows, 64, outputs, 64, limit)
            sizes.append(entry(ctypes.byref(p), 1))
        assert sizes == sorted(sizes, reverse=True) and sizes[0] > sizes[-1]
        least = rows * 256 * 2 * planes * matrices
        assert least <= sizes[-1] <= least + outputs * 64 * 2 * planes * matrices + rows * 1024 * planes + (1 << 20)
        assert sizes[0] <= (1 << 29) * (1 + 1 / planes) + outputs * 64 * 2 * planes * matrices + rows * 1024 * planes
