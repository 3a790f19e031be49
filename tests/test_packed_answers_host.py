"""Answers of a linear layer with many classes, as far as no GPU is needed: what is refused, and with which exception; modules; entries."""
import ctypes

import pytest
import torch

from hingetreefortorch_b200 import HingeTree as F, RandomHingeForest as R, _cabi
from test_dense_host import DenseProblem


class SampleProblem(ctypes.Structure):
    _fields_ = [("dtype", ctypes.c_int32), ("reserved", ctypes.c_int32), ("rows", ctypes.c_int64), ("classes", ctypes.c_int64), ("stride", ctypes.c_int64),
                ("temperature", ctypes.c_double), ("top_p", ctypes.c_double), ("min_p", ctypes.c_double), ("top_k", ctypes.c_int64),
                ("row_temperature", ctypes.c_void_p), ("row_top_p", ctypes.c_void_p), ("row_min_p", ctypes.c_void_p), ("row_top_k", ctypes.c_void_p)]


def test_packing_refuses():
    for bad in (torch.randn(4, 5).double(), torch.zeros(4, 5, dtype=torch.int32), torch.randn(5), torch.randn(0, 5), torch.randn(5, 0), torch.randn(2, 3, 4)):
        with pytest.raises(ValueError, match="Error: "):
            F.pack_mx4(bad)
    with pytest.raises(RuntimeError, match="CUDA devices only"):
        F.pack_mx4(torch.randn(4, 5))


def packed(outputs=4, features=40):
    blocks = -(-features // 32)
    return torch.zeros(outputs, 16 * blocks, dtype=torch.uint8), torch.zeros(outputs, blocks, dtype=torch.uint8)


def test_unpacking_refuses():
    codes, scales = packed()
    for args in [(codes.int(), scales, 40), (codes, scales.char(), 40), (codes, scales, 65), (codes, scales, 32), (codes, scales, 0), (codes[:3], scales, 40),
                 (codes[:, :16], scales, 40), (codes[0], scales[0], 40), (codes[:0], scales[:0], 40), (codes, scales, 40, torch.float64), (codes, scales, 40, torch.uint8)]:
        with pytest.raises(ValueError, match="Error: "):
            F.unpack_mx4(*args)
    with pytest.raises(RuntimeError, match="CUDA devices only"):
        F.unpack_mx4(codes, scales, 40)


def test_products_refuse():
    codes, scales = packed()
    x, b = torch.randn(3, 40), torch.randn(4)
    for args in [(x.double(), codes, scales), (x.int(), codes, scales), (x, codes, scales, b.half()), (x, codes, scales, b[:3]), (x, codes, scales, b.view(1, 4)),
                 (torch.randn(3, 65), codes, scales), (x, codes.int(), scales), (x, codes, scales[:, :1]), (torch.tensor(1.0), codes, scales),
                 (torch.randn(3, 0), codes, scales)]:
        with pytest.raises(ValueError, match="Error: "):
            F.linear_mx4(*args)
    with pytest.raises(RuntimeError, match="CUDA devices only"):
        F.linear_mx4(x, codes, scales, b)


def test_sampling_refuses():
    s, u = torch.randn(3, 7), torch.rand(3)
    for args in [(s.double(), u), (s.int(), u), (s, u.double()), (s, u[:2]), (s, u.view(3, 1)), (torch.randn(3, 0), u), (torch.tensor(1.0), u)]:
        with pytest.raises(ValueError, match="Error: "):
            F.sample_classes(*args)
    for bound in [dict(temperature=-0.1), dict(temperature=float("nan")), dict(temperature=float("inf")), dict(top_k=-1), dict(top_k=2.5), dict(top_p=1.1),
                  dict(top_p=-0.1), dict(top_p=float("nan")), dict(min_p=1.5), dict(min_p=-1.0), dict(temperature="hot"), dict(top_k=torch.ones(3)),
                  dict(temperature=torch.ones(3).double()), dict(top_p=torch.ones(2)), dict(min_p=torch.ones(3, 1)), dict(temperature=torch.ones(()))]:
        with pytest.raises(ValueError, match="Error: "):
            F.sample_classes(s, u, **bound)
    with pytest.raises(RuntimeError, match="CUDA devices only"):
        F.sample_classes(s, u, temperature=torch.ones(3), top_k=torch.ones(3, dtype=torch.long), top_p=torch.ones(3), min_p=torch.zeros(3))


def test_modules():
    head = R.PackedClasses(70, 5)
    assert sorted(head.state_dict()) == ["bias", "codes", "scales"] and head.codes.shape == (5, 48) and head.scales.shape == (5, 3)
    assert not list(head.parameters()) and "in_features=70" in repr(head)
    other = R.PackedClasses(70, 5, bias=False)
    assert sorted(other.state_dict()) == ["codes", "scales"] and other.to(torch.bfloat16).codes.dtype == torch.uint8
    with pytest.raises(RuntimeError, match="CUDA devices only"):
        head(torch.randn(2, 70))
    with pytest.raises(RuntimeError, match="CUDA devices only"):
        R.LinearClassLoss(5, 3).packed()
    with pytest.raises(RuntimeError, match="CUDA devices only"):
        R.LinearClassLoss(5, 3).sample(torch.randn(2, 5), torch.rand(2))
    forest = R.RandomHingeForestFusedLinear(5, 6, 3, 2, extra_outputs=2)
    with pytest.raises(RuntimeError, match="extra_outputs"):
        forest.sample(torch.randn(2, 5), torch.rand(2), packed=head)


def test_entries_screen_before_they_touch_a_device():
    lib = _cabi.library()
    null, size, i64, f64 = None, ctypes.c_size_t, ctypes.c_int64, ctypes.c_double
    host = (ctypes.c_char * 4096)()
    at = (ctypes.addressof(host) + 255) // 256 * 256
    ptr, odd = ctypes.c_void_p(at), ctypes.c_void_p(at + 4)
    for entry in (lambda dtype, outputs, features, stride, a=ptr: lib.ht_mx4_pack(dtype, ptr, i64(stride), i64(outputs), i64(features), a, ptr, null),
                  lambda dtype, outputs, features, stride, a=ptr: lib.ht_mx4_unpack(dtype, a, ptr, i64(outputs), i64(features), ptr, i64(stride), null)):
        for bad in ((3, 4, 5, 5), (-1, 4, 5, 5), (0, -1, 5, 5), (0, 4, 0, 5), (0, 4, 5, 4)):
            assert entry(*bad) == -1
        assert entry(0, 0, 5, 5) == 0 and entry(0, 4, 5, 5, odd) == -5 and entry(0, 4, 5, 5, null) == -1 and entry(0, 1 << 31, 5, 5) == -5
    lib.ht_linear_mx4_workspace_bytes.restype = size
    for change in [("dtype", 3), ("rows", -1), ("features", 0), ("outputs", 0), ("x_stride", 15)]:
        p = DenseProblem(1, 0, 8, 16, 32, 16, 0)
        setattr(p, *change)
        assert lib.ht_linear_mx4_workspace_bytes(ctypes.byref(p)) == 0
        assert lib.ht_linear_mx4(ctypes.byref(p), ptr, ptr, ptr, null, ptr, ptr, size(1 << 30), null, null) == -1
    p = DenseProblem(1, 0, 8, 16, 32, 16, 0)
    assert lib.ht_linear_mx4(ctypes.byref(p), odd, ptr, ptr, null, ptr, ptr, size(1 << 30), null, null) == -5
    assert lib.ht_linear_mx4(ctypes.byref(p), ptr, ptr, ptr, null, null, ptr, size(1 << 30), null, null) == -1
    assert lib.ht_linear_mx4(ctypes.byref(p), ptr, ptr, ptr, null, ptr, odd, size(1 << 30), null, null) == -4
    p = DenseProblem(1, 0, 0, 16, 32, 16, 0)
    assert lib.ht_linear_mx4(ctypes.byref(p), null, ptr, ptr, null, null, null, size(0), null, null) == 0
    for change in [("dtype", 3), ("rows", -1), ("classes", 0), ("stride", 6), ("temperature", -1.0), ("temperature", float("nan")), ("top_p", 2.0), ("min_p", -1.0), ("top_k", -1)]:
        p = SampleProblem(0, 0, 2, 7, 7, 1.0, 1.0, 0.0, 0)
        setattr(p, *change)
        assert lib.ht_sample_classes(ctypes.byref(p), ptr, ptr, ptr, ptr, null) == -1
    p = SampleProblem(0, 0, 2, 7, 7, 1.0, 1.0, 0.0, 0)
    assert lib.ht_sample_classes(ctypes.byref(p), ptr, ptr, null, ptr, null) == -1
    assert lib.ht_sample_classes(null, ptr, ptr, ptr, ptr, null) == -1
    p.rows = 0
    assert lib.ht_sample_classes(ctypes.byref(p), null, null, null, null, null) == 0
