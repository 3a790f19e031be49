"""Calls of the answers' functions that their documentation allows, at the ends of their arguments."""
import ctypes
import math
import sys

import pytest
import torch

from hingetreefortorch_b200 import HingeTree as F, RandomHingeForest as R, _cabi
from hingetreefortorch_b200._ext import hingetree_cpp
from test_dense_gpu import generator, lost, normal, within
from test_dense_host import DenseProblem
from test_packed_answers_gpu import check_linear

pytestmark = pytest.mark.gpu


def test_top_k_up_to_the_largest_whole_number():
    """Any number of classes from theirs on is all of them, as one for all rows and as one a row."""
    s, u = normal(generator(1), 5, 1000, scale=2.0), torch.rand(5, generator=generator(2), device="cuda")
    want = F.sample_classes(s, u, top_p=0.9)
    for k in (1000, 2 ** 31, 2 ** 53 + 1, 2 ** 62, 2 ** 63 - 513, sys.maxsize):
        for top_k in (k, torch.full((5,), k, device="cuda")):
            got = F.sample_classes(s, u, top_k=top_k, top_p=0.9)
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("kind", [torch.float32, torch.bfloat16, torch.float16])
def test_unpacked_zeros_have_the_sign_of_their_code(kind):
    """Under every scale and at every place of 8 codes, in rows that start on 16 bytes and on fewer; what is packed again is the same."""
    gen = generator(3)
    codes = torch.randint(0, 256, (255, 64), generator=gen, device="cuda", dtype=torch.int32).to(torch.uint8)
    codes[:, :16] = 0x80
    codes[:, 16:32] = 0x08
    scales = torch.arange(255, device="cuda", dtype=torch.uint8).view(255, 1).repeat(1, 4)
    each = torch.stack([codes & 15, codes >> 4], 2).flatten(1)
    for features in (128, 127, 101):
        got = F.unpack_mx4(codes, scales, features, dtype=kind)
        assert torch.equal(torch.signbit(got), each[:, :features] >= 8)
    w = torch.zeros(3, 64, dtype=kind, device="cuda")
    w[:, ::3] = -0.0
    w[1, 5], w[2, 6] = 1.0, -2.0 ** -14
    assert torch.equal(torch.signbit(F.unpack_mx4(*F.pack_mx4(w), 64, dtype=kind)), torch.signbit(w))


def test_packed_head_draws_for_features_that_require_a_gradient():
    """As the heads that it was packed from do: nothing drawn has a derivative."""
    gen = generator(4)
    head = R.LinearClassLoss(100, 300).cuda()
    packed = head.packed()
    x, u = normal(gen, 20, 100), torch.rand(20, generator=gen, device="cuda")
    want = packed.sample(x, u, top_k=5)
    for bounds in (dict(top_k=5), dict(top_k=5, temperature=torch.ones(20, device="cuda", requires_grad=True))):
        leaf = x.clone().requires_grad_()
        got = packed.sample(leaf, u, **bounds)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]) and not got[1].requires_grad
        head.sample(leaf, u, **bounds)
    forest = R.RandomHingeForestFusedLinear(12, 70, 30, 4).cuda()
    rows, v = torch.randn(9, 12, generator=gen, device="cuda"), torch.rand(9, generator=gen, device="cuda")
    packed = forest.packed_classes()
    features = forest._function.apply(rows, *forest._tree_params())
    assert features.requires_grad
    assert torch.equal(packed.sample(features, v)[0], forest.sample(rows, v, packed=packed)[0])
    with pytest.raises(RuntimeError, match="no derivative"):
        packed(features)


# ---- scores of many rows with little memory ----------------------------------------------------------------------------

def many_rows(rows, features, outputs):
    gen = generator(outputs)
    codes, scales = F.pack_mx4(normal(gen, outputs, features, scale=1 / math.sqrt(features)))
    return normal(gen, rows, features, kind=torch.bfloat16), codes, scales, normal(gen, outputs, scale=0.5, kind=torch.bfloat16)


def near(got, want):
    """Sums of the same products in another order: each is off by half a step of bf16, 2^-9, and by far less in its sums."""
    assert (got.float() - want.float()).norm() <= 2.0 ** -8 * want.float().norm()


def test_decoded_weights_within_a_limit():
    """Pieces of whole tiles, the last one ragged, and none at all; what lies behind the workspace's end stays as it was."""
    rows, features, outputs = 1100, 1024, 30011
    x, codes, scales, bias = many_rows(rows, features, outputs)
    want = check_linear(x, codes, scales, bias)
    lib = _cabi.library()
    lib.ht_linear_mx4_workspace_bytes.restype = ctypes.c_size_t
    at = lambda t: ctypes.c_void_p(t.data_ptr())
    for limit, least in ((0, 2 * features * outputs), (1 << 40, 2 * features * outputs), (40 << 20, 36 << 20), (20 << 20, 18 << 20), (10 << 20, 0), (1, 0)):
        p = DenseProblem(1, 0, rows, features, outputs, features, limit)
        size = lib.ht_linear_mx4_workspace_bytes(ctypes.byref(p))
        assert least <= size <= (limit if 1 < limit < 1 << 30 else least + 256), (limit, size)
        room = torch.full((size + 256,), 77, dtype=torch.uint8, device="cuda")
        got = torch.empty(rows, outputs, dtype=torch.bfloat16, device="cuda")
        stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
        assert lib.ht_linear_mx4(ctypes.byref(p), at(x), at(codes), at(scales), at(bias), at(got), at(room), ctypes.c_size_t(size), None, stream) == 0
        assert (room[size:] == 77).all()
        near(got, want)
        if size > 0:
            assert lib.ht_linear_mx4(ctypes.byref(p), at(x), at(codes), at(scales), at(bias), at(got), at(room), ctypes.c_size_t(size - 1), None, stream) == -4


def test_scores_without_room_for_decoded_weights():
    """246 MB of scores are to be had, 123 MB of decoded weights beside them are not: scores all the same."""
    x, codes, scales, bias = many_rows(4096, 2048, 30000)
    want = check_linear(x, codes, scales, bias)
    out = want.numel() * want.element_size()
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    total = torch.cuda.get_device_properties(0).total_memory
    torch.cuda.set_per_process_memory_fraction((torch.cuda.memory_reserved() + out + (60 << 20)) / total)
    try:
        got = F.linear_mx4(x, codes, scales, bias)
    finally:
        torch.cuda.set_per_process_memory_fraction(1.0)
    near(got, want)
    assert hingetree_cpp.pipeline_status() == 0


@pytest.mark.parametrize("rows", [3, 40])
def test_smallest_numbers_of_fp32(rows):
    """x as three bf16 numbers is exact from 2^-110 on; of what is smaller the third number leaves 2^-134, half of bf16's smallest.  Weights
    between 2^98 and 2^108 lift the products into fp32's range, where 2^-140 is no matter."""
    gen = generator(rows)
    features = 200
    codes = torch.randint(0, 256, (90, 16 * 7), generator=gen, device="cuda", dtype=torch.int32).to(torch.uint8)
    scales = torch.randint(225, 235, (90, 7), generator=gen, device="cuda", dtype=torch.int32).to(torch.uint8)
    w = F.unpack_mx4(codes, scales, features).double()
    for size, lost_of_x in ((2.0 ** -106, 0.0), (2.0 ** -118, 2.0 ** -134), (2.0 ** -128, 2.0 ** -134)):
        x = normal(gen, rows, features, scale=size)
        if size == 2.0 ** -106:
            x = torch.where(x.abs() < 2.0 ** -110, torch.zeros_like(x), x)
        got = F.linear_mx4(x, codes, scales)
        terms = x.double().abs() @ w.abs().t()
        within(got, x.double() @ w.t(), (lost(features) + 2.0 ** -23) * terms + lost_of_x * w.abs().sum(1) + 2.0 ** -135, torch.float32)
