"""Calls of the answers' functions that their documentation allows, at the ends of their arguments."""
import sys

import pytest
import torch

from hingetreefortorch_b200 import HingeTree as F, RandomHingeForest as R
from test_dense_gpu import generator, normal

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
