"""Calls of the answers' functions that their documentation allows, at the ends of their arguments."""
import sys

import pytest
import torch

from hingetreefortorch_b200 import HingeTree as F
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
