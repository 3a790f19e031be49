"""Draws under a top_p so near 1 that it cuts through a long tail of classes of little weight, against the definition.

The rows are ordered so that the ends of `uniform` show the border itself: with falling scores the last class that counts, drawn at 1, and with rising
ones the first, drawn at 0, are the lightest class of the prefix.  A class there weighs 1e-12 of the row or more.  The oracle's weights and sums are held
in 80 bits: in 64, 10 ** 5 additions of such classes to a sum of 1 may be off by 10 ** 5 halves of 2.2e-16, more than a class.  The operator's sums
are those of some hundred additions each, 1e-14.  Tolerances of the logarithm: test_packed_answers_gpu.py.
"""
import math

import numpy as np
import pytest
import torch

from hingetreefortorch_b200 import HingeTree as F
from test_dense_gpu import generator
from test_packed_answers_gpu import TYPES

pytestmark = pytest.mark.gpu


def border(scores, share, temperature=1.0, count=0):
    """top_p with which the class at `share` of all but the heaviest class's weight is the last of the first row's prefix."""
    v = np.sort(scores[0].double().cpu().numpy())[::-1]
    w = np.exp((v - v[0]) / temperature)[:count or None]
    upto = np.cumsum(w)
    at = max(int(np.searchsorted(upto, w[0] + share * (upto[-1] - w[0]))), 1)
    at = min(at, len(w) - 2)
    return float((upto[at - 1] + upto[at]) / 2 / upto[-1])


def draw(v, u, temperature, top_p, top_k=0, min_p=0.0):
    """The class drawn from one row, the logarithm of its share, and the mean of |y|, the exponents to base 2."""
    v = v.astype(np.longdouble)
    order = np.argsort(-v, kind="stable")
    w = np.exp((v[order] - v[order[0]]) / np.longdouble(temperature))
    n = min(top_k, len(v)) if top_k > 0 else len(v)
    upto = np.cumsum(w[:n])
    n = max(int((upto - w[:n] < np.longdouble(top_p) * upto[-1]).sum()), 1)
    n = max(int((w[:n] >= min_p).sum()), 1)
    held = np.sort(order[:n])
    y = (v[held] - v[order[0]]) / np.longdouble(temperature)
    w = np.exp(y)
    upto = np.cumsum(w)
    at = int(np.searchsorted(upto, np.longdouble(u) * upto[-1], side="right"))
    at = min(at, int(np.flatnonzero(w)[-1]))
    return int(held[at]), float(y[at] - np.log(upto[-1])), float((w * -y).sum() / upto[-1]) / math.log(2)


def check(scores, top_ps, temperature=1.0, **bounds):
    """Falling rows with uniform 1 and the number before it, rising ones with 0 and the number of its size, others with both; in clusters of 8, 4, 2
    CTAs a row and one alone; each call twice."""
    rows = torch.cat([scores, scores.flip(1), scores[:, torch.randperm(scores.size(1), device="cuda", generator=generator(1))]])
    uniform = torch.tensor([1.0, 0.0, 1.0], device="cuda")
    host = rows.double().cpu().numpy()
    for p in top_ps:
        for u in (uniform, (uniform - 2.0 ** -24).abs()):
            classes, logs, powers = (torch.tensor(v) for v in zip(*[draw(host[r], float(u[r]), temperature, p, **bounds) for r in range(3)]))
            for times in (1, 10, 15, 30):
                got = [F.sample_classes(rows.repeat(times, 1), u.repeat(times), temperature=temperature, top_p=p, **bounds) for _ in range(2)]
                assert all(torch.equal(a, b) for a, b in zip(*got))
                assert torch.equal(got[0][0].cpu(), classes.repeat(times)), (p, times, got[0][0][:3].tolist(), classes.tolist())
                off = (got[0][1].cpu().double() - logs.repeat(times)).abs() / (2.0 ** -24 * logs.abs() + 4.3e-7 + 1.25e-7 * powers).repeat(times)
                assert not (off > 1).any(), (p, times, off.max())


def falling(values, kind):
    return torch.sort(values, dim=1, descending=True)[0].to(kind)


NEAR = [0.99998, 0.999995, 1.0 - 2.0 ** -24]


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("classes,gap,sigma", [(20000, 20.0, 1.0), (20000, 24.0, 1.0), (50000, 22.35, 0.05), (50000, 23.0, 0.3), (131072, 24.0, 1.0),
                                               (131072, 26.0, 0.02), (262147, 22.5, 0.2), (262147, 23.0, 0.02)])
def test_one_class_above_a_long_background(kind, classes, gap, sigma):
    s = torch.randn(1, classes, generator=generator(classes), device="cuda") * sigma - gap
    s[:, 0] = 0.0
    s = falling(s, kind)
    check(s, NEAR + [border(s, share) for share in (0.2, 0.8)])


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("classes", [50000, 262144])
def test_one_class_above_a_flat_background(kind, classes):
    s = torch.rand(1, classes, generator=generator(classes), device="cuda") * 0.02 - 22.3
    s[:, 0] = 0.0
    s = falling(s, kind)
    check(s, [0.99997] + [border(s, share) for share in (0.05, 0.5, 0.95)])
    check(s * 2, [border(s * 2, 0.5, 2.0)], temperature=2.0)


@pytest.mark.parametrize("kind", TYPES)
def test_long_background_behind_top_k(kind):
    s = torch.randn(1, 60000, generator=generator(7), device="cuda") * 0.3 - 22.5
    s[:, 0] = 0.0
    s = falling(s, kind)
    for k in (201, 5000, 30000):
        check(s, [0.99999] + [border(s, share, count=k) for share in (0.3, 0.9)], top_k=k)
    check(s, [border(s, 0.5)], min_p=math.exp(-22.6))


@pytest.mark.parametrize("kind", TYPES)
def test_backgrounds_of_several_heights(kind):
    """Each of them weighs little beside the one above; many classes of one score, more than a list holds."""
    gen = generator(9)
    steps = torch.tensor([0.0, -5.0, -11.0, -18.0, -23.0, -25.0], device="cuda")
    which = torch.multinomial(torch.tensor([0.0005, 0.0005, 0.009, 0.09, 0.3, 0.6], device="cuda"), 40000, replacement=True, generator=gen).view(1, 40000)
    for spread in (0.0, 0.01, 0.5):
        s = falling(steps[which] + spread * torch.randn(1, 40000, generator=gen, device="cuda"), kind)
        check(s, NEAR + [border(s, 1.0 - left) for left in (1e-2, 1e-5, 1e-7)])


@pytest.mark.parametrize("kind", [torch.float32, torch.bfloat16])
def test_scores_of_every_size(kind):
    """Scores that lie evenly neither by value nor by their bits."""
    gen = generator(10)
    s = -torch.exp(torch.rand(1, 30000, generator=gen, device="cuda") * 64 - 60)
    s = falling(torch.cat([s, s - 22.0, s - 24.0], 1), kind)
    check(s, NEAR + [border(s, share) for share in (0.5, 0.9999)])
