"""The dense layers around a forest (gated_linear, linear_class_loss) against the same formulas in 64 bits.

Bounds, per element.  u: half a step of a type, finfo.eps / 2; fp32 operands are held to 2^-23 (three planes of 8 bits leave
2^-24, the products left out as much).  A sum of K products loses at most (K + 16) 2^-23 of the sum of their magnitudes (the tensor core
truncates when it adds).  So a score s is off by ds = (K + 16 + 2) 2^-23 sum |x||w|, a probability p by p (2 max ds + 2^-20) (exponent
and its argument, and the row's sum), and the gradient g of the scores, rounded to the operands' type, by
E = u |g| + p (2 max ds + 2^-20).  What is a sum of g's is off by E times the magnitudes of the other factor, the sum's own loss, and
the rounding of the result.  The projection's gradient goes the same way from its own terms.
"""
import math

import pytest
import torch

from hingetreefortorch_b200 import HingeTree as F, RandomHingeForest as R
from hingetreefortorch_b200._ext import hingetree_cpp

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]
TINY = {torch.float32: 1e-37, torch.bfloat16: 1e-37, torch.float16: 2.0 ** -25}  # half a step of the smallest numbers


def half_step(kind):
    return torch.finfo(kind).eps / 2


def operand_step(kind):
    return 2.0 ** -23 if kind == torch.float32 else half_step(kind)


def lost(terms):
    return (terms + 16) * 2.0 ** -23


def normal(gen, *shape, scale=1.0, kind=torch.float32):
    return (torch.randn(*shape, generator=gen, device="cuda") * scale).to(kind)


def generator(seed=0):
    return torch.Generator(device="cuda").manual_seed(seed)


def within(got, want, bound, kind):
    got = got.detach().double()
    slack = half_step(kind) * want.abs() + TINY[kind] + bound
    # The largest fp16 number is 65504 = (2 - 2^-10) 2^15 and the next step would be 65536: what is 65520 or more rounds to infinity, with
    # its sign.  Only where the exact value lies there, to within the bound, may the result be infinite.
    top = torch.finfo(kind).max
    beyond = want.abs() + bound >= top * (1 + half_step(kind) / 2)
    assert got.shape == want.shape and (torch.isfinite(got) | (beyond & (got == torch.copysign(torch.full_like(want, math.inf), want)))).all()
    finite = torch.isfinite(got)
    worst = ((got - want).abs() / slack)[finite].max().item() if finite.any() else 0.0
    assert worst <= 1.0, worst


# ---- class loss --------------------------------------------------------------------------------------------------------

def loss_inputs(kind, rows, features, classes, bias=True, ignored=False, seed=0):
    gen = generator(seed)
    x, w = normal(gen, rows, features, kind=kind), normal(gen, classes, features, scale=2 / math.sqrt(features), kind=kind)
    b = normal(gen, classes, scale=0.5, kind=kind) if bias else None
    t = torch.randint(0, classes, (rows,), generator=gen, device="cuda")
    if ignored:
        t[::3] = -100
    return x, w, b, t


def check_loss(x, w, b, t, reduction, grad=None, ignore=-100, run=None):
    """Loss and gradients of one call against the formulas in 64 bits; gives what the call gave."""
    kind = x.dtype
    leaves = [v.detach().requires_grad_() for v in (x, w) + ((b,) if b is not None else ())]
    loss = (run or F.linear_class_loss)(leaves[0], leaves[1], leaves[2] if b is not None else None, t, ignore_index=ignore, reduction=reduction)
    assert loss.dtype == torch.float32
    grads = torch.autograd.grad(loss, leaves, grad)
    counts = t != ignore
    X, W, B = (v.detach().double() if v is not None else None for v in (x, w, b))
    X = torch.where(counts[:, None], X, torch.zeros_like(X))
    s = X @ W.t() + (B if B is not None else 0.0)
    ds = lost(X.shape[1] + 2) * (X.abs() @ W.abs().t() + (B.abs() if B is not None else 0.0)).amax()
    lse = torch.logsumexp(s, 1)
    at = torch.where(counts, t, torch.zeros_like(t))
    rows = torch.where(counts, lse - s.gather(1, at[:, None])[:, 0], torch.zeros_like(lse))
    off = 2 * ds + 2.0 ** -20 + 2.0 ** -22 * lse.abs()
    n = counts.sum()
    if reduction == "none":
        within(loss, rows, off, torch.float32)
        upstream = (grad if grad is not None else torch.ones_like(rows)).double()
    else:
        total = rows.sum() / (n if reduction == "mean" else 1)
        within(loss, total, off * (1 if reduction == "mean" else n) if torch.is_tensor(off) and off.dim() == 0 else off.amax() * (1 if reduction == "mean" else n), torch.float32)
        one = grad.double() if grad is not None else torch.ones((), dtype=torch.float64, device="cuda")
        upstream = (one / (n if reduction == "mean" else 1)).expand(len(t))
    r = torch.where(counts, upstream, torch.zeros_like(rows))[:, None]
    p = torch.exp(s - lse[:, None])
    g = p.scatter_add(1, at[:, None], -torch.ones_like(r)) * r
    E = operand_step(kind) * g.abs() + p * r.abs() * (2 * ds + 2.0 ** -20)
    if kind == torch.float16:  # the smallest gradients that are held: 2^-25 of 2^14 times the largest factor
        E = E + 2.0 ** -38 * r.abs().amax()
    u = operand_step(kind) if kind == torch.float32 else 0.0  # x and w are split as well
    within(grads[0], g @ W, E @ W.abs() + (lost(W.shape[0]) + u) * (g.abs() @ W.abs()), kind)
    within(grads[1], g.t() @ X, E.t() @ X.abs() + (lost(X.shape[0]) + u) * (g.abs().t() @ X.abs()), kind)
    if b is not None:
        within(grads[2], g.sum(0), E.sum(0) + len(t) * 2.0 ** -24 * g.abs().sum(0), kind)
    return [loss.detach(), *grads]


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("rows,features,classes", [
    (1, 1, 1), (1, 64, 7), (2, 7, 2), (5, 16, 64), (9, 24, 1000), (17, 65, 255), (127, 64, 257), (128, 63, 256), (129, 130, 65), (300, 200, 513),
    (640, 40, 2049), (31, 1025, 50), (2, 2048, 33)])
@pytest.mark.parametrize("reduction", ["none", "mean", "sum"])
def test_class_loss(kind, rows, features, classes, reduction):
    x, w, b, t = loss_inputs(kind, rows, features, classes, bias=rows % 2 == 1, ignored=rows > 2)
    grad = normal(generator(5), rows, scale=3.0) if reduction == "none" else torch.tensor(0.37, device="cuda")
    if reduction == "none":
        grad[rows // 2] = 0.0
    check_loss(x, w, b, t, reduction, grad)
    with torch.no_grad():  # the call that is not differentiated gives the same
        again = F.linear_class_loss(x, w, b, t, reduction=reduction)
    assert torch.equal(again, F.linear_class_loss(x.requires_grad_(), w, b, t, reduction=reduction).detach())


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("rows,features,classes", [
    (8, 200, 40000),      # few rows, a warp for every 16 classes
    (8, 2700, 50), (8, 5400, 50), (8, 2660, 50), (7, 2900, 40), (14, 2500, 40), (30, 1240, 40), (29, 1300, 30),  # x about fills shared memory
    (16, 1030, 6000), (20, 500, 300), (32, 2050, 90), (24, 4096, 100), (31, 70, 5000),
    (33, 4, 17), (64, 1024, 2300), (65, 100, 4700), (100, 2048, 31), (128, 36, 1000), (77, 2052, 130), (90, 99, 600),
    (6000, 33, 70),       # few tiles of the weights' gradient, long sums over the rows
    (150, 48, 9000),      # and of the features'
    (2500, 300, 300), (1100, 65, 1500), (700, 520, 225)])
def test_class_loss_by_size(kind, rows, features, classes):
    """Sizes at which other kernels, tile shapes and cuts of the sums are taken."""
    x, w, b, t = loss_inputs(kind, rows, features, classes, bias=features % 2 == 0, ignored=rows % 2 == 1, seed=rows)
    check_loss(x, w, b, t, "mean")


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("act,rows,features,outputs", [
    ("silu", 8, 200, 20000), ("gelu", 16, 1030, 3000), ("relu", 20, 500, 150), ("sigmoid", 32, 2050, 45), ("gelu", 24, 4096, 50),
    ("silu", 33, 4, 9), ("gelu", 64, 1024, 1150), ("sigmoid", 65, 100, 2350), ("silu", 100, 2048, 16), ("relu", 128, 36, 500), ("gelu", 77, 2052, 65),
    ("silu", 90, 99, 300), ("gelu", 6000, 33, 35), ("silu", 150, 48, 5000), ("gelu", 2500, 300, 150), ("sigmoid", 1100, 65, 900), ("silu", 700, 520, 97)])
def test_gated_linear_by_size(kind, act, rows, features, outputs):
    check_gated(*gated_inputs(kind, rows, features, outputs, bias=features % 2 == 0, seed=rows), act)


@pytest.mark.parametrize("kind", TYPES)
def test_rows_that_do_not_count(kind):
    """Whatever an ignored row holds, nothing of it enters; none at all: NaN for a mean, and no gradient."""
    x, w, b, t = loss_inputs(kind, 200, 72, 300, ignored=True)
    clean = check_loss(x, w, b, t, "mean")
    dirty = x.clone()
    dirty[0], dirty[3], dirty[6, 5], dirty[9] = float("nan"), float("inf"), float("-inf"), torch.finfo(kind).max
    leaves = [v.requires_grad_() for v in (dirty, w, b)]
    loss = F.linear_class_loss(*leaves, t)
    for a, c in zip([loss.detach(), *torch.autograd.grad(loss, leaves)], clean):
        assert torch.equal(a, c)
    assert torch.equal(clean[1][::3], torch.zeros_like(clean[1][::3]))
    none = torch.full_like(t, 7)
    loss = F.linear_class_loss(*leaves, none, ignore_index=7)
    assert torch.isnan(loss) and all(torch.equal(g, torch.zeros_like(g)) for g in torch.autograd.grad(loss, leaves))
    assert F.linear_class_loss(*leaves, none, ignore_index=7, reduction="sum").item() == 0.0
    assert torch.equal(F.linear_class_loss(*leaves, none, ignore_index=7, reduction="none"), torch.zeros(200, device="cuda"))


@pytest.mark.parametrize("kind", TYPES)
def test_no_rows(kind):
    w, b = torch.randn(5, 3, device="cuda", dtype=kind, requires_grad=True), torch.randn(5, device="cuda", dtype=kind, requires_grad=True)
    x, t = torch.empty(0, 3, device="cuda", dtype=kind, requires_grad=True), torch.empty(0, dtype=torch.long, device="cuda")
    for reduction, value in (("mean", math.nan), ("sum", 0.0)):
        loss = F.linear_class_loss(x, w, b, t, reduction=reduction)
        assert math.isnan(loss.item()) if math.isnan(value) else loss.item() == value
        grads = torch.autograd.grad(loss, [x, w, b])
        assert grads[0].shape == (0, 3) and not grads[1].any() and not grads[2].any()
    assert F.linear_class_loss(x, w, b, t, reduction="none").shape == (0,)
    h = F.gated_linear(x, w, w)
    assert h.shape == (0, 5) and not torch.autograd.grad(h.sum(), w)[0].any()


@pytest.mark.parametrize("kind", TYPES)
def test_classes_that_a_bias_masks(kind):
    """A bias of -inf, or of the type's lowest value, takes classes out; all of them: no number, as the softmax has it."""
    x, w, b, t = loss_inputs(kind, 40, 32, 300)
    t = t % 100
    for low in (float("-inf"), torch.finfo(kind).min):
        masked = b.clone()
        masked[100:] = low
        loss = F.linear_class_loss(x, w, masked, t, reduction="none")
        within(loss, F.linear_class_loss(x, w[:100].contiguous(), b[:100].contiguous(), t, reduction="none").double(), 2.0 ** -20, torch.float32)
        leaves = [v.detach().requires_grad_() for v in (x, w, masked)]
        grads = torch.autograd.grad(F.linear_class_loss(*leaves, t), leaves)
        assert all(torch.isfinite(g).all() for g in grads) and not grads[1][100:].any() and not grads[2][100:].any()
    assert torch.isnan(F.linear_class_loss(x, w, torch.full_like(b, float("-inf")), t, reduction="none")).all()
    # lowest everywhere: the scores are that value and nothing else counts beside it (fp32 and bf16 sums do not leave it)
    even = F.linear_class_loss(x, w, torch.full_like(b, torch.finfo(torch.float32).min if kind == torch.float32 else torch.finfo(kind).min), t, reduction="none")
    assert torch.isfinite(even).all()
    if kind != torch.float16:
        within(even, torch.full((40,), math.log(300.0), dtype=torch.float64, device="cuda"), 2.0 ** -20, torch.float32)


def test_large_scores():
    """Scores of some thousands: one class takes all, and its row's loss is the distance in full."""
    for kind in TYPES:
        x, w, b, t = loss_inputs(kind, 64, 256, 130)
        check_loss(x, (w.float() * 60).to(kind), b, t, "mean")


def test_a_target_that_is_no_class():
    x, w, b, t = loss_inputs(torch.float32, 50, 20, 30)
    for wrong in (30, -1, 2 ** 40, -2 ** 62):
        bad = t.clone()
        bad[7] = wrong
        leaves = [v.detach().requires_grad_() for v in (x, w, b)]
        rows = F.linear_class_loss(*leaves, bad, reduction="none")
        assert torch.isnan(rows[7]) and torch.isfinite(rows).sum() == 49
        gx, gw, gb = torch.autograd.grad(rows.sum(), leaves)
        assert torch.isnan(gx[7]).all() and torch.isfinite(gx[:7]).all() and torch.isfinite(gx[8:]).all()
        assert torch.isnan(gw).all() and torch.isnan(gb).all()
        with pytest.raises(RuntimeError, match="neither a class"):
            hingetree_cpp.pipeline_status()
    assert hingetree_cpp.pipeline_status() == 0


# ---- gated projection ------------------------------------------------------------------------------------------------

def gate(a, act):
    if act == "relu":
        return a.clamp_min(0), (a > 0).double()
    if act == "gelu":
        phi = 0.5 * torch.erfc(-a / math.sqrt(2))
        return a * phi, phi + a * torch.exp(-a * a / 2) / math.sqrt(2 * math.pi)
    s = torch.sigmoid(a)
    return (s, s * (1 - s)) if act == "sigmoid" else (a * s, s * (1 + a * (1 - s)))


def gated_inputs(kind, rows, features, outputs, bias=True, seed=0):
    gen = generator(seed)
    x = normal(gen, rows, features, kind=kind)
    wg, wv = (normal(gen, outputs, features, scale=1.5 / math.sqrt(features), kind=kind) for _ in range(2))
    bg, bv = (normal(gen, outputs, scale=0.3, kind=kind) if bias else None for _ in range(2))
    return x, wg, wv, bg, bv, normal(gen, rows, outputs, scale=0.1, kind=kind)


def check_gated(x, wg, wv, bg, bv, dh, act):
    kind = x.dtype
    leaves = [v.detach().requires_grad_() for v in (x, wg, wv, bg, bv) if v is not None]
    named = iter(leaves)
    h = F.gated_linear(*[None if v is None else next(named) for v in (x, wg, wv, bg, bv)], activation=act)
    grads = torch.autograd.grad(h, leaves, dh)
    X, G, V, D = (v.detach().double() for v in (x, wg, wv, dh))
    a, u = X @ G.t(), X @ V.t()
    da_, du_ = (lost(X.shape[1] + 2) * (X.abs() @ M.abs().t()) for M in (G, V))
    if bg is not None:
        a, da_ = a + bg.double(), da_ + 2.0 ** -23 * bg.double().abs()
    if bv is not None:
        u, du_ = u + bv.double(), du_ + 2.0 ** -23 * bv.double().abs()
    g, slope = gate(a, act)
    # the activation and its slope as evaluated: 2^-21 in fp32 (a few roundings), 2^-17 where the result is rounded to 16 bits anyway
    eps = (2.0 ** -21 if kind == torch.float32 else 2.0 ** -17) * (1 + a.abs())
    within(h, g * u, (1.2 * da_ + eps) * u.abs() + (g.abs() + 1.2 * da_ + eps) * du_, kind)
    jump = (a.abs() <= da_).double() if act == "relu" else 0.0  # a slope that jumps where a may lie on either side
    ga, gu = D * u * slope, D * g
    Ea = operand_step(kind) * ga.abs() + D.abs() * (1.2 * du_ + u.abs() * (1.2 * da_ + eps + jump))
    Eu = operand_step(kind) * gu.abs() + D.abs() * (1.2 * da_ + eps)
    if kind == torch.float16:
        Ea, Eu = Ea + 2.0 ** -24 * D.abs().amax(), Eu + 2.0 ** -24 * D.abs().amax()
    split = operand_step(kind) if kind == torch.float32 else 0.0
    rows, outputs = dh.shape
    k = lost(2 * outputs) + split
    within(grads[0], ga @ G + gu @ V, Ea @ G.abs() + Eu @ V.abs() + k * (ga.abs() @ G.abs() + gu.abs() @ V.abs()), kind)
    k = lost(rows) + split
    within(grads[1], ga.t() @ X, Ea.t() @ X.abs() + k * (ga.abs().t() @ X.abs()), kind)
    within(grads[2], gu.t() @ X, Eu.t() @ X.abs() + k * (gu.abs().t() @ X.abs()), kind)
    rest = list(grads[3:])
    for bias, q, e in ((bg, ga, Ea), (bv, gu, Eu)):
        if bias is not None:
            within(rest.pop(0), q.sum(0), e.sum(0) + rows * 2.0 ** -24 * q.abs().sum(0), kind)
    return [h.detach(), *grads]


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("act", ["silu", "gelu", "relu", "sigmoid"])
@pytest.mark.parametrize("rows,features,outputs", [
    (1, 1, 1), (1, 64, 700), (2, 9, 64), (8, 33, 65), (16, 100, 129), (127, 128, 63), (130, 65, 257), (300, 257, 128), (513, 40, 1000), (3, 2048, 40)])
def test_gated_linear(kind, act, rows, features, outputs):
    args = gated_inputs(kind, rows, features, outputs, bias=rows != 127)
    check_gated(*args, act)
    with torch.no_grad():  # the call that is not differentiated gives the same
        again = F.gated_linear(*args[:5], activation=act)
    assert torch.equal(again, F.gated_linear(args[0].requires_grad_(), *args[1:5], activation=act).detach())


def test_one_bias_alone_and_some_gradients_alone():
    x, wg, wv, bg, bv, dh = gated_inputs(torch.bfloat16, 140, 72, 200)
    check_gated(x, wg, wv, bg, None, dh, "silu")
    check_gated(x, wg, wv, None, bv, dh, "silu")
    full = check_gated(x, wg, wv, bg, bv, dh, "silu")[1:]
    for wanted in ([0], [1], [2], [3], [4], [1, 4], [0, 2, 3]):
        args = [v.detach().requires_grad_(i in wanted) for i, v in enumerate((x, wg, wv, bg, bv))]
        h = F.gated_linear(*args)
        for i, g in zip(wanted, torch.autograd.grad(h, [args[i] for i in wanted], dh)):
            assert torch.equal(g, full[i])
    x, w, b, t = loss_inputs(torch.bfloat16, 140, 72, 200)
    full = check_loss(x, w, b, t, "mean")[1:]
    for wanted in ([0], [1], [2], [0, 2]):
        args = [v.detach().requires_grad_(i in wanted) for i, v in enumerate((x, w, b))]
        for i, g in zip(wanted, torch.autograd.grad(F.linear_class_loss(*args, t), [args[i] for i in wanted])):
            assert torch.equal(g, full[i])


def test_small_gradients_in_half_precision():
    """Upstream gradients near the smallest fp16 numbers: what they are summed into is as exact as elsewhere."""
    x, wg, wv, bg, bv, dh = gated_inputs(torch.float16, 700, 64, 90)
    check_gated(x, wg, wv, bg, bv, (dh.float() * 1e-4).half(), "silu")
    x, w, b, t = loss_inputs(torch.float16, 700, 64, 900)
    check_loss(x, w, b, t, "none", torch.full((700,), 1e-5, device="cuda"))
    check_loss(x, w, b, t, "none", torch.full((700,), 1e4, device="cuda"))


# ---- both ---------------------------------------------------------------------------------------------------------------

def both(x, w, b, t, reduction="mean", **options):
    """A pass through both operators on the same rows: {outputs and gradients}."""
    leaves = [v.detach().requires_grad_() for v in (x, w, b)]
    loss = F.linear_class_loss(*leaves, t, reduction=reduction)
    h = F.gated_linear(leaves[0], leaves[1], leaves[1], leaves[2], leaves[2])
    return [loss.detach(), h.detach(), *torch.autograd.grad(loss.sum(), leaves), *torch.autograd.grad(h.float().square().sum(), leaves)]


@pytest.mark.parametrize("kind", TYPES)
def test_strides_and_alignment(kind):
    """Rows apart, columns apart, an odd start, more dimensions, one row for all: the values count, not where they lie."""
    for rows in (3, 20, 200):
        x, w, b, t = loss_inputs(kind, rows, 40, 70)
        want = both(x, w, b, t)
        wide = torch.zeros(rows, 48, device="cuda", dtype=kind)
        wide[:, :40] = x
        odd = torch.zeros(rows * 40 + 1, device="cuda", dtype=kind)
        odd[1:] = x.flatten()
        ragged = torch.zeros(rows, 41, device="cuda", dtype=kind)
        ragged[:, 1:] = x
        narrow = torch.zeros(rows, 41, device="cuda", dtype=kind)  # rows apart by an odd number of values, the first one aligned
        narrow[:, :40] = x
        for view in (wide[:, :40], odd[1:].view(rows, 40), ragged[:, 1:], narrow[:, :40], x.t().contiguous().t()):
            assert torch.equal(view, x)
            for got, value in zip(both(view, w, b, t), want):
                assert torch.equal(got, value)
    x, w, b, t = loss_inputs(kind, 60, 40, 70)
    want = both(x, w, b, t)
    odd_w = torch.zeros(70 * 40 + 1, device="cuda", dtype=kind)
    odd_w[1:] = w.flatten()
    odd_b = torch.zeros(71, device="cuda", dtype=kind)
    odd_b[1:] = b
    for got, value in zip(both(x, odd_w[1:].view(70, 40), odd_b[1:], t), want):
        assert torch.equal(got, value)
    for got, value in zip(both(x, w.t().contiguous().t(), b, t), want):
        assert torch.equal(got, value)
    loss = F.linear_class_loss(x.view(3, 20, 40), w, b, t.view(3, 20), reduction="none")
    assert loss.shape == (3, 20) and torch.equal(loss.flatten(), F.linear_class_loss(x, w, b, t, reduction="none"))
    assert torch.equal(F.gated_linear(x.view(3, 20, 40), w, w, b, b), want[1].view(3, 20, 70))
    one = x[:1].expand(60, 40)
    assert torch.equal(F.gated_linear(one, w, w), F.gated_linear(one.contiguous(), w, w))
    row = F.gated_linear(x[5], w, w, b, b)  # a single sample, without a batch
    assert row.shape == (70,) and torch.allclose(row.float(), want[1][5].float(), rtol=2 * torch.finfo(kind).eps, atol=1e-5)
    assert F.linear_class_loss(x[5], w, b, t[5], reduction="none").shape == ()
    h = F.gated_linear(x.requires_grad_(), w, w)
    dh = torch.randn(70, 60, device="cuda").to(kind).t()  # an upstream gradient with its columns apart, and one number for all
    assert torch.equal(torch.autograd.grad(h, x, dh, retain_graph=True)[0], torch.autograd.grad(h, x, dh.contiguous(), retain_graph=True)[0])
    assert torch.equal(torch.autograd.grad(h.sum(), x, retain_graph=True)[0], torch.autograd.grad(h, x, torch.ones_like(h))[0])


@pytest.mark.parametrize("kind", TYPES)
def test_pieces_give_what_the_whole_gives(kind):
    """A bound on the scratch splits the outputs into pieces of 256: sums over the rows keep their bits, those over the outputs their bound."""
    x, w, b, t = loss_inputs(kind, 150, 72, 1000, ignored=True)
    args = gated_inputs(kind, 150, 72, 1000)
    whole, whole_gated = check_loss(x, w, b, t, "mean"), check_gated(*args, "gelu")
    hingetree_cpp.set_backward_scratch_limit(0)
    try:
        pieces, pieces_gated = check_loss(x, w, b, t, "mean"), check_gated(*args, "gelu")
    finally:
        hingetree_cpp.set_backward_scratch_limit(2 ** 63 - 1)
    for a, c in ((whole, pieces), (whole_gated, pieces_gated)):
        for i in [0, *range(2, len(a))]:
            assert torch.equal(a[i], c[i])


def test_the_same_call_gives_the_same_bits():
    for kind in TYPES:
        x, w, b, t = loss_inputs(kind, 1000, 136, 3001, ignored=True)
        first = both(x, w, b, t)
        junk = torch.full((1 << 26,), float("nan"), device="cuda")  # what a workspace holds before does not matter
        del junk
        for a, c in zip(first, both(x, w, b, t)):
            assert torch.equal(a, c)


def test_other_streams_and_captured_graphs():
    x, w, b, t = loss_inputs(torch.bfloat16, 260, 72, 500)
    want = both(x, w, b, t)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = both(x, w, b, t)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, c) for a, c in zip(got, want))
    # two captured steps, replayed in turn on new data
    graphs = []
    with torch.cuda.stream(side):
        for _ in range(2):
            leaves = [v.clone().requires_grad_() for v in (x, w, b)]

            def step(leaves=leaves):
                loss = F.linear_class_loss(*leaves, t)
                h = F.gated_linear(leaves[0], leaves[1], leaves[1], leaves[2], leaves[2])
                return [loss.detach(), h.detach(), *torch.autograd.grad(loss, leaves), *torch.autograd.grad(h.float().square().sum(), leaves)]

            step()
            graph = torch.cuda.CUDAGraph()
            torch.cuda.current_stream().synchronize()
            with torch.cuda.graph(graph, stream=side):
                out = step()
            graphs.append((graph, leaves, out))
    torch.cuda.synchronize()
    fresh = [loss_inputs(torch.bfloat16, 260, 72, 500, seed=k + 1)[:3] for k in range(2)]
    for (graph, leaves, _), values in zip(graphs, fresh):
        for leaf, value in zip(leaves, values):
            leaf.data.copy_(value)
    for order in ((0, 1), (1, 0)):
        for k in order:
            graphs[k][0].replay()
        torch.cuda.synchronize()
        for k in order:
            assert all(torch.equal(a, c) for a, c in zip(graphs[k][2], both(*fresh[k], t)))
    assert hingetree_cpp.pipeline_status() == 0


@pytest.mark.parametrize("kind", TYPES)
def test_what_is_kept_for_the_backward_does_not_change_it(kind):
    """Copies of operands that a forward leaves (fp32, and rows that do not start on 16 bytes): kept, made again, used twice."""
    x, w, b, t = loss_inputs(kind, 150, 75, 300, ignored=True)
    dh = normal(generator(4), 150, 300, kind=kind)

    def run(times):
        leaves = [v.detach().requires_grad_() for v in (x, w, b)]
        out = [F.linear_class_loss(*leaves, t), F.gated_linear(leaves[0], leaves[1], leaves[1], leaves[2], leaves[2])]
        return [[torch.autograd.grad(o, leaves, d, retain_graph=k + 1 < times) for k in range(times)] for o, d in zip(out, (None, dh))]

    kept = run(3)
    hingetree_cpp.set_save_forward(False)
    try:
        again = run(1)
    finally:
        hingetree_cpp.set_save_forward(True)
    for a, c in zip(kept, again):
        for grads in a:
            assert all(torch.equal(g, v) for g, v in zip(grads, c[0]))


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("apart", [75, 80, 83])
def test_hooks_may_lay_out_what_is_saved_anew(kind, apart):
    """Saved tensors that come back with other strides, from the host or in columns: the backward goes by what it is given."""
    x, w, b, t = loss_inputs(kind, 150, 75, 300, ignored=True)
    dh = normal(generator(4), 150, 300, kind=kind)
    wide = torch.zeros(150, apart, device="cuda", dtype=kind)
    wide[:, :75] = x

    def strided(v):
        if v.dim() != 2:
            return v
        home = torch.zeros(v.shape[0], 75 + (-apart) % 16, device="cuda", dtype=v.dtype)
        home[:, :75] = v
        return home[:, :75]

    def run():
        leaves = [wide.detach().requires_grad_(), w.detach().requires_grad_(), b.detach().requires_grad_()]
        rows = leaves[0][:, :75]
        out = [F.linear_class_loss(rows, leaves[1], leaves[2], t), F.gated_linear(rows, leaves[1], leaves[1], leaves[2], leaves[2])]
        return leaves, out

    leaves, out = run()
    want = [torch.autograd.grad(o, leaves, d) for o, d in zip(out, (None, dh))]
    for pack, unpack in ((lambda v: v.cpu(), lambda v: v.cuda()), (strided, lambda v: v), (lambda v: v.t().contiguous().t() if v.dim() == 2 else v, lambda v: v)):
        with torch.autograd.graph.saved_tensors_hooks(pack, unpack):
            leaves, out = run()
        for o, d, grads in zip(out, (None, dh), want):
            assert all(torch.equal(g, v) for g, v in zip(torch.autograd.grad(o, leaves, d), grads))


def test_calls_on_two_streams_at_once():
    """Large and small calls of either operator on two streams, alternately: nothing is shared that they could meet in."""
    cases = [loss_inputs(kind, rows, 136, 900, ignored=True, seed=rows) for kind in TYPES for rows in (5, 100, 900)]
    want = [both(*c) for c in cases]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = {}
    for turn in range(3):
        for k, c in enumerate(cases):
            with torch.cuda.stream(streams[(k + turn) % 2]):
                got[turn, k] = both(*c)
    torch.cuda.synchronize()
    for (_, k), values in got.items():
        assert all(torch.equal(a, v) for a, v in zip(values, want[k]))
    assert hingetree_cpp.pipeline_status() == 0


@pytest.mark.parametrize("rows", [1, 20, 100])
def test_captured_answers(rows):
    """Few rows, captured and replayed on new data, in inference mode too."""
    for kind in TYPES:
        x, w, b, t = loss_inputs(kind, rows, 72, 500)
        y, _, _, s = loss_inputs(kind, rows, 72, 500, seed=9)

        def answer():
            return F.linear_class_loss(x, w, b, t, reduction="none"), F.gated_linear(x, w, w, b, b), F.linear_class_loss(x, w, b, t)

        with torch.inference_mode():
            first = answer()
        graph = torch.cuda.CUDAGraph()
        with torch.no_grad(), torch.cuda.graph(graph):
            out = answer()
        graph.replay()
        assert all(torch.equal(a, c) for a, c in zip(out, first))
        x.copy_(y)
        t.copy_(s)
        graph.replay()
        assert all(torch.equal(a, c) for a, c in zip(out, answer()))


def test_transforms_are_refused():
    x, w, b, t = loss_inputs(torch.float32, 20, 8, 9)
    with pytest.raises(RuntimeError):
        torch.func.vmap(lambda v: F.gated_linear(v, w, w))(x.view(4, 5, 8))
    with pytest.raises((RuntimeError, NotImplementedError)):
        torch.func.jvp(lambda v: F.linear_class_loss(v, w, b, t), (x,), (torch.ones_like(x),))


def test_no_second_derivative():
    x, w, b, t = loss_inputs(torch.float32, 20, 8, 9)
    x.requires_grad_()
    for out in (F.linear_class_loss(x, w, b, t), F.gated_linear(x, w, w).sum()):
        with pytest.raises(RuntimeError, match="second derivative"):
            torch.autograd.grad(out, x, create_graph=True)


def test_gradients_against_differences():
    """Directional derivatives from differences of the operators themselves, fp32: a step of 2^-7 along a random direction, central
    differences, whose error is step^2 / 6 of the third derivative (here below 2^-9 of what is compared) and 2^-22 / 2^-7 of the value."""
    gen = generator(3)
    x, w, b, t = loss_inputs(torch.float32, 90, 33, 130, ignored=True)
    x2, wg, wv, bg, bv, dh = gated_inputs(torch.float32, 90, 33, 70)
    for leaves, value in (([x, w, b], lambda *v: F.linear_class_loss(*v, t, reduction="none").double().sum() / 60),
                          ([x2, wg, wv, bg, bv], lambda *v: (F.gated_linear(*v, activation="silu").double() * dh.double()).sum())):
        leaves = [v.detach().requires_grad_() for v in leaves]
        grads = torch.autograd.grad(value(*leaves), leaves)
        with torch.no_grad():
            for i, leaf in enumerate(leaves):
                direction = normal(gen, *leaf.shape) / math.sqrt(leaf.shape[-1])
                ends = [value(*[v + s * 2.0 ** -7 * direction if j == i else v for j, v in enumerate(leaves)]) for s in (1, -1)]
                difference = (ends[0] - ends[1]).item() * 2.0 ** 6
                along = (grads[i].double() * direction.double()).sum().item()
                size = (grads[i].double().norm() * direction.double().norm()).item()
                assert abs(difference - along) <= 2.0 ** -9 * max(size, abs(along)) + 2.0 ** -15 * abs(ends[0].item())


@pytest.mark.parametrize("kind", TYPES)
def test_modules_take_their_operators(kind):
    gated = R.GatedLinear(24, 40, activation="gelu").cuda().to(kind)
    head = R.LinearClassLoss(40, 11, ignore_index=3).cuda().to(kind)
    x, t = normal(generator(), 50, 24, kind=kind), torch.randint(0, 11, (50,), generator=generator(), device="cuda")
    h = gated(x)
    assert torch.equal(h, F.gated_linear(x, gated.gate_weight, gated.value_weight, gated.gate_bias, gated.value_bias, "gelu"))
    loss = head(h, t)
    assert torch.equal(loss, F.linear_class_loss(h, head.weight, head.bias, t, ignore_index=3))
    loss.backward()
    assert all(p.grad is not None and torch.isfinite(p.grad).all() for p in [*gated.parameters(), *head.parameters()])


@pytest.mark.parametrize("fern", [False, True])
@pytest.mark.parametrize("inner", [(), (3, 2)])
def test_front_forest_and_loss_together(fern, inner):
    """Gated front, forest with its linear layer, class loss: the step's loss and gradients are those of the parts (scores written, torch's
    loss), in fp32 to the parts' own rounding."""
    torch.manual_seed(0)
    front = R.GatedLinear(20, 48).cuda()
    forest = (R.RandomHingeFernFusedLinear if fern else R.RandomHingeForestFusedLinear)(48, 64, 37, 5).cuda()
    with torch.no_grad():  # thresholds among the features
        forest.thresholds.mul_(0.05)
        if not fern:
            forest.fix_thresholds()
    rows = (80, *inner)
    x = torch.randn(*rows, 20, device="cuda")
    t = torch.randint(0, 37, rows, device="cuda")
    t.view(-1)[::5] = -100
    params = [p for m in (front, forest) for p in m.parameters() if p.requires_grad]

    def features():
        h = front(x)
        return h if not inner else h.movedim(-1, 1).contiguous()

    loss = forest.class_loss(features(), t)
    grads = torch.autograd.grad(loss, params)
    f = features()
    trees = (R.RandomHingeFern if fern else R.RandomHingeForest)._function.apply(f, forest.thresholds, forest.ordinals, forest.weights)
    if inner:
        trees = trees.movedim(1, -1)
    scores = trees @ forest.linear_weights.t() + forest.linear_bias
    want = torch.nn.functional.cross_entropy(scores.reshape(-1, 37), t.reshape(-1))
    assert abs(loss.item() - want.item()) <= 1e-5 * abs(want.item())
    for got, value in zip(grads, torch.autograd.grad(want, params)):
        assert (got - value).norm() <= 2e-5 * value.norm() + 1e-12
    assert hingetree_cpp.pipeline_status() == 0


def test_a_traced_front_and_loss_compute_on_new_data():
    front, head = R.GatedLinear(12, 20).cuda(), R.LinearClassLoss(20, 6).cuda()

    class Net(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.front, self.head = front, head

        def forward(self, x, t):
            return self.head(self.front(x), t)

    gen = generator()
    x, y = normal(gen, 30, 12), normal(gen, 30, 12)
    t, s = (torch.randint(0, 6, (30,), generator=gen, device="cuda") for _ in range(2))
    traced = torch.jit.trace(Net(), (x, t), check_trace=False)
    assert torch.equal(traced(y, s), Net()(y, s))


@pytest.mark.parametrize("bias", [False, True])
def test_a_traced_front_is_differentiated(bias):
    front = R.GatedLinear(12, 20, bias=bias, activation="gelu").cuda()
    gen = generator()
    x, y = normal(gen, 30, 12), normal(gen, 30, 12)
    traced = torch.jit.trace(front, (x,), check_trace=False)
    params = list(front.parameters())
    for got, want in zip(torch.autograd.grad(traced(y).square().sum(), params), torch.autograd.grad(front(y).square().sum(), params)):
        assert torch.equal(got, want)


def test_half_a_million_rows_of_few_features():
    """Row counts far beyond a tile, and products of sizes beyond 2^31: offsets are 64 bits wide."""
    rows, features, classes = 530000, 8, 4100  # 2.2e9 scores
    x, w, b, t = loss_inputs(torch.bfloat16, rows, features, classes)
    loss = F.linear_class_loss(x, w, b, t, reduction="none")
    part = slice(rows - 300, rows)
    s = x[part].double() @ w.double().t() + b.double()
    within(loss[part], torch.logsumexp(s, 1) - s.gather(1, t[part, None])[:, 0], 2.0 ** -17, torch.float32)
    h = F.gated_linear(x, w, w, b, b)
    a = x[part].double() @ w.double().t() + b.double()
    within(h[part], gate(a, "silu")[0] * a, 2.0 ** -14 * (1 + a * a), torch.bfloat16)
