"""The dense layers around a forest over the range of their types.

Bounds are an element's own: what another row, output or feature holds does not widen them.  u: half a step of a type.  A sum of K
products loses at most (K + 16) 2^-23 of the sum of their magnitudes (the tensor core truncates when it adds).  fp16 gradients are held as
two bf16 numbers, 2^-17 of their size; one more factor of two is for the products of the two second ones, which are left out.
"""
import ctypes
import math
import os
import random
import subprocess
import sys
import threading

import pytest
import torch

from hingetreefortorch_b200 import HingeTree as F, RandomHingeForest as R, _cabi
from hingetreefortorch_b200._ext import hingetree_cpp
from test_dense_gpu import TYPES, check_gated, check_loss, gate, gated_inputs, generator, lost, loss_inputs, normal, within
from test_dense_host import DenseProblem

pytestmark = pytest.mark.gpu

HELD = {torch.float32: 2.0 ** -22, torch.bfloat16: 2.0 ** -9, torch.float16: 2.0 ** -16}


# ---- gradients of every size -------------------------------------------------------------------------------------------

def check_gated_gradients(x, wg, wv, dh, act):
    kind = x.dtype
    leaves = [v.detach().requires_grad_() for v in (x, wg, wv)]
    grads = torch.autograd.grad(F.gated_linear(*leaves, activation=act), leaves, dh)
    X, G, V, D = (v.detach().double() for v in (x, wg, wv, dh))
    a, u = X @ G.t(), X @ V.t()
    da, du = (lost(X.shape[1]) * (X.abs() @ M.abs().t()) for M in (G, V))
    g, slope = gate(a, act)
    eps = (2.0 ** -21 if kind == torch.float32 else 2.0 ** -17) * (1 + a.abs()) + 1.2 * da
    ga, gu = D * u * slope, D * g
    Ea = HELD[kind] * ga.abs() + D.abs() * (du + u.abs() * eps)
    Eu = HELD[kind] * gu.abs() + D.abs() * eps
    k = lost(2 * dh.shape[1]) + HELD[kind]
    within(grads[0], ga @ G + gu @ V, Ea @ G.abs() + Eu @ V.abs() + k * (ga.abs() @ G.abs() + gu.abs() @ V.abs()), kind)
    k = lost(dh.shape[0]) + HELD[kind]
    within(grads[1], ga.t() @ X, Ea.t() @ X.abs() + k * (ga.abs().t() @ X.abs()), kind)
    within(grads[2], gu.t() @ X, Eu.t() @ X.abs() + k * (gu.abs().t() @ X.abs()), kind)
    return grads


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("act", ["silu", "gelu", "relu"])
def test_large_projections_with_small_gradients(kind, act):
    """u act'(a) or act(a) far beyond 65504 / 2, where h and every gradient are numbers of the type (three rows: a
    weight's gradient is below 3 x 200 x 0.0019 x 40000 x 1.09 = 49704)."""
    x = torch.full((3, 1), 200.0, device="cuda", dtype=kind)
    grads = check_gated_gradients(x, torch.full((3, 1), 1 / 200, device="cuda", dtype=kind), torch.full((3, 1), 200.0, device="cuda", dtype=kind),
                                  torch.full((3, 3), 0.0019, device="cuda", dtype=kind), act)
    assert all(torch.isfinite(g).all() for g in grads)
    # act(a) itself: 60000 with a value of one in 32
    grads = check_gated_gradients(x, torch.full((3, 1), 300.0, device="cuda", dtype=kind), torch.full((3, 1), 1 / 6400, device="cuda", dtype=kind),
                                  torch.full((3, 3), 2.0 ** -12, device="cuda", dtype=kind), act)
    assert all(torch.isfinite(g).all() for g in grads)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("rows,features,outputs", [(64, 64, 90), (300, 72, 200), (9, 75, 33)])
def test_rows_whose_gradients_differ_in_size(kind, rows, features, outputs):
    """One row's gradients are a million times the others': each row's result is as exact as it would be alone."""
    x, wg, wv, _, _, dh = gated_inputs(kind, rows, features, outputs, bias=False)
    dh = dh.float() * 1e-2
    dh[rows // 2] *= 1e6
    for act in ("silu", "relu"):
        check_gated_gradients(x, wg, wv, dh.to(kind), act)


def check_loss_gradients(x, w, t, grad, ignore=-100):
    kind = x.dtype
    leaves = [v.detach().requires_grad_() for v in (x, w)]
    grads = torch.autograd.grad(F.linear_class_loss(*leaves, None, t, ignore_index=ignore, reduction="none"), leaves, grad)
    X, W = (v.detach().double() for v in (x, w))
    s = X @ W.t()
    ds = lost(X.shape[1]) * (X.abs() @ W.abs().t()).amax(1, keepdim=True)
    r = torch.where(t != ignore, grad.double(), 0.0)[:, None]
    p = torch.softmax(s, 1)
    g = p.scatter_add(1, torch.where(t != ignore, t, 0)[:, None], torch.full_like(r, -1.0)) * r
    E = HELD[kind] * g.abs() + r.abs() * (p * (2 * ds + 2.0 ** -20) + 2.0 ** -24)
    within(grads[0], g @ W, E @ W.abs() + (lost(W.shape[0]) + HELD[kind]) * (g.abs() @ W.abs()), kind)
    within(grads[1], g.t() @ X, E.t() @ X.abs() + (lost(X.shape[0]) + HELD[kind]) * (g.abs().t() @ X.abs()), kind)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("rows,features,classes", [(64, 64, 300), (200, 75, 1000)])
def test_losses_whose_gradients_differ_in_size(kind, rows, features, classes):
    x, w, _, t = loss_inputs(kind, rows, features, classes, bias=False)
    grad = normal(generator(2), rows).abs() * 1e-2 + 1e-3
    grad[::7] *= 1e6
    check_loss_gradients(x, w, t, grad)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("junk", [3e38, math.inf, math.nan])
def test_the_upstream_gradient_of_a_row_that_does_not_count(kind, junk):
    x, w, _, t = loss_inputs(kind, 100, 72, 300, bias=False, ignored=True)
    grad = torch.where(t == -100, torch.full((100,), junk, device="cuda"), torch.full((100,), 1e-3, device="cuda"))
    clean = torch.where(t == -100, torch.zeros_like(grad), grad)
    leaves = [v.detach().requires_grad_() for v in (x, w)]
    loss = F.linear_class_loss(*leaves, None, t, reduction="none")
    want = torch.autograd.grad(loss, leaves, clean, retain_graph=True)
    for got, value in zip(torch.autograd.grad(loss, leaves, grad), want):
        assert torch.equal(got, value)
    check_loss_gradients(x, w, t, clean)


# ---- values of every size ----------------------------------------------------------------------------------------------

@pytest.mark.parametrize("rows", [1, 20, 100, 300])
@pytest.mark.parametrize("features", [33, 64])
def test_the_largest_numbers(rows, features):
    """The largest fp32 numbers are numbers, however many rows there are: as a feature beside small weights, and as a weight."""
    top = torch.finfo(torch.float32).max
    gen = generator(rows)
    x, w = normal(gen, rows, features), normal(gen, 70, features, scale=1e-29)
    x[:, 3], x[0, 5], x[rows // 2, 7] = top, -top, float.fromhex("0x1.ffep127")  # (the last one: the first that rounds to infinity at 11 bits)
    zero, one = torch.zeros_like(w), torch.ones(70, device="cuda")
    s, ds = x.double() @ w.double().t(), lost(features) * (x.double().abs() @ w.double().abs().t())
    within(F.gated_linear(x, w, zero, None, one, "relu"), s.clamp_min(0), ds, torch.float32)
    t = torch.arange(rows, device="cuda") % 70
    loss = F.linear_class_loss(x, w, None, t, reduction="none")
    within(loss, torch.logsumexp(s, 1) - s.gather(1, t[:, None])[:, 0], 2 * ds.amax(1) + 2.0 ** -20, torch.float32)
    swapped = F.gated_linear(w[:rows % 70], x[:70], torch.zeros_like(x[:70]), None, one[:min(rows, 70)], "relu")  # weights and features change places
    within(swapped, s[:70, :rows % 70].t().clamp_min(0), ds[:70, :rows % 70].t(), torch.float32)


@pytest.mark.parametrize("kind", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows", [20, 400])
def test_the_tails_of_gelu(kind, rows):
    """The normal distribution function far out is as exact as in the middle: within 2^-15 of itself (its fit 2^-16.9, the exponential of up to 84,
    rounded as fp32, 2^-17.5, a quotient), then the type's rounding.  A value of 1024 lifts what fp16 would lose among its smallest numbers."""
    x = torch.linspace(-12.9, 12.9, rows, device="cuda").to(kind)[:, None].requires_grad_()
    one, zero = torch.ones(8, 1, device="cuda", dtype=kind), torch.zeros(8, 1, device="cuda", dtype=kind)
    h = F.gated_linear(x, one, zero, None, torch.full((8,), 1024.0, device="cuda", dtype=kind), "gelu")
    a = x.detach().double()
    phi, density = 0.5 * torch.erfc(-a / math.sqrt(2)), torch.exp(-a * a / 2) / math.sqrt(2 * math.pi)
    within(h, (1024 * a * phi).expand(-1, 8), 2.0 ** -15 * 1024 * a.abs() * phi, kind)
    dx, = torch.autograd.grad(h, x, torch.eye(8, device="cuda", dtype=kind)[:1].expand(rows, 8))
    within(dx, 1024 * (phi + a * density), (2.0 ** -15 + HELD[kind]) * 1024 * (phi + a.abs() * density), kind)


# ---- fp32 as exact as fp32 ---------------------------------------------------------------------------------------------
# In norm, for random numbers.  Three bf16 numbers a value and six products leave 2^-24 of a term.  The kernels for few rows add every 16 terms
# in fp32: a truncation of 2^-23 at the most, a rounding of 2^-24 at each of K / 16 additions in several strands; a sum of K fp32 products loses as much.
# Bound 2^-22.  The tiles add 16 times in the tensor core, which truncates each time, up to 2^-23 of half the sum on average: 2^-20, and
# 2^-22 for the rest.  (Two bf16 numbers and three products would be off by 4e-6, two TF32 numbers and three products by 2.6e-7.)

def off(got, want):
    return ((got.double() - want).norm() / want.norm()).item()


@pytest.mark.parametrize("rows,bound", [(1, 2.0 ** -22), (5, 2.0 ** -22), (13, 2.0 ** -22), (30, 2.0 ** -22), (64, 2.0 ** -22), (128, 2.0 ** -22),
                                        (129, 1.25 * 2.0 ** -20), (700, 1.25 * 2.0 ** -20)])
@pytest.mark.parametrize("features", [64, 336, 1024, 2048])
@pytest.mark.parametrize("one_sign", [False, True])
def test_fp32_products_in_norm(rows, bound, features, one_sign):
    gen = generator(rows + features)
    x, w = normal(gen, rows, features), normal(gen, 600, features, scale=features ** -0.5)
    if one_sign:
        x, w = x.abs(), w.abs()
    s = x.double() @ w.double().t()
    h = F.gated_linear(x, w, torch.zeros_like(w), None, torch.ones(600, device="cuda"), "relu")
    assert off(h, s.clamp_min(0)) <= bound
    # a loss of scores with that error: the score's own, and 2^-23 of rounding and exponentials
    t = torch.randint(0, 600, (rows,), generator=gen, device="cuda")
    want = torch.logsumexp(s, 1) - s.gather(1, t[:, None])[:, 0]
    error = (F.linear_class_loss(x, w, None, t, reduction="none").double() - want).norm() / (s.norm() / 600 ** 0.5 + want.norm())
    assert error <= 2 * bound


@pytest.mark.parametrize("rows,features,outputs", [(8, 1024, 1000), (100, 336, 500), (300, 200, 513), (1024, 784, 2048), (5000, 333, 700)])
def test_fp32_gradients_in_norm(rows, features, outputs):
    """Two products one after the other, each as above, and the activation's 2^-21."""
    x, wg, wv, bg, bv, dh = gated_inputs(torch.float32, rows, features, outputs)

    def gradients(*given):
        leaves = [v.detach().requires_grad_() for v in given[:-1]]
        x, wg, wv, bg, bv = leaves
        h = F.gated_linear(*leaves) if x.dtype == torch.float32 else torch.nn.functional.silu(x @ wg.t() + bg) * (x @ wv.t() + bv)
        return torch.autograd.grad(h, leaves, given[-1])

    for got, want in zip(gradients(x, wg, wv, bg, bv, dh), gradients(*(v.double() for v in (x, wg, wv, bg, bv, dh)))):
        assert off(got, want) <= 2.5 * 2.0 ** -20 + 2.0 ** -21
    x, w, b, t = loss_inputs(torch.float32, rows, features, outputs)
    grads = []
    for kind in (torch.float32, torch.float64):
        leaves = [v.detach().to(kind).requires_grad_() for v in (x, w, b)]
        loss = F.linear_class_loss(*leaves, t) if kind == torch.float32 else torch.nn.functional.cross_entropy(leaves[0] @ leaves[1].t() + leaves[2], t)
        grads.append(torch.autograd.grad(loss, leaves))
    for got, want in zip(*grads):  # (scores of some units: their error enters as it is)
        assert off(got, want) <= 4 * 1.25 * 2.0 ** -20


# ---- little memory -----------------------------------------------------------------------------------------------------

def test_a_backward_without_room_for_the_whole_gradient_takes_pieces():
    """105 MB of score gradients, 60 MB to be had: pieces, although the bound on the scratch would admit all."""
    x, w, _, t = loss_inputs(torch.bfloat16, 4096, 64, 12800, bias=False)
    leaves = [v.requires_grad_() for v in (x, w)]
    want = torch.autograd.grad(F.linear_class_loss(*leaves, None, t), leaves)
    loss = F.linear_class_loss(*leaves, None, t)
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    total = torch.cuda.get_device_properties(0).total_memory
    torch.cuda.set_per_process_memory_fraction((torch.cuda.memory_reserved() + (60 << 20)) / total)
    try:
        got = torch.autograd.grad(loss, leaves)
    finally:
        torch.cuda.set_per_process_memory_fraction(1.0)
    # the same products, added in fp32 in another order (dx piece by piece, dw by how many tiles a piece has): either is off by half a step
    # of bf16, 2^-9, and by far less in its sums, so they differ by 2^-8 at the most
    for a, b in zip(got, want):
        assert (a.float() - b.float()).norm() <= 2.0 ** -8 * b.float().norm()


# ---- targets that are no class -----------------------------------------------------------------------------------------

def test_a_bad_target_leaves_other_operators_alone():
    """A forest's first call on its ordinals reads the status word: it has its own result, and the flag waits for pipeline_status()."""
    x, w, _, t = loss_inputs(torch.float32, 20, 8, 9, bias=False)
    t[4] = 9
    assert hingetree_cpp.pipeline_status() == 0
    assert torch.isnan(F.linear_class_loss(x, w, None, t))
    forest = R.RandomHingeForest(8, 5, 3).cuda()
    first = forest(x)
    forest.ordinals.copy_(forest.ordinals.clone())  # (a new version: looked at again)
    assert torch.equal(forest(x), first)
    with pytest.raises(RuntimeError, match="neither a class"):
        hingetree_cpp.pipeline_status()
    assert hingetree_cpp.pipeline_status() == 0


FIRST_CALL = """
import torch
from hingetreefortorch_b200 import HingeTree as F
from hingetreefortorch_b200._ext import hingetree_cpp
x, w, t = torch.randn(200, 8, device="cuda"), torch.randn(9, 8, device="cuda"), torch.full((200,), 9, device="cuda")
torch.cuda.synchronize()
%s
torch.cuda.synchronize()
for _ in range(2):
    try:
        print("status", hingetree_cpp.pipeline_status())
    except RuntimeError as e:
        print("raised", "neither a class" in str(e))
"""


@pytest.mark.parametrize("call", [
    "graph = torch.cuda.CUDAGraph()\nwith torch.no_grad(), torch.cuda.graph(graph):\n    F.linear_class_loss(x, w, None, t)\ngraph.replay()",
    "with torch.inference_mode():\n    F.linear_class_loss(x, w, None, t)",
    "with torch.no_grad(), torch.cuda.stream(torch.cuda.Stream()):\n    F.linear_class_loss(x, w, None, t)"])
def test_a_bad_target_in_the_first_call_of_a_process(call):
    """Captured, in inference mode, on another stream: the flag is there afterwards, once."""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    run = subprocess.run([sys.executable, "-c", FIRST_CALL % call], cwd=root, capture_output=True, text=True, timeout=300)
    assert run.returncode == 0, run.stderr[-2000:]
    assert run.stdout.split("\n")[:2] == ["raised True", "status 0"]


# ---- threads -----------------------------------------------------------------------------------------------------------

def test_the_first_call_of_a_thread():
    """An entry of the library is the first that a thread asks of CUDA: nothing has made the device's context current there."""
    lib = _cabi.library()
    lib.ht_linear_class_loss_workspace_bytes.restype = ctypes.c_size_t
    x, w, _, t = loss_inputs(torch.bfloat16, 300, 64, 500, bias=False)
    p = DenseProblem(1, 0, 300, 64, 500, 64, 0)
    ws = torch.empty(lib.ht_linear_class_loss_workspace_bytes(ctypes.byref(p), 0), dtype=torch.uint8, device="cuda")
    loss = torch.zeros(300, device="cuda")
    torch.cuda.synchronize()
    status = []

    def call():
        at = [ctypes.c_void_p(v.data_ptr()) for v in (x, w, t, loss, ws)]
        status.append(lib.ht_linear_class_loss_forward(ctypes.byref(p), at[0], at[1], None, at[2], ctypes.c_int64(-100), 0, at[3], None, None, at[4],
                                                       ctypes.c_size_t(ws.numel()), None, None))

    thread = threading.Thread(target=call)
    thread.start()
    thread.join()
    torch.cuda.synchronize()
    assert status == [0] and torch.equal(loss, F.linear_class_loss(x, w, None, t, reduction="none"))


# ---- long sums ---------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("kind", TYPES)
def test_gradients_summed_over_many_rows_of_one_sign(kind):
    """400000 rows, every term positive and exact in the type: a weight's and a bias's gradient within one step of the sum."""
    rows = 400000
    x = (torch.randint(128, 256, (rows, 40), generator=generator(), device="cuda").float() / 128).to(kind)
    wg, bg = torch.zeros(64, 40, device="cuda", dtype=kind), torch.ones(64, device="cuda", dtype=kind)
    leaves = [v.clone().requires_grad_() for v in (wg, wg, bg, bg)]
    h = F.gated_linear(x, *leaves, "relu")
    grads = torch.autograd.grad(h, leaves, torch.full_like(h, 2.0 ** -14))
    step = 2.0 ** -19 if kind == torch.float32 else torch.finfo(kind).eps  # (fp32: 2^-23 of half of 256 terms' sums, 32 times: 2^-20)
    for got, want in zip(grads, [2.0 ** -14 * x.double().sum(0)] * 2 + [torch.full((), 2.0 ** -14 * rows, device="cuda", dtype=torch.float64)] * 2):
        assert ((got.double() - want).abs() <= step * want).all()


# ---- calls at random ---------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("seed", range(24))
def test_calls_at_random(seed):
    """Sizes, types, reductions, biases and strides drawn at random, against the formulas in 64 bits."""
    rng = random.Random(seed)

    def size(low, high):
        return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))

    rows, features, outputs, kind = size(1, 3000), size(1, 1500), size(1, 3000), rng.choice(TYPES)
    bias, act, reduction = rng.random() < 0.5, rng.choice(["silu", "gelu", "relu", "sigmoid"]), rng.choice(["none", "mean", "sum"])

    def strided(v):  # rows apart by a few more values than they have, or as they are
        home = torch.zeros(v.shape[0], v.shape[1] + rng.choice([0, 1, 3, 8]), device="cuda", dtype=kind)
        home[:, :v.shape[1]] = v
        return home[:, :v.shape[1]]

    x, wg, wv, bg, bv, dh = gated_inputs(kind, rows, features, outputs, bias=bias, seed=seed)
    check_gated(strided(x), wg, strided(wv), bg, bv, dh, act)
    x, w, b, t = loss_inputs(kind, rows, features, outputs, bias=bias, ignored=rows > 2 and rng.random() < 0.5, seed=seed)
    grad = normal(generator(seed), rows, scale=2.0) if reduction == "none" else torch.tensor(1.7, device="cuda")
    check_loss(strided(x), strided(w), b, t, reduction, grad)


# ---- forests with sparse gradients -------------------------------------------------------------------------------------

@pytest.mark.parametrize("sparse,dense", [(R.SparseRandomHingeForestFusedLinear, R.RandomHingeForestFusedLinear),
                                          (R.SparseRandomHingeFernFusedLinear, R.RandomHingeFernFusedLinear)])
def test_the_class_loss_of_a_sparse_forest_keeps_its_gradients_sparse(sparse, dense):
    """As forward() does: thresholds and leaf weights sparse, the linear layer's and x's dense, with the dense forest's values."""
    torch.manual_seed(1)
    forests = [sparse(10, 30, 6, 4).cuda(), dense(10, 30, 6, 4).cuda()]
    forests[1].load_state_dict(forests[0].state_dict())
    x, t = torch.randn(50, 10, device="cuda"), torch.randint(0, 6, (50,), device="cuda")
    inputs = [x.clone().requires_grad_() for _ in range(2)]
    losses = [f.class_loss(v, t) for f, v in zip(forests, inputs)]
    assert torch.equal(*losses)
    for loss in losses:
        loss.backward()
    for name, p in forests[0].named_parameters():
        if p.requires_grad:
            other = dict(forests[1].named_parameters())[name].grad
            assert p.grad.is_sparse == (name in ("thresholds", "weights")), name
            # the same terms, added in an order that is free
            assert torch.allclose(p.grad.to_dense(), other, rtol=1e-5, atol=1e-6 * other.abs().max().item())
    assert not inputs[0].grad.is_sparse and torch.allclose(inputs[0].grad, inputs[1].grad, rtol=1e-5, atol=1e-6)
