"""Answers of a linear layer with many classes (pack_mx4, unpack_mx4, linear_mx4, sample_classes) against their formulas in 64 bits.

Packing and unpacking are exact.  A score: a sum of K products loses at most (K + 16) 2^-23 of the sum of their magnitudes (the tensor core truncates when
it adds), fp32 x is held to 2^-23 (three bf16 numbers), and the result is rounded to its type.  A drawn class is the formula's: weights and sums are held
to some 1e-13 where that decides, and no case here comes that near to a border but where both sides are exact.  The logarithm of its share is rounded to
fp32, 2^-24 of it, and what counts may have been summed in fp32: w = 2^y, y = (s - m) / (T ln 2), with the hardware's exponential (2^-22 of w), sums of
8 (3 2^-24) and three roundings of y (3 2^-24 |y| ln 2 of w): 2^-22 + 3 2^-24 < 4.2e-7 and 3 2^-24 ln 2 < 1.25e-7 times the mean of |y|.
"""
import gc
import math

import pytest
import torch

from hingetreefortorch_b200 import HingeTree as F, RandomHingeForest as R
from hingetreefortorch_b200._ext import hingetree_cpp
from test_dense_gpu import generator, lost, normal, within

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]
NUMBERS = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


@pytest.fixture(scope="module", autouse=True)
def nothing_stays():
    """What these tests leave in the allocator's cache goes before those that count bytes."""
    yield
    gc.collect()
    torch.cuda.empty_cache()


# ---- packed weights ----------------------------------------------------------------------------------------------------

def pack(w):
    """codes [outputs, 32 blocks] one by one, scales [outputs, blocks], by distances in 64 bits."""
    outputs, features = w.shape
    blocks = -(-features // 32)
    v = torch.zeros(outputs, 32 * blocks, dtype=torch.float64, device=w.device)
    v[:, :features] = w.double()
    v = v.view(outputs, blocks, 32)
    top = v.abs().amax(2)
    broken = ~torch.isfinite(v).all(2)
    top = torch.where(broken | (top == 0), torch.full_like(top, 2.0 ** -149), top)
    scale = (torch.frexp(top)[1] - 1 - 2).clamp_min(-127)
    a = (torch.where(broken[:, :, None], torch.zeros_like(v), v).abs() * torch.exp2(-scale.double())[:, :, None])
    grid = torch.tensor(NUMBERS, dtype=torch.float64, device=w.device)
    order = torch.tensor([0, 2, 4, 6, 1, 3, 5, 7], device=w.device)  # of two as near the even one comes first
    code = order[(a[..., None] - grid[order]).abs().argmin(-1)]
    code = torch.where(broken[:, :, None], torch.zeros_like(code), code + 8 * torch.signbit(v))
    return code.flatten(1), torch.where(broken, torch.full_like(scale, 255), scale + 127)


def values(codes, scales, features):
    """In 64 bits, of codes as they are stored."""
    grid = torch.tensor(NUMBERS + [-n for n in NUMBERS], dtype=torch.float64, device=codes.device)
    v = grid[torch.stack([codes & 15, codes >> 4], 2).flatten(1).long()]
    power = torch.where(scales == 255, torch.full(scales.shape, math.nan, dtype=torch.float64, device=codes.device), torch.exp2(scales.double() - 127))
    return (v * power.repeat_interleave(32, 1))[:, :features]


def check_pack(w):
    codes, scales = F.pack_mx4(w)
    want, power = pack(w.contiguous())
    assert codes.dtype == scales.dtype == torch.uint8 and codes.is_contiguous() and scales.is_contiguous()
    assert torch.equal(scales.long(), power.long())
    assert torch.equal(torch.stack([codes & 15, codes >> 4], 2).flatten(1).long(), want)
    v = values(codes, scales, w.size(1))
    for kind in TYPES:
        got = F.unpack_mx4(codes, scales, w.size(1), dtype=kind)
        assert got.dtype == kind and torch.equal(torch.nan_to_num(got, 123.0), torch.nan_to_num(v.to(kind), 123.0))
    return codes, scales


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("outputs,features", [(1, 1), (3, 7), (2, 31), (5, 32), (4, 33), (7, 64), (129, 100), (33, 257), (1000, 40), (17, 1031), (2, 70001)])
def test_pack(kind, outputs, features):
    gen = generator(outputs)
    check_pack(normal(gen, outputs, features, kind=kind))
    spread = torch.exp2(torch.randint(-20, 15, (outputs, 1), generator=gen, device="cuda").float())
    check_pack((torch.randn(outputs, features, generator=gen, device="cuda") * spread).to(kind))


@pytest.mark.parametrize("kind", TYPES)
def test_pack_borders(kind):
    """Every midpoint and number with its neighbours, the smallest and largest numbers, zeros, blocks with an infinity or NaN."""
    rows = []
    near = torch.tensor(NUMBERS + [0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.0, 7.9])
    for power in (0, -8, 5, -14):
        base = (near * 2.0 ** power).to(kind)
        down, up = (torch.nextafter(base, torch.full_like(base, to)) for to in (-1e4, 1e4))
        for top in (4.0, 6.0, 7.5):  # what makes the scale 2 ** power
            for part in (base, down, up):
                block = torch.cat([part[:17], -part[:14], torch.tensor([top * 2.0 ** power], dtype=kind)])
                rows.append(torch.where(block.abs() < 8 * 2.0 ** power, block, torch.zeros_like(block)))
    info = torch.finfo(kind)
    rows += [torch.full((32,), v, dtype=kind) for v in (0.0, -0.0, info.tiny, info.max, -info.max, info.tiny * info.eps)]
    for bad in (math.inf, -math.inf, math.nan):
        row = torch.ones(32, dtype=kind)
        row[11] = bad
        rows.append(row)
    w = torch.stack(rows).cuda()
    codes, scales = check_pack(w)
    assert (scales[-3:] == 255).all() and not codes[-3:].any()
    check_pack(torch.cat([w, w.flip(0)[:, :9]], 1))


def test_pack_strides():
    wide = normal(generator(1), 40, 100)
    for w in (wide[:, :64], wide[:, 3:90], wide[::3], wide.t(), wide[:, ::2], wide[:1], wide[:, :1], wide[5:6].expand(4, 100), wide[:, :1].expand(40, 30)):
        codes, scales = check_pack(w)
        assert all(torch.equal(a, b) for a, b in zip((codes, scales), F.pack_mx4(w.contiguous())))
    leaf = wide.clone().requires_grad_()
    codes, scales = F.pack_mx4(leaf)
    assert not codes.requires_grad and torch.equal(codes, F.pack_mx4(wide)[0])


def test_unpack_every_code_and_scale():
    codes = torch.arange(256, device="cuda", dtype=torch.uint8).view(1, 256).repeat(256, 1)
    scales = torch.arange(256, device="cuda", dtype=torch.uint8).view(256, 1).repeat(1, 16)
    v = values(codes, scales, 512)
    for kind in TYPES:
        got = F.unpack_mx4(codes, scales, 512, dtype=kind)
        want = v.to(torch.float32).to(kind)  # (exact in fp32 but where it is too large for that)
        assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(torch.nan_to_num(got, 0.0), torch.nan_to_num(want, 0.0))


# ---- scores ------------------------------------------------------------------------------------------------------------

def check_linear(x, codes, scales, bias):
    kind, features = x.dtype, x.size(-1)
    result = got = F.linear_mx4(x, codes, scales, bias)
    w = values(codes, scales, features)
    want = x.double() @ w.t()
    terms = x.double().abs() @ w.abs().t()
    if bias is not None:
        want, terms = want + bias.double(), terms + bias.double().abs()
    assert got.dtype == kind and got.shape == (*x.shape[:-1], codes.size(0))
    finite = torch.isfinite(x).all(-1)  # a row of x with an infinity has sums of infinities and no numbers: nothing to compare
    if not finite.all():
        got, want, terms = got[finite], want[finite], terms[finite]
    # (within: half a step of the result's type besides; fp16 results may be infinite where the exact ones are beyond its numbers)
    within(got, want, (lost(features + 1) + (2.0 ** -23 if kind == torch.float32 else 0.0)) * terms, kind)
    return result


def linear_inputs(kind, rows, features, outputs, bias=True, seed=0):
    gen = generator(seed)
    x = normal(gen, rows, features, kind=kind)
    codes, scales = F.pack_mx4(normal(gen, outputs, features, scale=1 / math.sqrt(features)))
    return x, codes, scales, normal(gen, outputs, scale=0.5, kind=kind) if bias else None


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("rows,features,outputs", [
    (1, 1, 1), (1, 64, 7), (2, 7, 16), (3, 31, 17), (5, 32, 64), (8, 33, 100), (9, 127, 129), (16, 128, 1000), (17, 129, 33), (1, 784, 12700), (31, 1000, 257),
    (33, 255, 300), (64, 2048, 130), (65, 2049, 40), (7, 5000, 50), (100, 771, 1003), (127, 96, 500), (128, 128, 128), (129, 640, 260), (192, 64, 127), (193, 72, 129),
    (300, 513, 700), (400, 100, 3), (1, 40000, 20), (1000, 24, 2000)])
def test_linear(kind, rows, features, outputs):
    x, codes, scales, bias = linear_inputs(kind, rows, features, outputs, bias=rows % 2 == 1)
    first = check_linear(x, codes, scales, bias)
    assert torch.equal(first, F.linear_mx4(x, codes, scales, bias))


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("rows", [3, 40, 200])
def test_linear_by_scale(kind, rows):
    """Blocks of very different size, the smallest and largest powers of two among them, beside an x that keeps the products in range; a row that
    holds no number; codes of which every one occurs."""
    gen = generator(rows)
    codes = torch.randint(0, 256, (90, 64), generator=gen, device="cuda", dtype=torch.int32).to(torch.uint8)
    for low, high, size in ((100, 140, 1.0), (0, 40, 2.0 ** 15), (135, 165, 1.0), (190, 254, 2.0 ** -14)):
        scales = torch.randint(low, high, (90, 4), generator=gen, device="cuda", dtype=torch.int32).to(torch.uint8)
        x = normal(gen, rows, 128, scale=size, kind=kind)
        if kind == torch.float16 and low >= 135:  # results beyond fp16's numbers
            scales[:, :] = scales // 32 + 120
        if kind != torch.float16 and high == 254:
            x = x * 2.0 ** -90
        check_linear(x, codes, scales, None)
    scales[7, 2] = 255
    got = F.linear_mx4(x, codes, scales)
    assert torch.isnan(got[:, 7]).all() and not torch.isnan(got[:, :7]).any() and not torch.isnan(got[:, 8:]).any()


@pytest.mark.parametrize("rows,features,outputs,apart", [(1024, 1024, 10007, 1024), (1100, 519, 20011, 519), (2050, 200, 26000, 211), (5000, 2049, 1001, 2056)])
def test_linear_of_many_rows(rows, features, outputs, apart):
    """bf16 rows and products enough that the weights are decoded once, into memory; blocks of every size, one that holds no number."""
    gen = generator(rows)
    wide = normal(gen, rows, apart, kind=torch.bfloat16)
    codes, scales = F.pack_mx4(normal(gen, outputs, features, scale=1 / math.sqrt(features)))
    bias = normal(gen, outputs, scale=0.5, kind=torch.bfloat16)
    first = check_linear(wide[:, :features], codes, scales, bias)
    assert torch.equal(first, F.linear_mx4(wide[:, :features].contiguous(), codes, scales, bias))
    for low, high, size in ((0, 40, 2.0 ** 15), (190, 254, 2.0 ** -104)):
        scales = torch.randint(low, high, scales.shape, generator=gen, device="cuda", dtype=torch.int32).to(torch.uint8)
        check_linear(wide[:, :features] * size, codes, scales, None)
    scales[7, -1] = 255
    got = F.linear_mx4(wide[:, :features] * size, codes, scales)
    assert torch.isnan(got[:, 7]).all() and not torch.isnan(got[:, :7]).any() and not torch.isnan(got[:, 8:]).any()
    assert hingetree_cpp.pipeline_status() == 0


@pytest.mark.parametrize("kind", TYPES)
def test_linear_strides_and_shapes(kind):
    x, codes, scales, bias = linear_inputs(kind, 60, 200, 90)
    wide = normal(generator(2), 60, 211, kind=kind)
    for rows in (2, 60):
        for v in (wide[:rows, :200], wide[:rows, 3:203], wide[:rows, 8:208], wide[:, :200][:rows].t().contiguous().t()):
            got = check_linear(v, codes, scales, bias)
            assert torch.equal(got, F.linear_mx4(v.contiguous(), codes, scales, bias))
    y = F.linear_mx4(x, codes, scales, bias)
    assert torch.equal(F.linear_mx4(x.view(3, 4, 5, 200), codes, scales, bias), y.view(3, 4, 5, 90))
    assert F.linear_mx4(x[5], codes, scales, bias).shape == (90,)
    assert F.linear_mx4(x[:0], codes, scales, bias).shape == (0, 90) and F.linear_mx4(x[:0].view(0, 3, 200), codes, scales).shape == (0, 3, 90)
    odd = torch.zeros(codes.numel() + 5, dtype=torch.uint8, device="cuda")[5:].view_as(codes).copy_(codes)  # not on 16 bytes
    assert torch.equal(F.linear_mx4(x, odd, scales.t().contiguous().t(), bias), y)
    assert torch.equal(F.linear_mx4(wide[:7, :200].expand(7, 200)[:1].expand(9, 200), codes, scales), F.linear_mx4(wide[:1, :200].repeat(9, 1), codes, scales))


def test_no_derivatives():
    x, codes, scales, bias = linear_inputs(torch.float32, 4, 40, 9)
    with pytest.raises(RuntimeError, match="no derivative"):
        F.linear_mx4(x.requires_grad_(), codes, scales, bias)
    with pytest.raises(RuntimeError, match="no derivative"):
        F.linear_mx4(x.detach(), codes, scales, bias.requires_grad_())
    with pytest.raises(RuntimeError, match="no derivative"):
        F.sample_classes(x, torch.rand(4, device="cuda"))
    with torch.no_grad():
        y = F.linear_mx4(x, codes, scales, bias)
        F.sample_classes(x, torch.rand(4, device="cuda"))
    assert not y.requires_grad
    with pytest.raises(RuntimeError, match="no derivative"):
        torch.func.jvp(lambda v: F.linear_mx4(v, codes, scales), (x.detach(),), (torch.ones_like(x),))


# ---- draws -------------------------------------------------------------------------------------------------------------

def draw(scores, uniform, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """The definition, row by row, in 64 bits on the host."""
    import numpy as np
    s, u = scores.double().cpu().numpy(), uniform.double().cpu().numpy()
    rows = [v.double().cpu().numpy() if torch.is_tensor(v) else np.full(len(u), float(v)) for v in (temperature, top_k, top_p, min_p)]
    classes, logs, powers = np.full(len(u), -1, dtype=np.int64), np.full(len(u), np.nan), np.zeros(len(u))
    for r, (t, k, p, least) in enumerate(zip(*rows)):
        v = s[r]
        if np.isnan(v).any() or not np.isfinite(v.max()) or not (0 <= t < math.inf) or not 0 <= u[r] <= 1 or p != p or least != least:
            continue
        order = np.argsort(-v, kind="stable")
        if t == 0:
            order, w = order[:1], np.ones(1)
        else:
            w = np.exp((v[order] - v.max()) / t)
        n = len(order) if k < 1 else min(int(k), len(order))
        before = np.concatenate([[0.0], np.cumsum(w[:n])[:-1]])
        if p < 1:
            n = max(int((before < p * w[:n].sum()).sum()), 1)
        n = max(int((w[:n] >= least).sum()), 1)
        held = np.sort(order[:n])
        weight = np.exp((v[held] - v.max()) / t) if t > 0 else np.ones(1)
        upto = np.cumsum(weight)
        at = int(np.searchsorted(upto, u[r] * upto[-1], side="right"))
        if at == len(held):
            at = int(np.flatnonzero(weight > 0)[-1])
        # (not the logarithm of the weight, which may be a subnormal number of few bits)
        classes[r], logs[r] = held[at], (v[held[at]] - v.max()) / (t if t > 0 else 1.0) - np.log(upto[-1])
        some = weight > 0
        powers[r] = (weight[some] * np.abs(v[held][some] - v.max())).sum() / (t if t > 0 else 1.0) / math.log(2) / upto[-1]
    return torch.from_numpy(classes), torch.from_numpy(logs), torch.from_numpy(powers)


def check_draw(scores, uniform, **bounds):
    got, logs = F.sample_classes(scores, uniform, **bounds)
    want, exact, powers = draw(scores, uniform, **bounds)
    assert got.dtype == torch.int64 and logs.dtype == torch.float32
    wrong = (got.cpu() != want).nonzero()[:, 0]
    assert len(wrong) == 0, [(int(r), int(got[r]), int(want[r])) for r in wrong[:5]]
    logs = logs.cpu().double()
    assert torch.equal(torch.isnan(logs), torch.isnan(exact))
    off = (logs - exact).abs() / (2.0 ** -24 * exact.abs() + 4.3e-7 + 1.25e-7 * powers)
    assert not (off > 1).any(), off.max()
    # the same rows in larger batches, where fewer CTAs share a row
    for times in (30, 80):
        if scores.dim() == 2 and 0 < len(scores) < times and not any(torch.is_tensor(v) for v in bounds.values()):
            k = -(-times // len(scores))
            more, more_logs = F.sample_classes(scores.repeat(k, 1), uniform.repeat(k), **bounds)
            assert torch.equal(more, got.repeat(k))
            assert not ((more_logs.cpu().double() - exact.repeat(k)).abs() > (2.0 ** -24 * exact.abs() + 4.3e-7 + 1.25e-7 * powers).repeat(k)).any()
    return got, logs


BOUNDS = [dict(), dict(temperature=0.7, top_k=5), dict(top_p=0.9), dict(temperature=1.5, top_p=0.999), dict(min_p=0.05), dict(top_k=50, top_p=0.5, min_p=0.01),
          dict(temperature=0.0), dict(top_k=1), dict(top_p=0.0), dict(top_k=700, temperature=3.0), dict(top_k=3000, top_p=0.95), dict(top_k=1 << 40), dict(min_p=1.0),
          dict(temperature=100.0, top_p=0.6), dict(temperature=0.01), dict(top_k=2000, min_p=1e-4), dict(temperature=50.0, top_k=2500, top_p=0.7)]


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("classes", [1, 2, 7, 8, 9, 31, 100, 127, 1000, 1025, 4097, 20000])
def test_sample(kind, classes):
    gen = generator(classes)
    rows = 24 if classes < 5000 else 6
    scores = normal(gen, rows, classes, scale=2.5, kind=kind)
    uniform = torch.rand(rows, generator=gen, device="cuda")
    for bounds in BOUNDS:
        check_draw(scores, uniform, **bounds)


@pytest.mark.parametrize("kind,classes", [(torch.float32, 50000), (torch.bfloat16, 100003), (torch.float32, 131072), (torch.float16, 262147)])
def test_sample_many_classes(kind, classes):
    """With the row in shared memory and without."""
    gen = generator(3)
    scores = normal(gen, 3, classes, scale=2.0, kind=kind)
    uniform = torch.rand(3, generator=gen, device="cuda")
    for bounds in BOUNDS:
        check_draw(scores, uniform, **bounds)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("name", ["equal", "few", "rising", "falling", "offset", "masked", "lowest", "two", "large"])
def test_sample_of_hard_rows(kind, name):
    gen = generator(5)
    rows, classes = 8, 5003
    s = torch.randn(rows, classes, generator=gen, device="cuda") * 2
    if name == "equal":
        s = torch.full_like(s, 1.25)
    elif name == "few":  # many equal scores
        s = (s / 2).round()
    elif name in ("rising", "falling"):
        s = torch.sort(s, dim=1, descending=name == "falling")[0]
    elif name == "offset":
        s = s + 1000.0
    elif name == "masked":
        s[torch.rand(rows, classes, generator=gen, device="cuda") < 0.99] = -math.inf
        s[3, :-1] = -math.inf
        s[3, -1] = -7.0
        s[4] = -math.inf
    elif name == "lowest":
        s[torch.rand(rows, classes, generator=gen, device="cuda") < 0.99] = torch.finfo(kind).min
        s[4] = torch.finfo(kind).min
    elif name == "two":
        s = torch.where(s > 4, torch.ones_like(s), torch.zeros_like(s))
    elif name == "large":
        s = s * (2000.0 if kind == torch.float16 else 1e30)
    uniform = torch.rand(rows, generator=gen, device="cuda")
    uniform[0], uniform[1] = 0.0, 1.0
    uniform[2] = 1.0 - 2.0 ** -24
    for bounds in BOUNDS:
        check_draw(s.to(kind), uniform, **bounds)


@pytest.mark.parametrize("kind", TYPES)
def test_sample_at_the_ends_of_the_temperature(kind):
    gen = generator(11)
    s, u = normal(gen, 10, 3001, scale=2.0, kind=kind), torch.rand(10, generator=gen, device="cuda")
    s[3] = (s[3] * 2).round()  # equal scores at the top as well
    for t in (1e-45, 1e-38, 1e-30, 1e-3, 1e3, 1e30, 3e38):
        for bounds in (dict(), dict(top_p=0.7), dict(top_k=300, top_p=0.9), dict(min_p=0.5)):
            check_draw(s, u, temperature=torch.full((10,), t, device="cuda"), **bounds)
            check_draw(s, u, temperature=t, **bounds)


def test_sample_rows_without_an_answer():
    s = torch.randn(12, 300, device="cuda", generator=generator(1))
    s[0, 7], s[1, 7], s[2], s[3, 299] = math.nan, math.inf, -math.inf, math.nan
    u = torch.full((12,), 0.3, device="cuda")
    u[4], u[5], u[6] = math.nan, -0.1, 1.5
    t = torch.ones(12, device="cuda")
    t[7], t[8], t[9] = -1.0, math.inf, math.nan
    p = torch.full((12,), 0.9, device="cuda")
    p[10] = math.nan
    for bounds in (dict(), dict(top_k=torch.full((12,), 7, device="cuda")), dict(top_p=p), dict(min_p=1 - p)):
        got, logs = check_draw(s, u, temperature=t, **bounds)
        assert (got[:10] == -1).all() and torch.isnan(logs[:10]).all() and got[11] >= 0


@pytest.mark.parametrize("kind", TYPES)
def test_sample_with_bounds_for_each_row(kind):
    gen = generator(8)
    rows, classes = 200, 1500
    s, u = normal(gen, rows, classes, scale=3.0, kind=kind), torch.rand(rows, generator=gen, device="cuda")

    def some(low, high, *others):
        v = low + (high - low) * torch.rand(rows, generator=gen, device="cuda")
        which = torch.randint(0, 2 * len(others), (rows,), generator=gen, device="cuda")
        for i, o in enumerate(others):
            v = torch.where(which == i, torch.full_like(v, o), v)
        return v

    check_draw(s, u, temperature=some(0.3, 2.0, 0.0, 1.0), top_k=some(1, 1600, 0, -5, 1).long(), top_p=some(0.1, 1.0, 1.0, 0.0, 2.0, -1.0),
               min_p=some(0.0, 0.2, 0.0, 1.0, 3.0, -1.0))
    # the same numbers as one for all and as one a row
    for bounds in (dict(temperature=0.75, top_k=40, top_p=0.875, min_p=0.03125),):
        each = {k: torch.full((rows,), v, device="cuda") for k, v in bounds.items()}
        one, all_ = F.sample_classes(s, u, **bounds), F.sample_classes(s, u, **each)
        assert torch.equal(one[0], all_[0]) and torch.equal(one[1], all_[1])


@pytest.mark.parametrize("kind", TYPES)
def test_sample_strides_and_shapes(kind):
    wide = normal(generator(2), 30, 1013, scale=2.0, kind=kind)
    u = torch.rand(30, generator=generator(3), device="cuda")
    for s in (wide[:, :1000], wide[:, 1:1001], wide[:, 5:], wide[::2], wide[:, ::2], wide[:, :60].t()[:30], wide[4:5].expand(30, 1013)):
        for bounds in (dict(), dict(top_k=20, top_p=0.8), dict(top_p=0.97)):
            got = check_draw(s, u[:len(s)], **bounds)
            again = F.sample_classes(s.contiguous(), u[:len(s)], **bounds)
            assert torch.equal(got[0], again[0])
    got, logs = F.sample_classes(wide.view(2, 3, 5, 1013), u.view(2, 3, 5), top_k=torch.full((2, 3, 5), 9, device="cuda"))
    want = F.sample_classes(wide, u, top_k=9)
    assert torch.equal(got.flatten(), want[0]) and torch.equal(logs.flatten(), want[1]) and got.shape == (2, 3, 5)
    one = F.sample_classes(wide[3], u[3], top_k=9)
    assert one[0].shape == () and one[0] == want[0][3]
    assert F.sample_classes(wide[:0], u[:0])[0].shape == (0,)


# ---- together ----------------------------------------------------------------------------------------------------------

def answer(x, w, bias, u):
    codes, scales = F.pack_mx4(w)
    scores = F.linear_mx4(x, codes, scales, bias)
    return [codes, scales, scores, *F.sample_classes(scores, u, temperature=0.8, top_k=40, top_p=0.9), *F.sample_classes(scores, u, top_p=0.95)]


@pytest.mark.parametrize("kind", TYPES)
def test_an_answer_on_streams_and_in_captured_graphs(kind):
    for rows in (1, 12, 200):
        gen = generator(rows)
        sets = [(normal(gen, rows, 200, kind=kind), normal(gen, 900, 200, scale=0.2, kind=kind), normal(gen, 900, kind=kind), torch.rand(rows, generator=gen, device="cuda"))
                for _ in range(2)]
        want = [answer(*s) for s in sets]
        scores = want[0][2]
        assert all(torch.equal(a, b) for a, b in zip(want[0][3:5], check_draw(scores, sets[0][3], temperature=0.8, top_k=40, top_p=0.9)) if a.dtype == torch.int64)
        streams = [torch.cuda.Stream() for _ in range(2)]
        torch.cuda.synchronize()
        got = []
        for turn in range(3):
            for k in range(2):
                with torch.cuda.stream(streams[(k + turn) % 2]):
                    got.append((k, answer(*sets[k])))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for k, out in got for a, b in zip(out, want[k]))
        held = [tuple(v.clone() for v in sets[0]) for _ in range(2)]
        graphs = []
        for s in held:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                out = answer(*s)
            graphs.append((graph, out))
        for s, new in zip(held, sets):
            for a, b in zip(s, new):
                a.copy_(b)
        for order in ((0, 1), (1, 0), (0, 1)):
            for k in order:
                graphs[k][0].replay()
        torch.cuda.synchronize()
        for k in range(2):
            assert all(torch.equal(a, b) for a, b in zip(graphs[k][1], want[k]))
    assert hingetree_cpp.pipeline_status() == 0


def test_modules_answer():
    gen = generator(6)
    for kind in TYPES:
        head = R.LinearClassLoss(100, 300).cuda().to(kind)
        packed = head.packed()
        x, u = normal(gen, 20, 100, kind=kind), torch.rand(20, generator=gen, device="cuda")
        codes, scales = F.pack_mx4(head.weight)
        assert torch.equal(packed(x), F.linear_mx4(x, codes, scales, head.bias.detach())) and torch.equal(packed.scores(x), packed(x))
        assert torch.equal(packed.sample(x, u, top_k=5)[0], F.sample_classes(packed(x), u, top_k=5)[0])
        assert torch.equal(head.sample(x, u, 0.5, 0, 0.9)[0], F.sample_classes(head.scores(x).detach(), u, 0.5, 0, 0.9)[0])
        copy = R.PackedClasses(100, 300).cuda().to(kind)
        copy.load_state_dict(packed.state_dict())
        assert torch.equal(copy(x), packed(x))
    for kind in (R.RandomHingeForestFusedLinear, R.RandomHingeFernFusedLinear):
        forest = kind(12, 70, 30, 4).cuda()
        x, u = torch.randn(9, 12, generator=gen, device="cuda"), torch.rand(9, generator=gen, device="cuda")
        assert torch.equal(forest.sample(x, u, top_p=0.8)[0], F.sample_classes(forest(x).detach(), u, top_p=0.8)[0])
        packed = forest.packed_classes()
        features = forest._function.apply(x, *forest._tree_params()).detach()
        assert torch.equal(forest.sample(x, u, packed=packed)[0], F.sample_classes(packed(features), u)[0])
        image, v = torch.randn(2, 12, 3, 4, generator=gen, device="cuda"), torch.rand(2, 3, 4, generator=gen, device="cuda")
        for p in (None, packed):
            classes, logs = forest.sample(image, v, packed=p)
            assert classes.shape == logs.shape == (2, 3, 4)
            rows = forest.sample(image.movedim(1, -1).reshape(24, 12).contiguous(), v.flatten(), packed=p)
            assert (rows[0] == classes.flatten()).float().mean() > 0.9  # (scores may differ in their last bit)


def test_traced_scores():
    x, codes, scales, bias = linear_inputs(torch.float32, 4, 40, 9)
    traced = torch.jit.trace(lambda v: F.linear_mx4(v, codes, scales, bias), (x,))
    other = torch.randn_like(x)
    assert torch.equal(traced(other), F.linear_mx4(other, codes, scales, bias))
    with pytest.raises(RuntimeError):
        torch.jit.trace(lambda v: F.sample_classes(v, torch.zeros(4, device="cuda"))[1], (x,))
