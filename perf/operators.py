"""The dense ends of a forest model as programs use them: a gated projection in front of a forest, and the class loss of a linear
layer behind one, each for answering and for training.

Fields of a case:

  op        "loss": linear_class_loss, x [rows, features] times w [outputs, features] as class scores, softmax cross entropy;
            "gated": gated_linear, act(x wg^T + bg) * (x wv^T + bv) with [outputs, features] weights
  train     gradients of everything that takes one come too; a loss is then the mean over the rows that count, otherwise one per row
  dtype     "f32", "bf16" or "f16"
  bias      whether the linear layers have one;  ignored: whether every eighth row or so has no class (loss)
  act       activation of the gate: "silu", "gelu", "relu" or "sigmoid" (gated)
"""
import math

import torch

own = False

DEVICE = "cuda"
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
IGNORED = -100


def _loss(name, rows, features, outputs, train, dtype, bias=True, ignored=False):
    return {"name": name, "op": "loss", "rows": rows, "features": features, "outputs": outputs, "train": train, "dtype": dtype,
            "bias": bias, "ignored": ignored, "act": ""}


def _gated(name, rows, features, outputs, train, dtype, bias=True, act="silu"):
    return {"name": name, "op": "gated", "rows": rows, "features": features, "outputs": outputs, "train": train, "dtype": dtype,
            "bias": bias, "ignored": False, "act": act}


def listed():
    return [
        # one sample's answer, scored against its class: the features of 1024 trees, a thousand classes
        _loss("loss_one_row", 1, 1024, 1000, False, "f32"),
        # a small batch of answers over many classes: the weights are read once for all of them
        _loss("loss_few_rows", 16, 1024, 50000, False, "bf16"),
        # an ordinary training step of a classifier on forest features, in the forest's own type
        _loss("loss_train_f32", 8192, 1024, 1000, True, "f32"),
        # many classes at sizes that divide by nothing, rows without a class among them
        _loss("loss_train_ragged", 1003, 771, 10007, True, "f16", ignored=True),
        # evaluation on a held-out set: the loss of every row
        _loss("loss_evaluate", 8192, 784, 21841, False, "bf16", ignored=True),
        # the largest training step: the scores alone would take 1.6 GB in 16 bits
        _loss("loss_train_large", 16384, 1024, 50000, True, "bf16", bias=False),
        # one sample through the gated front of a forest
        _gated("gated_one_row", 1, 784, 12700, False, "bf16"),
        # a small batch in the forest's own type
        _gated("gated_few_rows", 100, 1000, 700, False, "f32", act="gelu"),
        # training of a front for 100 trees of depth 7, one feature per decision, in the forest's own type
        _gated("gated_train_f32", 4096, 784, 2048, True, "f32"),
        # training at sizes that divide by nothing
        _gated("gated_train_ragged", 1555, 333, 1001, True, "f16", act="gelu"),
        # scoring of a large data set
        _gated("gated_predict", 65536, 784, 4096, False, "bf16", bias=False, act="sigmoid"),
        # training of the front of 8192 rows to 100 trees of depth 7, one feature per decision
        _gated("gated_train_large", 8192, 784, 12700, True, "bf16", bias=False),
    ]


def _log_uniform(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    top = {op: max(work(c)["flops"] for c in listed() if c["op"] == op) for op in ("loss", "gated")}
    while True:
        train = rng.random() < 0.6
        case = {"op": rng.choice(["loss", "gated"]), "rows": _log_uniform(rng, 16 if train else 1, 16384 if train else 65536),
                "features": _log_uniform(rng, 24, 2048), "train": train, "dtype": rng.choice(["f32", "bf16", "f16"]),
                "bias": rng.random() < 0.5, "ignored": False, "act": ""}
        if case["op"] == "loss":
            case["outputs"], case["ignored"] = _log_uniform(rng, 10, 50000), rng.random() < 0.4
        else:
            case["outputs"], case["act"] = _log_uniform(rng, 24, 12700), rng.choice(["silu", "gelu", "relu", "sigmoid"])
        if rng.random() < 0.5:  # whole multiples of what rows are usually padded to
            case["features"], case["outputs"] = -(-case["features"] // 8) * 8, -(-case["outputs"] // 8) * 8
        if work(case)["flops"] * (6 if case["dtype"] == "f32" else 1) <= top[case["op"]]:
            return case


def prepare(case, seed):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(seed)
    rows, features, outputs, kind = case["rows"], case["features"], case["outputs"], TYPES[case["dtype"]]

    def normal(*shape, scale=1.0):
        return (torch.randn(*shape, generator=g, device=DEVICE) * scale).to(kind)

    state = {"case": case, "x": normal(rows, features)}
    if case["op"] == "loss":
        state["w"] = normal(outputs, features, scale=2.0 / math.sqrt(features))
        state["b"] = normal(outputs, scale=0.5) if case["bias"] else None
        state["target"] = torch.randint(0, outputs, (rows,), generator=g, device=DEVICE)
        if case["ignored"]:
            state["target"][torch.rand(rows, generator=g, device=DEVICE) < 0.125] = IGNORED
        state["leaves"] = [state["x"], state["w"]] + ([state["b"]] if case["bias"] else [])
    else:
        state["wg"], state["wv"] = (normal(outputs, features, scale=1.0 / math.sqrt(features)) for _ in range(2))
        state["bg"], state["bv"] = (normal(outputs, scale=0.3) if case["bias"] else None for _ in range(2))
        state["leaves"] = [state["x"], state["wg"], state["wv"]] + ([state["bg"], state["bv"]] if case["bias"] else [])
        if case["train"]:
            state["grad"] = normal(rows, outputs, scale=0.1)
    if case["train"]:
        for leaf in state["leaves"]:
            leaf.requires_grad_()
    return state


def run(state):
    case = state["case"]
    if own:
        return _own_loss(state) if case["op"] == "loss" else _own_gated(state)
    with torch.no_grad():
        return _plain_loss(state) if case["op"] == "loss" else _plain_gated(state)


# ---- the framework's operators ---------------------------------------------------------------------------------------

def _own_loss(state):
    from hingetreefortorch_b200 import HingeTree
    if not state["case"]["train"]:
        return HingeTree.linear_class_loss(state["x"], state["w"], state["b"], state["target"], ignore_index=IGNORED, reduction="none")
    loss = HingeTree.linear_class_loss(state["x"], state["w"], state["b"], state["target"], ignore_index=IGNORED, reduction="mean")
    return [loss.detach(), *torch.autograd.grad(loss, state["leaves"])]


def _own_gated(state):
    from hingetreefortorch_b200 import HingeTree
    h = HingeTree.gated_linear(state["x"], state["wg"], state["wv"], state["bg"], state["bv"], activation=state["case"]["act"])
    return [h.detach(), *torch.autograd.grad(h, state["leaves"], state["grad"])] if state["case"]["train"] else h


# ---- their plain forms -----------------------------------------------------------------------------------------------

def _plain_loss(state):
    kind, x, w, target = state["x"].dtype, state["x"].float(), state["w"].float(), state["target"]
    counts = target != IGNORED
    at = torch.where(counts, target, torch.zeros_like(target))[:, None]
    scores = x @ w.t()
    if state["b"] is not None:
        scores += state["b"].float()
    of_target = scores.gather(1, at)
    top = scores.amax(1, keepdim=True)
    scores = scores.sub_(top).exp_()
    total = scores.sum(1, keepdim=True)
    loss = torch.where(counts[:, None], total.log() + top - of_target, torch.zeros_like(total))[:, 0]
    if not state["case"]["train"]:
        return loss
    valid = counts.sum()
    p = scores.div_(total)
    p.scatter_add_(1, at, torch.full_like(total, -1.0))
    p *= (counts / valid)[:, None]
    grads = [p @ w, p.t() @ x] + ([p.sum(0)] if state["b"] is not None else [])
    return [loss.sum() / valid, *(v.to(kind) for v in grads)]


def _gate(a, act):
    """The activation and its derivative."""
    if act == "relu":
        return a.clamp_min(0.0), (a > 0).to(a.dtype)
    if act == "gelu":
        phi = 0.5 * (1.0 + torch.erf(a * math.sqrt(0.5)))
        return a * phi, phi + a * torch.exp(-0.5 * a * a) / math.sqrt(2.0 * math.pi)
    s = 1.0 / (1.0 + torch.exp(-a))
    return (s, s * (1.0 - s)) if act == "sigmoid" else (a * s, s * (1.0 + a * (1.0 - s)))


def _plain_gated(state):
    kind, x, wg, wv = state["x"].dtype, state["x"].float(), state["wg"].float(), state["wv"].float()
    a, u = x @ wg.t(), x @ wv.t()
    if state["bg"] is not None:
        a, u = a + state["bg"].float(), u + state["bv"].float()
    gate, slope = _gate(a, state["case"]["act"])
    h = (gate * u).to(kind)
    if not state["case"]["train"]:
        return h
    g = state["grad"].float()
    da, du = g * u * slope, g * gate
    grads = [da @ wg + du @ wv, da.t() @ x, du.t() @ x] + ([da.sum(0), du.sum(0)] if state["bg"] is not None else [])
    return [h, *(v.to(kind) for v in grads)]


# ---- the same in 64 bits, from the definitions, by automatic differentiation -----------------------------------------

def exact(case, seed):
    state = prepare(case, seed)
    wide = [leaf.detach().double().requires_grad_(case["train"]) for leaf in state["leaves"]]
    if case["op"] == "loss":
        rows = torch.nonzero(state["target"] != IGNORED)[:, 0]
        s = torch.addmm(wide[2], wide[0], wide[1].t()) if case["bias"] else torch.mm(wide[0], wide[1].t())
        each = torch.logsumexp(s, 1)[rows] - s[rows, state["target"][rows]]
        if not case["train"]:
            return torch.zeros(case["rows"], dtype=torch.float64, device=DEVICE).index_add(0, rows, each)
        out = each.mean()
        return [out.detach(), *torch.autograd.grad(out, wide)]
    gate, value = (torch.addmm(b, wide[0], w.t()) if case["bias"] else torch.mm(wide[0], w.t())
                   for w, b in zip(wide[1:3], wide[3:5] if case["bias"] else (None, None)))
    if case["act"] == "silu":
        gate = gate * torch.sigmoid(gate)
    elif case["act"] == "gelu":
        gate = gate * 0.5 * torch.erfc(-gate / math.sqrt(2.0))
    elif case["act"] == "relu":
        gate = torch.maximum(gate, torch.zeros_like(gate))
    else:
        gate = torch.sigmoid(gate)
    out = gate * value
    return [out.detach(), *torch.autograd.grad(out, wide, state["grad"].double())] if case["train"] else out


def work(case):
    rows, features, outputs = case["rows"], case["features"], case["outputs"]
    size = 4 if case["dtype"] == "f32" else 2
    products = 1 if case["op"] == "loss" else 2  # projections of x
    flops = 2.0 * products * rows * features * outputs * (3 if case["train"] else 1)
    leaves = rows * features + products * outputs * (features + (1 if case["bias"] else 0))
    moved = size * leaves * (2 if case["train"] else 1)  # inputs, and a gradient of each
    if case["op"] == "loss":
        moved += 8 * rows + 4 * (1 if case["train"] else rows)
    else:
        moved += size * rows * outputs * (2 if case["train"] else 1)
    return {"bytes": float(moved), "flops": flops}
