"""Answers from a linear layer of many classes behind a forest, as programs make them: its weights held as microscaled 4-bit numbers,
the class scores of rows under such weights, and a class drawn from a row of scores with given random numbers.

Fields of a case:

  op        "pack": pack_mx4 of weights [outputs, features] and unpack_mx4 of what it gives, the values that are held
            "linear": linear_mx4, x [rows, features] times packed weights [outputs, features], with a bias
            "sample": sample_classes from scores [rows, outputs]
  dtype     "f32", "bf16" or "f16": of the weights (pack), x (linear) or scores (sample)
  bias      whether the linear layer has one
  temperature, top_k, top_p, min_p   of a sampling call, top_k 0: all classes; each_row: every row has its own of all four
  spread    of the scores that are sampled from, as a standard deviation
"""
import math

import torch

own = False

DEVICE = "cuda"
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
NUMBERS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _case(name, op, rows, features, outputs, dtype, bias=False, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, each_row=False, spread=0.0):
    return {"name": name, "op": op, "rows": rows, "features": features, "outputs": outputs, "dtype": dtype, "bias": bias,
            "temperature": temperature, "top_k": top_k, "top_p": top_p, "min_p": min_p, "each_row": each_row, "spread": spread}


def listed():
    return [
        # a head of 50000 classes on the features of 1024 trees, packed once after training
        _case("pack_large", "pack", 0, 1024, 50000, "f32"),
        # weights at sizes that divide by nothing
        _case("pack_ragged", "pack", 0, 771, 10007, "f16"),
        # one sample's scores
        _case("linear_one_row", "linear", 1, 784, 12700, "bf16", bias=True),
        # a small batch of answers over many classes: the weights are read once for all of them
        _case("linear_few_rows", "linear", 16, 1024, 50000, "bf16"),
        # a batch in the forest's own type
        _case("linear_f32", "linear", 2048, 1024, 1000, "f32", bias=True),
        # sizes that divide by nothing
        _case("linear_ragged", "linear", 333, 771, 10007, "f16", bias=True),
        # scoring of a data set over many classes
        _case("linear_large", "linear", 8192, 1024, 50000, "bf16"),
        # one sample's answer
        _case("sample_one_row", "sample", 1, 0, 50000, "bf16", temperature=0.8, top_k=50, top_p=0.9, spread=3.0),
        # a small batch, the likeliest classes that hold most of the weight
        _case("sample_few_rows", "sample", 16, 0, 21841, "f32", temperature=0.7, top_p=0.95, spread=2.0),
        # a batch of answers with every bound
        _case("sample_batch", "sample", 256, 0, 50000, "bf16", top_k=1000, top_p=0.95, min_p=0.02, spread=2.5),
        # requests of many callers in one batch, each with bounds of its own
        _case("sample_each_row", "sample", 1003, 0, 10007, "f32", temperature=0.9, top_k=100, top_p=0.9, min_p=0.01, each_row=True, spread=2.0),
        # a data set's labels drawn from a model
        _case("sample_large", "sample", 4096, 0, 21841, "f16", spread=2.0),
    ]


def _log_uniform(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    top = {op: max(_cost(c) for c in listed() if c["op"] == op) for op in ("pack", "linear", "sample")}
    while True:
        op = rng.choice(["pack", "linear", "linear", "sample", "sample"])
        case = _case("", op, 0, 0, _log_uniform(rng, 24, 50000), rng.choice(["f32", "bf16", "f16"]))
        del case["name"]
        if op != "sample":
            case["features"] = _log_uniform(rng, 24, 2048)
        if op != "pack":
            case["rows"] = _log_uniform(rng, 1, 8192)
        if op == "linear":
            case["bias"] = rng.random() < 0.5
        if op == "sample":
            case["temperature"], case["spread"] = round(rng.uniform(0.5, 1.5), 2), round(rng.uniform(0.5, 4.0), 1)
            if rng.random() < 0.5:
                case["top_k"] = min(_log_uniform(rng, 1, 2000), case["outputs"])
            if rng.random() < 0.6:
                case["top_p"] = round(rng.uniform(0.3, 0.99), 2)
            if rng.random() < 0.3:
                case["min_p"] = round(rng.uniform(0.001, 0.3), 3)
            case["each_row"] = rng.random() < 0.3
        elif rng.random() < 0.5:  # whole multiples of what rows are usually padded to
            case["features"], case["outputs"] = -(-case["features"] // 8) * 8, -(-case["outputs"] // 8) * 8
        if _cost(case) <= top[op]:
            return case


def _cost(case):
    w = work(case)
    return max(w["bytes"], w["flops"] * (3 if case["dtype"] == "f32" else 2 if case["dtype"] == "f16" else 1) / 200.0)


def prepare(case, seed):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(seed)
    rows, features, outputs, kind = case["rows"], case["features"], case["outputs"], TYPES[case["dtype"]]

    def normal(*shape, scale=1.0):
        return (torch.randn(*shape, generator=g, device=DEVICE) * scale).to(kind)

    state = {"case": case}
    if case["op"] == "pack":
        state["w"] = normal(outputs, features, scale=1.0 / math.sqrt(features))
    elif case["op"] == "linear":
        state["x"] = normal(rows, features)
        state["codes"], state["scales"] = _pack(torch.randn(outputs, features, generator=g, device=DEVICE) / math.sqrt(features))
        state["bias"] = normal(outputs, scale=0.5) if case["bias"] else None
    else:
        state["scores"] = normal(rows, outputs, scale=case["spread"])
        state["uniform"] = torch.rand(rows, generator=g, device=DEVICE)
        bounds = {k: case[k] for k in ("temperature", "top_k", "top_p", "min_p")}
        if case["each_row"]:  # some callers without a bound, some that ask for the likeliest class
            def some(value, low, high, otherwise, part=0.25):
                v = value * (low + (high - low) * torch.rand(rows, generator=g, device=DEVICE))
                return torch.where(torch.rand(rows, generator=g, device=DEVICE) < part, torch.full_like(v, otherwise), v)
            bounds["temperature"] = some(case["temperature"], 0.7, 1.3, 0.0, 0.125)
            bounds["top_k"] = some(float(case["top_k"]), 0.2, 2.0, 0.0).long()
            bounds["top_p"] = some(case["top_p"], 0.5, 1.0, 1.0)
            bounds["min_p"] = some(case["min_p"], 0.2, 2.0, 0.0)
        state["bounds"] = bounds
    return state


def run(state):
    op = state["case"]["op"]
    if own:
        return _own(op, state)
    return {"pack": _plain_pack, "linear": _plain_linear, "sample": _plain_sample}[op](state)


# ---- the framework's operators ---------------------------------------------------------------------------------------

def _own(op, state):
    from hingetreefortorch_b200 import HingeTree
    if op == "pack":
        codes, scales = HingeTree.pack_mx4(state["w"])
        return HingeTree.unpack_mx4(codes, scales, state["w"].size(1), dtype=torch.bfloat16)
    if op == "linear":
        return HingeTree.linear_mx4(state["x"], state["codes"], state["scales"], state["bias"])
    return HingeTree.sample_classes(state["scores"], state["uniform"], **state["bounds"])


# ---- their plain forms -----------------------------------------------------------------------------------------------

def _pack(w):
    """Codes, two to a byte, the first in the low half, and a power of two for each 32 features: [outputs, 16 blocks], [outputs, blocks]."""
    outputs, features = w.shape
    blocks = -(-features // 32)
    v = torch.zeros(outputs, 32 * blocks, device=w.device)
    v[:, :features] = w
    v = v.view(outputs, blocks, 32)
    field = (v.abs().amax(2).view(torch.int32) >> 23) - 2  # the exponent of the largest, less that of 6.0
    scale = field.clamp_min(0)
    a = v.double().abs() * torch.exp2(127.0 - scale.double())[:, :, None]
    a = torch.where(a < 2, (2 * a).round() / 2, torch.where(a < 4, a.round(), 2 * (a / 2).round())).clamp_max(6.0).float()
    code = (2 * a).long()  # twice the value counts 0, 1, 2, 3, 4, 6, 8, 12
    code = torch.where(code <= 4, code, torch.where(code == 6, torch.full_like(code, 5), torch.where(code == 8, torch.full_like(code, 6), torch.full_like(code, 7))))
    code = (code + 8 * torch.signbit(v)).to(torch.uint8).view(outputs, 16 * blocks, 2)
    return code[:, :, 0] | (code[:, :, 1] << 4), scale.to(torch.uint8)


def _unpack(codes, scales, features):
    numbers = torch.tensor(NUMBERS + tuple(-n for n in NUMBERS), device=codes.device)
    v = torch.stack([numbers[(codes & 15).long()], numbers[(codes >> 4).long()]], 2).view(codes.size(0), -1, 32)
    return (v * torch.exp2(scales.float() - 127.0)[:, :, None]).flatten(1)[:, :features]


def _plain_pack(state):
    return _unpack(*_pack(state["w"].float()), state["w"].size(1)).to(torch.bfloat16)


def _plain_linear(state):
    x = state["x"]
    y = x.float() @ _unpack(state["codes"], state["scales"], x.size(1)).t()
    if state["bias"] is not None:
        y += state["bias"].float()
    return y.to(x.dtype)


def _wide(bounds, like):
    """Each bound as one number a row, in 64 bits."""
    return {k: (v.double() if torch.is_tensor(v) else torch.full_like(like, float(v)))[:, None] for k, v in bounds.items()}


def _plain_sample(state):
    s = state["scores"].double()
    b = _wide(state["bounds"], state["uniform"].double())
    s, index = torch.sort(s, dim=1, descending=True, stable=True)
    greedy = b["temperature"] == 0
    t = torch.where(greedy, torch.ones_like(b["temperature"]), b["temperature"])
    x = (s - s[:, :1]) / t
    w = torch.exp(x)
    place = torch.arange(s.size(1), device=s.device)
    w = torch.where((place < b["top_k"]) | (b["top_k"] <= 0), w, torch.zeros_like(w))
    before = torch.cumsum(w, 1) - w
    keep = (before < b["top_p"] * w.sum(1, keepdim=True)) | (b["top_p"] >= 1) | (place == 0)
    keep &= (w >= b["min_p"]) & ((place == 0) | ~greedy)
    w = torch.where(keep, w, torch.zeros_like(w))
    by_class = torch.zeros_like(w).scatter_(1, index, w)
    upto = torch.cumsum(by_class, 1)
    drawn = (upto > state["uniform"].double()[:, None] * upto[:, -1:]).int().argmax(1)
    chosen = state["scores"].double().gather(1, drawn[:, None])
    return drawn, (((chosen - s[:, :1]) / t) - torch.log(upto[:, -1:]))[:, 0].float()


# ---- the same in 64 bits, from the definitions -----------------------------------------------------------------------

def _exact_values(codes, scales, features):
    nibbles = torch.stack([codes.int() % 16, codes.int() // 16], 2).flatten(1)
    sign, exponent, half = nibbles // 8, (nibbles // 2) % 4, nibbles % 2
    a = torch.where(exponent == 0, 0.5 * half, (1.0 + 0.5 * half) * torch.pow(2.0, exponent.double() - 1.0)).double()
    power = torch.pow(torch.tensor(2.0, dtype=torch.float64, device=codes.device), scales.double() - 127.0)
    return (torch.where(sign == 1, -a, a) * power.repeat_interleave(32, 1))[:, :features]


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "pack":  # the nearest of the numbers by their distances, of two as near the one whose code is even
        w = state["w"].double()
        grid = torch.tensor(NUMBERS, dtype=torch.float64, device=w.device)
        out = torch.empty_like(w)
        for first in range(0, w.size(1), 32):
            block = w[:, first:first + 32]
            top = block.abs().amax(1, keepdim=True)
            power = torch.pow(2.0, torch.where(top > 0, torch.floor(torch.log2(top)) - 2, torch.full_like(top, -127.0)).clamp_min(-127.0))
            distance = ((block.abs() / power)[:, :, None] - grid).abs()
            order = torch.tensor([0, 2, 4, 6, 1, 3, 5, 7], device=w.device)
            out[:, first:first + 32] = torch.copysign(grid[order[distance[:, :, order].argmin(2)]] * power, block)
        return out
    if case["op"] == "linear":
        w = _exact_values(state["codes"], state["scales"], case["features"])
        y = torch.mm(state["x"].double(), w.t())
        return y if state["bias"] is None else y + state["bias"].double()
    s, b = state["scores"].double(), _wide(state["bounds"], state["uniform"].double())
    rank = torch.argsort(torch.argsort(-s, dim=1, stable=True), dim=1)
    top = s.amax(1, keepdim=True)
    t = b["temperature"].clamp_min(1e-300)
    logs = torch.where(b["temperature"] == 0, torch.where(rank == 0, 0.0, -math.inf), (s - top) / t)
    count = torch.where(b["top_k"] > 0, b["top_k"], torch.full_like(b["top_k"], float(s.size(1))))
    logs = torch.where(rank < count, logs, -math.inf)
    share = torch.softmax(logs, 1)
    ordered = torch.zeros_like(share).scatter_(1, rank, share)
    sums = torch.cumsum(ordered, 1)
    enough = torch.searchsorted(sums, b["top_p"].contiguous()) + 1  # classes until the sum is there
    count = torch.minimum(count, torch.where(b["top_p"] >= 1, count, enough.double()))
    logs = torch.where((rank < count.clamp_min(1)) & ((logs >= torch.log(b["min_p"])) | (rank == 0)), logs, -math.inf)
    logs = logs - torch.logsumexp(logs, 1, keepdim=True)
    upto = torch.cumsum(torch.exp(logs), 1)
    drawn = torch.searchsorted(upto, state["uniform"].double()[:, None] * upto[:, -1:], right=True).clamp_max(s.size(1) - 1)
    return None, logs.gather(1, drawn)[:, 0]


def work(case):
    rows, features, outputs = case["rows"], case["features"], case["outputs"]
    size = 4 if case["dtype"] == "f32" else 2
    packed = outputs * -(-features // 32) * 17
    if case["op"] == "pack":  # the packed form is written and read again
        return {"bytes": float(outputs * features * (size + 2) + 2 * packed), "flops": float(4 * outputs * features)}
    if case["op"] == "linear":
        return {"bytes": float(packed + size * (rows * (features + outputs) + (outputs if case["bias"] else 0))),
                "flops": 2.0 * rows * features * outputs}
    return {"bytes": float(rows * (outputs * size + 4 + 12 + (20 if case["each_row"] else 0))), "flops": float(4 * rows * outputs)}
