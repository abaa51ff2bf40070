"""Cases of the 8-bit and grouped linear layers: what is timed, on what inputs, and what the answers are.

Four operators, all of y = act(x w^T + bias) over rows ("tokens": an image's pooled features, a pixel of a feature map):

  quantize   rows of floats -> 8-bit codes and one scale for each row
  linear_i8  float rows -> codes -> product with 8-bit weights (a scale for each output channel) -> bias, activation -> floats
  group      the group (hash head, expert) of each row -> rows in the order of their groups, and where each group begins
  grouped    `group`, then the product of each row with its own group's weights, ragged numbers of rows, rows without a group left alone

Where `own` is false, run() computes them with elementary torch operations; where it is true, with pixelbox_amd.linear.
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BYTES = {"f32": 4, "bf16": 2, "f16": 2, "i8": 1}


def listed():
    return [
        # the pooled features of one image, ahead of an 8-bit head
        {"name": "quantize-1x1280-f32", "op": "quantize", "m": 1, "k": 1280, "type": "f32"},
        # the 4 x 4 maps of 512 images, 1280 channels behind the head convolution
        {"name": "quantize-8192x1280-f32", "op": "quantize", "m": 8192, "k": 1280, "type": "f32"},
        # the hash layer of one image: Linear(1280, 256) + tanh, latency only
        {"name": "linear_i8-1x256x1280-f32", "op": "linear_i8", "m": 1, "n": 256, "k": 1280, "type": "f32", "bias": True, "act": "tanh"},
        # sixteen rows through a square layer: the weights' bytes are what it costs
        {"name": "linear_i8-16x4096x4096-bf16", "op": "linear_i8", "m": 16, "n": 4096, "k": 4096, "type": "bf16", "bias": False, "act": "none"},
        # nothing a multiple of anything
        {"name": "linear_i8-777x1003x1289-f16", "op": "linear_i8", "m": 777, "n": 1003, "k": 1289, "type": "f16", "bias": True, "act": "silu"},
        # the matrix cores' case: a large batch through a wide layer
        {"name": "linear_i8-8192x8192x8192-bf16", "op": "linear_i8", "m": 8192, "n": 8192, "k": 8192, "type": "bf16", "bias": False, "act": "none"},
        # a batch of 512 images over eight hash heads
        {"name": "group-512-of-8", "op": "group", "m": 512, "groups": 8, "skew": 0.5, "none": 0.0},
        # many rows over many groups, one in ten without a group
        {"name": "group-131072-of-256", "op": "group", "m": 131072, "groups": 256, "skew": 0.5, "none": 0.1},
        # eight hash heads on one backbone: 512 images, each with the head of its collection
        {"name": "grouped-512-of-8-256x1280-f32", "op": "grouped", "m": 512, "groups": 8, "n": 256, "k": 1280, "type": "f32", "bias": True, "act": "tanh",
         "skew": 0.5, "none": 0.0},
        # a few rows over many experts: about half of the groups are empty, most others hold one row
        {"name": "grouped-32-of-64-2048x2048-bf16", "op": "grouped", "m": 32, "groups": 64, "n": 2048, "k": 2048, "type": "bf16", "bias": False, "act": "silu",
         "skew": 0.5, "none": 0.0},
        # ragged and odd, 8-bit, one row in twenty without a group
        {"name": "grouped-3001-of-17-1000x1285-i8", "op": "grouped", "m": 3001, "groups": 17, "n": 1000, "k": 1285, "type": "i8", "bias": True, "act": "silu",
         "skew": 1.0, "none": 0.05},
        # a large batch over 32 experts
        {"name": "grouped-16384-of-32-4096x4096-f16", "op": "grouped", "m": 16384, "groups": 32, "n": 4096, "k": 4096, "type": "f16", "bias": False, "act": "none",
         "skew": 0.25, "none": 0.0},
    ]


def _size(rng, lo, hi):
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    return min(max(v, lo), hi)


def draw(rng):
    op = rng.choice(["quantize", "linear_i8", "linear_i8", "group", "grouped", "grouped", "grouped"])
    if op == "quantize":
        return {"op": op, "m": _size(rng, 1, 8192), "k": _size(rng, 32, 8192), "type": rng.choice(["f32", "bf16", "f16"])}
    if op == "linear_i8":
        return {"op": op, "m": _size(rng, 1, 8192), "n": _size(rng, 32, 8192), "k": _size(rng, 32, 8192), "type": rng.choice(["f32", "bf16", "f16"]),
                "bias": rng.random() < 0.5, "act": rng.choice(["none", "silu", "tanh"])}
    if op == "group":
        return {"op": op, "m": _size(rng, 1, 131072), "groups": _size(rng, 1, 256), "skew": rng.choice([0.0, 0.5, 1.0]), "none": rng.choice([0.0, 0.1])}
    m, n, k, groups = _size(rng, 1, 16384), _size(rng, 32, 4096), _size(rng, 32, 4096), _size(rng, 1, 64)
    while groups > 1 and groups * n * k > 1 << 27:
        groups //= 2
    while m > 1 and m * n * k > 1 << 35:
        m //= 2
    return {"op": op, "m": m, "groups": groups, "n": n, "k": k, "type": rng.choice(["f32", "bf16", "f16", "i8"]), "bias": rng.random() < 0.5,
            "act": rng.choice(["none", "silu", "tanh"]), "skew": rng.choice([0.0, 0.5, 1.0]), "none": rng.choice([0.0, 0.05])}


def _shares(case):
    """How often a row falls into each group: 1 / (g + 1)^skew, scaled to what the rows without a group leave."""
    w = [(g + 1.0) ** -case["skew"] for g in range(case["groups"])]
    return [(1.0 - case["none"]) * v / sum(w) for v in w]


def work(case):
    m = case["m"]
    if case["op"] == "quantize":
        k = case["k"]
        return {"bytes": m * k * (BYTES[case["type"]] + 1) + 4 * m, "flops": 0}
    if case["op"] == "group":
        return {"bytes": 4 * m + 4 * m + 4 * (case["groups"] + 1), "flops": 0}
    n, k = case["n"], case["k"]
    if case["op"] == "linear_i8":
        size = BYTES[case["type"]]
        return {"bytes": m * k * size + n * k + 4 * n + (4 * n if case["bias"] else 0) + m * n * size, "flops": 2 * m * n * k}
    shares = _shares(case)
    met = sum(1.0 - (1.0 - p) ** m for p in shares)  # groups that some row falls into, on average
    rows = m * sum(shares)
    x = 4 if case["type"] in ("f32", "i8") else 2
    weights = met * n * (k * BYTES[case["type"]] + (4 if case["type"] == "i8" else 0) + (4 if case["bias"] else 0))
    return {"bytes": 4 * m + rows * k * x + weights + rows * n * x, "flops": 2 * rows * n * k}


def _rows(gen, m, k, dtype):
    """Activations: rows of different strength, a few channels far stronger than the rest."""
    x = torch.randn(m, k, generator=gen, device="cuda", dtype=torch.float32)
    x *= torch.exp(0.5 * torch.randn(m, 1, generator=gen, device="cuda"))
    loud = torch.rand(1, k, generator=gen, device="cuda") < 0.01
    return torch.where(loud, 6.0 * x, x).to(dtype)


def _codes(w):
    """Weights in 8 bits, one scale for each output channel (the last axis is summed over)."""
    scale = (w.abs().amax(-1).double() / 127).float()
    codes = torch.empty(w.shape, dtype=torch.int8, device=w.device)
    torch.clamp(torch.round(w / scale[..., None]), -127, 127, out=w)
    codes.copy_(w)
    return codes, scale


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    m = case["m"]
    s = {"case": case}
    if case["op"] == "quantize":
        s["x"] = _rows(gen, m, case["k"], DTYPES[case["type"]])
        s["codes"] = torch.empty(m, case["k"], dtype=torch.int8, device="cuda")
        s["scale"] = torch.empty(m, dtype=torch.float32, device="cuda")
        return s
    if case["op"] in ("group", "grouped"):
        groups = case["groups"]
        ends = torch.tensor(_shares(case), dtype=torch.float64).cumsum(0).to("cuda")
        at = torch.rand(m, generator=gen, device="cuda", dtype=torch.float64)
        group = torch.searchsorted(ends, at, right=True)
        s["group"] = torch.where(at < ends[-1], group.clamp(max=groups - 1), torch.full_like(group, -1)).to(torch.int32)
        s["offsets"] = torch.empty(groups + 1, dtype=torch.int32, device="cuda")
        s["order"] = torch.empty(m, dtype=torch.int32, device="cuda")
        # the room that the plain form pads every group to (a program knows its batch's largest group)
        s["largest"] = int(torch.bincount(s["group"].long() + 1, minlength=groups + 1)[1:].max())
        if case["op"] == "group":
            return s
    n, k = case["n"], case["k"]
    i8 = case["op"] == "linear_i8" or case["type"] == "i8"
    dtype = DTYPES[case["type"]] if case["type"] != "i8" else torch.float32
    s["x"] = _rows(gen, m, k, dtype)
    shape = (n, k) if case["op"] == "linear_i8" else (case["groups"], n, k)
    w = torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32).mul_(k ** -0.5)
    if i8:
        s["w"], s["w_scale"] = _codes(w)
        s["codes"] = torch.empty(m, k, dtype=torch.int8, device="cuda")
        s["scale"] = torch.empty(m, dtype=torch.float32, device="cuda")
    else:
        s["w"] = w.to(dtype)
    del w
    s["bias"] = torch.randn(shape[:-1], generator=gen, device="cuda", dtype=torch.float32).mul_(0.1) if case["bias"] else None
    s["y"] = torch.zeros(m, n, dtype=dtype, device="cuda")
    return s


# ---- the plain forms ------------------------------------------------------------------------------------------------------------------

def _plain_quantize(x):
    """scale = max(|x|) / 127, at least the smallest normal number; code = x / scale to the nearest whole number, halves to the even one.
    The quotient is taken in 64 bits: next to a half, 32 bits would round to another code."""
    x = x.float()
    scale = (x.abs().amax(1).double() / 127).float().clamp_min(2.0 ** -126)
    return torch.round(x.double() / scale.double()[:, None]).float(), scale


def _plain_act(y, act):
    if act == "silu":
        return y / (1 + torch.exp(-y))
    if act == "tanh":
        return torch.tanh(y)
    return y


def _plain_group(group, groups):
    key = torch.where((group >= 0) & (group < groups), group, torch.full_like(group, groups)).long()
    order = torch.argsort(key, stable=True)
    offsets = torch.searchsorted(key[order].contiguous(), torch.arange(groups + 1, device=key.device))
    return offsets.to(torch.int32), order.to(torch.int32)


def _plain_grouped(s, case):
    """Every group padded to the largest one's rows, one batched product."""
    groups, largest = case["groups"], max(s["largest"], 1)
    offsets, order = _plain_group(s["group"], groups)
    place = torch.arange(case["m"], device="cuda")
    group = s["group"][order.long()].long()
    has = (group >= 0) & (group < groups)
    slot = torch.where(has, group * largest + place - offsets.long()[group.clamp(0, groups - 1)], torch.full_like(group, groups * largest))
    x = s["x"].float()
    if case["type"] == "i8":
        x, scale = _plain_quantize(x)
    padded = torch.zeros(groups * largest + 1, case["k"], dtype=torch.float32, device="cuda")
    padded[slot] = x[order.long()]
    y = torch.bmm(padded[:-1].view(groups, largest, case["k"]), s["w"].float().transpose(1, 2).contiguous())
    if case["type"] == "i8":
        row_scale = torch.zeros(groups * largest + 1, dtype=torch.float32, device="cuda")
        row_scale[slot] = scale[order.long()]
        y = y * row_scale[:-1].view(groups, largest, 1) * s["w_scale"][:, None, :]
    if s["bias"] is not None:
        y = y + s["bias"][:, None, :]
    y = _plain_act(y, case["act"]).reshape(groups * largest, case["n"])
    y = torch.cat([y, torch.zeros(1, case["n"], dtype=y.dtype, device="cuda")])  # what a row without a group keeps: s["y"] is zero there
    out = torch.empty(case["m"], case["n"], dtype=s["y"].dtype, device="cuda")
    out[order.long()] = y[slot].to(out.dtype)
    return out


def _plain(s):
    case = s["case"]
    if case["op"] == "quantize":
        codes, scale = _plain_quantize(s["x"])
        return codes * scale[:, None], scale
    if case["op"] == "group":
        return _plain_group(s["group"], case["groups"])
    if case["op"] == "grouped":
        return _plain_grouped(s, case)
    codes, scale = _plain_quantize(s["x"])
    y = torch.matmul(codes, s["w"].float().t()) * scale[:, None] * s["w_scale"]
    if s["bias"] is not None:
        y = y + s["bias"]
    return _plain_act(y, case["act"]).to(s["y"].dtype)


# ---- the framework's -------------------------------------------------------------------------------------------------------------------

def _own(s):
    from pixelbox_amd import linear

    case = s["case"]
    if case["op"] == "group":
        return linear.group_rows(s["group"], case["groups"], offsets=s["offsets"], order=s["order"])
    if case["op"] == "grouped":
        linear.group_rows(s["group"], case["groups"], offsets=s["offsets"], order=s["order"])
        if case["type"] == "i8":
            linear.quantize_rows(s["x"], codes=s["codes"], scale=s["scale"])
            return linear.linear_grouped(s["codes"], s["w"], s["offsets"], rows=s["order"], x_scale=s["scale"], w_scale=s["w_scale"], bias=s["bias"],
                                         act=case["act"], out=s["y"])
        return linear.linear_grouped(s["x"], s["w"], s["offsets"], rows=s["order"], bias=s["bias"], act=case["act"], out=s["y"])
    linear.quantize_rows(s["x"], codes=s["codes"], scale=s["scale"])
    if case["op"] == "quantize":
        return torch.mul(s["codes"], s["scale"][:, None]), s["scale"]  # the values that the codes stand for
    return linear.linear_i8(s["codes"], s["scale"], s["w"], s["w_scale"], bias=s["bias"], act=case["act"], out=s["y"])


def run(state):
    return _own(state) if own else _plain(state)


# ---- from the definitions, in 64 bits ----------------------------------------------------------------------------------------------------

def _exact_codes(x):
    x = x.double()
    scale = torch.maximum((x.abs().max(dim=1).values / 127.0).float(), torch.tensor(torch.finfo(torch.float32).tiny, device=x.device)).double()
    return (x / scale.unsqueeze(1)).round(), scale


def _exact_linear(x, w, bias, act):
    y = x @ w.T
    if bias is not None:
        y += bias.double()
    if act == "tanh":
        return y.tanh()
    return y * y.sigmoid() if act == "silu" else y


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "quantize":
        codes, scale = _exact_codes(s["x"])
        return codes * scale.unsqueeze(1), scale
    if case["op"] == "group":
        return None  # whole numbers
    i8 = case["op"] == "linear_i8" or case["type"] == "i8"
    x = s["x"].double()
    if i8:
        codes, scale = _exact_codes(s["x"])
        x = codes * scale.unsqueeze(1)
    if case["op"] == "linear_i8":
        return _exact_linear(x, s["w"].double() * s["w_scale"].double().unsqueeze(1), s["bias"], case["act"])
    y = torch.zeros(case["m"], case["n"], dtype=torch.float64, device="cuda")
    for g in range(case["groups"]):
        rows = (s["group"] == g).nonzero().squeeze(1)
        if rows.numel():
            w = s["w"][g].double()
            if i8:
                w *= s["w_scale"][g].double().unsqueeze(1)
            y[rows] = _exact_linear(x[rows], w, s["bias"][g] if s["bias"] is not None else None, case["act"])
    return y
