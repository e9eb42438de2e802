"""What the group norm and the two fused matrix products are measured on.

``listed()`` names fixed cases, ``draw()`` makes more of the same ranges, ``prepare()`` makes a case's inputs
on the GPU, ``run()`` is one call: the plain form in elementary torch operations (32 bits, rounded once), or with
``own`` set the calls a user makes of ``distributed_machine_learning_amd.ops``. ``exact()`` computes the same in
64 bits from the definitions.
"""
import math
import random

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}
ACTS = ("none", "relu", "silu", "gelu", "gelu_tanh")


def listed():
    return [
        # one image's feature map in a residual stage: the smallest call, launch latency counts
        norm("norm one image", 1, 14, 14, 512, 32, "silu", "bf16"),
        # a batch of token sequences of an image transformer (14 x 14 patches and a class token), full precision
        norm("norm tokens fp32", 8, 1, 197, 768, 32, "none", "fp32"),
        # a 35 x 35 map of 288 channels read out of a wider concat buffer: nine channels a group
        norm("norm concat slice", 32, 35, 35, 288, 32, "gelu", "fp16", pitch=384),
        # residual stage 3 of a serving batch
        norm("norm batch 28x28", 128, 28, 28, 512, 32, "relu", "bf16"),
        # residual stage 2 of a serving batch of 256: the largest, far beyond the caches
        norm("norm batch 56x56", 256, 56, 56, 256, 32, "relu", "bf16"),
        # one image's classifier head: weight streaming for a single row, fp32 logits
        product("head one image", 1, 2048, 1000, "none", "bf16", out="fp32"),
        # nothing is a multiple of anything
        product("product odd sizes", 333, 1001, 517, "gelu", "fp16", residual=True),
        # the projection back of a transformer's feed-forward half for 32 images of 197 tokens, with its residual
        product("feed-forward out", 6304, 4096, 1024, "none", "bf16", residual=True),
        # a large batch's projection with its activation
        product("product large", 16384, 4096, 4096, "silu", "bf16"),
        # a few tokens over many experts: most groups are empty, weight streaming
        grouped("experts few tokens", 8, 64, 1024, 4096, "gelu_tanh", "bf16", mix=3),
        # one mixed batch's features, each job with a head of its own; padding rows behind the last job stay
        grouped("heads mixed batch", 256, 12, 2048, 1000, "none", "bf16", out="fp32", mix=5, spare=19),
        # a prompt's tokens over eight experts of uneven load
        grouped("experts prompt", 16384, 8, 1024, 4096, "silu", "bf16", mix=7),
    ]


def norm(name, n, h, w, c, groups, act, dtype, pitch=0):
    return {"name": name, "op": "group_norm", "n": n, "h": h, "w": w, "c": c, "groups": groups, "act": act,
            "dtype": dtype, "pitch": pitch or c}


def product(name, m, k, n, act, dtype, out="", residual=False, act_last=False):
    return {"name": name, "op": "linear", "m": m, "k": k, "n": n, "act": act, "dtype": dtype, "out": out or dtype,
            "residual": residual, "act_last": act_last}


def grouped(name, m, e, k, n, act, dtype, out="", residual=False, mix=1, spare=0):
    return {"name": name, "op": "grouped_linear", "m": m, "e": e, "k": k, "n": n, "act": act, "dtype": dtype,
            "out": out or dtype, "residual": residual, "mix": mix, "spare": spare}


def spread(rng, lo, hi):
    """A whole number between lo and hi, even over the logarithm, odd ones among them."""
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def width(rng, lo, hi):
    """A feature width: half of them multiples of 64, the others as they fall."""
    v = spread(rng, lo, hi)
    return max(64, v // 64 * 64) if rng.random() < 0.5 else v


def draw(rng):
    op = rng.choice(("group_norm", "linear", "grouped_linear"))
    dtype = rng.choice(("bf16", "bf16", "fp16"))
    act = rng.choice(ACTS)
    if op == "group_norm":
        dtype = rng.choice(("bf16", "bf16", "fp16", "fp32"))
        groups = rng.choice((1, 8, 16, 32, 32, 32, 64))
        c = groups * spread(rng, 1, max(1, 2048 // groups))
        side = rng.choice((7, 8, 14, 17, 28, 35, 56, 73))
        h, w = rng.choice(((side, side), (1, side * side), (1, spread(rng, 1, 4096)), (side, side + 1)))
        n = spread(rng, 1, max(1, min(512, 100_000_000 // (h * w * c))))
        pitch = c + rng.choice((0, 0, 8, 64, 3))
        return {k: v for k, v in norm("", n, h, w, c, groups, act, dtype, pitch).items() if k != "name"}
    out = rng.choice((dtype, dtype, "fp32"))
    k, n = width(rng, 16, 8192), width(rng, 16, 8192)
    if op == "linear":
        m = spread(rng, 1, max(1, min(16384, 270_000_000_000 // (k * n))))
        case = product("", m, k, n, act, dtype, out, rng.random() < 0.5, rng.random() < 0.3)
    else:
        e = spread(rng, 1, max(1, min(128, 270_000_000 // (k * n))))
        m = spread(rng, 1, max(1, min(16384, 68_000_000_000 // (k * n))))
        case = grouped("", m, e, k, n, act, dtype, out, rng.random() < 0.3, rng.randrange(1, 1 << 20),
                       rng.choice((0, 0, 1, 37)))
    return {k: v for k, v in case.items() if k != "name"}


def lengths(case):
    """Rows of each group: an uneven load, some groups without rows; they sum to the case's m less its spare rows."""
    rng = random.Random(case["mix"])
    e, rows = case["e"], max(0, case["m"] - case["spare"])
    load = [rng.random() ** 2 if rng.random() < 0.85 else 0.0 for _ in range(e)]
    load = load if sum(load) else [1.0] * e
    edges = [0]
    for v in load:
        edges.append(edges[-1] + v)
    edges = [round(rows * v / edges[-1]) for v in edges]
    return [b - a for a, b in zip(edges, edges[1:])]


def prepare(case, seed):
    gen = torch.Generator("cuda").manual_seed(seed)
    t = TYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(shape, generator=gen, device="cuda")

    if case["op"] == "group_norm":
        c = case["c"]
        # a convolution's output: each channel has a level and a spread of its own
        level, scale = normal(case["pitch"]), normal(case["pitch"]).mul_(0.5).exp_()
        buf = torch.empty((case["n"], case["h"], case["w"], case["pitch"]), device="cuda", dtype=t)
        for i in range(0, case["n"], 32):
            part = buf[i:i + 32]
            part.copy_(normal(*part.shape).mul_(scale).add_(level))
        return {"case": case, "x": buf[..., :c], "weight": 1 + 0.2 * normal(c), "bias": 0.2 * normal(c)}
    m, k, n = case["m"], case["k"], case["n"]
    to = TYPES[case["out"]]
    state = {"case": case, "x": normal(m, k).to(t)}
    if case["op"] == "linear":
        state["weight"] = (normal(n, k) * k ** -0.5).to(t)
        state["bias"] = 0.5 * normal(n)
    else:
        state["weight"] = torch.empty((case["e"], n, k), device="cuda", dtype=t)
        for w in state["weight"]:
            w.copy_(normal(n, k) * k ** -0.5)
        state["bias"] = 0.5 * normal(case["e"], n)
        sizes = lengths(case)
        state["sizes"] = sizes  # the batch's makeup, as the program that sorted the rows knows it
        state["ends"] = torch.tensor(sizes).cumsum(0).to(torch.int32).cuda()
        state["out"] = normal(m, n).to(to)  # rows behind the last group keep this
    state["residual"] = normal(m, n).to(to) if case["residual"] else None
    return state


def run(state):
    case = state["case"]
    if own:
        return run_own(case, state)
    if case["op"] == "group_norm":
        return plain_norm(case, state)
    if case["op"] == "linear":
        y = state["x"].float() @ state["weight"].float().t()
        return epilogue(case, y, state["bias"], state["residual"])
    return plain_grouped(case, state)


def run_own(case, s):
    from distributed_machine_learning_amd import ops

    if case["op"] == "group_norm":
        return ops.group_norm(s["x"], case["groups"], s["weight"], s["bias"], 1e-5, act=case["act"])
    if case["op"] == "linear":
        return ops.linear(s["x"], s["weight"], s["bias"], act=case["act"], residual=s["residual"],
                          act_last=case["act_last"], out_dtype=TYPES[case["out"]])
    return ops.grouped_linear(s["x"], s["weight"], s["ends"], s["bias"], act=case["act"], residual=s["residual"],
                              out=s["out"])


def activate(v, act):
    if act == "relu":
        return v.clamp(min=0)
    if act == "silu":
        return v / (1 + torch.exp(-v))
    if act == "gelu":
        return 0.5 * v * (1 + torch.erf(v * 0.5 ** 0.5))
    if act == "gelu_tanh":
        return 0.5 * v * (1 + torch.tanh((2 / math.pi) ** 0.5 * (v + 0.044715 * v * v * v)))
    return v


def epilogue(case, y, bias, residual):
    y = y + bias
    if residual is not None and case.get("act_last"):
        return activate(y + residual.float(), case["act"]).to(TYPES[case["out"]])
    y = activate(y, case["act"])
    return (y if residual is None else y + residual.float()).to(TYPES[case["out"]])


def plain_norm(case, s):
    n, c, g = case["n"], case["c"], case["groups"]
    x = s["x"].float().reshape(n, -1, g, c // g)
    d = x - x.mean((1, 3), keepdim=True)
    y = (d * torch.rsqrt(d.square().mean((1, 3), keepdim=True) + 1e-5)).reshape(s["x"].shape)
    return activate(y * s["weight"] + s["bias"], case["act"]).to(s["x"].dtype)


def plain_grouped(case, s):
    """The groups that have rows as one batch of products, each padded to the longest."""
    sizes, x, ends = s["sizes"], s["x"], s["ends"].long()
    rows = sum(sizes)
    y = s["out"].clone()
    if not rows:
        return y
    used = torch.tensor([i for i, v in enumerate(sizes) if v], device="cuda")
    r = torch.arange(rows, device="cuda")
    group = torch.searchsorted(ends, r, right=True)
    start = torch.cat([ends.new_zeros(1), ends[:-1]])
    slot = torch.searchsorted(used, group) * max(sizes) + r - start[group]
    padded = x.new_zeros((len(used) * max(sizes), case["k"]), dtype=torch.float32)
    padded[slot] = x[:rows].float()
    w = s["weight"][used].float().transpose(1, 2).contiguous()
    got = torch.bmm(padded.view(len(used), max(sizes), -1), w).reshape(-1, case["n"])[slot]
    residual = s["residual"]
    y[:rows] = epilogue(case, got, s["bias"][group], None if residual is None else residual[:rows])
    return y


def work(case):
    size = SIZE[case["dtype"]]
    if case["op"] == "group_norm":
        values = case["n"] * case["h"] * case["w"] * case["c"]
        return {"bytes": 2 * values * size + 8 * case["c"], "flops": 8 * values}
    sizes = lengths(case) if case["op"] == "grouped_linear" else [case["m"]]
    rows, used = sum(sizes), sum(v > 0 for v in sizes)
    outs = rows * case["n"] * SIZE[case["out"]] * (2 if case["residual"] else 1)
    return {"bytes": (rows * case["k"] + used * case["n"] * case["k"]) * size + outs + 4 * used * case["n"] + 4,
            "flops": 2 * rows * case["n"] * case["k"] + 4}


def exact(case, seed):
    """The definitions in 64 bits, one sample or one group at a time."""
    s = prepare(case, seed)

    def act(v):
        if case["act"] == "relu":
            return torch.where(v > 0, v, torch.zeros_like(v))
        if case["act"] == "silu":
            return v * torch.sigmoid(v)
        if case["act"] == "gelu":
            return v * torch.special.ndtr(v)
        if case["act"] == "gelu_tanh":
            return v * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (v + 0.044715 * v ** 3))
        return v

    x = s["x"]
    if case["op"] == "group_norm":
        y = torch.empty(x.shape, device="cuda", dtype=torch.float64)
        step, per = max(1, 60_000_000 // (case["h"] * case["w"] * case["c"])), case["c"] // case["groups"]
        w, b = s["weight"].double(), s["bias"].double()
        for i in range(0, case["n"], step):
            v = x[i:i + step].double().unflatten(-1, (case["groups"], per))
            var, mean = torch.var_mean(v, dim=(1, 2, 4), unbiased=False, keepdim=True)
            y[i:i + step] = act(((v - mean) / torch.sqrt(var + 1e-5)).flatten(-2) * w + b)
        return y
    sizes = s.get("sizes", [case["m"]])
    weight = s["weight"] if case["op"] == "grouped_linear" else s["weight"][None]
    bias = s["bias"].reshape(weight.shape[0], -1).double()
    y = s["out"].double() if "out" in s else torch.empty((case["m"], case["n"]), device="cuda", dtype=torch.float64)
    a = 0
    for e, rows in enumerate(sizes):
        if not rows:
            continue
        v = torch.mm(x[a:a + rows].double(), weight[e].double().t()) + bias[e]
        r = s["residual"][a:a + rows].double() if s["residual"] is not None else 0.0
        y[a:a + rows] = act(v + r) if case.get("act_last") else act(v) + r
        a += rows
    return y
