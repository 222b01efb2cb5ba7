"""Operators on 4-bit rows with a scale per 32 values (microscaled e2m1), as a server with 4-bit weights calls them: rounding rows to them and
back, a feed-forward's gated activation that ends in such rows, and the product of such rows with such a weight."""
from __future__ import annotations

import math

import torch

own = False
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SIZE = {"bf16": 2, "f16": 2, "f32": 4}
LIMIT = 7.0                                                     # of the clamped activation


def listed():
    return [
        # one decoded token's activations on their way into a product
        {"name": "round_token", "work": "round", "rows": 1, "cols": 4096, "dtype": "bf16", "out": "bf16"},
        # nothing divides anything: the last block of a row is short
        {"name": "round_odd", "work": "round", "rows": 203, "cols": 1999, "dtype": "f16", "out": "f16"},
        # a layer's gate and up projection brought to 4 bits when a model is loaded, and looked at
        {"name": "round_weight", "work": "round", "rows": 28672, "cols": 4096, "dtype": "bf16", "out": "bf16"},
        # the activation of a loaded server's decode step
        {"name": "glu_batch", "work": "glu", "rows": 64, "cols": 14336, "dtype": "bf16", "act": "silu"},
        # an odd hidden width, 32-bit projections, the tanh form of gelu
        {"name": "glu_odd", "work": "glu", "rows": 37, "cols": 5001, "dtype": "f32", "act": "gelu_tanh"},
        # the activation of a long prompt's portion
        {"name": "glu_prompt", "work": "glu", "rows": 4096, "cols": 14336, "dtype": "bf16", "act": "silu"},
        # one decoded token through a square projection of a 4096-wide model
        {"name": "linear_token", "work": "linear", "rows": 1, "k": 4096, "n": 4096, "dtype": "bf16", "out": "bf16", "bias": False, "given": False},
        # gate and up projection of a loaded server's decode step
        {"name": "linear_batch", "work": "linear", "rows": 64, "k": 4096, "n": 28672, "dtype": "bf16", "out": "bf16", "bias": False, "given": False},
        # output projection onto a large vocabulary for 37 sequences, logits in 32 bits
        {"name": "linear_head", "work": "linear", "rows": 37, "k": 3584, "n": 152064, "dtype": "bf16", "out": "f32", "bias": False, "given": False},
        # odd inner and outer sizes, a bias, half precision
        {"name": "linear_odd", "work": "linear", "rows": 203, "k": 1999, "n": 5001, "dtype": "f16", "out": "f16", "bias": True, "given": False},
        # a prompt's portion through a down projection, its rows in 4 bits already, as the activation leaves them
        {"name": "linear_down", "work": "linear", "rows": 1531, "k": 14336, "n": 4096, "dtype": "bf16", "out": "bf16", "bias": False, "given": True},
        # a long prompt through a gate and up projection: the largest product
        {"name": "linear_prompt", "work": "linear", "rows": 4096, "k": 3584, "n": 37888, "dtype": "bf16", "out": "bf16", "bias": False, "given": False},
    ]


def _spread(rng, lo, hi):
    """a whole number, even over the logarithm"""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["linear", "linear", "linear", "round", "glu"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    if kind == "linear":
        k, n = _spread(rng, 64, 14336), _spread(rng, 64, 65536)
        if rng.random() < 0.5:
            k, n = max(1, k // 64) * 64, max(1, n // 64) * 64
        return {"work": kind, "rows": _spread(rng, 1, max(1, min(4096, (1 << 38) // (k * n)))), "k": k, "n": n, "dtype": dtype,
                "out": rng.choice(["bf16", "f16", "f32"]), "bias": rng.random() < 0.5, "given": rng.random() < 0.25}
    cols = _spread(rng, 32, 16384)
    if rng.random() < 0.5:
        cols = cols // 32 * 32
    rows = _spread(rng, 1, min(16384, (1 << 26) // cols))
    if kind == "round":
        return {"work": kind, "rows": rows, "cols": cols, "dtype": dtype, "out": rng.choice(["bf16", "f32"])}
    return {"work": kind, "rows": rows, "cols": cols, "dtype": dtype, "act": rng.choice(["silu", "silu", "gelu_tanh", "relu", "swish_clamp"])}


def _activations(rows, k, dtype, g):
    """normed rows with a few channels that stand out, as a transformer's have them"""
    x = torch.randn(rows, k, device="cuda", generator=g)
    x *= 1.0 + 15.0 * (torch.rand(k, device="cuda", generator=g) < 0.004).float()
    return x.to(DTYPES[dtype])


def _rows4(n, k, middle, g):
    """a 4-bit checkpoint's rows: two values a byte, whole blocks (the last one's end holds zeros), and a byte of scale per block"""
    blocks = (k + 31) // 32
    q = torch.randint(0, 256, (n, blocks * 16), dtype=torch.uint8, device="cuda", generator=g)
    if k % 32:
        q[:, (k + 1) // 2:] = 0
        if k % 2:
            q[:, k // 2] &= 15
    return q, torch.randint(middle - 1, middle + 2, (n, blocks), dtype=torch.uint8, device="cuda", generator=g)


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    s = {"case": case}
    if case["work"] == "round":
        s["x"] = _activations(case["rows"], case["cols"], case["dtype"], g)
        return s
    if case["work"] == "glu":
        s["x"] = (torch.randn(case["rows"], 2 * case["cols"], device="cuda", generator=g) * 2.0).to(DTYPES[case["dtype"]])
        return s
    if case["given"]:
        s["x"], s["x_scale"] = _rows4(case["rows"], case["k"], 125, g)
    else:
        s["x"], s["x_scale"] = _activations(case["rows"], case["k"], case["dtype"], g), None
    s["w"], s["scale"] = _rows4(case["n"], case["k"], 126 - round(0.5 * math.log2(case["k"])), g)
    s["bias"] = torch.randn(case["n"], device="cuda", generator=g) if case["bias"] else None
    if own:                                                     # the weight as a program keeps it
        from fastllm_b200 import ops
        s["weight"] = ops.weight4(s["w"], s["scale"])
    return s


def _round4(x):
    """x in 64 bits -> the values that its 4-bit rows stand for, and the scales' bytes.  In 64 bits, since a value next to a border decides."""
    rows, k = x.shape
    b = torch.nn.functional.pad(x, (0, -k % 32)).reshape(rows, -1, 32)
    most = b.abs().amax(-1, keepdim=True)
    e = torch.where(most > 0, torch.frexp(most).exponent - 3, -127).clamp(min=-127)           # floor(log2 a) - 2
    v = torch.ldexp(b, -e)
    step = torch.ldexp(torch.ones_like(v), (torch.frexp(v).exponent - 2).clamp(min=-1))
    v = (torch.round(v / step) * step).clamp(-6.0, 6.0)
    return torch.ldexp(v, e).reshape(rows, -1)[:, :k], (e[..., 0] + 127).to(torch.uint8)


def _values(q, scale, k):
    """the values that 4-bit rows stand for"""
    table = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device=q.device)
    table = torch.cat([table, -table])
    v = table[torch.stack([q & 15, q >> 4], -1).long()].reshape(len(q), -1, 32)
    return torch.ldexp(v, scale.int()[..., None] - 127).reshape(len(q), -1)[:, :k]


def _activation(x, act):
    g, u = x.double().chunk(2, -1)
    if act == "silu":
        return g / (1.0 + torch.exp(-g)) * u
    if act == "gelu_tanh":
        return g / (1.0 + torch.exp(-2.0 * math.sqrt(2.0 / math.pi) * (g + 0.044715 * g * g * g))) * u
    if act == "relu":
        return g.clamp(min=0.0) * u
    g = g.clamp(max=LIMIT)
    return g / (1.0 + torch.exp(-1.702 * g)) * (u.clamp(-LIMIT, LIMIT) + 1.0)


def run(state):
    case = state["case"]
    if own:
        from fastllm_b200 import ops
        if case["work"] == "linear":
            return ops.linear4(state["x"], state["weight"], state["bias"], x_scale=state["x_scale"], out_dtype=DTYPES[case["out"]])
        if case["work"] == "round":
            q, scale = ops.quantize4(state["x"])
            return {"values": ops.dequantize4(q, scale, cols=case["cols"], dtype=DTYPES[case["out"]]), "scale": scale}
        q, scale = ops.glu4(state["x"], case["act"], limit=LIMIT)
        return {"values": ops.dequantize4(q, scale, cols=case["cols"], dtype=torch.bfloat16), "scale": scale}
    if case["work"] == "round":
        values, scale = _round4(state["x"].double())
        return {"values": values.to(DTYPES[case["out"]]), "scale": scale}
    if case["work"] == "glu":
        values, scale = _round4(_activation(state["x"], case["act"]))
        return {"values": values.to(torch.bfloat16), "scale": scale}
    x = _values(state["x"], state["x_scale"], case["k"]) if case["given"] else _round4(state["x"].double())[0].float()
    y = x @ _values(state["w"], state["scale"], case["k"]).T
    return (y if state["bias"] is None else y + state["bias"]).to(DTYPES[case["out"]])


def _bytes4(rows, cols):
    return rows * ((cols + 31) // 32) * 17


def work(case):
    r = case["rows"]
    if case["work"] == "linear":
        k, n = case["k"], case["n"]
        rows = _bytes4(r, k) if case["given"] else r * k * SIZE[case["dtype"]]
        return {"bytes": rows + _bytes4(n, k) + r * n * SIZE[case["out"]] + (4 * n if case["bias"] else 0), "flops": 2.0 * r * n * k}
    c = case["cols"]
    if case["work"] == "round":                                 # there and back: the 4-bit rows are written and read
        return {"bytes": r * c * (SIZE[case["dtype"]] + SIZE[case["out"]]) + 2 * _bytes4(r, c), "flops": 4.0 * r * c}
    return {"bytes": r * c * (2 * SIZE[case["dtype"]] + 2) + 2 * _bytes4(r, c), "flops": 12.0 * r * c}


def _exact_round4(x):
    """by the borders between neighbours: each belongs to the neighbour with the even mantissa"""
    rows, k = x.shape
    blocks = (k + 31) // 32
    b = x.new_zeros(rows, blocks * 32)
    b[:, :k] = x
    b = b.view(rows, blocks, 32)
    most = torch.linalg.vector_norm(b, ord=math.inf, dim=-1)
    e = torch.floor(torch.log2(most))                           # put right where the logarithm's rounding crossed a whole number
    e = torch.where(torch.pow(2.0, e) > most, e - 1.0, torch.where(torch.pow(2.0, e + 1.0) <= most, e + 1.0, e))
    e = torch.where(most > 0, e - 2.0, -127.0).clamp(min=-127.0)
    m = b.abs() / torch.pow(torch.tensor(2.0, dtype=x.dtype, device=x.device), e)[..., None]
    v = torch.zeros_like(m)
    for border, up, above in ((0.25, 0.5, False), (0.75, 0.5, True), (1.25, 0.5, False), (1.75, 0.5, True), (2.5, 1.0, False), (3.5, 1.0, True), (5.0, 2.0, False)):
        v += up * ((m >= border) if above else (m > border))
    return (torch.sign(b) * v * torch.pow(torch.tensor(2.0, dtype=x.dtype, device=x.device), e)[..., None]).view(rows, -1)[:, :k].contiguous()


def _exact_values(q, scale, k):
    low, high = (q & 15).to(torch.int32), (q >> 4).to(torch.int32)
    c = torch.empty(q.shape[0], 2 * q.shape[1], dtype=torch.int32, device=q.device)
    c[:, 0::2], c[:, 1::2] = low, high
    m, e = (c & 1).double(), ((c >> 1) & 3).double()
    v = torch.where(e > 0, (1.0 + 0.5 * m) * torch.pow(2.0, e - 1.0), 0.5 * m) * torch.where(c > 7, -1.0, 1.0)
    v *= torch.pow(2.0, scale.double() - 127.0).repeat_interleave(32, dim=1)
    return v[:, :k]


def _exact_activation(x, act):
    f = x.shape[1] // 2
    g, u = x[:, :f].double(), x[:, f:].double()
    if act == "silu":
        return g * torch.sigmoid(g) * u
    if act == "gelu_tanh":
        return g * torch.sigmoid(1.5957691216057308 * g * (1.0 + 0.044715 * g * g)) * u
    if act == "relu":
        return torch.where(g > 0, g, 0.0) * u
    g = torch.minimum(g, torch.tensor(LIMIT, dtype=g.dtype, device=g.device))
    return g * torch.sigmoid(1.702 * g) * (u.clip(-LIMIT, LIMIT) + 1.0)


def exact(case, seed):
    s = prepare(case, seed)
    if case["work"] == "linear":
        x = _exact_values(s["x"], s["x_scale"], case["k"]) if case["given"] else _exact_round4(s["x"].double())
        parts = [torch.mm(x, _exact_values(w, e, case["k"]).t()) for w, e in zip(torch.split(s["w"], 8192), torch.split(s["scale"], 8192))]
        y = torch.cat(parts, 1)
        return y if s["bias"] is None else y + s["bias"].double()
    parts = torch.split(s["x"], 4096)
    if case["work"] == "round":
        return {"values": torch.cat([_exact_round4(p.double()) for p in parts]), "scale": None}
    return {"values": torch.cat([_exact_round4(_exact_activation(p, case["act"])) for p in parts]), "scale": None}
