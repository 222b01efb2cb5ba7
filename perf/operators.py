"""Operators of the output side, as a server or a scoring job calls them: the matrix product in 8-bit integers with a scale per token and per
channel, the log probabilities of given tokens with entropy and top alternatives, and the two in a row (an 8-bit output projection whose
logits become log probabilities)."""
from __future__ import annotations

import math

import numpy as np
import torch

own = False
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SIZE = {"bf16": 2, "f16": 2, "f32": 4}


def listed():
    return [
        # one decoded token through a square projection of a 4096-wide model
        {"name": "linear_token", "work": "linear8", "rows": 1, "k": 4096, "n": 4096, "dtype": "bf16", "out": "bf16", "bias": False},
        # gate and up projection of a loaded server's decode step
        {"name": "linear_batch", "work": "linear8", "rows": 64, "k": 4096, "n": 28672, "dtype": "bf16", "out": "bf16", "bias": False},
        # output projection onto a large vocabulary for 37 sequences, logits in 32 bits
        {"name": "linear_head", "work": "linear8", "rows": 37, "k": 3584, "n": 152064, "dtype": "bf16", "out": "f32", "bias": False},
        # nothing divides anything: odd inner and outer sizes, a bias, half precision
        {"name": "linear_odd", "work": "linear8", "rows": 203, "k": 1999, "n": 5001, "dtype": "f16", "out": "f16", "bias": True},
        # a prompt's portion through a down projection: long sums, few output columns
        {"name": "linear_down", "work": "linear8", "rows": 1531, "k": 14336, "n": 4096, "dtype": "bf16", "out": "bf16", "bias": False},
        # a long prompt through a gate and up projection: the largest product
        {"name": "linear_prompt", "work": "linear8", "rows": 4096, "k": 3584, "n": 37888, "dtype": "bf16", "out": "bf16", "bias": False},
        # one chat's token with its five alternatives
        {"name": "logprobs_chat", "work": "logprobs", "rows": 1, "vocab": 32000, "dtype": "f32", "given": 1, "top": 5, "temperature": 1.0, "banned": 0.0},
        # a server's step: 64 sequences, twenty alternatives, half of the vocabulary ruled out by a grammar
        {"name": "logprobs_batch", "work": "logprobs", "rows": 64, "vocab": 152064, "dtype": "f32", "given": 1, "top": 20, "temperature": 1.0, "banned": 0.5},
        # multiple choice: four given answers per row, an odd vocabulary, half precision, a temperature
        {"name": "logprobs_choices", "work": "logprobs", "rows": 1000, "vocab": 32003, "dtype": "f16", "given": 4, "top": 5, "temperature": 0.7, "banned": 0.0},
        # scoring a long text: no alternatives
        {"name": "logprobs_text", "work": "logprobs", "rows": 2048, "vocab": 152064, "dtype": "bf16", "given": 1, "top": 0, "temperature": 1.0, "banned": 0.0},
        # scoring a short answer: output projection and log probabilities of its 19 tokens
        {"name": "score_answer", "work": "score", "rows": 19, "k": 2048, "vocab": 32000, "dtype": "bf16", "top": 5},
        # scoring a text's portion the same way
        {"name": "score_text", "work": "score", "rows": 777, "k": 4096, "vocab": 32000, "dtype": "bf16", "top": 5},
    ]


def _spread(rng, lo, hi):
    """a whole number, even over the logarithm"""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["linear8", "linear8", "logprobs", "logprobs", "score"])
    if kind == "linear8":
        k, n = _spread(rng, 256, 14336), _spread(rng, 256, 65536)
        if rng.random() < 0.5:
            k, n = max(1, k // 64) * 64, max(1, n // 64) * 64
        rows = _spread(rng, 1, max(1, min(4096, (1 << 38) // (k * n))))
        return {"work": kind, "rows": rows, "k": k, "n": n, "dtype": rng.choice(["bf16", "bf16", "f16", "f32"]),
                "out": rng.choice(["bf16", "f16", "f32"]), "bias": rng.random() < 0.5}
    if kind == "logprobs":
        vocab = _spread(rng, 500, 160000)
        return {"work": kind, "rows": _spread(rng, 1, min(4096, (1 << 28) // vocab)), "vocab": vocab, "dtype": rng.choice(["bf16", "f16", "f32"]),
                "given": rng.choice([1, 1, 2, 5]), "top": rng.choice([0, 1, 5, 20]), "temperature": rng.choice([1.0, 0.7, 1.3]),
                "banned": rng.choice([0.0, 0.0, 0.5, 0.99])}
    k, vocab = 64 * _spread(rng, 8, 64), _spread(rng, 2000, 64000)
    return {"work": kind, "rows": _spread(rng, 1, min(1024, (1 << 36) // (k * vocab))), "k": k, "vocab": vocab,
            "dtype": rng.choice(["bf16", "f16"]), "top": rng.choice([0, 5, 20])}


def _activations(rows, k, dtype, g):
    """normed rows with a few channels that stand out, as a transformer's have them"""
    x = torch.randn(rows, k, device="cuda", generator=g)
    x *= 1.0 + 15.0 * (torch.rand(k, device="cuda", generator=g) < 0.004).float()
    return x.to(DTYPES[dtype])


def _weight8(n, k, g):
    """an 8-bit checkpoint's matrix: whole numbers per channel and their scales; rows start on 16-byte borders"""
    w = torch.empty(n, (k + 15) // 16 * 16, dtype=torch.int8, device="cuda")
    w.random_(-127, 128, generator=g)
    scale = (0.5 + torch.rand(n, device="cuda", generator=g)) * (k ** -0.5 / 73.0)
    return w[:, :k], scale


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    s = {"case": case}
    if case["work"] == "logprobs":
        x = torch.randn(case["rows"], case["vocab"], device="cuda", generator=g) * 2.5
        x += 6.0 * (torch.rand(case["rows"], case["vocab"], device="cuda", generator=g) < 1e-3).float()
        if case["banned"]:
            x.masked_fill_(torch.rand(case["rows"], case["vocab"], device="cuda", generator=g) < case["banned"], -math.inf)
            x[:, 0] = 0.0                                       # (the end of the text is always allowed)
        s["logits"] = x.to(DTYPES[case["dtype"]])
        s["tokens"] = torch.randint(0, case["vocab"], (case["rows"], case["given"]), device="cuda", generator=g)
        s["tokens"][::2, 0] = s["logits"][::2].argmax(-1)       # half of the tokens are likely ones
        return s
    n = case["n"] if case["work"] == "linear8" else case["vocab"]
    s["x"] = _activations(case["rows"], case["k"], case["dtype"], g)
    s["w"], s["scale"] = _weight8(n, case["k"], g)
    s["bias"] = torch.randn(n, device="cuda", generator=g) if case.get("bias") else None
    if case["work"] == "score":
        s["scale"] = s["scale"] * 2.5
        s["tokens"] = torch.randint(0, n, (case["rows"],), device="cuda", generator=g)
    return s


def _quantize(x):
    """Whole numbers -127..127 per row and the row's scale; in 64 bits, where 127 x / max next to a half decides."""
    most = x.float().abs().amax(-1, keepdim=True)
    return torch.round(127.0 * x.double() / most.double()), (most.double() / 127.0).float()


def _linear8(x, w, scale, bias, dtype):
    """sums of whole numbers up to 2^28: in 64 bits"""
    q, xs = _quantize(x)
    y = (q @ w.double().T).float() * xs * scale
    return (y if bias is None else y + bias).to(dtype)


def _logprobs(x, tokens, top, temperature):
    x = x.float()
    z = x * (1.0 / temperature)
    most = z.amax(-1, keepdim=True)
    e = torch.exp(z - most)
    total = e.sum(-1, keepdim=True)
    log_z = most + torch.log(total)
    entropy = torch.log(total) - torch.where(e > 0, e * (z - most), 0.0).sum(-1, keepdim=True) / total
    given = tokens if tokens.ndim == 2 else tokens[:, None]
    lp = z.gather(1, given) - log_z
    out = {"logprob": lp.reshape(tokens.shape), "logsumexp": log_z[:, 0], "entropy": entropy[:, 0]}
    if top:
        ids = torch.sort(x, dim=-1, descending=True, stable=True).indices[:, :top]     # equal ones: the lowest index first
        out["top_ids"], out["top_logprobs"] = ids.int(), z.gather(1, ids) - log_z
    return out


def run(state):
    case = state["case"]
    if own:
        from fastllm_b200 import ops
        if case["work"] == "linear8":
            return ops.linear8(state["x"], state["w"], state["scale"], state["bias"], out_dtype=DTYPES[case["out"]])
        if case["work"] == "logprobs":
            r = ops.logprobs(state["logits"], state["tokens"], top=case["top"], temperature=case["temperature"])
        else:
            logits = ops.linear8(state["x"], state["w"], state["scale"], out_dtype=torch.float32)
            r = ops.logprobs(logits, state["tokens"], top=case["top"])
        out = {"logprob": r.logprob, "logsumexp": r.logsumexp, "entropy": r.entropy}
        if case["top"]:
            out["top_ids"], out["top_logprobs"] = r.top_ids, r.top_logprobs
        return out
    if case["work"] == "linear8":
        return _linear8(state["x"], state["w"], state["scale"], state["bias"], DTYPES[case["out"]])
    if case["work"] == "logprobs":
        return _logprobs(state["logits"], state["tokens"], case["top"], case["temperature"])
    return _logprobs(_linear8(state["x"], state["w"], state["scale"], None, torch.float32), state["tokens"], case["top"], 1.0)


def work(case):
    r = case["rows"]
    if case["work"] == "logprobs":
        v = case["vocab"]
        return {"bytes": r * (v * SIZE[case["dtype"]] + case["given"] * 12 + 8 + case["top"] * 8), "flops": 6.0 * r * v}
    k, n = case["k"], case["n"] if case["work"] == "linear8" else case["vocab"]
    moved = r * k * SIZE[case["dtype"]] + n * k + 4 * n
    if case["work"] == "linear8":
        return {"bytes": moved + r * n * SIZE[case["out"]] + (4 * n if case["bias"] else 0), "flops": 2.0 * r * n * k}
    return {"bytes": moved + r * (12 + 8 + case["top"] * 8), "flops": 2.0 * r * n * k + 6.0 * r * n}


def _exact_logits(x, w, scale, bias=None):
    """numpy-style: the nearest whole number of 127 x / max, halves to even, from the two neighbours' distances; then the products"""
    x = x.double()
    most = x.abs().amax(-1, keepdim=True)
    low = torch.floor(127.0 * x / most)
    over = 254.0 * x - (2.0 * low + 1.0) * most                 # the sign of 127 x / max - (low + 1/2)
    q = torch.where(over > 0, low + 1.0, torch.where(over < 0, low, low + torch.remainder(low, 2.0)))
    y = torch.mm(q, w.double().t()) * (most / 127.0)
    y *= scale.double()
    return y if bias is None else y + bias.double()


def _exact_logprobs(x, tokens, top, temperature):
    rows, got = [], []
    for part, given in zip(torch.split(x, 256), torch.split(tokens, 256)):
        z = part.double() / temperature
        log_z = torch.logsumexp(z, -1)
        p = torch.exp(z - log_z[:, None])
        rows.append((log_z, log_z - torch.nansum(p * z.masked_fill(p == 0, 0.0), -1)))
        got.append(torch.gather(z, 1, given.reshape(len(part), -1)) - log_z[:, None])
        if top:
            best = torch.topk(part.double(), top, dim=-1).values     # (values alone: ties do not matter)
            rows[-1] += (best / temperature - log_z[:, None],)
    out = {"logprob": torch.cat(got).reshape(tokens.shape), "logsumexp": torch.cat([r[0] for r in rows]), "entropy": torch.cat([r[1] for r in rows])}
    if top:
        out["top_ids"], out["top_logprobs"] = None, torch.cat([r[2] for r in rows])
    return {k: None if v is None else v.cpu().numpy().astype(np.float64) for k, v in out.items()}


def exact(case, seed):
    s = prepare(case, seed)
    if case["work"] == "logprobs":
        return _exact_logprobs(s["logits"], s["tokens"], case["top"], case["temperature"])
    y = _exact_logits(s["x"], s["w"], s["scale"], s["bias"])
    return y if case["work"] == "linear8" else _exact_logprobs(y, s["tokens"], case["top"], 1.0)
