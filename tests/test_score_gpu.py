"""GPU tests of log probabilities over a forward's logits (DeviceCache.logprobs, ContinuousBatcher, models.score, the command line) and of the
8-bit output projection of layered models.

Bounds: log probabilities are those of the logits that the same forward returned, in 64 bits, to (vocab / 256 + 80) u + 16 u max|z|, u = 2^-24 (sums in
32 bits, see test_ops_gpu.py); against an oracle's logits, whose positions agree to a relative rms error E, to 2 sqrt(vocab) E rms (a log probability moves by
twice the largest logit's error at most)."""
import json
import os
import subprocess

import numpy as np
import pytest

from fastllm_b200 import models
from fastllm_b200._lib import FastllmError
from oracle import rofetar as O
from oracle import synth

import test_rofetar_gpu as rofetar
from helpers import golden_weights, product_model

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def _lp(logits):
    z = np.asarray(logits, dtype=np.float64)
    m = z.max(-1, keepdims=True)
    return z - m - np.log(np.exp(z - m).sum(-1, keepdims=True))


def _check(r, logits, tokens, top):
    lp = _lp(logits)
    tol = (lp.shape[1] / 256 + 80) * U + 16 * U * np.abs(logits).max()
    if tokens is not None:
        t = np.asarray(tokens).reshape(len(lp), -1)
        want = np.where(t < 0, 0.0, np.take_along_axis(lp, np.maximum(t, 0), 1)).reshape(np.shape(tokens))
        assert r.logprob.shape == want.shape and np.abs(r.logprob - want).max() <= tol
    assert np.abs(r.logsumexp - (logits[:, 0] - lp[:, 0])).max() <= tol
    assert np.abs(r.entropy + (np.exp(lp) * lp).sum(1)).max() <= tol * (1 + np.abs(lp).max())
    ids = np.argsort(-logits.astype(np.float64), axis=1, kind="stable")[:, :top]
    assert np.array_equal(r.top_ids, ids) and (top == 0 or np.abs(r.top_logprobs - np.take_along_axis(lp, ids, 1)).max() <= tol)


# ---- over the last forward's logits ---------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("name", ["llama", "mistral", "qwen2", "mixtral"])
def test_last_forward_of_the_llama_family(name):
    cfg, w, _ = golden_weights(name)
    model, _ = product_model(cfg, w)
    prompt = synth.token_ids(3, cfg.vocab_size, (3, 7))
    cache = models.DeviceCache(model.dev, 3, 64)
    with pytest.raises(FastllmError, match="left logits of 0 rows"):
        cache.logprobs(rows=1)
    logits = cache.forward(prompt, 0)
    tokens = np.arange(12).reshape(3, 4) * 5
    tokens[1, 2] = -1
    _check(cache.logprobs(tokens, 8), logits, tokens, 8)
    _check(cache.logprobs(tokens[:2, 0], 0), logits[:2], tokens[:2, 0], 0)
    _check(cache.logprobs(top=32, rows=3), logits, None, 32)
    hot = cache.logprobs(tokens, 3, temperature=2.0)
    assert np.abs(hot.logprob - np.where(tokens < 0, 0, np.take_along_axis(_lp(logits / 2), np.maximum(tokens, 0), 1))).max() <= 1e-5
    step = cache.forward(np.asarray([[5], [6], [7]], dtype=np.uint32), 7)              # a step of single tokens, its logits this time
    _check(cache.logprobs([9, 8, 7], 5), step, [9, 8, 7], 5)
    got = cache.forward_greedy(np.asarray([[5], [6], [7]], dtype=np.uint32), 8)
    assert np.array_equal(cache.logprobs(rows=3, top=1).top_ids[:, 0], got)
    for bad in (dict(), dict(rows=4), dict(rows=1, top=33), dict(rows=1, top=-1), dict(rows=1, temperature=0.0), dict(tokens=[1, 2], rows=1), dict(rows=-1)):
        with pytest.raises(FastllmError):
            cache.logprobs(**bad)
    cache.decode_greedy_loop(got, 9, 3)
    with pytest.raises(FastllmError, match="left logits of 0 rows"):
        cache.logprobs(rows=1)


def test_last_forward_of_slots_and_of_one_row():
    cfg, w, _ = golden_weights("llama")
    model, _ = product_model(cfg, w)
    cache = models.DeviceCache(model.dev, 4, 64)
    logits = cache.forward_slots([2], synth.token_ids(1, cfg.vocab_size, (1, 9)), [0])
    _check(cache.logprobs([3], 4), logits, [3], 4)
    cache.forward_slots([0], synth.token_ids(2, cfg.vocab_size, (1, 4)), [0])
    logits = cache.forward_slots([0, 2], np.asarray([[7], [8]], dtype=np.uint32), [4, 9])
    _check(cache.logprobs([3, -1], 4), logits, [3, -1], 4)
    _check(cache.logprobs([3, -1], 4), logits, [3, -1], 4)             # (asked twice)
    with pytest.raises(FastllmError):
        cache.forward_slots([0], np.asarray([[cfg.vocab_size]], dtype=np.uint32), [5])     # refused before anything ran
    _check(cache.logprobs([3, -1], 4), logits, [3, -1], 4)


def test_logits_that_stay_on_the_device():
    cfg = rofetar.hybrid_cfg()
    _, model = rofetar.build(cfg, 3)
    toks = rofetar.tokens(cfg, 40)
    a, b = (model.new_device_cache(max_batch=2, max_seq=64) for _ in range(2))
    logits = a.forward_ragged([0, 1], [toks[:25], toks[25:]], [range(25), [3, 14]])
    assert b.forward_ragged([0, 1], [toks[:25], toks[25:]], [range(25), [3, 14]], fetch=False) is None
    tokens = np.arange(27) % cfg["vocab"]
    for c in (a, b):
        _check(c.logprobs(tokens, 6), logits, tokens, 6)
    for _ in range(4):                                                  # single tokens: eager, captured, replayed
        want = a.forward_ragged([1, 0], [[5], [6]])
        assert b.forward_ragged([1, 0], [[5], [6]], fetch=False) is None
        _check(b.logprobs([1, 2], 3), want, [1, 2], 3)
    assert np.array_equal(b.forward_ragged([0], [[9]]), a.forward_ragged([0], [[9]]))     # fetched again
    b.forward_ragged([0], [[9]], [[]], fetch=False)
    with pytest.raises(FastllmError, match="left logits of 0 rows"):
        b.logprobs(rows=1)


# ---- scoring and generation -----------------------------------------------------------------------------------------------------------
def _texts(cfg, sizes):
    return [rofetar.tokens(cfg, n, seed=70 + n) for n in sizes]


@pytest.mark.parametrize("portion", [8, 40, 512])
def test_score_against_the_oracle(portion):
    cfg = rofetar.hybrid_cfg()
    oracle, model = rofetar.build(cfg, 4)
    texts = _texts(cfg, [70, 1, 2, 33, 9])
    for t, s in zip(texts, models.score(model, texts, top=4, portion=portion)):
        assert s.logprobs.shape == (len(t) - 1,) and s.top_ids.shape == (len(t) - 1, 4)
        if len(t) < 2:
            continue
        ref = oracle.run(t)[:-1]
        lp = _lp(ref)
        tol = 2 * np.sqrt(cfg["vocab"]) * rofetar.TOL["f32"] * np.sqrt((ref ** 2).mean())
        assert np.abs(s.logprobs - lp[np.arange(len(t) - 1), t[1:]]).max() <= tol
        assert np.abs(s.top_logprobs - np.sort(lp, axis=1)[:, ::-1][:, :4]).max() <= tol
        assert s.total == pytest.approx(float(s.logprobs.sum()), rel=1e-5)


@pytest.mark.parametrize("chunk", [None, 16])
def test_generated_tokens_and_their_log_probabilities(chunk):
    """what generation tells of its tokens is what scoring the whole text tells of them"""
    cfg = rofetar.hybrid_cfg()
    _, model = rofetar.build(cfg, 5)
    prompts = _texts(cfg, [3, 40, 17, 8])
    new = lambda: models.ContinuousBatcher(model, max_batch=3, eos_token_id=None, prefill_chunk=chunk)  # noqa: E731
    plain = new().generate(prompts, 7)
    ids, told = new().generate(prompts, 7, logprobs=3)
    assert ids == plain
    scored = models.score(model, [p + i for p, i in zip(prompts, ids)], top=3)
    for p, about, s in zip(prompts, told, scored):
        n = len(p) - 1
        tol = 4 * np.sqrt(cfg["vocab"]) * rofetar.TOL["f32"] * max(1.0, np.abs(s.logprobs).max())
        assert np.abs(np.array([d["logprob"] for d in about]) - s.logprobs[n:]).max() <= tol
        assert np.abs(np.array([[v for _, v in d["top"]] for d in about]) - s.top_logprobs[n:]).max() <= tol
        assert all(d["top"][0][1] >= d["logprob"] - tol for d in about)


# ---- 8-bit output projection ----------------------------------------------------------------------------------------------------------
def _eight_bit_bound(h, w):
    """|y8 - h w^T| <= sum over j of |h_j| t / 2 + |w_j| s / 2 + s t / 4, s and t the steps of the row and of the channel; and what f32 rounds"""
    s, t = np.abs(h).max(1) / 127, np.abs(w).max(1) / 127
    k = h.shape[1]
    return np.abs(h).sum(1)[:, None] * t / 2 + np.abs(w).sum(1) * s[:, None] / 2 + k * s[:, None] * t / 4 + 1e-4


@pytest.mark.parametrize("width, vocab", [(48, 48), (64, 200), (40, 1000)])
def test_head_in_8_bits(width, vocab):
    """the head read off a model whose head is the identity (its logits are the normed rows), every position of a prompt and of single steps"""
    cfg = rofetar.config([rofetar.att(), rofetar.delta(mlp=rofetar.dense())], vocab=vocab, width=width)
    w = O.random_weights(cfg, 6)
    eye = dict(w, head=np.eye(vocab, width, dtype=np.float32))
    make = lambda ws, bits: models.RofetarWithConfig.initialize_model(cfg, {k: rofetar.to_bits(v) for k, v in ws.items()}, "bf16", head_bits=bits)[0]  # noqa: E731
    toks = rofetar.tokens(cfg, 150)
    rows = [model.new_device_cache(2, 256) for model in (make(eye, 16), make(w, 8), make(w, 16))]
    for step in [toks] + [[t] for t in (5, 6, 7, 8)]:
        h, y8, y16 = (c.forward_ragged([1], [step], [range(len(step))]) for c in rows)
        h = h[:, :width].astype(np.float64)
        far = np.abs(y8 - h @ w["head"].astype(np.float64).T)
        assert (far <= _eight_bit_bound(h, w["head"].astype(np.float64))).all()
        d = (y8 - y16).astype(np.float64)
        rms = np.sqrt((d ** 2).mean() / (y16.astype(np.float64) ** 2).mean())
        assert 1e-5 < rms < 0.03        # (steps of a 127th of the largest of a row: 1 % where that is four times the rms)
    _check(rows[1].logprobs([3], 5), y8, [3], 5)


def test_tied_head_in_8_bits():
    """the embedding table itself stays as it is; looped layers, every position of a prompt, then single steps"""
    import test_latodra_gpu as latodra
    from oracle import latodra as OL
    cfg = latodra.deep_cfg(vocab=96)
    w = OL.random_weights(cfg, 8)
    make = lambda bits: models.LatodraWithConfig.initialize_model(cfg, {k: latodra.to_bits(v) for k, v in w.items()}, "bf16", head_bits=bits)[0]  # noqa: E731
    a, b = (make(bits).new_device_cache(2, 128) for bits in (16, 8))
    for step in [latodra.tokens(cfg, 60)] + [[t] for t in (5, 6, 7, 8)]:
        y16, y8 = (c.forward_ragged([0], [step], [range(len(step))]).astype(np.float64) for c in (a, b))
        assert 1e-5 < np.sqrt(((y8 - y16) ** 2).mean() / (y16 ** 2).mean()) < 0.03
    assert a.model.streamed_bytes() - b.model.streamed_bytes() == 96 * 32


def test_head_in_8_bits_streams_less_and_is_refused_elsewhere():
    cfg = rofetar.config([rofetar.att()], vocab=96, width=32)
    w = {k: rofetar.to_bits(v) for k, v in O.random_weights(cfg, 7).items()}
    make = lambda bits, dtype="bf16": models.RofetarWithConfig.initialize_model(cfg, w, dtype, head_bits=bits)[0]  # noqa: E731
    assert make(16).dev.streamed_bytes() - make(8).dev.streamed_bytes() == 96 * 32
    for bits, dtype in ((8, "f32"), (4, "bf16"), (7, "bf16"), (-8, "bf16")):
        with pytest.raises(FastllmError, match="head_bits"):
            make(bits, dtype)


def test_command_line(tmp_path):
    """generate --logprobs --head-bits and score, as processes"""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    cfg = rofetar.hybrid_cfg()
    w = O.random_weights(cfg, 29)
    rofetar._write_checkpoint(tmp_path / "m", cfg, w)
    prompts = _texts(cfg, [3, 20])

    def run(*args):
        r = subprocess.run(["python3", "-m", "fastllm_b200", *args, "--model", str(tmp_path / "m")], capture_output=True, text=True, timeout=600, cwd=root,
                           env=dict(os.environ, PYTHONPATH=root))
        assert r.returncode == 0, r.stderr[-2000:]
        return [json.loads(line) for line in r.stdout.splitlines() if line.startswith("{")]

    ids = [a for p in prompts for a in ("--prompt-ids", ",".join(map(str, p)))]
    plain = run("generate", *ids, "--dtype", "f32", "--max-tokens", "5")
    told = run("generate", *ids, "--dtype", "f32", "--max-tokens", "5", "--logprobs", "2")
    assert [d["generated"] for d in plain] == [d["generated"] for d in told] and "logprobs" not in plain[0]
    texts = [p + d["generated"] for p, d in zip(prompts, told)]
    ids = [a for t in texts for a in ("--ids", ",".join(map(str, t)))]
    for d, s, p in zip(told, run("score", *ids, "--dtype", "f32", "--top", "2"), prompts):
        assert np.abs(np.array([x["logprob"] for x in d["logprobs"]]) - s["logprobs"][len(p) - 1:]).max() < 1e-2
        assert len(s["top"]) == len(s["logprobs"]) == len(s["ids"]) - 1 and s["total"] == pytest.approx(sum(s["logprobs"]), rel=1e-4)
    for a, b in zip(run("score", *ids), run("score", *ids, "--head-bits", "8")):
        assert a["logprobs"] != b["logprobs"] and np.abs(np.subtract(a["logprobs"], b["logprobs"])).max() < 0.5
