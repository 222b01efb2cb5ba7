"""CPU tests of log probabilities above the caches: ContinuousBatcher.generate(logprobs=...) and models.score over stand-in caches."""
import zlib

import numpy as np
import pytest

from fastllm_b200 import models
from fastllm_b200._lib import FastllmError

VOCAB = 23


def _row(history):
    row = np.random.RandomState(zlib.crc32(np.asarray(history, dtype=np.uint32).tobytes())).standard_normal(VOCAB).astype(np.float32) * 2
    row[2] += 1.5
    return row


def _lp(row):
    z = row.astype(np.float64)
    return z - z.max() - np.log(np.exp(z - z.max()).sum())


class _Cache:
    """logits of a row are a function of its slot's tokens; remembers the last forward's, as a DeviceCache does"""
    ragged = True

    def __init__(self, slots):
        self.max_batch, self.hist, self.last, self.sizes, self.max_seq, self.vocab = slots, [[] for _ in range(slots)], None, [], 30, VOCAB
        if not self.ragged:
            self.forward_ragged = None

    def _feed(self, slot, toks, places):
        rows = []
        for k, t in enumerate(toks):
            self.hist[slot].append(int(t))
            if k in places:
                rows.append(_row(self.hist[slot]))
        return rows

    def forward_slots(self, slots, ids, rope_offsets):
        self.last = np.stack([r for s, t in zip(slots, np.asarray(ids)) for r in self._feed(s, t, [len(t) - 1])])
        return self.last

    def forward_ragged(self, slots, token_lists, want=None, fetch=True):
        assert len(set(slots)) == len(slots) and all(len(t) > 0 for t in token_lists)
        self.sizes.append(sum(len(t) for t in token_lists))
        rows = [r for s, t, w in zip(slots, token_lists, want) for r in self._feed(s, t, list(w))]
        self.last = np.stack(rows) if rows else np.empty((0, VOCAB), np.float32)
        return self.last if fetch else None

    def logprobs(self, tokens=None, top=0, temperature=1.0, rows=None):
        lp = np.stack([_lp(r) for r in self.last[:len(tokens)]])
        ids = np.argsort(-lp, axis=1, kind="stable")[:, :top]
        given = np.array([0.0 if t < 0 else lp[i, t] for i, t in enumerate(tokens)])
        return models.LogProbs(given, np.zeros(len(tokens)), -(np.exp(lp) * lp).sum(1), ids.astype(np.int32), np.take_along_axis(lp, ids, 1))

    def slot_len(self, slot):
        return len(self.hist[slot])

    def slot_reset(self, slot):
        assert self.hist[slot]
        self.hist[slot] = []


class _Model:
    arch = "llama"


def _prompts(sizes):
    return [np.random.default_rng(i).integers(3, VOCAB, n).tolist() for i, n in enumerate(sizes)]


@pytest.mark.parametrize("chunk", [None, 4])
@pytest.mark.parametrize("temperature", [0.0, 0.8])
def test_generate_tells_log_probabilities(chunk, temperature):
    """the ids are those without logprobs; every emitted token has its log probability and alternatives, the token that ends a text has none"""
    prompts = _prompts([5, 9, 1, 7, 3])
    new = lambda: models.ContinuousBatcher(_Model(), max_batch=3, eos_token_id=2, cache=_Cache(3), prefill_chunk=chunk)  # noqa: E731
    plain = new().generate(prompts, 6, temperature)
    ids, told = new().generate(prompts, 6, temperature, logprobs=4)
    assert ids == plain and len({len(i) for i in ids}) > 1
    for p, out, about in zip(prompts, ids, told):
        assert len(out) == len(about)
        for k, (tok, d) in enumerate(zip(out, about)):
            lp = _lp(_row(p + out[:k]))
            assert d["logprob"] == pytest.approx(lp[tok], abs=1e-6)
            best = np.argsort(-lp, kind="stable")[:4]
            assert [i for i, _ in d["top"]] == best.tolist() and [v for _, v in d["top"]] == pytest.approx(lp[best].tolist(), abs=1e-6)


def test_generate_tells_nothing_for_no_tokens():
    cb = models.ContinuousBatcher(_Model(), 2, cache=_Cache(2))
    assert cb.generate([], 4, logprobs=0) == ([], [])
    assert cb.generate([[3, 4]], 0, logprobs=0) == ([[]], [[]])


@pytest.mark.parametrize("slots, portion", [(1, 1), (1, 512), (3, 3), (3, 7), (2, 64)])
def test_score_in_portions(slots, portion):
    """texts of any length, one and no token among them, in portions that end anywhere"""
    texts = _prompts([5, 1, 0, 30, 2, 11, 7])
    cache = _Cache(slots)
    got = models.score(_Model(), texts, top=3, cache=cache, portion=portion)
    assert max(cache.sizes) <= portion and all(not h for h in cache.hist)
    assert sum(cache.sizes) == sum(max(0, len(t) - 1) for t in texts)
    for t, s in zip(texts, got):
        assert s.logprobs.shape == s.entropy.shape == (max(0, len(t) - 1),) and s.top_ids.shape == s.top_logprobs.shape == (max(0, len(t) - 1), 3)
        for i in range(len(t) - 1):
            lp = _lp(_row(t[:i + 1]))
            assert s.logprobs[i] == pytest.approx(lp[t[i + 1]], abs=1e-6)
            assert s.top_ids[i].tolist() == np.argsort(-lp, kind="stable")[:3].tolist()
        assert s.total == pytest.approx(float(np.sum(s.logprobs)), abs=1e-5)


def test_score_refusals():
    with pytest.raises(FastllmError, match="layered models only"):
        models.score(_Model(), [[3, 4]])
    with pytest.raises(FastllmError, match="at least one token"):
        models.score(_Model(), [[3, 4]], cache=_Cache(4), portion=3)
    for bad in ([3] * 32, [3, VOCAB], [3, -1]):
        with pytest.raises(FastllmError, match="longer than the cache"):
            models.score(_Model(), [[3, 4], bad], cache=_Cache(2))
    assert models.score(_Model(), [[3] * 31], cache=_Cache(1))[0].logprobs.shape == (30,)
    used = _Cache(2)
    used.forward_slots([1], [[5, 6]], [0])
    with pytest.raises(FastllmError, match="holds a sequence"):
        models.score(_Model(), [[3, 4]], cache=used)


def test_score_gives_its_slots_back_after_an_error():
    class _Broken(_Cache):
        def logprobs(self, *args, **kw):
            raise FastllmError(-2, "lost")

    cache = _Broken(2)
    with pytest.raises(FastllmError, match="lost"):
        models.score(_Model(), [[3, 4, 5], [6, 7, 8]], cache=cache)
    assert not any(cache.hist)


def test_head_bits_of_other_models_are_refused(tmp_path):
    (tmp_path / "config.json").write_text('{"architectures": ["LlamaForCausalLM"], "hidden_size": 64, "intermediate_size": 64, "vocab_size": 64, "num_hidden_layers": 1, '
                                          '"num_attention_heads": 4}')
    with pytest.raises(FastllmError, match="layered models only"):
        models.load_model(str(tmp_path), head_bits=8)
