"""CPU tests of what a generation or a scoring that was refused, or failed on its way, leaves behind (stand-in caches of test_score_cpu.py)."""
import pytest

from fastllm_b200 import models
from fastllm_b200._lib import FastllmError
from test_score_cpu import VOCAB, _Cache, _Model, _prompts


class _Failing(_Cache):
    """the call of `what` that comes after `good` of them fails, before or behind its work; slots that hold nothing can be given back"""

    def __init__(self, slots, what, good, behind, error):
        super().__init__(slots)
        self.what, self.good, self.behind, self.error = what, good, behind, error

    def _count(self, name, call):
        if name == self.what:
            self.good -= 1
            if self.good == -1 and not self.behind:
                raise self.error
        out = call()
        if name == self.what and self.good == -1:
            raise self.error
        return out

    def forward_slots(self, *a, **k):
        return self._count("forward", lambda: _Cache.forward_slots(self, *a, **k))

    def forward_ragged(self, *a, **k):
        return self._count("forward", lambda: _Cache.forward_ragged(self, *a, **k))

    def logprobs(self, *a, **k):
        return self._count("logprobs", lambda: _Cache.logprobs(self, *a, **k))

    def slot_reset(self, slot):
        self.hist[slot] = []


def _batcher(cache, chunk):
    return models.ContinuousBatcher(_Model(), max_batch=3, eos_token_id=2, cache=cache, prefill_chunk=chunk)


@pytest.mark.parametrize("chunk", [None, 4])
@pytest.mark.parametrize("top", [-1, 24, 33, 1 << 20])
def test_a_number_of_alternatives_is_refused_before_any_step(chunk, top):
    """24 are more than the vocabulary has"""
    cache = _Cache(3)
    with pytest.raises(FastllmError, match="alternatives"):
        _batcher(cache, chunk).generate(_prompts([5, 9, 1, 7, 3]), 6, logprobs=top)
    assert cache.last is None and not any(cache.hist)


@pytest.mark.parametrize("chunk", [None, 4])
@pytest.mark.parametrize("what", ["forward", "logprobs"])
@pytest.mark.parametrize("good", [0, 1, 2, 5])
@pytest.mark.parametrize("behind", [False, True])
@pytest.mark.parametrize("error", [FastllmError(-2, "lost"), KeyboardInterrupt()])
def test_a_generation_after_one_that_failed(chunk, what, good, behind, error):
    prompts = _prompts([5, 9, 1, 7, 3])
    want = _batcher(_Cache(3), chunk).generate(prompts, 6, logprobs=VOCAB)
    cache = _Failing(3, what, good, behind, error)
    cb = _batcher(cache, chunk)
    with pytest.raises(type(error)):
        cb.generate(prompts, 6, logprobs=3)
    assert not any(cache.hist)
    assert cb.generate(prompts, 6, logprobs=VOCAB) == want


def test_a_cache_that_gives_nothing_back_shows_its_first_error():
    class _Lost(_Failing):
        def slot_reset(self, slot):
            raise FastllmError(-2, "poisoned")

    with pytest.raises(FastllmError, match="lost"):
        _batcher(_Lost(3, "forward", 2, True, FastllmError(-2, "lost")), 4).generate(_prompts([5, 9]), 6)


@pytest.mark.parametrize("top", [-1, 24, 33])
def test_scoring_refuses_a_number_of_alternatives_before_any_step(top):
    cache = _Cache(2)
    with pytest.raises(FastllmError, match="alternatives"):
        models.score(_Model(), [[3, 4]], top=top, cache=cache)
    assert cache.last is None


@pytest.mark.parametrize("what", ["forward", "logprobs"])
@pytest.mark.parametrize("good", [0, 2])
@pytest.mark.parametrize("error", [FastllmError(-2, "lost"), MemoryError(), KeyboardInterrupt()])
def test_a_scoring_after_one_that_failed(what, good, error):
    texts = _prompts([5, 9, 1, 7, 3])
    want = [s.total for s in models.score(_Model(), texts, cache=_Cache(2), portion=4)]
    cache = _Failing(2, what, good, True, error)
    with pytest.raises(type(error)):
        models.score(_Model(), texts, cache=cache, portion=4)
    assert not any(cache.hist)
    assert [s.total for s in models.score(_Model(), texts, cache=cache, portion=4)] == want
