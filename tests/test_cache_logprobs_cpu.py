"""CPU tests of what DeviceCache.logprobs hands to the library (a stand-in for it)."""
import ctypes as C

import numpy as np
import pytest

from fastllm_b200 import models
from fastllm_b200._lib import FastllmError


class _Lib:
    def fl_cache_logprobs(self, cache, rows, tokens, given, temperature, top, *out):
        n = rows * given
        self.rows, self.given = rows, given
        self.tokens = None if tokens is None else np.array((C.c_int32 * n).from_address(tokens.value))
        return 0


def _cache():
    cache = models.DeviceCache.__new__(models.DeviceCache)
    cache.lib, cache.h = _Lib(), None
    return cache


@pytest.mark.parametrize("kind", [np.int8, np.int16, np.int32, np.int64, np.uint8, np.uint32, np.uint64])
def test_tokens_of_any_whole_type(kind):
    """those that 32 bits do not hold are none of the vocabulary's: neither wrapped round into it nor, from above, into padding"""
    info = np.iinfo(kind)
    values = [v for v in (0, 5, 127, 30000, 2 ** 31 - 1, 2 ** 31, 2 ** 32 - 1, 2 ** 32 + 5, 2 ** 40, 2 ** 63 - 1, -1, -100, -2 ** 31, -2 ** 31 - 7, -2 ** 32 + 5, -2 ** 40)
              if info.min <= v <= info.max]
    cache = _cache()
    r = cache.logprobs(np.array(values, dtype=kind))
    assert r.logprob.shape == (len(values),) and (cache.lib.rows, cache.lib.given) == (len(values), 1)
    for v, got in zip(values, cache.lib.tokens):
        assert got < 0 if v < 0 else got == min(v, 2 ** 31 - 1), (v, got)


def test_tokens_that_are_no_whole_numbers_are_refused():
    for bad in ([1.5, 2.0], np.zeros(2, np.float32), np.array([True, False]), np.array(["a"])):
        with pytest.raises(FastllmError, match="whole numbers"):
            _cache().logprobs(bad)


def test_shapes():
    cache = _cache()
    tokens = np.arange(12, dtype=np.int64).reshape(3, 4)[:, ::2]
    assert cache.logprobs(tokens).logprob.shape == (3, 2) and cache.lib.tokens.tolist() == [0, 2, 4, 6, 8, 10]
    assert cache.logprobs([]).logprob.shape == (0,) and cache.logprobs(rows=2).logprob is None
    with pytest.raises(FastllmError, match="shape"):
        cache.logprobs(np.zeros((1, 1, 1), np.int32))
