"""CPU tests of the operators' refusals: every argument check answers on the host, before any device is asked for."""
import ctypes as C

import pytest
import torch

from fastllm_b200 import _lib, ops
from fastllm_b200._lib import FastllmError

P = 1 << 20             # an address that no call below gets far enough to use


def _linear8(**change):
    a = dict(x=P, x_dtype=1, ldx=64, x_scale=None, w=P, ldw=64, w_scale=P, bias=None, rows=5, n=32, k=64, y=P, y_dtype=1, ldy=32, workspace=P, workspace_bytes=1 << 20)
    a.update(change)
    return _lib.load().fl_linear8(*a.values(), None)


def _logprobs(**change):
    a = dict(logits=P, dtype=0, rows=4, vocab=100, ld=100, tokens=P, token_bytes=8, given=1, temperature=1.0, top=5, logprob=P, logsumexp=P, entropy=P, top_ids=P,
             top_logprobs=P)
    a.update(change)
    return _lib.load().fl_logprobs(*a.values(), None)


def _quantize(**change):
    a = dict(x=P, dtype=1, rows=4, cols=64, ldx=64, q=P, ldq=64, scale=P)
    a.update(change)
    return _lib.load().fl_quantize_rows(*a.values(), None)


def _refused(rc, word):
    assert rc == -1, rc
    assert word in _lib.load().fl_last_error().decode(), _lib.load().fl_last_error()


@pytest.mark.parametrize("change, word", [
    (dict(x_dtype=7), "activations"), (dict(y_dtype=3), "results"), (dict(rows=-1), "rows"), (dict(rows=(1 << 30) + 1), "rows"), (dict(n=0), "n from"), (dict(k=0), "k from"),
    (dict(k=131072, ldx=131072, ldw=131072), "k from"), (dict(ldx=63), "row stride"), (dict(ldw=48), "row stride"), (dict(ldy=31), "row stride"),
    (dict(x=None), "NULL"), (dict(w=None), "NULL"), (dict(w_scale=None), "NULL"), (dict(y=None), "NULL"), (dict(x_scale=P), "x_scale"),
    (dict(x_dtype=3, ldx=64), "x_scale"), (dict(w=P + 8), "16-byte"), (dict(ldw=72), "16-byte"), (dict(x_dtype=3, x_scale=P, x=P + 4), "16-byte"),
    (dict(x_dtype=3, x_scale=P, ldx=72), "16-byte"), (dict(x=P + 1), "aligned"), (dict(y=P + 1), "aligned"), (dict(w_scale=P + 2), "aligned"), (dict(bias=P + 1), "aligned"),
    (dict(workspace=None), "workspace"), (dict(workspace=P + 16), "workspace"), (dict(workspace_bytes=5 * 64 + 192 + 19), "workspace")])
def test_linear8_refuses(change, word):
    _refused(_linear8(**change), word)


@pytest.mark.parametrize("change, word", [
    (dict(dtype=3), "logits"), (dict(rows=-1), "rows"), (dict(vocab=0), "vocabulary"), (dict(vocab=(1 << 20) + 1, ld=1 << 21), "vocabulary"), (dict(ld=99), "row stride"),
    (dict(given=-1), "given"), (dict(token_bytes=2), "given"), (dict(top=-1), "alternatives"), (dict(top=33), "alternatives"), (dict(vocab=4, top=5), "alternatives"),
    (dict(temperature=0.0), "temperature"), (dict(temperature=-1.0), "temperature"), (dict(temperature=float("nan")), "temperature"),
    (dict(temperature=float("inf")), "temperature"), (dict(temperature=1e-300), "temperature"), (dict(temperature=1e300), "temperature"), (dict(logits=None), "NULL"),
    (dict(tokens=None), "NULL"), (dict(logprob=None), "NULL"), (dict(top_ids=None), "NULL"), (dict(top_logprobs=None), "NULL"), (dict(logits=P + 2), "aligned"),
    (dict(tokens=P + 4), "aligned"), (dict(top_ids=P + 2), "aligned"), (dict(entropy=P + 1), "aligned")])
def test_logprobs_refuses(change, word):
    _refused(_logprobs(**change), word)


@pytest.mark.parametrize("change, word", [
    (dict(dtype=3), "f32, bf16 or f16"), (dict(rows=-1), "rows"), (dict(cols=0), "columns"), (dict(cols=131072, ldx=131072, ldq=131072), "columns"), (dict(ldx=63), "row stride"),
    (dict(ldq=63), "row stride"), (dict(x=None), "NULL"), (dict(q=None), "NULL"), (dict(scale=None), "NULL"), (dict(x=P + 1), "aligned"), (dict(scale=P + 2), "aligned")])
def test_quantize_rows_refuses(change, word):
    _refused(_quantize(**change), word)


def test_no_rows_is_no_work():
    assert _linear8(rows=0, x=None, y=None, workspace=None) == 0
    assert _logprobs(rows=0, logits=None) == 0
    assert _quantize(rows=0, x=None) == 0


def test_workspace_size():
    """the rule that ops.py keeps too"""
    n = C.c_size_t()
    lib = _lib.load()
    for rows in (0, 1, 2, 3, 4, 5, 9, 128, 300):
        for k in (1, 17, 100, 2048, 4096, 4097, 8192, 8193, 10922, 10923, 16384, 16385, 32768, 32769):
            want = 0 if rows <= 2 and rows * rows * k <= 16384 else (rows * ((k + 15) // 16 * 16) + 255) // 256 * 256 + 4 * rows
            assert lib.fl_linear8_workspace(rows, k, 1, C.byref(n)) == 0 and n.value == want, (rows, k)
            assert lib.fl_linear8_workspace(rows, k, 3, C.byref(n)) == 0 and n.value == 0
    _refused(lib.fl_linear8_workspace(1, 0, 1, C.byref(n)), "k from")
    _refused(lib.fl_linear8_workspace(1, 1, 9, C.byref(n)), "activations")
    _refused(lib.fl_linear8_workspace(1, 1, 1, None), "NULL")


def test_tensors_off_the_gpu_are_refused():
    x, w, s = torch.zeros(2, 16), torch.zeros(4, 16, dtype=torch.int8), torch.ones(4)
    for call in (lambda: ops.quantize_rows(x), lambda: ops.linear8(x, w, s), lambda: ops.logprobs(x)):
        with pytest.raises(FastllmError, match="no CPU fallback"):
            call()


def test_types_are_refused():
    x = torch.zeros(2, 16)
    with pytest.raises(FastllmError, match="activations"):
        ops.linear8(x.double(), x.to(torch.int8), x[0])
    with pytest.raises(FastllmError, match="int8 matrix"):
        ops.linear8(x, x, x[0])
    with pytest.raises(FastllmError, match="logits are"):
        ops.logprobs(x.double())
    with pytest.raises(FastllmError, match="rows are wanted"):
        ops.quantize_rows(x.long())
