"""Operators on device memory: torch tensors in, torch tensors out, on the current stream of their device.

    quantize_rows(x)                          rows as 8-bit whole numbers with a scale each
    linear8(x, weight, weight_scale, bias)    matrix product in 8-bit integers with a scale per token and per channel
    logprobs(logits, tokens, top=K)           log probabilities of given tokens, log-sum-exp, entropy, the K most likely alternatives
    check()                                   raises when a product that has run is not valid

Thin over the C ABI (include/fastllm_b200.h, "operators on device memory", which states the formulas and what NaN, infinities, padding and
rows without probabilities give).  Calls are asynchronous, allocate their results (and linear8 its workspace) with torch, and can be captured into a CUDA graph.
No autograd: results do not require gradients.
"""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from . import _lib
from ._lib import FastllmError

_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda dev: torch.cuda.current_stream(dev).cuda_stream)      # (without the Stream object around it)
_bound = [None]             # the device of the last call
_FLOATS = {torch.float32: _lib.FL_DTYPE_F32, torch.bfloat16: _lib.FL_DTYPE_BF16, torch.float16: _lib.FL_DTYPE_F16}
_TYPES = {**_FLOATS, torch.int8: _lib.FL_DTYPE_I8}
_TOKENS = {torch.int32: 4, torch.int64: 8}
MAX_TOP = 32


def _refuse(msg: str):
    raise FastllmError(-1, msg)


def _device(t: torch.Tensor, what: str) -> int:
    """the tensor's device, which is (or becomes) the one this process is bound to"""
    dev = t.get_device()
    if dev != _bound[0]:
        if dev < 0:
            _refuse(f"{what}: tensors live on the GPU (there is no CPU fallback), got one on {t.device}")
        _lib.init(dev)
        _bound[0] = dev
    return dev


def _rows(t: torch.Tensor, what: str) -> torch.Tensor:
    """[..., cols] as [rows, cols] without a copy"""
    if t.ndim == 0:
        _refuse(f"{what}: a tensor of at least one dimension is wanted")
    if t.shape[-1] > 1 and t.stride(-1) != 1:
        _refuse(f"{what}: the last dimension is not dense")
    if t.ndim == 2:
        return t
    if t.ndim == 1:
        return t[None]
    try:
        return t.view(-1, t.shape[-1])
    except RuntimeError:
        _refuse(f"{what}: the leading dimensions do not have one row stride")


def _same(dev: int, t: Optional[torch.Tensor], what: str, name: str):
    if t is not None and t.get_device() != dev:
        _refuse(f"{what}: {name} lives on {t.device}, the first tensor on cuda:{dev}")


def _vector(t: Optional[torch.Tensor], n: int, dev: int, what: str, name: str):
    if t is None:
        return None
    if t.dtype != torch.float32 or t.numel() != n or not t.is_contiguous():
        _refuse(f"{what}: {name} is a dense f32 tensor of {n} entries, got {t.dtype} {tuple(t.shape)}")
    if t.get_device() != dev:
        _same(dev, t, what, name)
    return t.data_ptr()


def quantize_rows(x: torch.Tensor):
    """[..., cols] f32 / bf16 / f16 -> (q int8 [..., cols], scale f32 [...]): q * scale is x to half a step of max|x| / 127.  q's rows
    start on 16-byte borders (its row stride is cols rounded up to 16), as linear8 wants a weight's or 8-bit activations' rows."""
    if x.dtype not in _FLOATS:
        _refuse(f"quantize_rows: f32, bf16 or f16 rows are wanted, got {x.dtype}")
    dev = _device(x, "quantize_rows")
    x2 = _rows(x, "quantize_rows")
    rows, cols = x2.shape
    step = (cols + 15) // 16 * 16
    q = torch.empty((rows, step), dtype=torch.int8, device=x.device)
    scale = torch.empty(x.shape[:-1], dtype=torch.float32, device=x.device)
    _lib.check(_lib.load().fl_quantize_rows(x2.data_ptr(), _FLOATS[x.dtype], rows, cols, x2.stride(0), q.data_ptr(), step, scale.data_ptr(),
                                            _stream(dev)))
    q = q[:, :cols]
    return (q if x.ndim == 2 else q.unflatten(0, x.shape[:-1]) if x.ndim > 2 else q[0]), scale


def linear8(x: torch.Tensor, weight: torch.Tensor, weight_scale: torch.Tensor, bias: Optional[torch.Tensor] = None, *,
            x_scale: Optional[torch.Tensor] = None, out_dtype: Optional[torch.dtype] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """y[..., i] = (sum_j q[..., j] weight[i, j]) scale[...] weight_scale[i] (+ bias[i]), the sum exact in 32-bit integers.

    x [..., k]: f32 / bf16 / f16, rounded per row as quantize_rows does; or int8 with x_scale [...] (rows on 16-byte borders).
    weight int8 [n, k] with rows on 16-byte borders, weight_scale f32 [n], bias f32 [n] or None.  out_dtype: f32 / bf16 / f16 (default: x's
    type, f32 for int8 rows); out: where the result goes, [..., n] with a dense last dimension, not overlapping an input."""
    what = "linear8"
    x_type = _TYPES.get(x.dtype)
    if x_type is None:
        _refuse(f"{what}: activations are f32, bf16, f16 or int8, got {x.dtype}")
    if weight.dtype != torch.int8 or weight.ndim != 2:
        _refuse(f"{what}: the weight is an int8 matrix [n, k], got {weight.dtype} {tuple(weight.shape)}")
    dev = x.get_device()
    if dev != _bound[0]:
        _device(x, what)
    x2 = x if x.ndim == 2 and x.stride(1) == 1 else _rows(x, what)
    rows, k = x2.shape
    n, wk = weight.shape
    ldw, w_step = weight.stride()
    if wk != k or (k > 1 and w_step != 1):
        _refuse(f"{what}: the weight is [n, {k}] with a dense last dimension, got {tuple(weight.shape)}")
    if weight.get_device() != dev:
        _same(dev, weight, what, "the weight")
    ws_ptr = _vector(weight_scale, n, dev, what, "weight_scale")
    xs_ptr = None if x_scale is None else _vector(x_scale, rows, dev, what, "x_scale")
    bias_ptr = None if bias is None else _vector(bias, n, dev, what, "bias")
    if out is not None:
        if out.shape != x.shape[:-1] + (n,) or (out_dtype is not None and out.dtype != out_dtype):
            _refuse(f"{what}: out is {tuple(x.shape[:-1] + (n,))}, got {tuple(out.shape)} {out.dtype}")
        _same(dev, out, what, "out")
        out_dtype = out.dtype
    elif out_dtype is None:
        out_dtype = torch.float32 if x_type == _lib.FL_DTYPE_I8 else x.dtype
    y_type = _FLOATS.get(out_dtype)
    if y_type is None:
        _refuse(f"{what}: results are f32, bf16 or f16, got {out_dtype}")
    if out is None:
        y2 = x.new_empty((rows, n), dtype=out_dtype)
        out, ldy = (y2 if x.ndim == 2 else y2.view(x.shape[:-1] + (n,))), n
    else:
        y2 = _rows(out, what)
        ldy = y2.stride(0)
    lib = _lib.load()
    # (fl_linear8_workspace's rule)
    room = 0 if x_type == _lib.FL_DTYPE_I8 or rows <= 2 and rows * rows * k <= 16384 else (rows * ((k + 15) // 16 * 16) + 255) // 256 * 256 + 4 * rows
    work = work_ptr = None
    if room:
        work = x.new_empty(room, dtype=torch.uint8)
        work_ptr = work.data_ptr()
    rc = lib.fl_linear8(x2.data_ptr(), x_type, x2.stride(0), xs_ptr, weight.data_ptr(), ldw, ws_ptr, bias_ptr, rows, n, k, y2.data_ptr(), y_type, ldy, work_ptr, room,
                        _stream(dev))
    if rc:
        _lib.check(rc)
    return out


def check():
    """Raises FastllmError when a product since the last check gave up on a wait inside its kernel, once (fl_operators_check; the next linear8 would raise it too).
    To be asked after a synchronize, or after the replay of a graph has been waited for."""
    _lib.check(_lib.load().fl_operators_check())


class LogProbs(NamedTuple):
    logprob: Optional[torch.Tensor]         # as tokens; None without tokens
    logsumexp: torch.Tensor                 # [...]
    entropy: torch.Tensor                   # [...]
    top_ids: Optional[torch.Tensor]         # int32 [..., top]; None with top = 0
    top_logprobs: Optional[torch.Tensor]    # [..., top]


def logprobs(logits: torch.Tensor, tokens: Optional[torch.Tensor] = None, top: int = 0, temperature: float = 1.0) -> LogProbs:
    """Log probabilities of softmax(logits / temperature) over the last dimension, without writing the distribution.

    logits [..., vocab] f32 / bf16 / f16; tokens [...] or [..., m] int32 / int64, negative ones are padding (0); top: 0 to 32 alternatives,
    the most likely first, the lowest index first among equals.  All results f32 (top_ids int32)."""
    what = "logprobs"
    if logits.dtype not in _FLOATS:
        _refuse(f"{what}: logits are f32, bf16 or f16, got {logits.dtype}")
    dev = logits.get_device()
    if dev != _bound[0]:
        _device(logits, what)
    x = logits if logits.ndim == 2 and logits.stride(1) == 1 else _rows(logits, what)
    rows, vocab = x.shape
    lead = logits.shape[:-1]
    given, tok, tok_ptr, width = 0, None, None, 4
    if tokens is not None:
        if tokens.get_device() != dev:
            _same(dev, tokens, what, "tokens")
        width = _TOKENS.get(tokens.dtype)
        if width is None:
            _refuse(f"{what}: tokens are int32 or int64, got {tokens.dtype}")
        if tokens.shape == lead:
            given = 1
        elif tokens.ndim == len(lead) + 1 and tokens.shape[:-1] == lead:
            given = tokens.shape[-1]
        else:
            _refuse(f"{what}: tokens are {tuple(lead)} or {tuple(lead)} + (m,), got {tuple(tokens.shape)}")
        tok = tokens if tokens.is_contiguous() else tokens.contiguous()
        tok_ptr = tok.data_ptr()
    if not 0 <= top <= MAX_TOP:
        _refuse(f"{what}: from 0 to {MAX_TOP} alternatives, got {top}")
    # all results in one piece of memory: an allocation each would take as long as the launch
    mem = x.new_empty(rows * (given + 2 + 2 * top), dtype=torch.float32)
    at, step = mem.data_ptr(), 4 * rows
    rc = _lib.load().fl_logprobs(x.data_ptr(), _FLOATS[logits.dtype], rows, vocab, x.stride(0), tok_ptr if given else None, width, given, temperature, top,
                                 at + 2 * step if given else None, at, at + step, at + (2 + given) * step if top else None, at + (2 + given + top) * step if top else None,
                                 _stream(dev))
    if rc:
        _lib.check(rc)

    if len(lead) == 1:
        lp = None if tok is None else mem.as_strided(tokens.shape, (1,) if tokens.ndim == 1 else (given, 1), 2 * rows)
        lse, ent, ids, tlp = mem.as_strided(lead, (1,), 0), mem.as_strided(lead, (1,), rows), None, None
        if top:
            ids = mem.view(torch.int32).as_strided((rows, top), (top, 1), (2 + given) * rows)
            tlp = mem.as_strided((rows, top), (top, 1), (2 + given + top) * rows)
        return LogProbs(lp, lse, ent, ids, tlp)
    lse, ent, lp, ids, tlp = mem.split_with_sizes([rows, rows, given * rows, top * rows, top * rows])
    return LogProbs(None if tok is None else lp.view(tokens.shape), lse.view(lead), ent.view(lead), ids.view(torch.int32).view(lead + (top,)) if top else None,
                    tlp.view(lead + (top,)) if top else None)
