"""Operators on device memory: torch tensors in, torch tensors out, on the current stream of their device.

    quantize_rows(x)                          rows as 8-bit whole numbers with a scale each
    linear8(x, weight, weight_scale, bias)    matrix product in 8-bit integers with a scale per token and per channel
    logprobs(logits, tokens, top=K)           log probabilities of given tokens, log-sum-exp, entropy, the K most likely alternatives

Thin over the C ABI (include/fastllm_b200.h, "operators on device memory", which states the formulas and what NaN, infinities, padding and
rows without probabilities give).  Calls are asynchronous, allocate their results (and linear8 its workspace) with torch, and can be captured into a CUDA graph.
No autograd: results do not require gradients.
"""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from . import _lib
from ._lib import FastllmError

_FLOATS = {torch.float32: _lib.FL_DTYPE_F32, torch.bfloat16: _lib.FL_DTYPE_BF16, torch.float16: _lib.FL_DTYPE_F16}
MAX_TOP = 32


def _refuse(msg: str):
    raise FastllmError(-1, msg)


def _device(t: torch.Tensor, what: str) -> int:
    """the tensor's device, which is (or becomes) the one this process is bound to"""
    if t.device.type != "cuda":
        _refuse(f"{what}: tensors live on the GPU (there is no CPU fallback), got one on {t.device}")
    _lib.init(t.device.index)
    return t.device.index


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


def _same(device: torch.device, what: str, **tensors):
    for name, t in tensors.items():
        if t is not None and t.device != device:
            _refuse(f"{what}: {name} lives on {t.device}, the first tensor on {device}")


def _vector(t: Optional[torch.Tensor], n: int, what: str, name: str):
    if t is None:
        return None
    if t.dtype != torch.float32 or t.numel() != n or not t.is_contiguous():
        _refuse(f"{what}: {name} is a dense f32 tensor of {n} entries, got {t.dtype} {tuple(t.shape)}")
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
                                            torch.cuda.current_stream(dev).cuda_stream))
    q = q[:, :cols]
    return (q if x.ndim == 2 else q.unflatten(0, x.shape[:-1]) if x.ndim > 2 else q[0]), scale


def linear8(x: torch.Tensor, weight: torch.Tensor, weight_scale: torch.Tensor, bias: Optional[torch.Tensor] = None, *,
            x_scale: Optional[torch.Tensor] = None, out_dtype: Optional[torch.dtype] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """y[..., i] = (sum_j q[..., j] weight[i, j]) scale[...] weight_scale[i] (+ bias[i]), the sum exact in 32-bit integers.

    x [..., k]: f32 / bf16 / f16, rounded per row as quantize_rows does; or int8 with x_scale [...] (rows on 16-byte borders).
    weight int8 [n, k] with rows on 16-byte borders, weight_scale f32 [n], bias f32 [n] or None.  out_dtype: f32 / bf16 / f16 (default: x's
    type, f32 for int8 rows); out: where the result goes, [..., n] with a dense last dimension, not overlapping an input."""
    what = "linear8"
    x_type = _lib.FL_DTYPE_I8 if x.dtype == torch.int8 else _FLOATS.get(x.dtype)
    if x_type is None:
        _refuse(f"{what}: activations are f32, bf16, f16 or int8, got {x.dtype}")
    if weight.dtype != torch.int8 or weight.ndim != 2:
        _refuse(f"{what}: the weight is an int8 matrix [n, k], got {weight.dtype} {tuple(weight.shape)}")
    dev = _device(x, what)
    x2 = x if x.ndim == 2 and x.stride(1) == 1 else _rows(x, what)
    rows, k = x2.shape
    n = weight.shape[0]
    if weight.shape[1] != k or (k > 1 and weight.stride(1) != 1):
        _refuse(f"{what}: the weight is [n, {k}] with a dense last dimension, got {tuple(weight.shape)}")
    _same(x.device, what, weight=weight, weight_scale=weight_scale, bias=bias, x_scale=x_scale, out=out)
    if out is not None:
        if out.shape != x.shape[:-1] + (n,) or (out_dtype is not None and out.dtype != out_dtype):
            _refuse(f"{what}: out is {tuple(x.shape[:-1] + (n,))}, got {tuple(out.shape)} {out.dtype}")
        y2 = _rows(out, what)
    else:
        out = torch.empty(x.shape[:-1] + (n,), dtype=out_dtype or (torch.float32 if x_type == _lib.FL_DTYPE_I8 else x.dtype), device=x.device)
        y2 = out if out.ndim == 2 else out.view(rows, n)
    if out.dtype not in _FLOATS:
        _refuse(f"{what}: results are f32, bf16 or f16, got {out.dtype}")
    step = (k + 15) // 16 * 16
    room = 0 if x_type == _lib.FL_DTYPE_I8 else (rows * step + 255) // 256 * 256 + 4 * rows       # (fl_linear8_workspace's rule)
    ws = torch.empty(room, dtype=torch.uint8, device=x.device) if room else None
    _lib.check(_lib.load().fl_linear8(x2.data_ptr(), x_type, x2.stride(0), _vector(x_scale, rows, what, "x_scale"), weight.data_ptr(), weight.stride(0),
                                      _vector(weight_scale, n, what, "weight_scale"), _vector(bias, n, what, "bias"), rows, n, k, y2.data_ptr(), _FLOATS[out.dtype],
                                      y2.stride(0), ws.data_ptr() if room else None, room, torch.cuda.current_stream(dev).cuda_stream))
    return out


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
    dev = _device(logits, what)
    x = logits if logits.ndim == 2 and logits.stride(1) == 1 else _rows(logits, what)
    rows, vocab = x.shape
    lead = logits.shape[:-1]
    given, lp, tok, width = 0, None, None, 4
    if tokens is not None:
        _same(logits.device, what, tokens=tokens)
        if tokens.dtype not in (torch.int32, torch.int64):
            _refuse(f"{what}: tokens are int32 or int64, got {tokens.dtype}")
        if tokens.shape == lead:
            given = 1
        elif tokens.ndim == len(lead) + 1 and tokens.shape[:-1] == lead:
            given = tokens.shape[-1]
        else:
            _refuse(f"{what}: tokens are {tuple(lead)} or {tuple(lead)} + (m,), got {tuple(tokens.shape)}")
        tok = tokens.contiguous()
        width = 4 if tok.dtype == torch.int32 else 8
        lp = torch.empty(tokens.shape, dtype=torch.float32, device=logits.device)
    lse = torch.empty(lead, dtype=torch.float32, device=logits.device)
    ent = torch.empty(lead, dtype=torch.float32, device=logits.device)
    ids = tlp = None
    if top > 0:
        ids = torch.empty(lead + (top,), dtype=torch.int32, device=logits.device)
        tlp = torch.empty(lead + (top,), dtype=torch.float32, device=logits.device)
    _lib.check(_lib.load().fl_logprobs(x.data_ptr(), _FLOATS[logits.dtype], rows, vocab, x.stride(0), tok.data_ptr() if given else None, width, given, temperature, top,
                                       lp.data_ptr() if given else None, lse.data_ptr(), ent.data_ptr(), ids.data_ptr() if top > 0 else None,
                                       tlp.data_ptr() if top > 0 else None, torch.cuda.current_stream(dev).cuda_stream))
    return LogProbs(lp, lse, ent, ids, tlp)
