"""GPU tests of the operators on device memory against their definitions in 64 bits.

Tolerances count roundings: u = 2^-24 is half a step of f32, half = finfo(type).eps / 2 that of the result's type."""
import math
import os
import subprocess
import sys

import pytest
import torch

from fastllm_b200 import ops
from fastllm_b200._lib import FastllmError

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
FLOATS = [torch.bfloat16, torch.float16, torch.float32]


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


# ---- rounding of rows ---------------------------------------------------------------------------------------------------------------
def _exact_rows(x):
    """127 x / max to the nearest whole number, halves to even: the sign of 254 x - (2 low + 1) max in 64 bits is exact (24 + 8 bits a side)"""
    x = x.double()
    most = x.abs().amax(-1, keepdim=True)
    safe = torch.where(most > 0, most, 1.0)
    low = torch.floor(127.0 * x / safe)
    over = 254.0 * x - (2.0 * low + 1.0) * safe
    q = torch.where(over > 0, low + 1, torch.where(over < 0, low, low + torch.remainder(low, 2.0)))
    return q, most[..., 0]


def _check_rows(x, q, scale):
    want, most = _exact_rows(x)
    assert torch.equal(q.double(), want)
    assert torch.equal(scale, (most / 127.0).float())


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("rows, cols", [(1, 1), (3, 2), (5, 15), (2, 16), (4, 17), (7, 255), (3, 256), (2, 1000), (2, 1999), (5, 4096), (3, 5001), (2, 14336), (1, 16384), (2, 20000), (1, 131071)])
def test_quantize_rows(dtype, rows, cols):
    x = (torch.randn(rows, cols, device="cuda", generator=_gen(cols)) * 3).to(dtype)
    q, scale = ops.quantize_rows(x)
    assert q.shape == x.shape and q.dtype == torch.int8 and scale.shape == (rows,) and q.stride(0) % 16 == 0
    _check_rows(x, q, scale)


@pytest.mark.parametrize("dtype", FLOATS)
def test_quantize_rows_at_the_borders(dtype):
    """every half between whole numbers and its neighbours on both sides; for f32 maxima whose quotients are no short fractions"""
    halves = (torch.arange(-127, 127, device="cuda") + 0.5).float()
    rows = []
    for most in (127.0, 254.0, 127.0 / 64, 1.0, 0.3, 100.0):
        r = (halves * (most / 127.0)).to(dtype)
        up, down = torch.nextafter(r, torch.full_like(r, math.inf)), torch.nextafter(r, torch.full_like(r, -math.inf))
        rows.append(torch.cat([r, up, down, torch.tensor([most], device="cuda").to(dtype)]).clamp(-most, most))
    x = torch.stack(rows)
    _check_rows(x, *ops.quantize_rows(x))


def test_quantize_rows_of_any_size():
    tiny = torch.finfo(torch.float32).smallest_normal
    base = torch.randn(9, 300, device="cuda", generator=_gen(1))
    base = base / base.abs().amax(-1, keepdim=True)
    x = base * torch.tensor([1e-44, 1e-41, tiny, 1e-37, 1e-30, 1e-20, 1e20, 1e38, 3.4e38], device="cuda")[:, None]
    q, scale = ops.quantize_rows(x)
    _check_rows(x, q, scale)
    h = torch.tensor([[2.0 ** -24, 2.0 ** -23, 0, -2.0 ** -24], [65504, -65504, 1, 0]], device="cuda").half()
    _check_rows(h, *ops.quantize_rows(h))


@pytest.mark.parametrize("dtype", FLOATS)
def test_quantize_rows_without_a_scale(dtype):
    x = torch.randn(5, 333, device="cuda", generator=_gen(2)).to(dtype)
    x[0] = 0
    x[1] = -0.0
    x[2, 100] = math.nan
    x[3, 332] = -math.inf
    q, scale = ops.quantize_rows(x)
    assert (q[:4] == 0).all() and (scale[:2] == 0).all() and scale[2:4].isnan().all()
    _check_rows(x[4:], q[4:], scale[4:])


def test_quantize_rows_strides_and_shapes():
    base = torch.randn(2, 6, 7, 100, device="cuda", generator=_gen(3)).bfloat16()
    x = base[:, :, 3, 1:98]                     # rows that start on odd elements, one row stride
    with pytest.raises(FastllmError, match="leading dimensions"):
        ops.quantize_rows(base[:, :4, 3, :])
    q, scale = ops.quantize_rows(x)
    assert q.shape == x.shape and scale.shape == x.shape[:-1]
    _check_rows(x, q, scale)
    q, scale = ops.quantize_rows(x[0, 0])
    assert q.shape == (97,) and scale.shape == ()
    with pytest.raises(FastllmError, match="not dense"):
        ops.quantize_rows(base[0, 0, :, ::2])
    q, scale = ops.quantize_rows(base[:, :0, 3, 1:98])
    assert q.shape == (2, 0, 97) and scale.shape == (2, 0)


# ---- the product --------------------------------------------------------------------------------------------------------------------
def _weight(n, k, seed):
    g = _gen(seed)
    w = torch.empty(n, (k + 15) // 16 * 16, dtype=torch.int8, device="cuda").random_(-128, 128, generator=g)      # (garbage behind the rows)
    return w[:, :k], (0.5 + torch.rand(n, device="cuda", generator=g)) * 0.01


def _check_product(y, q, xs, w, ws, bias):
    """sum exact (|sum| < 2^31); to f32, times xs, times ws: three roundings; the row's own scale one; plus bias one; to y's type one"""
    prod = (q.double() @ w.double().T) * xs.double()[:, None] * ws.double()
    want = prod if bias is None else prod + bias.double()
    half = torch.finfo(y.dtype).eps / 2
    least = torch.finfo(y.dtype).smallest_normal * torch.finfo(y.dtype).eps / 2          # half a step of the smallest numbers
    tol = 1.001 * (4 * U * prod.abs() + (U + half) * (want.abs() + 4 * U * prod.abs())) + least
    far = (y.double() - want).abs()
    assert y.shape == want.shape and bool((far <= tol).all()), float((far / tol).max())


SIZES = [(1, 1, 1), (1, 128, 128), (2, 5, 17), (3, 129, 15), (7, 64, 16), (8, 1000, 127), (9, 127, 129), (16, 256, 1000), (17, 130, 640), (31, 4096, 256), (33, 96, 2050),
         (64, 257, 513), (65, 5001, 96), (100, 640, 4096), (127, 384, 300), (128, 128, 1280), (129, 333, 128), (203, 1001, 1999), (255, 512, 160), (256, 256, 512),
         (257, 300, 400), (511, 2049, 144), (700, 200, 4097), (1025, 1030, 272), (1500, 777, 130), (2100, 2500, 64)]


@pytest.mark.parametrize("rows, n, k", SIZES)
@pytest.mark.parametrize("dtype", FLOATS)
def test_linear8(rows, n, k, dtype):
    x = (torch.randn(rows, k, device="cuda", generator=_gen(rows)) * 2).to(dtype)
    w, ws = _weight(n, k, n)
    bias = torch.randn(n, device="cuda", generator=_gen(k)) if (rows + n) % 2 else None
    y = ops.linear8(x, w, ws, bias)
    assert y.dtype == dtype
    q, most = _exact_rows(x)
    _check_product(y, q, most / 127.0, w, ws, bias)


@pytest.mark.parametrize("rows, n, k", [(1, 5000, 4096), (1, 9, 16384), (1, 20000, 100), (1, 1, 16385), (2, 100, 4096), (2, 4097, 2050), (2, 333, 4001), (2, 40, 4097), (4, 700, 8192),
                                        (4, 130, 8193), (4, 6000, 513), (5, 700, 2048)])
@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("shift", [0, 1])
def test_linear8_tokens(rows, n, k, dtype, shift):
    """a token or a few, on both sides of the line to products that round their rows beforehand; rows that start on odd elements"""
    store = (torch.randn(rows, k + 8, device="cuda", generator=_gen(rows + k)) * 2).to(dtype)
    x = store[:, shift:k + shift]
    w, ws = _weight(n, k, n)
    bias = torch.randn(n, device="cuda", generator=_gen(k)) if rows % 2 else None
    q, most = _exact_rows(x)
    for out in (dtype, torch.float32):
        _check_product(ops.linear8(x, w, ws, bias, out_dtype=out), q, most / 127.0, w, ws, bias)


@pytest.mark.parametrize("rows", [1, 40, 300, 1200])
@pytest.mark.parametrize("out_dtype", FLOATS)
def test_linear8_types_of_the_result(rows, out_dtype):
    x = torch.randn(rows, 272, device="cuda", generator=_gen(rows)).half()
    w, ws = _weight(390, 272, 5)
    y = ops.linear8(x, w, ws, out_dtype=out_dtype)
    assert y.dtype == out_dtype
    q, most = _exact_rows(x)
    _check_product(y, q, most / 127.0, w, ws, None)


@pytest.mark.parametrize("rows", [1, 5, 20, 140, 260, 1100])
def test_linear8_of_8_bit_rows(rows):
    """whole numbers given with their scales, garbage between the rows"""
    k, n = 333, 260
    store = torch.empty(rows, 400, dtype=torch.int8, device="cuda").random_(-128, 128, generator=_gen(rows))
    x, xs = store[:, :k], torch.rand(rows, device="cuda", generator=_gen(7)) + 0.1
    w, ws = _weight(n, k, 6)
    y = ops.linear8(x, w, ws, x_scale=xs)
    assert y.dtype == torch.float32
    _check_product(y, x, xs, w, ws, None)


@pytest.mark.parametrize("rows", [1, 70, 300, 1030])
def test_linear8_of_the_largest_sums(rows):
    """k = 131071 of -128 times -128 and 127: sums up to 2^31 - 16384, which 32-bit floats would not hold"""
    k = 131071
    store = torch.full((rows, k + 1), -128, dtype=torch.int8, device="cuda")
    w = torch.full((3, k + 1), -128, dtype=torch.int8, device="cuda")
    w[1] = 127
    w[2, ::2] = 127
    one = torch.ones(max(rows, 3), device="cuda")
    y = ops.linear8(store[:, :k], w[:, :k], one[:3], x_scale=one[:rows])
    sums = [16384 * k, -128 * 127 * k, 16384 * (k // 2) - 128 * 127 * (k // 2 + 1)]
    assert torch.equal(y, torch.tensor(sums, device="cuda").float().expand(rows, 3))


@pytest.mark.parametrize("rows", [3, 100, 300, 1111])
def test_linear8_rows_without_a_scale(rows):
    x = torch.randn(rows, 200, device="cuda", generator=_gen(9)).bfloat16()
    x[0] = 0
    x[1, 7] = math.nan
    x[2, 199] = math.inf
    w, ws = _weight(150, 200, 10)
    bias = torch.randn(150, device="cuda", generator=_gen(11))
    y = ops.linear8(x, w, ws, bias, out_dtype=torch.float32)
    assert torch.equal(y[0], bias) and y[1:3].isnan().all()
    if rows > 3:
        q, most = _exact_rows(x[3:])
        _check_product(y[3:], q, most / 127.0, w, ws, bias)


@pytest.mark.parametrize("rows", [1, 6, 90, 200, 280, 1040])
def test_linear8_writes_its_rows_and_nothing_else(rows):
    """strided input and result: rows behind the last one and columns behind the row stay as they were"""
    k, n = 160, 190
    x = torch.randn(rows + 2, 3, k + 5, device="cuda", generator=_gen(12)).bfloat16()[:, 1, 3:k + 3]
    w, ws = _weight(n, k, 13)
    store = torch.full((rows + 2, n + 9), 7.0, device="cuda", dtype=torch.bfloat16)
    out = ops.linear8(x[:rows], w, ws, out=store[:rows, 1:n + 1])
    assert out.data_ptr() == store[:, 1:].data_ptr()
    q, most = _exact_rows(x[:rows])
    _check_product(out, q, most / 127.0, w, ws, None)
    assert (store[rows:] == 7).all() and (store[:, 0] == 7).all() and (store[:, n + 1:] == 7).all()


def test_linear8_shapes_and_refusals():
    w, ws = _weight(40, 32, 14)
    x = torch.randn(2, 3, 32, device="cuda", generator=_gen(15)).bfloat16()
    assert torch.equal(ops.linear8(x, w, ws).view(6, 40), ops.linear8(x.view(6, 32), w, ws))
    assert torch.equal(ops.linear8(x[0, 0], w, ws), ops.linear8(x[0], w, ws)[0])
    assert ops.linear8(x[:, :0], w, ws).shape == (2, 0, 40)
    for bad in (lambda: ops.linear8(x, w[:, 1:], ws), lambda: ops.linear8(x, w, ws[:39]), lambda: ops.linear8(x, w, ws.half()), lambda: ops.linear8(x, w, ws, ws[::2]),
                lambda: ops.linear8(x, w.t(), ws), lambda: ops.linear8(x, w, ws.cpu()), lambda: ops.linear8(x, w, ws, x_scale=ws), lambda: ops.linear8(x.char(), w, ws),
                lambda: ops.linear8(x[..., ::2], w, ws), lambda: ops.linear8(x, w, ws, out=torch.empty(2, 3, 41, device="cuda")),
                lambda: ops.linear8(x, w, ws, out_dtype=torch.float64), lambda: ops.linear8(x, w, ws, out_dtype=torch.int8)):
        with pytest.raises(FastllmError):
            bad()
    odd = torch.zeros(40, 33, dtype=torch.int8, device="cuda")
    with pytest.raises(FastllmError, match="16-byte"):
        ops.linear8(x, odd[:, :32], ws)


def test_linear8_far_offsets():
    """weights and results whose offsets pass 2^31 bytes"""
    n, k = 9, 64
    stride = (1 << 31) // 8 + 16
    store = torch.zeros(8 * stride + k, dtype=torch.int8, device="cuda")
    w = store.as_strided((n, k), (stride, 1))
    w.random_(-128, 128, generator=_gen(16))
    ws = torch.rand(n, device="cuda", generator=_gen(17))
    x = torch.randn(20, k, device="cuda", generator=_gen(18)).bfloat16()
    q, most = _exact_rows(x)
    _check_product(ops.linear8(x, w, ws), q, most / 127.0, w, ws, None)
    far = store.view(torch.bfloat16)[: 8 * (stride // 2) + n].as_strided((9, n), (stride // 2, 1))
    del store
    dense = w.clone().contiguous()
    y = ops.linear8(x[:9], dense, ws, out=far)
    _check_product(y, q[:9], most[:9] / 127.0, dense, ws, None)


# ---- log probabilities --------------------------------------------------------------------------------------------------------------
def _check_logprobs(r, x, tokens, top, temperature):
    """z = x / T: two roundings (none for T = 1), d = z - max: one; sums of at most vocab / 256 + 64 terms in a row per thread and a tree behind;
    exp and log 2 steps each.  Relative error of the sum: (chain + 8) u, and what the rounded exponents bring, 2 u |z| + u |d| at most.  The
    entropy's second sum weighs that with 1 + E|d|."""
    v, zr = x.shape[-1], 0.0 if temperature == 1.0 else 2 * U
    z = x.double() / temperature
    good = ~(z.isnan().any(-1) | (z == math.inf).any(-1))
    none = (z == -math.inf).all(-1)
    m = torch.where(none | ~good, 0.0, z.amax(-1))
    e = torch.exp(z - m[:, None])
    log_s = torch.where(none, 0.0, e.sum(-1).log())
    lp = torch.where(none[:, None], -math.inf, z - m[:, None] - log_s[:, None])
    d = torch.where(e > 0, z - m[:, None], 0.0)
    far = (e * d.abs()).sum(-1) / e.sum(-1).clamp(min=1e-300)
    lse, ent = torch.where(none, -math.inf, m + log_s), log_s + far
    zmax = torch.where(e > 0, z.abs(), 0.0).amax(-1)
    rel = (v / 256 + 64 + 8) * U + zr * zmax + U * d.abs().amax(-1)
    rel = rel + 4 * U * (log_s.abs() + 1)

    def near(got, want, tol, rows):
        got, want, tol = got[rows].double(), want[rows], tol.expand_as(want)[rows]
        fine = want.isfinite()
        assert torch.equal(got[~fine], want[~fine]), (got[~fine], want[~fine])
        bad = (got[fine] - want[fine]).abs() > tol[fine]
        assert not bad.any(), (got[fine][bad][:5], want[fine][bad][:5], tol[fine][bad][:5])

    def lp_tol(want, zs):
        size = torch.where(zs.isfinite(), zs.abs(), 0.0)
        return rel[:, None] + 4 * U * torch.where(want.isfinite(), want.abs(), 0.0) + zr * (size + zmax[:, None])

    near(r.logsumexp, lse, rel + torch.where(none, 0.0, (4 * U + zr) * lse.abs()), good)
    near(r.entropy, ent, (1 + far) * rel + 8 * U * (far + log_s.abs() + 1), good)
    assert r.logsumexp[~good].isnan().all() and r.entropy[~good].isnan().all()
    if tokens is not None:
        t2 = tokens.reshape(len(x), -1)
        got = r.logprob.reshape(len(x), -1)
        inside = (t2 >= 0) & (t2 < v)
        at = t2.clamp(0, v - 1).long()
        want = lp.gather(1, at)
        near(torch.where(inside, got, 0.0), torch.where(inside, want, 0.0), lp_tol(want, z.gather(1, at)), good)
        assert (got[t2 < 0] == 0).all() and got[t2 >= v].isnan().all() and got[~good][inside[~good]].isnan().all()
    if top:
        ids = torch.sort(x.float(), dim=-1, descending=True, stable=True).indices[:, :top]
        assert torch.equal(r.top_ids[good].long(), ids[good])
        want = lp.gather(1, ids)
        near(r.top_logprobs, want, lp_tol(want, z.gather(1, ids)), good)
        assert (r.top_ids[~good] == -1).all() and r.top_logprobs[~good].isnan().all()


@pytest.mark.parametrize("rows, vocab, top", [(1, 1, 1), (2, 1, 0), (3, 2, 2), (1, 31, 31), (5, 33, 32), (2, 255, 5), (3, 256, 20), (4, 257, 1), (1, 1000, 32), (9, 2049, 5), (1, 32000, 5),
                                              (2, 32003, 20), (7, 30522, 0), (40, 5001, 7), (200, 999, 3), (300, 4100, 32), (1000, 515, 5), (3, 152064, 20), (150, 152064, 8), (1, 1 << 20, 32)])
@pytest.mark.parametrize("dtype", FLOATS)
def test_logprobs(rows, vocab, top, dtype):
    g = _gen(vocab + rows)
    x = (torch.randn(rows, vocab, device="cuda", generator=g) * 3).to(dtype)
    tokens = torch.randint(0, vocab, (rows,), device="cuda", generator=g)
    _check_logprobs(ops.logprobs(x, tokens, top), x, tokens, top, 1.0)


@pytest.mark.parametrize("temperature", [0.05, 0.7, 1.0, 3.0, 1e4])
@pytest.mark.parametrize("dtype", FLOATS)
def test_logprobs_temperature(temperature, dtype):
    g = _gen(20)
    x = (torch.randn(6, 5000, device="cuda", generator=g) * 4).to(dtype)
    tokens = torch.randint(0, 5000, (6, 3), device="cuda", generator=g).int()
    r = ops.logprobs(x, tokens, 5, temperature)
    assert r.logprob.shape == (6, 3)
    _check_logprobs(r, x, tokens, 5, temperature)


@pytest.mark.parametrize("vocab", [40, 700, 32003, 152064])
@pytest.mark.parametrize("dtype", FLOATS)
def test_logprobs_masks(vocab, dtype):
    """rows with -infinity or the type's lowest value nearly everywhere, everywhere, in front, behind, alone at a place"""
    low = torch.finfo(dtype).min
    x = (torch.randn(12, vocab, device="cuda", generator=_gen(21)) * 3).to(dtype)
    x[0] = -math.inf
    x[1] = low
    x[2, 1:] = -math.inf
    x[3, :-1] = -math.inf
    x[4, : vocab // 2] = -math.inf
    x[5, vocab // 2:] = low
    x[6, torch.rand(vocab, device="cuda", generator=_gen(22)) < 0.99] = -math.inf
    x[7, vocab // 3] = math.nan
    x[8, vocab - 1] = math.inf
    x[9] = 0
    x[10] = math.nan
    x[11, :] = -math.inf
    x[11, vocab // 2] = low
    tokens = torch.randint(0, vocab, (12, 2), device="cuda", generator=_gen(23))
    tokens[2] = 0
    tokens[3] = vocab - 1
    for top in (0, 1, 20):
        _check_logprobs(ops.logprobs(x, tokens, top), x, tokens, top, 1.0)


def test_logprobs_tokens_outside():
    x = torch.randn(4, 100, device="cuda", generator=_gen(24))
    x[3] = math.nan
    for kind in (torch.int32, torch.int64):
        tokens = torch.tensor([[-1, 5], [100, -100], [99, 0], [-1, 3]], device="cuda", dtype=kind)
        _check_logprobs(ops.logprobs(x, tokens, 3), x, tokens, 3, 1.0)
    tokens = torch.tensor([1 << 40, -(1 << 40), 2, -1], device="cuda")
    _check_logprobs(ops.logprobs(x, tokens, 3), x, tokens, 3, 1.0)


@pytest.mark.parametrize("rows", [2, 9, 10, 60, 75, 89, 100, 120, 148, 149, 222, 223, 445, 592, 593])
@pytest.mark.parametrize("dtype", FLOATS)
def test_logprobs_row_counts(rows, dtype):
    """every number of blocks that a row is shared by, rows that start on no 16-byte border, a value alone behind the last chunk"""
    g = _gen(28)
    for vocab in (32001, 33025, 9000):
        x = (torch.randn(rows, vocab + 2, device="cuda", generator=g) * 3).to(dtype)[:, 1:vocab + 1]
        tokens = torch.randint(0, vocab, (rows, 2), device="cuda", generator=g)
        for top in (0, 7, 32):
            _check_logprobs(ops.logprobs(x, tokens, top), x, tokens, top, 1.0)


@pytest.mark.parametrize("rows, vocab", [(2, 40), (4, 1000), (4, 32003), (30, 32003), (4, 152064), (700, 5001)])
@pytest.mark.parametrize("dtype", FLOATS)
def test_logprobs_few_allowed(rows, vocab, dtype):
    """fewer logits above -infinity than alternatives are wanted, as many, and more than the tables hold: the lowest indices fill up"""
    g = _gen(27)
    values = (torch.randn(rows, vocab, device="cuda", generator=g) * 3).to(dtype)
    tokens = torch.randint(0, vocab, (rows,), device="cuda", generator=g)
    at = torch.rand(rows, vocab, device="cuda", generator=g).argsort(-1)
    for allowed in (0, 1, 3, 19, 20, 21, 33, 64, 250, 257, 300):
        x = torch.where(at < allowed, values, -math.inf)                 # anywhere
        x[1::4] = torch.where(torch.arange(vocab, device="cuda") < allowed, values[1::4], -math.inf)
        x[2::4] = torch.where(torch.arange(vocab, device="cuda") >= vocab - allowed, values[2::4], -math.inf)
        if rows > 3:
            x[3, vocab // 2] = math.nan
        for top in (1, 20, 32):
            _check_logprobs(ops.logprobs(x, tokens, top), x, tokens, top, 1.0)


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("vocab", [300, 5001, 152064])
def test_logprobs_many_equal(vocab, dtype):
    """few distinct values, rising and falling rows: the lowest index first, whatever the order they are met in"""
    g = _gen(25)
    x = torch.empty(7, vocab, device="cuda")
    x[0] = torch.randint(0, 3, (vocab,), device="cuda", generator=g).float()
    x[1] = torch.arange(vocab, device="cuda") / 1000.0
    x[2] = -torch.arange(vocab, device="cuda") / 1000.0
    x[3] = torch.where(torch.rand(vocab, device="cuda", generator=g) < 0.5, 0.0, -0.0)
    x[4] = -5.0
    x[4, vocab - 30:] = 4.0
    x[5] = 1.0
    x[5, :10] = 0.5
    x[6] = (torch.arange(vocab, device="cuda") % 97).float()
    x = x.to(dtype)
    for top in (1, 5, 32):
        _check_logprobs(ops.logprobs(x, None, top), x, None, top, 1.0)


def test_logprobs_strides_and_shapes():
    g = _gen(26)
    for dtype in FLOATS:
        store = (torch.randn(5, 3, 2030, device="cuda", generator=g) * 3).to(dtype)
        x = store[:, 1, 7:2010]
        tokens = torch.randint(0, x.shape[1], (2, 5), device="cuda", generator=g).t()       # (a view that is not dense)
        _check_logprobs(ops.logprobs(x, tokens, 6), x, tokens, 6, 1.0)
        r = ops.logprobs(store, top=4)
        assert r.logprob is None and r.logsumexp.shape == (5, 3) and r.top_ids.shape == (5, 3, 4)
        r = ops.logprobs(store[0, 0], tokens[0, 0])
        assert r.logprob.shape == () and r.top_ids is None
        assert ops.logprobs(store[:, :0], top=2).top_ids.shape == (5, 0, 2)
        assert ops.logprobs(x, tokens[:, :0]).logprob.shape == (5, 0)
    for bad in (lambda: ops.logprobs(x[:, ::2]), lambda: ops.logprobs(x, tokens[:4]), lambda: ops.logprobs(x, tokens.float()), lambda: ops.logprobs(x, tokens.cpu()),
                lambda: ops.logprobs(x, top=33), lambda: ops.logprobs(x, top=-1), lambda: ops.logprobs(x, temperature=0.0)):
        with pytest.raises(FastllmError):
            bad()


def test_logprobs_far_offsets():
    """rows whose offsets pass 2^31 elements"""
    vocab, stride = 1000, (1 << 31) // 4 + 1
    store = torch.zeros(4 * stride + vocab, dtype=torch.bfloat16, device="cuda")
    x = store.as_strided((5, vocab), (stride, 1))
    x.copy_(torch.randn(5, vocab, device="cuda", generator=_gen(27)) * 3)
    tokens = torch.arange(5, device="cuda") * 190
    _check_logprobs(ops.logprobs(x, tokens, 5), x, tokens, 5, 1.0)


# ---- together, on streams, in graphs ------------------------------------------------------------------------------------------------
def _score(x, w, ws, tokens, top=5):
    return ops.logprobs(ops.linear8(x, w, ws, out_dtype=torch.float32), tokens, top)


@pytest.mark.parametrize("rows", [1, 19, 150, 300, 1100])
def test_product_then_logprobs(rows):
    """an 8-bit output projection and the probabilities of its logits: the logits are off by at most 5 u of their size (see _check_product), which
    moves a log probability by as much as the largest logit's and its own error"""
    x = torch.randn(rows, 512, device="cuda", generator=_gen(28)).bfloat16()
    w, ws = _weight(3001, 512, 29)
    tokens = torch.randint(0, 3001, (rows,), device="cuda", generator=_gen(30))
    r = _score(x, w, ws, tokens)
    q, most = _exact_rows(x)
    z = (q @ w.double().T) * (most / 127.0)[:, None] * ws.double()
    want = torch.log_softmax(z, -1)
    tol = (3001 / 256 + 80) * U + 16 * U * z.abs().amax()
    assert float((r.logprob.double() - want.gather(1, tokens[:, None])[:, 0]).abs().max()) <= tol
    assert float((r.top_logprobs.double() - want.sort(-1, descending=True).values[:, :5]).abs().max()) <= tol


def test_same_bits_every_time():
    x = torch.randn(70, 1000, device="cuda", generator=_gen(31)).bfloat16()
    w, ws = _weight(5000, 1000, 32)
    first = ops.linear8(x, w, ws)
    lp = ops.logprobs(first, top=20)
    for _ in range(5):
        assert torch.equal(first, ops.linear8(x, w, ws))
        for a, b in zip(lp, ops.logprobs(first, top=20)):
            assert a is None and b is None or torch.equal(a, b)


def test_other_streams():
    """calls on several streams at once, each behind its own input"""
    w, ws = _weight(4000, 600, 33)
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    got = []
    for i in range(9):
        s = streams[i % 3]
        with torch.cuda.stream(s):
            x = torch.randn((1, 50, 400)[i % 3], 600, device="cuda", generator=_gen(34 + i)).bfloat16()
            tokens = torch.arange(len(x), device="cuda")
            got.append((x, tokens, _score(x, w, ws, tokens)))
    torch.cuda.synchronize()
    for x, tokens, r in got:
        for a, b in zip(r, _score(x, w, ws, tokens)):
            assert torch.equal(a, b)


@pytest.mark.parametrize("rows", [1, 60, 300])
def test_first_call_inside_a_capture(rows):
    """a process whose first calls are captured: set-up and loading do not break the capture"""
    code = """
import torch
from fastllm_b200 import ops
rows = %d
g = torch.Generator(device="cuda"); g.manual_seed(1)
x = torch.randn(rows, 200, device="cuda", generator=g).bfloat16()
w = torch.empty(900, 208, dtype=torch.int8, device="cuda").random_(-127, 128, generator=g)[:, :200]
s = torch.rand(900, device="cuda", generator=g)
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    y = ops.linear8(x, w, s, out_dtype=torch.float32)
    r = ops.logprobs(y, top=5)
graph.replay()
torch.cuda.synchronize()
y2 = ops.linear8(x, w, s, out_dtype=torch.float32)
r2 = ops.logprobs(y2, top=5)
assert torch.equal(y, y2) and torch.equal(r.logsumexp, r2.logsumexp) and torch.equal(r.top_ids, r2.top_ids)
print("same")
""" % rows
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300, cwd=root, env=dict(os.environ, PYTHONPATH=root))
    assert r.returncode == 0 and r.stdout.strip() == "same", r.stderr[-2000:]


@pytest.mark.parametrize("rows", [1, 60, 300, 1100])
def test_graphs(rows):
    """two captured graphs, replayed on new inputs and side by side"""
    w, ws = _weight(2000, 256, 50)
    graphs = []
    _score(torch.ones(rows, 256, device="cuda").bfloat16(), w, ws, torch.zeros(rows, dtype=torch.int64, device="cuda"))
    for i in range(2):
        x = torch.zeros(rows, 256, device="cuda", dtype=torch.bfloat16)
        tokens = torch.zeros(rows, dtype=torch.int64, device="cuda")
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            r = _score(x, w, ws, tokens)
        graphs.append((g, x, tokens, r, torch.cuda.Stream()))
    for step in range(3):
        for i, (g, x, tokens, r, s) in enumerate(graphs):
            x.copy_(torch.randn(rows, 256, device="cuda", generator=_gen(60 + 2 * step + i)))
            tokens.random_(0, 2000, generator=_gen(70 + 2 * step + i))
        torch.cuda.synchronize()
        for g, x, tokens, r, s in graphs:
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for g, x, tokens, r, s in graphs:
            for a, b in zip(r, _score(x, w, ws, tokens)):
                assert torch.equal(a, b)
