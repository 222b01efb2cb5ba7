"""GPU tests of the operators on 4-bit rows against their definitions in 64 bits.

Roundings to 4 bits are compared bit for bit; other tolerances count roundings: half = finfo(type).eps / 2 is half a step of the result's type."""
import math
import os
import subprocess
import sys

import pytest
import torch

from fastllm_b200 import _lib, ops
from fastllm_b200._lib import FastllmError

pytestmark = pytest.mark.gpu
FLOATS = [torch.bfloat16, torch.float16, torch.float32]
E2M1 = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]
ACTS = ["silu", "gelu_tanh", "relu", "swish_clamp"]


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _codes4(h, bad):
    """numbers in 64 bits [rows, k] -> (codes [rows, 32 blocks], scales [rows, blocks]): the nearest e2m1 by the borders between neighbours, a border itself to
    the even mantissa.  bad: blocks [rows, blocks] without a scale"""
    rows, k = h.shape
    b = torch.nn.functional.pad(h, (0, -k % 32)).view(rows, -1, 32)
    a = b.abs().amax(-1)
    e = torch.where(a > 0, torch.frexp(a).exponent - 3, -127).clamp(min=-127)
    t = torch.ldexp(b.abs(), -e[..., None])
    code = torch.zeros_like(t)
    for border, above in ((0.25, False), (0.75, True), (1.25, False), (1.75, True), (2.5, False), (3.5, True), (5.0, False)):
        code += (t >= border) if above else (t > border)
    code += 8 * (torch.signbit(b))
    scale = torch.where(bad, 255, e + 127)
    return torch.where(bad[..., None], 0, code).view(rows, -1).to(torch.uint8), scale.to(torch.uint8)


def _bad(x):
    rows, k = x.shape
    return ~torch.nn.functional.pad(x.float(), (0, -k % 32)).view(rows, -1, 32).isfinite().all(-1)


def _unpack(q):
    return torch.stack([q & 15, q >> 4], -1).flatten(-2)


def _same_codes(got, want):
    """equal but for the sign of a zero"""
    return torch.equal(torch.where(got == 8, 0, got), torch.where(want == 8, 0, want))


def _check_rows(x, q, scale):
    assert q.dtype == scale.dtype == torch.uint8 and q.shape[:-1] == scale.shape[:-1] == x.shape[:-1] and q.shape[-1] == 16 * scale.shape[-1] == 16 * ((x.shape[-1] + 31) // 32)
    x2, q2, s2 = x.reshape(-1, x.shape[-1]), q.reshape(-1, q.shape[-1]), scale.reshape(-1, scale.shape[-1])
    bad = _bad(x2)
    want, s = _codes4(torch.nan_to_num(x2.double(), 0.0, 0.0, 0.0), bad)
    assert torch.equal(s2, s)
    assert _same_codes(_unpack(q2), want)


def _values(q, scale):
    """in 64 bits"""
    table = torch.tensor(E2M1, device="cuda", dtype=torch.float64)
    v = torch.cat([table, -table])[_unpack(q).long()].unflatten(-1, (-1, 32))
    s = torch.where(scale == 255, math.nan, torch.ldexp(torch.ones_like(scale, dtype=torch.float64), scale.int() - 127))
    return (v * s[..., None]).flatten(-2)


# ---- rounding and back --------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("rows, cols", [(1, 1), (3, 2), (5, 31), (2, 32), (4, 33), (7, 255), (3, 256), (2, 257), (2, 1000), (2, 1999), (5, 4096), (3, 5001), (2, 14336), (1, 131073), (400, 96), (1, 1 << 20)])
def test_quantize4(dtype, rows, cols):
    x = (torch.randn(rows, cols, device="cuda", generator=_gen(cols)) * 3).to(dtype)
    _check_rows(x, *ops.quantize4(x))


@pytest.mark.parametrize("dtype", FLOATS)
def test_quantize4_at_the_borders(dtype):
    """every border between neighbours and the numbers next to it, at several scales; block maxima next to powers of two"""
    borders = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 7.0], device="cuda")
    rows = []
    for size in (1.0, 2.0 ** -9, 2.0 ** 7):
        r = (borders * size).to(dtype)
        up, down = torch.nextafter(r, torch.full_like(r, math.inf)), torch.nextafter(r, torch.full_like(r, -math.inf))
        for most in (4.0, 7.99):
            rows.append(torch.cat([r.clamp(max=most * size), up.clamp(max=most * size), down, -r[:4], torch.tensor([most * size], device="cuda").to(dtype)]))
        for top in (4.0, 8.0):
            t = torch.tensor([top * size], device="cuda").to(dtype)
            for m in (t, torch.nextafter(t, torch.zeros_like(t)), torch.nextafter(t, 2 * t)):
                rows.append(torch.cat([r / 4, -r / 2, m, torch.zeros(13, device="cuda", dtype=dtype)]).clamp(-m.item(), m.item())[:32])
    for r in rows:
        _check_rows(r[None], *ops.quantize4(r[None]))
        _check_rows(-r[None], *ops.quantize4(-r[None]))


def test_quantize4_of_any_size():
    tiny = torch.finfo(torch.float32).smallest_normal
    base = torch.randn(10, 300, device="cuda", generator=_gen(1))
    base = base / base.abs().amax(-1, keepdim=True)
    x = base * torch.tensor([1e-45, 1e-44, 1e-41, tiny, 4 * tiny, 1e-30, 1e-20, 1e20, 1e38, 3.4e38], device="cuda")[:, None]
    _check_rows(x, *ops.quantize4(x))
    h = torch.tensor([[2.0 ** -24, 2.0 ** -23, 0, -2.0 ** -24], [65504, -65504, 1, 0]], device="cuda").half()
    _check_rows(h, *ops.quantize4(h))


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("shift", [0, 1])
def test_quantize4_without_a_scale(dtype, shift):
    x = torch.randn(6, 340, device="cuda", generator=_gen(2)).to(dtype)[:, shift:333 + shift]
    x[0] = 0
    x[1] = -0.0
    x[2, 100] = math.nan
    x[3, 332] = -math.inf
    x[4, 64:96] = 0
    q, scale = ops.quantize4(x)
    _check_rows(x, q, scale)
    assert (scale[:2] == 0).all() and scale[2, 3] == 255 and scale[3, 10] == 255 and (scale == 255).sum() == 2 and scale[4, 2] == 0


def test_quantize4_strides_and_shapes():
    base = torch.randn(2, 6, 7, 100, device="cuda", generator=_gen(3)).bfloat16()
    x = base[:, :, 3, 1:98]                     # rows that start on odd elements, one row stride
    with pytest.raises(FastllmError, match="leading dimensions"):
        ops.quantize4(base[:, :4, 3, :])
    _check_rows(x, *ops.quantize4(x))
    q, scale = ops.quantize4(x[0, 0])
    assert q.shape == (64,) and scale.shape == (4,)
    _check_rows(x[0, 0], q, scale)
    with pytest.raises(FastllmError, match="not dense"):
        ops.quantize4(base[0, 0, :, ::2])
    q, scale = ops.quantize4(base[:, :0, 3, 1:98])
    assert q.shape == (2, 0, 64) and scale.shape == (2, 0, 4)
    assert ops.dequantize4(q, scale, 97).shape == (2, 0, 97)


@pytest.mark.parametrize("dtype", FLOATS)
def test_dequantize4_of_every_code(dtype):
    """16 numbers at 256 scales: rounded once"""
    scale = torch.arange(256, device="cuda").to(torch.uint8)[:, None]
    q = torch.arange(16, device="cuda").to(torch.uint8) * 17
    q = q.repeat(256, 1)
    y = ops.dequantize4(q, scale, dtype=dtype)
    want = _values(q, scale)
    f32 = want.float()                          # exact but for what passes its largest number
    assert ((f32.double() == want) | f32.isinf() | f32.isnan()).all()
    assert y.shape == (256, 32) and y[255].isnan().all() and torch.equal(y[:255], f32[:255].to(dtype))


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("rows, cols", [(1, 1), (3, 31), (2, 32), (5, 33), (7, 1999), (3, 4096), (300, 250)])
def test_dequantize4(dtype, rows, cols):
    blocks = (cols + 31) // 32
    store = torch.randint(0, 256, (rows, blocks * 16 + 32), device="cuda", generator=_gen(cols), dtype=torch.uint8)
    q, scale = store[:, 16:16 + blocks * 16], torch.randint(100, 130, (rows, blocks + 3), device="cuda", generator=_gen(rows), dtype=torch.uint8)[:, 1:blocks + 1]
    y = ops.dequantize4(q, scale, cols, dtype)
    assert torch.equal(y, _values(q, scale)[:, :cols].to(dtype))
    if cols % 32 == 0:
        assert torch.equal(ops.dequantize4(q, scale, dtype=dtype), y)
    for bad in (cols + 32, cols - 32, 0):
        if not 32 * blocks - 32 < bad <= 32 * blocks:
            with pytest.raises(FastllmError, match="columns"):
                ops.dequantize4(q, scale, bad)


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("cols, shift", [(96, 0), (70, 1), (33, 3), (1999, 2), (1, 5)])
def test_rows_with_room_between_them(dtype, cols, shift):
    """row strides on all sides, by the C ABI: what lies behind a row and behind the last row stays as it was"""
    rows, blocks, kind = 9, (cols + 31) // 32, {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}[dtype]
    lib, stream = _lib.load(), torch.cuda.current_stream().cuda_stream
    x = (torch.randn(rows, cols + 7, device="cuda", generator=_gen(cols)) * 3).to(dtype)[:, shift:cols + shift]
    q = torch.full((rows + 1, blocks * 16 + 48), 77, dtype=torch.uint8, device="cuda")
    scale = torch.full((rows + 1, blocks + 5), 77, dtype=torch.uint8, device="cuda")
    y = torch.full((rows + 1, cols + 9), 7.0, dtype=dtype, device="cuda")
    assert lib.fl_quantize4(x.data_ptr(), kind, rows, cols, x.stride(0), q[:, 16:].data_ptr(), q.stride(0), scale[:, shift:].data_ptr(), scale.stride(0), stream) == 0
    assert lib.fl_dequantize4(q[:, 16:].data_ptr(), q.stride(0), scale[:, shift:].data_ptr(), scale.stride(0), rows, cols, y[:, shift:].data_ptr(), kind, y.stride(0), stream) == 0
    inner, s = q[:rows, 16:16 + blocks * 16], scale[:rows, shift:shift + blocks]
    _check_rows(x, inner, s)
    assert torch.equal(y[:rows, shift:shift + cols], _values(inner, s)[:, :cols].to(dtype))
    inner.fill_(77), s.fill_(77), y[:rows, shift:shift + cols].fill_(7.0)
    assert (q == 77).all() and (scale == 77).all() and (y == 7).all()


# ---- the gated activation -----------------------------------------------------------------------------------------------------------
def _activation(x, act, limit):
    g, u = x.double().chunk(2, -1)
    if act == "silu":
        return g / (1.0 + torch.exp(-g)) * u
    if act == "gelu_tanh":
        return g / (1.0 + torch.exp(-2.0 * math.sqrt(2.0 / math.pi) * (g + 0.044715 * g ** 3))) * u
    if act == "relu":
        return g.clamp(min=0) * u
    g = g.clamp(max=limit)
    return g / (1.0 + torch.exp(-1.702 * g)) * (u.clamp(-limit, limit) + 1.0)


def _check_glu(x, act, q, scale, limit=7.0):
    f = x.shape[-1] // 2
    x2 = x.reshape(-1, 2 * f)
    h = _activation(x2, act, limit)
    bad = _bad(x2[:, :f]) | _bad(x2[:, f:]) | _bad(torch.where(h.abs() >= 2.0 ** 128, math.inf, 0.0))
    want, s = _codes4(torch.where(h.isfinite(), h, 0.0), bad)
    assert torch.equal(scale.reshape(s.shape), s)
    assert _same_codes(_unpack(q.reshape(len(s), -1)), want)


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("rows, f", [(1, 1), (2, 7), (3, 32), (5, 33), (2, 1000), (7, 2048), (37, 5001), (64, 4096), (2, 14336)])
def test_glu4(act, dtype, rows, f):
    x = (torch.randn(rows, 2 * f, device="cuda", generator=_gen(f)) * 3).to(dtype)
    _check_glu(x, act, *ops.glu4(x, act))


@pytest.mark.parametrize("act", ACTS)
def test_glu4_of_many(act):
    """so many numbers that some lie next to a border: 64 million, of which f32's exponential would put hundreds on the wrong side"""
    for seed in range(4):
        x = torch.randn(1024, 32768, device="cuda", generator=_gen(seed)) * 2
        _check_glu(x, act, *ops.glu4(x, act))


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("dtype", FLOATS)
def test_glu4_extremes(act, dtype):
    """gates from far below to far above, blocks whose results are all tiny, products that pass f32's range, numbers that are none"""
    big = min(torch.finfo(dtype).max, 1e30)
    x = torch.randn(16, 2 * 320, device="cuda", generator=_gen(4)).to(dtype)
    g, u = x[:, :320], x[:, 320:]
    g[0] = torch.linspace(-200, 200, 320, device="cuda").to(dtype)
    g[1] = torch.linspace(-120, -20, 320, device="cuda").to(dtype)
    g[2] = -30.0
    g[3] = 0.0
    g[4] = torch.linspace(0, 60, 320, device="cuda").to(dtype)
    u[4] = 1.25
    g[5] *= 1e-3
    u[5] *= 1e-3
    g[6], u[6] = big, big
    g[7, 5], u[7, 40] = math.nan, math.nan
    g[8, 5], u[8, 40], g[8, 100] = math.inf, -math.inf, -math.inf
    u[9] = -1.0
    u[10] = torch.linspace(-1.01, -0.99, 320, device="cuda").to(dtype)
    g[11] = -big
    u[12] = 0.0
    g[13] *= torch.finfo(dtype).smallest_normal
    g[14], u[14] = 40.0, 1.0
    g[15], u[15] = 1.0, 5.0 / torch.arange(1, 321, device="cuda").to(dtype)
    _check_glu(x, act, *ops.glu4(x, act))


def test_glu4_limits_strides_and_shapes():
    base = (torch.randn(2, 6, 7, 100, device="cuda", generator=_gen(5)) * 4).bfloat16()
    x = base[:, :, 3, 1:99]
    for limit in (0.5, 7.0, 100.0):
        _check_glu(x, "swish_clamp", *ops.glu4(x, "swish_clamp", limit=limit), limit)
    for act in ACTS:
        _check_glu(x, act, *ops.glu4(x, act))
    q, scale = ops.glu4(x[0, 0])
    assert q.shape == (32,) and scale.shape == (2,)
    assert ops.glu4(x[:, :0])[0].shape == (2, 0, 32)
    for bad in (lambda: ops.glu4(x[..., 1:]), lambda: ops.glu4(x, "gelu"), lambda: ops.glu4(x, "swish_clamp", limit=-1.0), lambda: ops.glu4(x[..., ::2])):
        with pytest.raises(FastllmError):
            bad()


# ---- the product --------------------------------------------------------------------------------------------------------------------
def _rows4(n, k, middle, seed):
    """4-bit rows with garbage behind their last column and between the rows"""
    g, blocks = _gen(seed), (k + 31) // 32
    q = torch.randint(0, 256, (n, blocks * 16 + 16), dtype=torch.uint8, device="cuda", generator=g)
    scale = torch.randint(middle - 3, middle + 4, (n, blocks + 1), dtype=torch.uint8, device="cuda", generator=g)
    return q[:, :blocks * 16], scale[:, 1:]


def _check_product(y, x, w, bias):
    """x, w in 64 bits.  Products of two e2m1 and two powers of two are exact.  A step of 64 products is summed with at most a step of f32 (2^-23) lost at each addition, and
    so is its sum's way into the accumulator, k / 64 times: (64 + k / 64) 2^-23 of the sum of magnitudes.  Then the bias (2^-24) and one rounding to y's type."""
    k = x.shape[1]
    want, size = x @ w.T, x.abs() @ w.abs().T
    tol = (64 + k / 64) * 2.0 ** -23 * size
    if bias is not None:
        want = want + bias.double()
    half = torch.finfo(y.dtype).eps / 2
    least = torch.finfo(y.dtype).smallest_normal * half
    tol = 1.001 * (tol + (half + (2.0 ** -24 if bias is not None else 0.0)) * (want.abs() + tol)) + least
    far = (y.double() - want).abs()
    assert y.shape == want.shape and bool((far <= tol).all()), float((far / tol).max())


SIZES = [(1, 1, 1), (1, 128, 128), (2, 5, 17), (3, 129, 15), (7, 64, 32), (8, 1000, 127), (9, 127, 129), (16, 256, 1000), (17, 130, 640), (31, 4096, 256), (33, 96, 2050),
         (64, 257, 513), (65, 5001, 96), (100, 640, 4096), (127, 384, 300), (128, 128, 1280), (129, 333, 128), (203, 1001, 1999), (255, 512, 160), (256, 256, 512),
         (257, 300, 400), (511, 2049, 144), (700, 200, 4097), (1025, 1030, 272), (1500, 777, 130), (2100, 2500, 64)]


def _exact_x(x):
    code, scale = _codes4(x.double(), _bad(x))
    q = code.view(len(x), -1, 2)
    return _values((q[..., 0] | q[..., 1] << 4), scale)


@pytest.mark.parametrize("rows, n, k", SIZES)
@pytest.mark.parametrize("dtype", FLOATS)
def test_linear4(rows, n, k, dtype):
    x = (torch.randn(rows, k, device="cuda", generator=_gen(rows)) * 2).to(dtype)
    q, scale = _rows4(n, k, 122, n)
    bias = torch.randn(n, device="cuda", generator=_gen(k)) if (rows + n) % 2 else None
    y = ops.linear4(x, ops.weight4(q, scale), bias)
    assert y.dtype == dtype
    _check_product(y, _exact_x(x), _values(q, scale), bias)


@pytest.mark.parametrize("rows", list(range(1, 20)) + [30, 63] + list(range(129, 260, 9)) + list(range(300, 1000, 67)))
def test_linear4_row_counts(rows):
    """every way to round the rows and to cut them into tiles, rows that start on odd elements, as many columns as no tile divides"""
    n, k = 300, 545
    x = (torch.randn(rows, k + 3, device="cuda", generator=_gen(rows)) * 2).to(FLOATS[rows % 3])[:, rows % 4:][:, :k]
    q, scale = _rows4(n, k, 122, n)
    xq, xs = ops.quantize4(x)
    y = ops.linear4(x, ops.weight4(q, scale), out_dtype=torch.float32)
    _check_product(y, _exact_x(x), _values(q, scale), None)
    if rows > 2:                                # (a token or two are summed in another order)
        assert torch.equal(y, ops.linear4(xq, ops.weight4(q, scale), x_scale=xs))


@pytest.mark.parametrize("rows, n", [(1, 40), (2, 300), (7, 140), (40, 130), (100, 129), (150, 520)])
def test_linear4_of_long_rows(rows, n):
    """long sums: many k blocks of a cluster's part, more groups than a word of their count holds"""
    k = 200003
    x = torch.randn(rows, k, device="cuda", generator=_gen(rows)).bfloat16()
    q, scale = _rows4(n, k, 118, n)
    _check_product(ops.linear4(x, ops.weight4(q, scale), out_dtype=torch.float32), _exact_x(x), _values(q, scale), None)


@pytest.mark.parametrize("rows, n", [(1, 70000), (3, 70000), (20, 40000), (300, 40000)])
def test_linear4_of_wide_matrices(rows, n):
    """more weight tiles than blocks that run at once"""
    k = 96
    x = torch.randn(rows, k, device="cuda", generator=_gen(rows)).half()
    q, scale = _rows4(n, k, 122, n)
    _check_product(ops.linear4(x, ops.weight4(q, scale)), _exact_x(x), _values(q, scale), None)


@pytest.mark.parametrize("rows, n, k", SIZES)
def test_linear4_of_4_bit_rows(rows, n, k):
    x, xs = _rows4(rows, k, 127, rows)
    q, scale = _rows4(n, k, 122, n)
    y = ops.linear4(x, ops.weight4(q, scale), x_scale=xs)
    assert y.dtype == torch.float32
    _check_product(y, _values(x, xs), _values(q, scale), None)


@pytest.mark.parametrize("rows", [1, 20, 100, 300, 1200])
@pytest.mark.parametrize("k", [64, 480, 4096])
def test_linear4_of_whole_numbers_is_exact(rows, k):
    """sums of quarters up to 36 k < 2^22: nothing is lost in 24 bits, in whatever order"""
    n = 300
    x = torch.randint(0, 256, (rows, k // 2), dtype=torch.uint8, device="cuda", generator=_gen(rows))
    q = torch.randint(0, 256, (n, k // 2), dtype=torch.uint8, device="cuda", generator=_gen(k))
    one = torch.full((max(rows, n), k // 32), 127, dtype=torch.uint8, device="cuda")
    y = ops.linear4(x, ops.weight4(q, one[:n]), x_scale=one[:rows])
    assert torch.equal(y.double(), _values(x, one[:rows]) @ _values(q, one[:n]).T)


@pytest.mark.parametrize("rows", [1, 9, 40, 70, 128, 200, 600])
def test_linear4_takes_every_block_at_its_scale(rows):
    """one column alone is not zero, and every block has a scale of its own: a scale read from the wrong place shows at once"""
    n, blocks = 140, 19
    k = 32 * blocks
    code = torch.randint(1, 8, (rows, blocks), device="cuda", generator=_gen(rows)).to(torch.uint8)
    xs = torch.randint(110, 140, (rows, blocks), device="cuda", generator=_gen(rows + 1)).to(torch.uint8)
    q = torch.randint(0, 256, (n, k // 2), dtype=torch.uint8, device="cuda", generator=_gen(rows + 2))
    scale = torch.randint(110, 140, (n, blocks), device="cuda", generator=_gen(rows + 3)).to(torch.uint8)
    w = ops.weight4(q, scale)
    wv = _values(q, scale)
    for b in range(blocks):
        x = torch.zeros(rows, k // 2, dtype=torch.uint8, device="cuda")
        x[:, 16 * b + 5] = code[:, b] << 4
        y = ops.linear4(x, w, x_scale=xs)
        assert torch.equal(y.double(), _values(x, xs) @ wv.T), b


@pytest.mark.parametrize("rows", [1, 40, 300, 1200])
@pytest.mark.parametrize("out_dtype", FLOATS)
def test_linear4_types_of_the_result(rows, out_dtype):
    x = torch.randn(rows, 272, device="cuda", generator=_gen(rows)).half()
    q, scale = _rows4(390, 272, 122, 5)
    y = ops.linear4(x, ops.weight4(q, scale), out_dtype=out_dtype)
    assert y.dtype == out_dtype
    _check_product(y, _exact_x(x), _values(q, scale), None)


@pytest.mark.parametrize("rows", [1, 2, 9, 40, 200, 500])
def test_linear4_of_far_scales(rows):
    """scales from the least to the largest: their product may be anything as long as the results are numbers of f32, and zeros stay zeros at any scale"""
    n, blocks = 130, 12
    g = _gen(rows)
    x = torch.randint(0, 256, (rows, 16 * blocks), dtype=torch.uint8, device="cuda", generator=g)
    q = torch.randint(0, 256, (n, 16 * blocks), dtype=torch.uint8, device="cuda", generator=g)
    xs = torch.tensor([0, 1, 40, 90, 127, 127, 180, 230, 253, 254, 120, 254], dtype=torch.uint8, device="cuda").repeat(rows, 1)
    ws = torch.tensor([240, 230, 200, 164, 127, 120, 70, 20, 1, 0, 254, 254], dtype=torch.uint8, device="cuda").repeat(n, 1)
    x[:, 16 * 10:16 * 11] = 0                   # zeros beside 2^120
    q[:, 16 * 11:] = 0                          # zeros whose scales' product is no number of f32
    y = ops.linear4(x, ops.weight4(q, ws), x_scale=xs)
    _check_product(y, _values(x, xs), _values(q, ws), None)
    v = _values(x, xs).float()                  # (the same numbers, rounded here; infinite ones would cost their rows)
    v = torch.where(v.isinf(), 1e38, v)
    w2, s2 = q.clone(), ws.clone()
    w2[:, 16 * 9:16 * 10] = 0
    s2[:, 9] = 254
    _check_product(ops.linear4(v, ops.weight4(w2, s2)), _exact_x(v), _values(w2, s2), None)


@pytest.mark.parametrize("rows", [1, 2, 3, 20, 200])
@pytest.mark.parametrize("low", [-147, -140, -130])
@pytest.mark.parametrize("of_x", [-127, -100, -60, -20])
def test_linear4_of_numbers_below_the_smallest_normal_one(rows, low, of_x):
    """scales whose product is below f32's range where the results are not: quarters of 2^low, up to 36 k of them, are all f32 numbers"""
    n, k = 150, 320
    of_w = low - of_x
    q = torch.randint(0, 256, (n, k // 2), dtype=torch.uint8, device="cuda", generator=_gen(rows))
    xq = torch.randint(0, 256, (rows, k // 2), dtype=torch.uint8, device="cuda", generator=_gen(rows + 1))
    xq[:, ::16] = 0xF7                          # (a block's largest number is 6, so that rounding finds its scale again)
    scale, xs = (torch.full((r, k // 32), 127 + e, dtype=torch.uint8, device="cuda") for r, e in ((n, of_w), (rows, of_x)))
    w, xv = ops.weight4(q, scale), _values(xq, xs)
    want = xv @ _values(q, scale).T
    assert want.abs().max() < 2.0 ** -110 and torch.equal(want.float().double(), want)
    assert torch.equal(ops.linear4(xv.float(), w).double(), want)
    assert torch.equal(ops.linear4(xq, w, x_scale=xs).double(), want)


@pytest.mark.parametrize("rows", [3, 100, 300, 1111])
def test_linear4_rows_without_a_scale(rows):
    """a row with a NaN or an infinity is NaN, a row of zeros the bias, the other rows are their own; likewise a weight row"""
    x = torch.randn(rows, 200, device="cuda", generator=_gen(9)).bfloat16()
    x[0] = 0
    x[1, 7] = math.nan
    x[2, 199] = math.inf
    q, scale = _rows4(150, 200, 122, 10)
    q, scale = q.clone(), scale.clone()
    bias = torch.randn(150, device="cuda", generator=_gen(11))
    y = ops.linear4(x, ops.weight4(q, scale), bias, out_dtype=torch.float32)
    assert torch.equal(y[0], bias) and y[1:3].isnan().all()
    if rows > 3:
        _check_product(y[3:], _exact_x(x[3:]), _values(q, scale), bias)
    scale[77, 4] = 255
    y2 = ops.linear4(x, ops.weight4(q, scale), bias, out_dtype=torch.float32)
    assert y2[:, 77].isnan().all()
    keep = torch.arange(150, device="cuda") != 77
    assert torch.equal(y2[3:, keep], y[3:, keep]) and torch.equal(y2[0, keep], y[0, keep])


@pytest.mark.parametrize("rows", [1, 2])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_linear4_of_a_token_without_a_scale(rows, bad):
    """as rows among more: NaN for a row with a NaN or an infinity and for a weight row without a scale, also where the other side's block holds zeros"""
    x = torch.randn(3, 200, device="cuda", generator=_gen(9)).bfloat16()
    x[:, 128:160] = 0
    x[rows - 1, 7] = bad
    q, scale = _rows4(150, 200, 122, 10)
    q, scale = q.clone(), scale.clone()
    q[5, :16] = 0
    scale[77, 4] = 255
    w = ops.weight4(q, scale)
    y, all_of_them = ops.linear4(x[:rows], w, out_dtype=torch.float32), ops.linear4(x, w, out_dtype=torch.float32)
    assert y[rows - 1].isnan().all() and all_of_them[rows - 1].isnan().all() and y[:, 77].isnan().all() and all_of_them[:, 77].isnan().all()
    keep = torch.arange(150, device="cuda") != 77
    if rows == 2:
        _check_product(y[:1, keep], _exact_x(x[:1]), _values(q, scale)[keep], None)


@pytest.mark.parametrize("rows", [1, 6, 90, 200, 280, 1040])
def test_linear4_writes_its_rows_and_nothing_else(rows):
    """strided input and result: rows behind the last one and columns behind the row stay as they were"""
    k, n = 160, 190
    x = torch.randn(rows + 2, 3, k + 5, device="cuda", generator=_gen(12)).bfloat16()[:, 1, 3:k + 3]
    q, scale = _rows4(n, k, 122, 13)
    store = torch.full((rows + 2, n + 9), 7.0, device="cuda", dtype=torch.bfloat16)
    out = ops.linear4(x[:rows], ops.weight4(q, scale), out=store[:rows, 1:n + 1])
    assert out.data_ptr() == store[:, 1:].data_ptr()
    _check_product(out, _exact_x(x[:rows]), _values(q, scale), None)
    assert (store[rows:] == 7).all() and (store[:, 0] == 7).all() and (store[:, n + 1:] == 7).all()


def test_linear4_shapes_and_refusals():
    q, scale = ops.quantize4(torch.randn(40, 64, device="cuda", generator=_gen(14)))
    w = ops.weight4(q, scale)
    x = torch.randn(2, 3, 64, device="cuda", generator=_gen(15)).bfloat16()
    assert torch.equal(ops.linear4(x, w).view(6, 40), ops.linear4(x.view(6, 64), w))
    assert torch.equal(ops.linear4(x[0, 0], w), ops.linear4(x[0], w)[0])
    assert ops.linear4(x[:, :0], w).shape == (2, 0, 40)
    xq, xs = ops.quantize4(x)
    assert torch.equal(ops.linear4(xq, w, x_scale=xs, out_dtype=torch.bfloat16), ops.linear4(x, w))
    assert torch.equal(ops.linear4(x[..., :50], w), ops.linear4(torch.nn.functional.pad(x[..., :50], (0, 14)), w))      # (a last block that is not whole)
    bias = torch.zeros(40, device="cuda")
    for bad in (lambda: ops.linear4(x[..., :32], w), lambda: ops.linear4(x, q), lambda: ops.linear4(x, w, bias[:39]), lambda: ops.linear4(x, w, bias.half()), lambda: ops.linear4(xq, w),
                lambda: ops.linear4(x, w, x_scale=xs), lambda: ops.linear4(xq, w, x_scale=xs[..., :1]), lambda: ops.linear4(xq, w, x_scale=xs.int()), lambda: ops.linear4(x[..., ::2], w),
                lambda: ops.linear4(x, w, out=torch.empty(2, 3, 41, device="cuda")), lambda: ops.linear4(x, w, out_dtype=torch.float64), lambda: ops.linear4(x, w, bias.cpu()),
                lambda: ops.weight4(q[:, :16], scale), lambda: ops.weight4(q, scale.cpu()), lambda: ops.weight4(q[:0], scale[:0]), lambda: ops.weight4(q[:, ::2], scale[:, :1])):
        with pytest.raises(FastllmError):
            bad()
    odd = torch.zeros(40, 40, dtype=torch.uint8, device="cuda")
    with pytest.raises(FastllmError, match="16-byte"):
        ops.linear4(x, ops.weight4(odd[:, :32], scale))


def test_linear4_far_offsets():
    """weights and results whose offsets pass 2^31 bytes"""
    n, k = 9, 64
    stride = (1 << 31) // 8 + 16
    store = torch.zeros(8 * stride + k, dtype=torch.uint8, device="cuda")
    q = store.as_strided((n, k // 2), (stride, 1))
    q.random_(0, 256, generator=_gen(16))
    scale = torch.randint(120, 125, (n, 2), device="cuda", generator=_gen(17)).to(torch.uint8)
    x = torch.randn(200, k, device="cuda", generator=_gen(18)).bfloat16()
    for rows in (1, 20, 200):
        _check_product(ops.linear4(x[:rows], ops.weight4(q, scale)), _exact_x(x[:rows]), _values(q, scale), None)
    far = store.view(torch.bfloat16)[: 8 * (stride // 2) + n].as_strided((9, n), (stride // 2, 1))
    del store
    dense = q.clone().contiguous()
    y = ops.linear4(x[:9], ops.weight4(dense, scale), out=far)
    _check_product(y, _exact_x(x[:9]), _values(dense, scale), None)


def _far(rows, cols, dtype):
    """rows on 16-byte borders whose last one lies behind 2^31 elements"""
    step = (1 << 31) // (rows - 1) // 16 * 16 + 16
    return torch.empty((rows - 1) * step + cols, dtype=dtype, device="cuda").as_strided((rows, cols), (step, 1))


@pytest.mark.parametrize("rows", [2, 9, 40, 140])
@pytest.mark.parametrize("out_dtype", [torch.bfloat16, torch.float32])
def test_linear4_far_results(rows, out_dtype):
    """every kernel's way of storing"""
    n, k = 256, 320
    x = torch.randn(rows, k, device="cuda", generator=_gen(rows)).bfloat16()
    q, scale = _rows4(n, k, 122, 5)
    out = _far(rows, n, out_dtype)
    ops.linear4(x, ops.weight4(q, scale), out=out)
    _check_product(out, _exact_x(x), _values(q, scale), None)


@pytest.mark.parametrize("rows", [2, 9, 40, 140])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32, torch.uint8])
def test_linear4_far_activations(rows, dtype):
    """every kernel's way of loading; of rows in 4 bits already (uint8) their scales too"""
    n, k = 200, 320
    w = ops.weight4(*_rows4(n, k, 122, 6))
    x = torch.randn(rows, k, device="cuda", generator=_gen(rows))
    x, xs = ops.quantize4(x) if dtype == torch.uint8 else (x.to(dtype), None)
    far, far_scale = _far(rows, x.shape[1], dtype), None
    far.copy_(x)
    if xs is not None:
        far_scale = _far(rows, xs.shape[1], dtype)
        far_scale.copy_(xs)
    assert torch.equal(ops.linear4(far, w, x_scale=far_scale), ops.linear4(x, w, x_scale=xs))


@pytest.mark.parametrize("dtype", FLOATS)
def test_far_rows_there_and_back(dtype):
    x = torch.randn(3, 96, device="cuda", generator=_gen(7)).to(dtype)
    far = _far(3, 96, dtype)
    far.copy_(x)
    for call in (ops.quantize4, ops.glu4):
        for a, b in zip(call(far), call(x)):
            assert torch.equal(a, b)
    q, scale = ops.quantize4(x)
    far_q, far_scale = _far(3, 48, torch.uint8), _far(3, 3, torch.uint8)
    far_q.copy_(q), far_scale.copy_(scale)
    assert torch.equal(ops.dequantize4(far_q, far_scale, dtype=dtype), ops.dequantize4(q, scale, dtype=dtype))
    far.fill_(7)
    kind, lib = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}[dtype], _lib.load()
    assert lib.fl_dequantize4(q.data_ptr(), 48, scale.data_ptr(), 3, 3, 96, far.data_ptr(), kind, far.stride(0), torch.cuda.current_stream().cuda_stream) == 0
    assert torch.equal(far, ops.dequantize4(q, scale, dtype=dtype))
    far_q.fill_(77), far_scale.fill_(77)
    assert lib.fl_quantize4(x.data_ptr(), kind, 3, 96, 96, far_q.data_ptr(), far_q.stride(0), far_scale.data_ptr(), far_scale.stride(0), torch.cuda.current_stream().cuda_stream) == 0
    assert torch.equal(far_q, q) and torch.equal(far_scale, scale)


# ---- together, on streams, in graphs ------------------------------------------------------------------------------------------------
def _feed_forward(x, w_in, w_out, act="silu"):
    """a feed-forward with 4-bit weights: two products with the activation between them"""
    h, hs = ops.glu4(ops.linear4(x, w_in, out_dtype=torch.float32), act)
    return ops.linear4(h, w_out, x_scale=hs, out_dtype=torch.bfloat16)


def _weights(width, hidden, seed):
    g = _gen(seed)
    first, second = torch.randn(2 * hidden, width, device="cuda", generator=g) * width ** -0.5, torch.randn(width, hidden, device="cuda", generator=g) * hidden ** -0.5
    return [(ops.quantize4(w), ops.weight4(*ops.quantize4(w))) for w in (first, second)]


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("rows", [1, 19, 150, 700])
def test_feed_forward(rows, act):
    """each operator on what the one before it left, as it is used"""
    (w1, w_in), (w2, w_out) = _weights(512, 1000, 20)
    x = torch.randn(rows, 512, device="cuda", generator=_gen(21)).bfloat16()
    y = ops.linear4(x, w_in, out_dtype=torch.float32)
    _check_product(y, _exact_x(x), _values(*w1), None)
    h, hs = ops.glu4(y, act)
    _check_glu(y, act, h, hs)
    out = ops.linear4(h, w_out, x_scale=hs, out_dtype=torch.bfloat16)
    _check_product(out, _values(h, hs), _values(*w2), None)
    assert torch.equal(out, _feed_forward(x, w_in, w_out, act))


def test_parts_of_a_weight_that_do_not_belong_together():
    """refused before a kernel is launched: it would read past their ends"""
    x = torch.randn(3, 500, device="cuda")
    w = ops.weight4(*_rows4(300, 500, 122, 3))
    for bad in (w._replace(tiles=w.tiles[:-1024]), w._replace(q=w.q[:40]), w._replace(q=w.q[:, :-16]), w._replace(q=w.q[:, :-1]), w._replace(q=w.q.t().contiguous().t()),
                w._replace(tiles=w.tiles[:1].expand(w.tiles.shape)), w._replace(tiles=w.tiles.cpu()), w._replace(q=w.q.cpu())):
        with pytest.raises(FastllmError, match="belong together|lives on|has 15 blocks"):
            ops.linear4(x, bad)


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("shift", [0, 1, 2, 3, 4, 5, 7])
def test_what_lies_beside_the_rows_does_not_matter(dtype, shift):
    """rows between numbers that are none, from every place within 16 bytes"""
    rows, k = 24, 250
    store = torch.full((rows, k + 11), math.nan, device="cuda").to(dtype)
    x = store[:, shift:k + shift]
    x.copy_(torch.randn(rows, k, device="cuda", generator=_gen(shift)) * 2)
    dense = x.clone()
    _check_rows(x, *ops.quantize4(x))
    for a, b in zip(ops.glu4(x), ops.glu4(dense)):
        assert torch.equal(a, b)
    q, scale = _rows4(200, k, 122, 3)
    w = ops.weight4(q, scale)
    for r in (1, 2, 9, 24):
        assert torch.equal(ops.linear4(x[:r], w), ops.linear4(dense[:r], w)) and not ops.linear4(x[:r], w).isnan().any()


def test_same_bits_every_time():
    (_, w_in), (_, w_out) = _weights(640, 3000, 22)
    for rows in (1, 70, 400):
        x = torch.randn(rows, 640, device="cuda", generator=_gen(23)).bfloat16()
        first = _feed_forward(x, w_in, w_out)
        for _ in range(5):
            assert torch.equal(first, _feed_forward(x, w_in, w_out))


def test_other_streams():
    """calls on several streams at once, each behind its own input"""
    (_, w_in), (_, w_out) = _weights(600, 2000, 24)
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    got = []
    for i in range(9):
        with torch.cuda.stream(streams[i % 3]):
            x = torch.randn((1, 50, 400)[i % 3], 600, device="cuda", generator=_gen(34 + i)).bfloat16()
            got.append((x, _feed_forward(x, w_in, w_out)))
    torch.cuda.synchronize()
    for x, y in got:
        assert torch.equal(y, _feed_forward(x, w_in, w_out))
    ops.check()


@pytest.mark.parametrize("rows", [1, 60, 300, 1100])
def test_graphs(rows):
    """two captured graphs, replayed on new inputs and side by side"""
    (_, w_in), (_, w_out) = _weights(256, 700, 25)
    graphs = []
    for i in range(2):
        x = torch.zeros(rows, 256, device="cuda", dtype=torch.bfloat16)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            y = _feed_forward(x, w_in, w_out)
        graphs.append((g, x, y, torch.cuda.Stream()))
    for step in range(3):
        for i, (g, x, y, s) in enumerate(graphs):
            x.copy_(torch.randn(rows, 256, device="cuda", generator=_gen(60 + 2 * step + i)))
        torch.cuda.synchronize()
        for g, x, y, s in graphs:
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for g, x, y, s in graphs:
            assert torch.equal(y, _feed_forward(x, w_in, w_out))
    ops.check()


HEAD = """
import threading
import torch
from fastllm_b200 import _lib, ops
g = torch.Generator(device="cuda"); g.manual_seed(1)
x = torch.randn(300, 200, device="cuda", generator=g).bfloat16()
w = ops.Weight4(*[torch.randint(118, 124, s, dtype=torch.uint8, device="cuda", generator=g) for s in ((900, 112), (8 * 1024,), (900, 7))])
calls = {"rows": lambda: ops.quantize4(x), "back": lambda: (ops.dequantize4(w.q, w.scale),), "glu": lambda: ops.glu4(x), "weight": lambda: ops.weight4(w.q, w.scale)[1:2],
         "token": lambda: (ops.linear4(x[:1], w),), "self": lambda: (ops.linear4(x[:9], w),), "few": lambda: (ops.linear4(x[:60], w),), "pair": lambda: (ops.linear4(x, w),)}
same = lambda a, b: all(torch.equal(u, v) for u, v in zip(a, b))
_lib.init(0)                        # the process is bound, no operator has run
"""


def _run(code):
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", HEAD + code], capture_output=True, text=True, timeout=300, cwd=root, env=dict(os.environ, PYTHONPATH=root))
    assert r.returncode == 0 and r.stdout.strip() == "same", r.stderr[-2000:]


@pytest.mark.parametrize("name", ["rows", "back", "glu", "weight", "token", "self", "few", "pair"])
def test_first_call_of_a_bound_process_inside_a_capture(name):
    """set-up and loading do not break the capture"""
    _run("""
call = calls[%r]
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    y = call()
graph.replay()
torch.cuda.synchronize()
assert same(y, call())
ops.check()
print("same")
""" % name)


def test_first_calls_in_several_threads():
    _run("""
got = {}
gate = threading.Barrier(16)
def work(i, name):
    gate.wait()
    with torch.cuda.stream(torch.cuda.Stream()):
        got[i, name] = calls[name]()
        torch.cuda.current_stream().synchronize()
torch.cuda.synchronize()
threads = [threading.Thread(target=work, args=(i, n)) for i in range(2) for n in calls]
[t.start() for t in threads]
[t.join() for t in threads]
assert len(got) == 16 and all(same(y, calls[n]()) for (_, n), y in got.items())
ops.check()
print("same")
""")
