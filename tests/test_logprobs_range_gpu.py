"""GPU tests of log probabilities over rows whose numbers are far from 0, against their definition in 64 bits (bounds: see test_ops_gpu.py)."""
import pytest
import torch

from fastllm_b200 import ops
from test_ops_gpu import FLOATS, _check_logprobs, _gen

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("rows, vocab", [(700, 40), (3000, 7), (2000, 300), (1200, 2100), (300, 40), (3, 40)])
def test_rows_summed_anew_are_the_same_every_time(rows, vocab, dtype):
    """short rows of one block, most of whose warps have nothing to add up, between rows that are summed once"""
    low = torch.finfo(dtype).min
    x = (torch.randn(rows, vocab, device="cuda", generator=_gen(1)) * 3).to(dtype)
    x[::3] = low
    tokens = torch.randint(0, vocab, (rows,), device="cuda", generator=_gen(2))
    for top, temperature in ((0, 1.0), (5, 1.0), (5, 1e4)):
        first = ops.logprobs(x, tokens, top, temperature)
        _check_logprobs(first, x, tokens, top, temperature)
        for _ in range(30):
            for a, b in zip(first, ops.logprobs(x, tokens, top, temperature)):
                assert a is b is None or torch.equal(a, b)


def _fill(x, mask, g):
    """24 kinds of rows, again and again: each of eight numbers as a run in front, behind, at random places"""
    rows, vocab = x.shape
    at = torch.arange(vocab, device="cuda")
    for i in range(min(rows, 24)):
        value = mask[i // 3]
        if i % 3 == 0:
            x[i::24, : vocab - vocab // 7 - 1] = value
        elif i % 3 == 1:
            x[i::24, vocab // 9 + 1:] = value
        else:
            x[i::24] = torch.where((torch.rand(vocab, device="cuda", generator=g) < 0.97) & (at != vocab // 2), value, x[i::24])
    return x


@pytest.mark.parametrize("rows, vocab", [(24, 40), (24, 4100), (700, 2500), (24, 32003), (48, 152064)])
@pytest.mark.parametrize("temperature", [1.0, 0.3, 0.1])
@pytest.mark.parametrize("dtype", FLOATS)
def test_masks_of_finite_numbers(rows, vocab, temperature, dtype):
    """one block a row and several; what a mask is written with reaches from -1e4 to the type's lowest value"""
    g = _gen(3)
    most = -torch.finfo(dtype).min
    mask = [-min(v, most) for v in (1e4, 1e9, 3e9, 1e10, 1e12, 1e20, 1e29, 1e30)]
    x = _fill((torch.randn(rows, vocab, device="cuda", generator=g) * 3).to(dtype), mask, g)
    tokens = torch.randint(0, vocab, (rows, 3), device="cuda", generator=g)
    for top in (0, 7):
        _check_logprobs(ops.logprobs(x, tokens, top, temperature), x, tokens, top, temperature)


@pytest.mark.parametrize("rows, vocab", [(20, 33), (20, 5000), (650, 700), (20, 32003)])
@pytest.mark.parametrize("temperature", [1.0, 0.3, 0.1, 25.0])
@pytest.mark.parametrize("dtype", FLOATS)
def test_rows_around_any_number(rows, vocab, temperature, dtype):
    """all of a row beside one number, of one value or a few steps of its type apart; the numbers around which rows are summed twice among them"""
    line = 2.0 ** 27 * temperature * 0.6931471805599453
    most = torch.finfo(dtype).max / 2
    g = _gen(4)
    x = torch.empty(rows, vocab, device="cuda")
    for i in range(20):
        at = [1e10, 1e12, 1e20, 1e37, line * 0.5, line * 0.99, line, line * 1.01, line * 2, line * 4][i // 2] * (-1) ** i
        at = max(min(at, most), -most)
        step = abs(at) * torch.finfo(dtype).eps
        x[i::20] = at + step * torch.randint(-3, 4, x[i::20].shape, device="cuda", generator=g) if i % 4 < 2 else at
    x = x.to(dtype)
    tokens = torch.randint(0, vocab, (rows, 3), device="cuda", generator=g)
    for top in (0, 7):
        _check_logprobs(ops.logprobs(x, tokens, top, temperature), x, tokens, top, temperature)


@pytest.mark.parametrize("temperature", [1e-30, 1e-20, 1e-9, 1e-5, 1e4, 1e20, 1e30])
@pytest.mark.parametrize("vocab", [40, 700, 32003])
@pytest.mark.parametrize("dtype", FLOATS)
def test_masks_at_any_temperature(vocab, temperature, dtype):
    low = torch.finfo(dtype).min
    x = (torch.randn(10, vocab, device="cuda", generator=_gen(5)) * 3).to(dtype)
    x[0] = -torch.inf
    x[1] = low if temperature > 1e-2 else -60000.0              # (its quotient is a number of 32 bits)
    x[2, 1:] = -torch.inf
    x[3, : vocab // 2] = -torch.inf
    x[4, torch.rand(vocab, device="cuda", generator=_gen(6)) < 0.99] = -torch.inf
    x[4, vocab // 2] = 0
    x[5, vocab // 3] = torch.nan
    x[6] = -torch.inf
    x[6, vocab // 3] = torch.nan
    x[7, vocab - 1] = torch.inf
    x[8] = torch.nan
    x[9] = -0.0
    tokens = torch.randint(0, vocab, (10, 2), device="cuda", generator=_gen(7))
    for top in (0, 7):
        _check_logprobs(ops.logprobs(x, tokens, top, temperature), x, tokens, top, temperature)


@pytest.mark.parametrize("temperature", [1e36, 1e37, 1e38])
@pytest.mark.parametrize("vocab", [40, 32003])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_differences_past_the_largest_number(vocab, temperature, dtype):
    """numbers of both signs whose difference is none of 32 bits, over temperatures that bring it back"""
    x = ((torch.rand(6, vocab, device="cuda", generator=_gen(8)) * 2 - 1) * 3.3e38).to(dtype)
    x[3, vocab // 2] = -torch.inf
    x[4] = x[4].abs()
    x[5] = -x[5].abs()
    tokens = torch.randint(0, vocab, (6, 4), device="cuda", generator=_gen(9))
    for top in (0, 7):
        _check_logprobs(ops.logprobs(x, tokens, top, temperature), x, tokens, top, temperature)
