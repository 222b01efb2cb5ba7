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
