"""GPU test of the memory that an 8-bit output projection takes."""
import gc

import pytest
import torch

from fastllm_b200 import models

import test_rofetar_gpu as rofetar
from test_score_gpu import _check

pytestmark = pytest.mark.gpu
VOCAB, WIDTH = 100000, 512


def _held(bits):
    """bytes of the device that a model of mostly its embedding and head takes"""
    cfg = rofetar.config([rofetar.att()], vocab=VOCAB, width=WIDTH)
    gc.collect()
    torch.cuda.synchronize()
    before = torch.cuda.mem_get_info()[0]
    model = models.RofetarWithConfig.initialize_model(cfg, None, "bf16", head_bits=bits)[0]
    after = torch.cuda.mem_get_info()[0]
    cache = model.new_device_cache(1, 64)
    logits = cache.forward_ragged([0], [[5, 6, 7]], [range(3)])
    _check(cache.logprobs([1, 2, 3], 5), logits, [1, 2, 3], 5)
    return before - after


def test_the_16_bit_matrix_is_given_back():
    torch.zeros(1, device="cuda")
    _held(16), _held(8)                             # (what a process takes once)
    assert _held(16) - _held(8) >= VOCAB * WIDTH - (4 << 20)        # a byte a weight less, to two pieces of what the driver hands out
