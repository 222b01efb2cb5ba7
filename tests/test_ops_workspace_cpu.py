"""Workspaces of products: one for any number of rows up to N is as large as that of N; the layered models take theirs by the same rule."""
import ctypes as C
from pathlib import Path

import pytest

from fastllm_b200 import _lib

CSRC = Path(__file__).resolve().parent.parent / "fastllm_b200" / "csrc"


@pytest.mark.parametrize("k", [1, 15, 2048, 4096, 4097, 8192, 16384, 16385, 131071])
@pytest.mark.parametrize("dtype", [0, 1, 2])
def test_fewer_rows_need_no_more(k, dtype):
    n, most = C.c_size_t(), 0
    for rows in range(0, 700):
        assert _lib.load().fl_linear8_workspace(rows, k, dtype, C.byref(n)) == 0
        assert n.value >= most
        most = n.value


def test_the_head_takes_its_workspace_by_the_rule():
    body = (CSRC / "fl_layered.cu").read_text()
    assert "y.head8_ws.alloc(linear8_workspace(N, m.W));" in body and "y.head8_ws.p, y.head8_ws.n, c.step_failed.p);" in body
    call = (CSRC / "fl_ops.cu").read_text().split("void op_linear8(", 1)[1].split("\n}\n", 1)[0]
    assert call.index("workspace_bytes >= linear8_workspace(rows, k)") < call.index("run_linear8(")


def test_memory_for_log_probabilities_that_cannot_be_had_does_not_cost_the_cache():
    """taken outside what marks the cache as lost after a CUDA error; the next call asks for both buffers again"""
    body = (CSRC / "fl_lib.cu").read_text().split("FL_EXPORT int fl_cache_logprobs(", 1)[1].split("FL_API_END", 1)[0]
    guarded = [part.split("} catch", 1)[0] for part in body.split("    try {\n")[1:]]
    assert len(guarded) == 2 and body.count(".alloc(") == 2 and not any(".alloc(" in part for part in guarded)
    assert "c->lp_dev.n < tok + res || c->lp_host.n < tok + res" in body and body.index("cudaStreamSynchronize") < body.index(".alloc(")
