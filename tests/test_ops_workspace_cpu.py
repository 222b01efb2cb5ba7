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
