"""A product whose kernel gave up on a wait: told of once, by the next product or when asked (CPU: no kernel is made to fail)."""
import shutil
import subprocess
from pathlib import Path

import pytest

from fastllm_b200 import _lib, ops

CSRC = Path(__file__).resolve().parent.parent / "fastllm_b200" / "csrc"
PROGRAM = r"""
#include "failed_word.hpp"
int main() {
    fl::FailedWord none, w;
    int word = 0;
    w.word = &word;
    if (none.take() || w.take()) return 1;
    for (int i = 0; i < 2; ++i) {               // a process goes on after it
        word = 1;
        if (!w.take() || w.take() || word != 0) return 2;
    }
    return 0;
}
"""


@pytest.mark.skipif(shutil.which("g++") is None, reason="no g++")
def test_a_failure_is_told_once(tmp_path):
    (tmp_path / "t.cpp").write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-O1", f"-I{CSRC}", str(tmp_path / "t.cpp"), "-o", str(tmp_path / "t")], check=True)
    assert subprocess.run([str(tmp_path / "t")]).returncode == 0


def test_products_and_the_check_ask_the_word_that_kernels_set():
    source = (CSRC / "fl_ops.cu").read_text()
    check = source.split("static void check_op_failed(", 1)[1].split("\n}\n", 1)[0]
    assert "g_op_failed.take()" in check and source.count("g_op_failed.take()") == 1
    linear8 = source.split("FL_EXPORT int fl_linear8(", 1)[1].split("\n}\n", 1)[0]
    assert linear8.index("check_op_failed();") < linear8.index("run_linear8(") and "g_op_failed.word)" in linear8
    assert "check_op_failed();" in source.split("FL_EXPORT int fl_operators_check(", 1)[1].split("\n}\n", 1)[0]


def test_nothing_has_failed_before_anything_ran():
    assert _lib.load().fl_operators_check() == 0
    ops.check()
