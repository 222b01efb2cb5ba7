"""The C++ mirror's log probabilities over a stand-in for the library: what it hands over, and what it refuses itself."""
import shutil
import subprocess
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parent.parent
PROGRAM = r"""
#include "fastllm_host.hpp"
#include <cstdlib>
static int calls = 0;
extern "C" const char* fl_last_error(void) { return "library"; }
extern "C" int fl_cache_logprobs(fl_cache*, int rows, const int32_t* tokens, int given, double, int top, float* logprob, float*, float*, int32_t* top_ids, float*) {
    ++calls;
    for (int i = 0; i < rows * given; ++i) logprob[i] = (float)tokens[i];
    for (int i = 0; i < rows * top; ++i) top_ids[i] = i;
    return FL_OK;
}
int main() {
    using fastllm::logprobs;
    const fastllm::LogProbs r = logprobs(nullptr, 3, {1, 2, 3, 4, 5, 6}, 2);
    if (calls != 1 || r.logprob != std::vector<float>{1, 2, 3, 4, 5, 6} || r.logsumexp.size() != 3 || r.entropy.size() != 3 || r.top_ids.size() != 6) return 1;
    if (logprobs(nullptr, 2, {}, 0).logprob.size() != 0 || logprobs(nullptr, 0, {}, 5).top_ids.size() != 0 || calls != 3) return 2;
    auto refused = [](int rows, std::vector<int32_t> tokens, int top) {
        try { logprobs(nullptr, rows, tokens, top); } catch (const fastllm::Error& e) { return e.code == FL_ERR_INVALID; } catch (...) {}
        return false;
    };
    if (!refused(3, {1, 2, 3, 4}, 0) || !refused(4, {1, 2, 3}, 0) || !refused(0, {1}, 0) || !refused(-1, {}, 0) || !refused(-2, {1, 2}, 0)) return 3;      // (no row without its tokens' numbers)
    if (!refused(1, {1}, -1) || !refused(1, {1}, 33) || calls != 3) return 4;
    return 0;
}
"""


@pytest.mark.skipif(shutil.which("g++") is None, reason="no g++")
def test_log_probabilities(tmp_path):
    (tmp_path / "t.cpp").write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-O1", f"-I{ROOT / 'host'}", str(tmp_path / "t.cpp"), "-o", str(tmp_path / "t")], check=True)
    assert subprocess.run([str(tmp_path / "t")]).returncode == 0
