"""GPU tests of the operators' set-up: a process's first call may be one of any operator, inside a capture or in several threads at once."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEAD = """
import threading
import torch
from fastllm_b200 import _lib, ops
g = torch.Generator(device="cuda"); g.manual_seed(1)
x = torch.randn(300, 200, device="cuda", generator=g).bfloat16()
w = torch.empty(900, 208, dtype=torch.int8, device="cuda").random_(-127, 128, generator=g)[:, :200]
s = torch.rand(900, device="cuda", generator=g)
calls = {"rows": lambda: ops.quantize_rows(x), "token": lambda: (ops.linear8(x[:1], w, s),), "few": lambda: (ops.linear8(x[:60], w, s),), "pair": lambda: (ops.linear8(x, w, s),),
         "logprobs": lambda: ops.logprobs(x.float(), top=5)}
same = lambda a, b: all(u is v is None or torch.equal(u, v) for u, v in zip(a, b))
_lib.init(0)                        # the process is bound, no operator has run
"""


def _run(code):
    r = subprocess.run([sys.executable, "-c", HEAD + code], capture_output=True, text=True, timeout=300, cwd=ROOT, env=dict(os.environ, PYTHONPATH=ROOT))
    assert r.returncode == 0 and r.stdout.strip() == "same", r.stderr[-2000:]


@pytest.mark.parametrize("name", ["rows", "token", "few", "pair", "logprobs"])
def test_first_call_of_a_bound_process_inside_a_capture(name):
    _run("""
call = calls[%r]
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    y = call()
graph.replay()
torch.cuda.synchronize()
assert same(y, call())
print("same")
""" % name)


def test_first_calls_in_several_threads():
    _run("""
got = {}
gate = threading.Barrier(10)
def work(i, name):
    gate.wait()
    with torch.cuda.stream(torch.cuda.Stream()):
        got[i, name] = calls[name]()
        torch.cuda.current_stream().synchronize()
torch.cuda.synchronize()
threads = [threading.Thread(target=work, args=(i, n)) for i in range(2) for n in calls]
[t.start() for t in threads]
[t.join() for t in threads]
assert len(got) == 10 and all(same(y, calls[n]()) for (_, n), y in got.items())
print("same")
""")


def test_products_that_ran_are_valid():
    """by calls and by a replayed graph"""
    _run("""
got = [calls[n]() for n in ("token", "few", "pair")]
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    again = [calls[n]() for n in ("token", "few", "pair")]
graph.replay()
torch.cuda.synchronize()
ops.check()
assert all(same(a, b) for a, b in zip(got, again))
print("same")
""")
