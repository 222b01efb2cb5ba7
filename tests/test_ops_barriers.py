"""Barriers inside the operators' kernels, read out of the sources: what one warp may still be reading is not written by another."""
from pathlib import Path

CSRC = Path(__file__).resolve().parent.parent / "fastllm_b200" / "csrc"


def test_the_sums_taken_anew_wait_for_readers_of_the_old_ones():
    """logprobs_kernel, a row far from 0: all warps have joined `part` (with one block per row no other barrier follows that) before any of them writes to it"""
    body = (CSRC / "logprobs.cuh").read_text().split(") logprobs_kernel(", 1)[1]
    again = body.split("    if (far) {\n", 1)[1].split("    } else {\n", 1)[0]
    assert body.count("    if (far) {\n") == 1 and again.count("part[warp] = ") == 1
    assert again.index("__syncthreads();") < again.index("part[warp] = ") < again.rindex("__syncthreads();") < again.index("part[i]")
