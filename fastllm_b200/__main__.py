"""Command line of the package.

    python -m fastllm_b200 generate --model DIR --prompt-ids 5,17,3 [--prompt-ids ...] [--max-tokens N] [--temperature T]
                                    [--dtype bf16|f32] [--max-batch B] [--prefill-chunk C] [--eos ID] [--logprobs K] [--head-bits 8|16]
    python -m fastllm_b200 score    --model DIR --ids 5,17,3 [--ids ...] [--top K] [--dtype bf16|f32] [--head-bits 8|16]
    python -m fastllm_b200 trace    --model DIR --dtype bfloat16|float32 --out DIR --max-tokens N      (same as bin/trace_run)

`generate` loads the model the registry picks for DIR/config.json and continues every prompt (token ids in, token ids out: the
tokenizer stays with the server above this library) through the continuous batcher; one JSON line per prompt, with --logprobs also every
token's log probability and its K most likely alternatives.  `score` prints, per text, the log probability of every token but the first given
those before it (layered models); a number that is none, as that of a token of probability 0, is null.  --head-bits 8: output projection in 8-bit integers (layered models, bf16).
"""
from __future__ import annotations

import argparse
import json
import math
import sys


def _json(value) -> str:
    """JSON has no infinities and no NaN (a token of probability 0, a row without probabilities): null"""
    def plain(v):
        if isinstance(v, float):
            return v if math.isfinite(v) else None
        if isinstance(v, dict):
            return {k: plain(x) for k, x in v.items()}
        return [plain(x) for x in v] if isinstance(v, (list, tuple)) else v
    return json.dumps(plain(value), allow_nan=False)


def _generate(argv) -> int:
    ap = argparse.ArgumentParser(prog="python -m fastllm_b200 generate")
    ap.add_argument("--model", required=True)
    ap.add_argument("--prompt-ids", action="append", required=True, help="comma-separated token ids; repeat for several prompts")
    ap.add_argument("--max-tokens", type=int, default=16)
    ap.add_argument("--temperature", type=float, default=0.0)
    ap.add_argument("--dtype", default="bf16")
    ap.add_argument("--max-batch", type=int, default=4)
    ap.add_argument("--prefill-chunk", type=int, default=None)
    ap.add_argument("--eos", type=int, default=None)
    ap.add_argument("--device", type=int, default=0)
    ap.add_argument("--logprobs", type=int, default=None, help="alternatives to report per token, 0 to 32")
    ap.add_argument("--head-bits", type=int, default=16, choices=[8, 16])
    a = ap.parse_args(argv)
    from . import build
    build.build_library()
    from . import models
    prompts = [[int(t) for t in p.split(",") if t.strip()] for p in a.prompt_ids]
    model, _ = models.load_model(a.model, a.dtype, a.device, a.head_bits)
    batcher = models.ContinuousBatcher(model, max_batch=a.max_batch, eos_token_id=a.eos, prefill_chunk=a.prefill_chunk)
    got = batcher.generate(prompts, a.max_tokens, a.temperature, a.logprobs)
    told = [None] * len(prompts)
    if a.logprobs is not None:
        got, told = got
    for p, ids, about in zip(prompts, got, told):
        line = {"prompt": p, "generated": [int(t) for t in ids]}
        print(_json(line if about is None else {**line, "logprobs": about}))
    return 0


def _score(argv) -> int:
    ap = argparse.ArgumentParser(prog="python -m fastllm_b200 score")
    ap.add_argument("--model", required=True)
    ap.add_argument("--ids", action="append", required=True, help="a text's comma-separated token ids; repeat for several texts")
    ap.add_argument("--top", type=int, default=0, help="alternatives to report per token, 0 to 32")
    ap.add_argument("--dtype", default="bf16")
    ap.add_argument("--device", type=int, default=0)
    ap.add_argument("--head-bits", type=int, default=16, choices=[8, 16])
    a = ap.parse_args(argv)
    from . import build
    build.build_library()
    from . import models
    texts = [[int(t) for t in p.split(",") if t.strip()] for p in a.ids]
    model, _ = models.load_model(a.model, a.dtype, a.device, a.head_bits)
    for t, s in zip(texts, models.score(model, texts, a.top)):
        line = {"ids": t, "logprobs": [float(v) for v in s.logprobs], "total": s.total}
        if a.top:
            line["top"] = [[(int(i), float(v)) for i, v in zip(*row)] for row in zip(s.top_ids, s.top_logprobs)]
        print(_json(line))
    return 0


def main(argv=None) -> int:
    argv = list(sys.argv[1:] if argv is None else argv)
    if not argv or argv[0] in ("-h", "--help"):
        print(__doc__)
        return 0
    if argv[0] == "generate":
        return _generate(argv[1:])
    if argv[0] == "score":
        return _score(argv[1:])
    if argv[0] == "trace":
        from . import trace_runner
        return trace_runner.main(argv[1:])
    print(f"unknown command {argv[0]!r}\n{__doc__}", file=sys.stderr)
    return 2


if __name__ == "__main__":
    sys.exit(main())
