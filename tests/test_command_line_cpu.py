"""CPU test of what the commands print: JSON that any reader takes, also for tokens of probability 0 and rows without probabilities."""
import json

import numpy as np
import pytest

from fastllm_b200 import __main__ as cli
from fastllm_b200 import models

INF, NAN = float("inf"), float("nan")


def _strict(line):
    def refuse(name):
        raise AssertionError(name)
    return json.loads(line, parse_constant=refuse)


class _Batcher:
    def __init__(self, *a, **k):
        pass

    def generate(self, prompts, max_tokens, temperature, logprobs):
        about = [{"logprob": -0.5, "top": [(4, -0.5), (7, -INF)]}, {"logprob": NAN, "top": [(-1, NAN), (-1, NAN)]}]
        return ([[4, 9]], [about]) if logprobs is not None else [[4, 9]]


@pytest.fixture
def stand_ins(monkeypatch):
    monkeypatch.setattr(models, "load_model", lambda *a, **k: (None, None))
    monkeypatch.setattr(models, "ContinuousBatcher", _Batcher)
    f = np.float32
    one = models.Scored(np.array([-1.5, -INF], f), np.zeros(2, f), np.array([[1, 2], [3, 4]], np.int32), np.array([[-1.5, -2], [-0.0, -INF]], f))
    monkeypatch.setattr(models, "score", lambda model, texts, top: [one])


def test_generate(stand_ins, capsys):
    assert cli.main(["generate", "--model", "x", "--prompt-ids", "5,6", "--logprobs", "2"]) == 0
    assert _strict(capsys.readouterr().out) == {"prompt": [5, 6], "generated": [4, 9], "logprobs": [{"logprob": -0.5, "top": [[4, -0.5], [7, None]]},
                                                                                                    {"logprob": None, "top": [[-1, None], [-1, None]]}]}
    assert cli.main(["generate", "--model", "x", "--prompt-ids", "5,6"]) == 0
    assert _strict(capsys.readouterr().out) == {"prompt": [5, 6], "generated": [4, 9]}


def test_score(stand_ins, capsys):
    assert cli.main(["score", "--model", "x", "--ids", "5,1,3", "--top", "2"]) == 0
    assert _strict(capsys.readouterr().out) == {"ids": [5, 1, 3], "logprobs": [-1.5, None], "total": None, "top": [[[1, -1.5], [2, -2.0]], [[3, 0.0], [4, None]]]}
