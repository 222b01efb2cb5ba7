"""Where the operators set themselves up, read out of the sources: by the first call that launches one, not for processes that never do."""
import re
from pathlib import Path

CSRC = Path(__file__).resolve().parent.parent / "fastllm_b200" / "csrc"


def _body(source, head):
    return source.split(head, 1)[1].split("\n}\n", 1)[0]


def test_fl_init_sets_up_no_operator():
    """about forty kernels would be loaded, and a device without pairs of SMs refused, for embeddings too"""
    init = (CSRC / "fl_lib.cu").read_text().split("FL_EXPORT int fl_init(", 1)[1].split("FL_API_END", 1)[0]
    assert "ops" not in init and "set_up" not in init


def test_every_way_to_an_operator_sets_up_first():
    source = (CSRC / "fl_ops.cu").read_text()
    heads = re.findall(r"\n(?:FL_EXPORT int|void) ((?:fl|op)_\w+)\(", source)
    for name in ("fl_linear8_workspace", "fl_operators_check"):         # (these launch nothing)
        heads.remove(name)
    assert sorted(heads) == sorted(["fl_quantize_rows", "fl_linear8", "fl_logprobs", "op_quantize_rows", "op_linear8", "op_logprobs"])
    for name in heads:
        body = _body(source, f" {name}(")
        launch = re.search(r"\n    (?:else )?(?:if \(.*\) )?(?:run_linear8|run_logprobs<\w+>|quantize_rows)\(", body)
        assert 0 <= body.index("set_up();") < launch.start(), name


def test_a_device_without_pairs_is_refused_where_they_are_needed():
    source = (CSRC / "fl_ops.cu").read_text()
    assert "FL_CHECK" not in _body(source, "static void set_up(") and "g_pair_clusters >= 1" in _body(source, "static void launch_pair(")
