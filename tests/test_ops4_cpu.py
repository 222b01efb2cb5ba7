"""CPU tests of the refusals of the operators on 4-bit rows: every argument check answers on the host, before any device is asked for."""
import ctypes as C
import re
from pathlib import Path

import pytest
import torch

from fastllm_b200 import _lib, ops
from fastllm_b200._lib import FastllmError

P = 1 << 20             # an address that no call below gets far enough to use
CSRC = Path(__file__).resolve().parent.parent / "fastllm_b200" / "csrc"


def _quantize4(**change):
    a = dict(x=P, dtype=1, rows=4, cols=70, ldx=70, q=P, ldq=48, scale=P, lds=3)
    a.update(change)
    return _lib.load().fl_quantize4(*a.values(), None)


def _dequantize4(**change):
    a = dict(q=P, ldq=48, scale=P, lds=3, rows=4, cols=70, y=P, dtype=1, ldy=70)
    a.update(change)
    return _lib.load().fl_dequantize4(*a.values(), None)


def _glu4(**change):
    a = dict(x=P, dtype=1, rows=4, cols=70, ldx=140, act=4, limit=7.0, q=P, ldq=48, scale=P, lds=3)
    a.update(change)
    return _lib.load().fl_glu4(*a.values(), None)


def _weight4(**change):
    a = dict(scale=P, lds=3, n=40, k=70, tiles=P)
    a.update(change)
    return _lib.load().fl_weight4(*a.values(), None)


def _linear4(**change):
    a = dict(x=P, x_dtype=1, ldx=70, x_scale=None, lds=0, w=P, ldw=48, w_tiles=P, bias=None, rows=5, n=32, k=70, y=P, y_dtype=1, ldy=32, workspace=P, workspace_bytes=1 << 20)
    a.update(change)
    return _lib.load().fl_linear4(*a.values(), None)


def _refused(rc, word):
    assert rc == -1, rc
    assert word in _lib.load().fl_last_error().decode(), _lib.load().fl_last_error()


@pytest.mark.parametrize("change, word", [
    (dict(dtype=3), "f32, bf16 or f16"), (dict(dtype=4), "f32, bf16 or f16"), (dict(rows=-1), "rows"), (dict(rows=(1 << 30) + 1), "rows"), (dict(cols=0), "columns"),
    (dict(cols=(1 << 20) + 1, ldx=1 << 21, ldq=1 << 21, lds=1 << 21), "columns"), (dict(ldx=69), "row stride"), (dict(ldq=32), "row stride"), (dict(lds=2), "row stride"),
    (dict(x=None), "NULL"), (dict(q=None), "NULL"), (dict(scale=None), "NULL"), (dict(x=P + 1), "aligned"), (dict(q=P + 8), "16-byte"), (dict(ldq=56), "16-byte")])
def test_quantize4_refuses(change, word):
    _refused(_quantize4(**change), word)


@pytest.mark.parametrize("change, word", [
    (dict(dtype=3), "f32, bf16 or f16"), (dict(rows=-1), "rows"), (dict(cols=0), "columns"), (dict(cols=(1 << 20) + 1, ldy=1 << 21), "columns"), (dict(ldy=69), "row stride"),
    (dict(ldq=32), "row stride"), (dict(lds=2), "row stride"), (dict(y=None), "NULL"), (dict(q=None), "NULL"), (dict(scale=None), "NULL"), (dict(y=P + 1), "aligned"),
    (dict(q=P + 8), "16-byte"), (dict(ldq=56), "16-byte")])
def test_dequantize4_refuses(change, word):
    _refused(_dequantize4(**change), word)


@pytest.mark.parametrize("change, word", [
    (dict(dtype=3), "f32, bf16 or f16"), (dict(act=2), "activation"), (dict(act=5), "activation"), (dict(act=0, limit=0.0), "limit"), (dict(act=0, limit=float("nan")), "limit"),
    (dict(act=0, limit=float("inf")), "limit"), (dict(rows=-1), "rows"), (dict(cols=0), "columns"), (dict(ldx=139), "row stride"), (dict(ldq=32), "row stride"),
    (dict(lds=2), "row stride"), (dict(x=None), "NULL"), (dict(q=None), "NULL"), (dict(scale=None), "NULL"), (dict(x=P + 1), "aligned"), (dict(q=P + 8), "16-byte"),
    (dict(ldq=56), "16-byte")])
def test_glu4_refuses(change, word):
    _refused(_glu4(**change), word)


@pytest.mark.parametrize("change, word", [(dict(n=0), "n from"), (dict(k=0), "k from"), (dict(k=(1 << 20) + 1, lds=1 << 20), "k from"), (dict(lds=2), "row stride"), (dict(scale=None), "NULL"),
                                          (dict(tiles=None), "NULL"), (dict(tiles=P + 8), "16-byte")])
def test_weight4_refuses(change, word):
    _refused(_weight4(**change), word)


@pytest.mark.parametrize("change, word", [
    (dict(x_dtype=3), "activations"), (dict(x_dtype=7), "activations"), (dict(y_dtype=3), "results"), (dict(y_dtype=4), "results"), (dict(rows=-1), "rows"),
    (dict(rows=(1 << 30) + 1), "rows"), (dict(n=0), "n from"), (dict(k=0), "k from"), (dict(k=(1 << 20) + 1, ldx=1 << 21, ldw=1 << 20), "k from"), (dict(ldx=69), "row stride"),
    (dict(ldw=32), "row stride"), (dict(ldy=31), "row stride"), (dict(x=None), "NULL"), (dict(w=None), "NULL"), (dict(w_tiles=None), "NULL"), (dict(y=None), "NULL"),
    (dict(x_scale=P), "x_scale"), (dict(x_dtype=4, ldx=48), "x_scale"), (dict(w=P + 8), "16-byte"), (dict(ldw=56), "16-byte"), (dict(w_tiles=P + 8), "16-byte"),
    (dict(x_dtype=4, x_scale=P, lds=3, ldx=47), "row stride"), (dict(x_dtype=4, x_scale=P, lds=2, ldx=48), "row stride"), (dict(x_dtype=4, x_scale=P, lds=3, ldx=48, x=P + 4), "16-byte"),
    (dict(x_dtype=4, x_scale=P, lds=3, ldx=56), "16-byte"), (dict(x=P + 1), "aligned"), (dict(y=P + 1), "aligned"), (dict(bias=P + 1), "aligned"), (dict(rows=17, workspace=None), "workspace"),
    (dict(rows=17, workspace=P + 16), "workspace"), (dict(rows=17, workspace_bytes=1024 + 1024 - 1), "workspace"), (dict(rows=17, x_dtype=4, x_scale=P, lds=3, ldx=48, workspace=None), "workspace"), (dict(rows=1 << 21, n=1 << 20, ldy=1 << 20), "2^40")])
def test_linear4_refuses(change, word):
    _refused(_linear4(**change), word)


def test_no_rows_is_no_work():
    assert _quantize4(rows=0, x=None) == 0
    assert _dequantize4(rows=0, y=None) == 0
    assert _glu4(rows=0, x=None) == 0
    assert _linear4(rows=0, x=None, y=None, workspace=None) == 0


def test_sizes():
    n = C.c_size_t()
    lib = _lib.load()
    for rows in (1, 127, 128, 129, 500):
        for k in (1, 32, 33, 256, 257, 4096):
            assert lib.fl_weight4_bytes(rows, k, C.byref(n)) == 0 and n.value == (rows + 127) // 128 * ((k + 255) // 256) * 1024
    _refused(lib.fl_weight4_bytes(0, 1, C.byref(n)), "n from")
    _refused(lib.fl_weight4_bytes(1, 1, None), "NULL")
    _refused(lib.fl_linear4_workspace(1, 0, 1, C.byref(n)), "k from")
    _refused(lib.fl_linear4_workspace(1, 1, 3, C.byref(n)), "activations")
    _refused(lib.fl_linear4_workspace(1, 1, 1, None), "NULL")


@pytest.mark.parametrize("k", [1, 31, 32, 33, 256, 257, 4096, 8193, 1 << 20])
@pytest.mark.parametrize("dtype", [0, 1, 2, 4])
def test_workspace_of_fewer_rows_is_no_larger(k, dtype):
    """and it is ops.py's rule"""
    n, most = C.c_size_t(), 0
    for rows in range(0, 700):
        assert _lib.load().fl_linear4_workspace(rows, k, dtype, C.byref(n)) == 0
        assert n.value >= most and n.value == ops._room4(rows, (k + 31) // 32, dtype == 4)
        most = n.value


def test_tensors_off_the_gpu_are_refused():
    x, q, s = torch.zeros(2, 64), torch.zeros(2, 32, dtype=torch.uint8), torch.zeros(2, 2, dtype=torch.uint8)
    w = ops.Weight4(q, s, s)
    for call in (lambda: ops.quantize4(x), lambda: ops.dequantize4(q, s), lambda: ops.glu4(x), lambda: ops.weight4(q, s), lambda: ops.linear4(x, w)):
        with pytest.raises(FastllmError, match="no CPU fallback"):
            call()


def test_types_are_refused():
    x, q = torch.zeros(2, 64), torch.zeros(2, 32, dtype=torch.uint8)
    for call, word in ((lambda: ops.quantize4(x.double()), "rows are wanted"), (lambda: ops.dequantize4(q, q, dtype=torch.float64), "results are"), (lambda: ops.glu4(x.long()), "rows are wanted"),
                       (lambda: ops.glu4(x, "relu2"), "activation"), (lambda: ops.weight4(q[0], q[0]), "matrix"), (lambda: ops.linear4(x.double(), q), "activations are"),
                       (lambda: ops.linear4(x, q), "weight4")):
        with pytest.raises(FastllmError, match=word):
            call()


def _by_hand(monkeypatch, n=300, blocks=16):
    """a weight's parts as weight4 makes them; tensors here pass for ones on the device, and a call that gets as far as the library fails"""
    monkeypatch.setattr(ops, "_bound", [-1])
    monkeypatch.setattr(_lib, "load", lambda: pytest.fail("not refused"))
    return ops.Weight4(torch.zeros(n, 16 * blocks, dtype=torch.uint8), torch.zeros((n + 127) // 128 * ((blocks + 7) // 8) * 1024, dtype=torch.uint8), torch.zeros(n, blocks, dtype=torch.uint8))


@pytest.mark.parametrize("part", ["q", "tiles"])
@pytest.mark.parametrize("dtype", [torch.int8, torch.int32, torch.float32, torch.bfloat16])
def test_a_weight_of_other_types_is_refused(monkeypatch, part, dtype):
    """strides count elements and the kernel bytes: it would read other numbers"""
    w = _by_hand(monkeypatch)
    with pytest.raises(FastllmError, match="belong together"):
        ops.linear4(torch.zeros(3, 512), w._replace(**{part: getattr(w, part).to(dtype)}))


@pytest.mark.parametrize("change", [
    lambda w: dict(q=w.q[:-1]), lambda w: dict(scale=w.scale[:-1]), lambda w: dict(scale=w.scale[:128]), lambda w: dict(scale=w.scale[:, :-1]), lambda w: dict(q=w.q[:, :-16]),
    lambda w: dict(q=w.q[:, :-1]), lambda w: dict(tiles=w.tiles[:2]), lambda w: dict(tiles=w.tiles.flatten()[:-1024]), lambda w: dict(tiles=w.tiles.view(2, 3, 1024)),
    lambda w: dict(tiles=w.tiles.view(6, 1024)), lambda w: dict(tiles=w.tiles[:1].expand(3, 2, 1024))],
    ids=["rows", "scales", "scales of fewer tiles", "scales of fewer blocks", "columns", "half a block", "tiles", "flat tiles", "tiles of another weight", "tiles of another shape", "tiles that repeat"])
def test_parts_of_different_weights_are_refused(monkeypatch, change):
    """also where no kernel would read out of bounds: 3 x 2 tiles are as many as 2 x 3, and other numbers"""
    w = _by_hand(monkeypatch)
    w = w._replace(tiles=w.tiles.view(3, 2, 1024))
    with pytest.raises(FastllmError, match="belong together"):
        ops.linear4(torch.zeros(3, 512), w._replace(**change(w)))


def test_parts_of_one_weight_go_through(monkeypatch):
    """tiles as weight4 shapes them, or the bytes that fl_weight4 wrote; rows with room between them"""
    w = _by_hand(monkeypatch)

    class Called(Exception):
        pass

    def load():
        raise Called

    monkeypatch.setattr(_lib, "load", load)
    wide = torch.zeros(300, 512, dtype=torch.uint8)
    for good in (w, w._replace(tiles=w.tiles.view(3, 2, 1024)), w._replace(q=wide[:, :256]), w._replace(scale=wide[:, 1:17])):
        with pytest.raises(Called):
            ops.linear4(torch.zeros(3, 512), good)


def test_every_way_to_an_operator_sets_up_first():
    source = (CSRC / "fl_ops4.cu").read_text()
    heads = re.findall(r"\n(?:FL_EXPORT int|void) ((?:fl|op)_\w+)\(", source)
    for name in ("fl_weight4_bytes", "fl_linear4_workspace"):           # (these launch nothing)
        heads.remove(name)
    for name in heads:
        body = source.split(f" {name}(", 1)[1].split("\n}\n", 1)[0]
        launch = re.search(r"\n    (?:run_linear4|quantize4|glu4|arrange4|by_type)\(", body)
        assert 0 <= body.index("set_up();") < launch.start(), name


def test_waits_inside_the_products_end():
    """every wait has a limit; a block that gave up goes through the same barriers as the others, reports it and leaves its copies time to land"""
    source = (CSRC / "linear4.cuh").read_text()
    assert re.search(r"\bmbar_wait\(", source) is None and source.count("if (!ok) op_give_up(g.failed);") == 3
    wide = source.split("l4_store_wide(const Linear4Args& g", 1)[1].split("\n}\n", 1)[0]
    assert wide.count("bar.sync") == 2 and " ok" not in wide
    assert "for (int c = cs * 16; c < last_col; c += 64)" in source


def test_a_product_that_gave_up_is_told_of():
    """the word that the kernels set goes into every product, is asked for before the next one is launched, and by the check, which takes it whatever the 8-bit products' word says"""
    source, ops8 = (CSRC / "fl_ops4.cu").read_text(), (CSRC / "fl_ops.cu").read_text()
    assert source.count("g_op4_failed.take()") == 1 and "bool products4_failed() { return g_op4_failed.take(); }" in source
    linear4 = source.split("FL_EXPORT int fl_linear4(", 1)[1].split("\n}\n", 1)[0]
    told = linear4.index("FL_CHECK(!products4_failed(), FL_ERR_CUDA,")
    assert linear4.index("set_up();") < told < linear4.index("run_linear4(") and linear4.split("run_linear4(", 1)[1].split(";", 1)[0].endswith("g_op4_failed.word)")
    run = source.split("static void run_linear4(", 1)[1].split("\n}\n", 1)[0]
    assert run.count("Linear4Args a{") == run.count(", failed, ") == 3
    check = ops8.split("FL_EXPORT int fl_operators_check(", 1)[1].split("\n}\n", 1)[0]
    assert check.index("= products4_failed();") < check.index("check_op_failed();") < check.index("FL_CHECK(!of4, FL_ERR_CUDA,")
