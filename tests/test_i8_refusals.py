"""The 8-bit projections' argument checks, on the CPU: every refusal returns before
any device work, so the stand-in addresses below are never dereferenced and no GPU
is needed."""
import os

import pytest

import myos
from myos import _lib

BASE = 1 << 40  # aligned stand-in address
F32, F16, BF16 = 0, 1, 2


@pytest.fixture(scope="module", autouse=True)
def built():
    import build as pkg_build

    pkg_build.build()


def norm(**over):
    a = dict(q=BASE, q_stride=1536, scales=BASE + (1 << 20), total=None, total_stride=0, x=BASE + (2 << 20),
             dtype=F32, x_stride=1536, residual=BASE + (3 << 20), residual_stride=1536, gamma=BASE + (4 << 20),
             eps=1e-6, rows=4, width=1536)
    a.update(over)
    return _lib.load().myos_dev_add_norm_quant(
        a["q"], a["q_stride"], a["scales"], a["total"], a["total_stride"], a["x"], a["dtype"], a["x_stride"],
        a["residual"], a["residual_stride"], a["gamma"], a["eps"], a["rows"], a["width"], None)


def rows(swiglu=False, **over):
    a = dict(q=BASE, q_stride=1536, scales=BASE + (1 << 20), x=BASE + (2 << 20), dtype=BF16,
             x_stride=3200 if swiglu else 1536, rows=4, width=1536)
    a.update(over)
    f = _lib.load().myos_dev_swiglu_quant if swiglu else _lib.load().myos_dev_quant_rows
    return f(a["q"], a["q_stride"], a["scales"], a["x"], a["dtype"], a["x_stride"], a["rows"], a["width"], None)


def swiglu(**over):
    return rows(True, **over)


def product(**over):
    a = dict(out=BASE, dtype=F32, out_stride=300, a=BASE + (1 << 30), a_stride=512, a_scales=BASE + (2 << 30),
             w=BASE + (3 << 30), w_stride=512, w_scales=BASE + (4 << 30), bias=None, rows=4, k=500, channels=300)
    a.update(over)
    return _lib.load().myos_dev_matmul_i8(
        a["out"], a["dtype"], a["out_stride"], a["a"], a["a_stride"], a["a_scales"], a["w"], a["w_stride"],
        a["w_scales"], a["bias"], a["rows"], a["k"], a["channels"], None)


@pytest.mark.parametrize("call", [norm, rows, swiglu])
@pytest.mark.parametrize("over,code", [
    (dict(q=None), _lib.ERR_ARG), (dict(scales=None), _lib.ERR_ARG), (dict(x=None), _lib.ERR_ARG),
    (dict(dtype=F16), _lib.ERR_ARG), (dict(dtype=3), _lib.ERR_ARG), (dict(dtype=-1), _lib.ERR_ARG),
    (dict(width=0), _lib.ERR_SHAPE), (dict(width=131072, q_stride=1 << 20, x_stride=1 << 20, residual_stride=1 << 20), _lib.ERR_SHAPE),
    (dict(q_stride=1535), _lib.ERR_SHAPE), (dict(x_stride=1535), _lib.ERR_SHAPE), (dict(rows=1 << 31), _lib.ERR_SHAPE),
    (dict(x_stride=1 << 50), _lib.ERR_SHAPE), (dict(q_stride=1 << 50), _lib.ERR_SHAPE),
    (dict(x=BASE + 1), _lib.ERR_ARG), (dict(scales=BASE + 2), _lib.ERR_ARG),
], ids=lambda x: str(x))
def test_row_refusals(call, over, code):
    if "residual_stride" in over and call is not norm:
        over = {k: v for k, v in over.items() if k != "residual_stride"}
    assert call(**over) == code


@pytest.mark.parametrize("over,code", [
    (dict(gamma=None), _lib.ERR_ARG), (dict(eps=-1.0), _lib.ERR_ARG), (dict(eps=float("nan")), _lib.ERR_ARG),
    (dict(gamma=BASE + 1), _lib.ERR_ARG), (dict(residual=BASE + 2), _lib.ERR_ARG), (dict(total=BASE + 2, total_stride=1536), _lib.ERR_ARG),
    (dict(residual_stride=1535), _lib.ERR_SHAPE), (dict(total=BASE + (5 << 20), total_stride=1535), _lib.ERR_SHAPE),
    (dict(residual_stride=1 << 50), _lib.ERR_SHAPE),
    (dict(total=BASE + (3 << 20), total_stride=1600), _lib.ERR_ARG),             # in place with another stride
    (dict(total=BASE + (2 << 20), total_stride=1600), _lib.ERR_ARG),
    (dict(total=BASE + (2 << 20), total_stride=1536, dtype=BF16), _lib.ERR_ARG),  # in place of bf16 rows
    (dict(total=BASE + (2 << 20), total_stride=1536, dtype=BF16, rows=1), _lib.ERR_ARG),
], ids=lambda x: str(x))
def test_norm_refusals(over, code):
    assert norm(**over) == code


def test_a_gate_row_is_twice_as_wide():
    assert swiglu(width=1500, x_stride=2999) == _lib.ERR_SHAPE


@pytest.mark.parametrize("over,code", [
    (dict(out=None), _lib.ERR_ARG), (dict(a=None), _lib.ERR_ARG), (dict(a_scales=None), _lib.ERR_ARG),
    (dict(w=None), _lib.ERR_ARG), (dict(w_scales=None), _lib.ERR_ARG), (dict(dtype=F16), _lib.ERR_ARG),
    (dict(dtype=7), _lib.ERR_ARG), (dict(k=0), _lib.ERR_SHAPE),
    (dict(k=131072, a_stride=131072, w_stride=131072), _lib.ERR_SHAPE),
    (dict(a_stride=496), _lib.ERR_SHAPE), (dict(w_stride=496), _lib.ERR_SHAPE), (dict(out_stride=299), _lib.ERR_SHAPE),
    (dict(a_stride=1 << 45), _lib.ERR_SHAPE), (dict(w_stride=1 << 45), _lib.ERR_SHAPE), (dict(out_stride=1 << 45), _lib.ERR_SHAPE),
    (dict(rows=0x7fffff01), _lib.ERR_SHAPE), (dict(channels=0x7fffff01, out_stride=1 << 32), _lib.ERR_SHAPE),
    (dict(a_stride=504), _lib.ERR_ARG), (dict(w_stride=504), _lib.ERR_ARG), (dict(a=BASE + 8), _lib.ERR_ARG),
    (dict(w=BASE + 8), _lib.ERR_ARG), (dict(out=BASE + 2), _lib.ERR_ARG), (dict(out=BASE + 1, dtype=BF16), _lib.ERR_ARG),
    (dict(a_scales=BASE + 2), _lib.ERR_ARG), (dict(w_scales=BASE + 2), _lib.ERR_ARG), (dict(bias=BASE + 2), _lib.ERR_ARG),
], ids=lambda x: str(x))
def test_product_refusals(over, code):
    assert product(**over) == code


def test_no_rows_is_no_work():
    assert norm(rows=0, q=None, gamma=None) == _lib.OK
    assert rows(rows=0, q=None) == _lib.OK
    assert swiglu(rows=0, x=None) == _lib.OK
    assert product(rows=0, a=None) == _lib.OK
    assert product(channels=0, w=None) == _lib.OK


@pytest.mark.skipif(os.path.exists("/dev/nvidiactl") or os.path.exists("/dev/nvidia0"), reason="no-GPU behaviour")
def test_no_gpu_is_an_error():
    for st in (norm(), rows(), swiglu(), product()):
        assert st == _lib.ERR_CUDA


def test_the_python_layer_refuses_host_tensors():
    torch = pytest.importorskip("torch")
    from myos import dev

    q, s, x = torch.zeros(4, 64, dtype=torch.int8), torch.zeros(4), torch.zeros(4, 64)
    for call in (lambda: dev.quant_rows(q, s, x), lambda: dev.swiglu_quant(q, s, x), lambda: dev.add_norm_quant(q, s, x, s),
                 lambda: dev.matmul_i8(x, q, s, q, s)):
        with pytest.raises(myos.MyosError) as e:
            call()
        assert e.value.code == _lib.ERR_ARG
