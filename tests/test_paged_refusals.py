"""The paged serving operators' argument checks, on the CPU: every refusal
returns before any device work, so the stand-in addresses below are never
dereferenced and no GPU is needed. Also the layout of the two argument structs
and the rotary table."""
import ctypes as C
import os
import shutil
import subprocess

import numpy as np
import pytest

import myos
from myos import _lib

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
BASE = 1 << 40  # aligned stand-in address


@pytest.fixture(scope="module", autouse=True)
def built():
    import build as pkg_build

    pkg_build.build()


def kv(**over):
    a = dict(k=BASE, v=BASE + (1 << 30), page_stride=2 * 16 * 128, head_stride=16 * 128,
             slot_stride=128, num_pages=64, page_size=16, num_kv_heads=2, head_dim=128,
             kv_dtype=_lib.KV_BF16, reserved=0)
    a.update(over)
    return _lib.PagedKV(*[a[n] for n, _ in _lib.PagedKV._fields_])


BAD_KV = [
    (dict(k=None), _lib.ERR_ARG), (dict(v=None), _lib.ERR_ARG), (dict(kv_dtype=2), _lib.ERR_ARG),
    (dict(kv_dtype=-1), _lib.ERR_ARG), (dict(reserved=1), _lib.ERR_ARG),
    (dict(k=BASE + 8), _lib.ERR_ARG), (dict(slot_stride=132), _lib.ERR_ARG),
    (dict(num_pages=0), _lib.ERR_SHAPE), (dict(page_size=0), _lib.ERR_SHAPE),
    (dict(page_size=65537), _lib.ERR_SHAPE), (dict(num_kv_heads=0), _lib.ERR_SHAPE),
    (dict(head_dim=0), _lib.ERR_SHAPE), (dict(head_dim=100), _lib.ERR_SHAPE),
    (dict(head_dim=264), _lib.ERR_SHAPE), (dict(slot_stride=64), _lib.ERR_SHAPE),
    (dict(page_stride=0), _lib.ERR_SHAPE), (dict(page_stride=1 << 60), _lib.ERR_SHAPE),
]


def attn(cache=None, **over):
    a = dict(out=BASE, out_stride=12 * 128, lse=None, q=BASE + (1 << 20), q_stride=12 * 128,
             nseq=4, hq=12, table=BASE + (1 << 22), table_stride=8, max_blocks=8,
             lens=BASE + (1 << 23), scale=0.1, window=0, work=BASE + (1 << 24),
             work_bytes=_lib.PAGED_WORK_BYTES)
    a.update(over)
    c = cache or kv()
    return _lib.load().myos_dev_paged_attn(
        a["out"], a["out_stride"], a["lse"], a["q"], a["q_stride"], a["nseq"], a["hq"], C.byref(c),
        a["table"], a["table_stride"], a["max_blocks"], a["lens"], a["scale"], a["window"],
        a["work"], a["work_bytes"], None)


@pytest.mark.parametrize("over,code", BAD_KV, ids=lambda x: str(x))
def test_a_cache_out_of_form_is_refused(over, code):
    assert attn(kv(**over)) == code
    assert store(kv(**over)) == code


@pytest.mark.parametrize("over,code", [
    (dict(out=None), _lib.ERR_ARG), (dict(q=None), _lib.ERR_ARG), (dict(table=None), _lib.ERR_ARG),
    (dict(lens=None), _lib.ERR_ARG), (dict(work=None), _lib.ERR_ARG),
    (dict(hq=13), _lib.ERR_SHAPE), (dict(hq=0), _lib.ERR_SHAPE), (dict(hq=18), _lib.ERR_SHAPE),
    (dict(q_stride=128), _lib.ERR_SHAPE), (dict(out_stride=128), _lib.ERR_SHAPE),
    (dict(max_blocks=0), _lib.ERR_SHAPE), (dict(table_stride=7), _lib.ERR_SHAPE),
    (dict(max_blocks=1 << 30, table_stride=1 << 30), _lib.ERR_SHAPE),
    (dict(max_blocks=1 << 20, table_stride=1 << 20, nseq=4096), _lib.ERR_SHAPE),  # 2^32 tiles of 32 keys
    (dict(q=BASE + 4), _lib.ERR_ARG), (dict(out=BASE + 8), _lib.ERR_ARG),
    (dict(q_stride=12 * 128 + 2), _lib.ERR_ARG), (dict(lens=BASE + 2), _lib.ERR_ARG),
    (dict(work=BASE + 4), _lib.ERR_ARG),
    (dict(work_bytes=_lib.PAGED_WORK_BYTES - 1), _lib.ERR_SCRATCH_LIMIT),
], ids=lambda x: str(x))
def test_attention_refusals(over, code):
    assert attn(**over) == code


def store(cache=None, **over):
    a = dict(q=BASE, q_stride=12 * 128, qkv=BASE + (1 << 20), qkv_stride=16 * 128, rows=4, hq=12,
             qg=None, kg=None, eps=1e-6, cos=BASE + (1 << 22), sin=BASE + (1 << 23), num_pos=100,
             rot=128, pos=BASE + (1 << 24), slots=BASE + (1 << 25))
    a.update(over)
    c = cache or kv()
    return _lib.load().myos_dev_qk_norm_rope_store(
        a["q"], a["q_stride"], a["qkv"], a["qkv_stride"], a["rows"], a["hq"], C.byref(c), a["qg"],
        a["kg"], a["eps"], a["cos"], a["sin"], a["num_pos"], a["rot"], a["pos"], a["slots"], None)


@pytest.mark.parametrize("over,code", [
    (dict(q=None), _lib.ERR_ARG), (dict(qkv=None), _lib.ERR_ARG), (dict(slots=None), _lib.ERR_ARG),
    (dict(cos=None), _lib.ERR_ARG), (dict(pos=None), _lib.ERR_ARG), (dict(hq=0), _lib.ERR_SHAPE),
    (dict(rot=130), _lib.ERR_SHAPE), (dict(rot=136), _lib.ERR_SHAPE), (dict(rot=4), _lib.ERR_SHAPE),
    (dict(num_pos=0), _lib.ERR_SHAPE), (dict(q_stride=64), _lib.ERR_SHAPE),
    (dict(qkv_stride=12 * 128), _lib.ERR_SHAPE), (dict(q=BASE + 4), _lib.ERR_ARG),
    (dict(qkv_stride=16 * 128 + 1), _lib.ERR_ARG), (dict(qg=BASE + 2), _lib.ERR_ARG),
    (dict(slots=BASE + 4), _lib.ERR_ARG), (dict(cos=BASE + 4), _lib.ERR_ARG),
    (dict(q=BASE + (1 << 20)), _lib.ERR_ARG),  # in place with another row stride
], ids=lambda x: str(x))
def test_store_refusals(over, code):
    assert store(**over) == code


def tables(**over):
    names = ("table", "ctx", "new", "free", "num_free", "slots", "pos", "seq", "lens", "starts", "result")
    a = {n: BASE + (i << 20) for i, n in enumerate(names)}
    a.update(stride=8, blocks=8, nseq=4, cap=64, page=16, pages=64, rows=16)
    a.update(over)
    return _lib.load().myos_dev_paged_tables(
        a["table"], a["stride"], a["blocks"], a["ctx"], a["new"], a["nseq"], a["free"], a["cap"],
        a["num_free"], a["page"], a["pages"], a["slots"], a["pos"], a["seq"], a["rows"], a["lens"],
        a["starts"], a["result"], None)


@pytest.mark.parametrize("over,code", [
    (dict(table=None), _lib.ERR_ARG), (dict(ctx=None), _lib.ERR_ARG), (dict(free=None), _lib.ERR_ARG),
    (dict(num_free=None), _lib.ERR_ARG), (dict(slots=None), _lib.ERR_ARG), (dict(result=None), _lib.ERR_ARG),
    (dict(slots=BASE + 4), _lib.ERR_ARG), (dict(pos=BASE + 2), _lib.ERR_ARG),
    (dict(lens=BASE + (1 << 20)), _lib.ERR_ARG),          # the lengths it reads
    (dict(result=BASE + (4 << 20)), _lib.ERR_ARG),        # the free count it reads
    (dict(result=BASE + (4 << 20) - 4), _lib.ERR_ARG),
    (dict(nseq=16385), _lib.ERR_SHAPE), (dict(page=0), _lib.ERR_SHAPE), (dict(page=70000), _lib.ERR_SHAPE),
    (dict(blocks=0), _lib.ERR_SHAPE), (dict(stride=7), _lib.ERR_SHAPE), (dict(rows=1 << 31), _lib.ERR_SHAPE),
], ids=lambda x: str(x))
def test_table_refusals(over, code):
    assert tables(**over) == code


def logits(c=None, **over):
    a = dict(out=BASE, out_stride=1000, x=BASE + (1 << 30), x_stride=1000, rows=4, vocab=1000, ids=None)
    a.update(over)
    s = _lib.LogitControls(**c) if c else None
    return _lib.load().myos_dev_logit_controls(a["out"], a["out_stride"], a["x"], a["x_stride"], a["rows"],
                                               a["vocab"], C.byref(s) if s else None, a["ids"], None)


@pytest.mark.parametrize("c,over,code", [
    (None, dict(x=None), _lib.ERR_ARG), (None, dict(out=None), _lib.ERR_ARG),
    (None, dict(x=BASE + 2), _lib.ERR_ARG), (None, dict(vocab=0), _lib.ERR_SHAPE),
    (None, dict(x_stride=999), _lib.ERR_SHAPE), (None, dict(out_stride=999), _lib.ERR_SHAPE),
    (None, dict(out=BASE + (1 << 30), out_stride=1004), _lib.ERR_ARG),
    (dict(repetition=BASE), {}, _lib.ERR_ARG),   # penalties without a history
    (dict(history=BASE, history_width=8, history_stride=7), {}, _lib.ERR_SHAPE),
    (dict(history=BASE, history_width=1 << 31, history_stride=1 << 31), {}, _lib.ERR_SHAPE),
    (dict(bias_starts=BASE, bias_ids=BASE, bias_vals=BASE, num_bias=1 << 31), {}, _lib.ERR_SHAPE),
    (dict(bias_starts=BASE), {}, _lib.ERR_ARG),
    (dict(bias_starts=BASE + 1, bias_ids=BASE, bias_vals=BASE), {}, _lib.ERR_ARG),
    (dict(mask=BASE, mask_stride=31, num_masks=4), {}, _lib.ERR_SHAPE),
    (dict(mask=BASE, mask_stride=32, num_masks=3), {}, _lib.ERR_SHAPE),  # a mask per row, one short
], ids=lambda x: str(x))
def test_logit_refusals(c, over, code):
    assert logits(c, **over) == code


def test_no_rows_is_no_work():
    assert attn(nseq=0, out=None) == _lib.OK
    assert store(rows=0, q=None) == _lib.OK
    assert tables(nseq=0, table=None) == _lib.OK
    assert logits(rows=0, x=None) == _lib.OK


@pytest.mark.skipif(os.path.exists("/dev/nvidiactl") or os.path.exists("/dev/nvidia0"), reason="no-GPU behaviour")
def test_no_gpu_is_an_error():
    for st in (attn(), store(), tables(), logits()):
        assert st == _lib.ERR_CUDA


def test_python_layer_refuses_host_tensors():
    torch = pytest.importorskip("torch")
    from myos import dev

    x = torch.zeros(2, 4, 16, 64)
    with pytest.raises(myos.MyosError) as e:
        dev.PagedKV(x, x)
    assert e.value.code == _lib.ERR_ARG
    with pytest.raises(myos.MyosError) as e:
        dev.logit_controls(x[0, 0], x[0, 0])
    assert e.value.code == _lib.ERR_ARG


def test_struct_layouts_match_the_header(tmp_path):
    if not shutil.which("gcc"):
        pytest.skip("gcc not available")
    structs = {"myos_paged_kv": _lib.PagedKV, "myos_logit_controls_args": _lib.LogitControls}
    lines = ['#include <stdio.h>', '#include <stddef.h>', '#include "myos_cuda.h"', "int main(void) {"]
    for cname, py in structs.items():
        lines.append('printf("%s %%zu\\n", sizeof(%s));' % (cname, cname))
        lines += ['printf("%s.%s %%zu\\n", offsetof(%s, %s));' % (cname, f, cname, f) for f, _ in py._fields_]
    lines += ['printf("work %u\\n", MYOS_PAGED_WORK_BYTES);', "return 0;", "}"]
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    src.write_text("\n".join(lines))
    subprocess.run(["gcc", "-std=c11", "-I", os.path.join(REPO, "include"), str(src), "-o", str(exe)], check=True)
    got = dict(x.split() for x in subprocess.run([str(exe)], capture_output=True, text=True,
                                                 check=True).stdout.splitlines())
    assert int(got["work"]) == _lib.PAGED_WORK_BYTES
    for cname, py in structs.items():
        assert int(got[cname]) == C.sizeof(py), cname
        for f, _ in py._fields_:
            assert int(got[f"{cname}.{f}"]) == getattr(py, f).offset, (cname, f)


def test_rust_structs_match_the_header():
    from test_rust_shim import c_struct, rust_struct

    for s in ("myos_paged_kv", "myos_logit_controls_args"):
        assert c_struct(s) == rust_struct(s), s


def test_rope_table_is_the_reference_row():
    """Against rope.rs:186-194 in f32 steps; cosf and sinf are off by at most a
    step of the result (2^-24 below 1), numpy's f64 functions of the same f32
    angle by far less."""
    pytest.importorskip("torch")
    from myos import dev

    cs, sn = dev.rope_table(300, 64, 10000.0)
    inv = np.float32(1) / np.power(np.float64(10000.0), np.arange(32, dtype=np.float32) * 2 / np.float32(64))
    angle = (np.arange(300, dtype=np.float64)[:, None] * inv[None, :])
    # powf and the two f32 roundings: the angle is off by at most 3 * 2^-24 of itself
    tol = 3 * 2.0**-24 * np.abs(angle) + 2.0**-23
    assert (np.abs(cs - np.cos(angle)) <= tol).all() and (np.abs(sn - np.sin(angle)) <= tol).all()
    assert _lib.load().myos_rope_table(None, None, 4, 64, 1e4) == _lib.ERR_ARG
    with pytest.raises(myos.MyosError):
        dev.rope_table(4, 7, 1e4)
