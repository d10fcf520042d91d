"""CPU: argument checks of the 8-bit layer operators run before any launch and
need no GPU; the ctypes mirror of zkv_fp8_weight has the C compiler's layout."""
import ctypes
import os
import shutil
import subprocess

import pytest
import torch

from conftest import ROOT
from zoomkv_revision_b200 import _lib, ops

OK, ARG, ALIGN, CAPACITY, UNSUPPORTED = 0, 1, 2, 3, 5


def weight(**kw):
    d = dict(w=0x10000, scale=0x20000, ld=256, rows=192, k=256, parts=1)
    d.update(kw)
    return _lib.ZkvFp8Weight(**d)


BAD_WEIGHTS = [
    (dict(w=None), ARG), (dict(scale=None), ARG), (dict(rows=0), ARG), (dict(k=0), ARG), (dict(ld=240), ARG),
    (dict(parts=0), ARG), (dict(parts=3), ARG), (dict(k=248), UNSUPPORTED), (dict(rows=200, parts=2), UNSUPPORTED),
    (dict(w=0x10008), ALIGN), (dict(ld=264), ALIGN), (dict(rows=2 ** 31), CAPACITY),
    (dict(k=2 ** 25, ld=2 ** 25), CAPACITY), (dict(ld=2 ** 33), CAPACITY),
]


def linear(w, x=0x1000, x_ld=256, xs=0x2000, st=1, sb=4, tokens=4, out=0x3000, ld=192, dtype=0):
    return _lib.lib().zkv_fp8_linear(x, x_ld, xs, st, sb, tokens, ctypes.addressof(w), out, ld, dtype, None, None)


def swiglu(w, x=0x1000, x_ld=256, xs=0x2000, st=1, sb=4, tokens=4, out=0x3000, ld=192, os=0x4000, ot=1, ob=4):
    return _lib.lib().zkv_fp8_swiglu(x, x_ld, xs, st, sb, tokens, ctypes.addressof(w), out, ld, os, ot, ob, None, None)


@pytest.mark.parametrize("bad,code", BAD_WEIGHTS)
def test_weight_fields(bad, code):
    w = weight(**bad)
    assert _lib.lib().zkv_fp8_weight_init(ctypes.addressof(w)) == code
    assert linear(w, x_ld=2 ** 26, ld=2 ** 32) == code
    assert swiglu(w, x_ld=2 ** 26, ld=2 ** 32) == code


COMMON = [(dict(x=None), ARG), (dict(xs=None), ARG), (dict(out=None), ARG), (dict(tokens=-1), ARG), (dict(x_ld=240), ARG),
          (dict(ld=176), ARG), (dict(st=-1), ARG), (dict(sb=-1), ARG), (dict(x=0x1008), ALIGN), (dict(x_ld=264), ALIGN),
          (dict(tokens=2 ** 31), CAPACITY), (dict(x_ld=2 ** 33), CAPACITY), (dict(tokens=0), OK)]


@pytest.mark.parametrize("bad,code", COMMON + [(dict(dtype=2), ARG), (dict(dtype=-1), ARG), (dict(out=0x3001), ALIGN),
                                               (dict(out=0x3002, dtype=3), ALIGN)])
def test_linear_arguments(bad, code):
    assert linear(weight(), **bad) == code
    assert linear(weight(parts=2), **bad) != OK


@pytest.mark.parametrize("bad,code", COMMON + [(dict(os=None), ARG), (dict(ot=0), ARG), (dict(ob=0), ARG),
                                               (dict(out=0x3008), ALIGN), (dict(ld=200), ALIGN)])
def test_swiglu_arguments(bad, code):
    assert swiglu(weight(parts=2), **bad) == code
    assert swiglu(weight(), **bad) != OK


ROWS = [(dict(x=None), ARG), (dict(out=None), ARG), (dict(scale=None), ARG), (dict(tokens=-1), ARG), (dict(dim=0), ARG),
        (dict(x_ld=100), ARG), (dict(out_ld=100), ARG), (dict(dtype=2), ARG), (dict(dtype=3), ARG), (dict(st=0), ARG),
        (dict(sb=0), ARG), (dict(dim=120), UNSUPPORTED), (dict(x=0x1008), ALIGN), (dict(x_ld=132), ALIGN),
        (dict(out=0x3008), ALIGN), (dict(out_ld=136), ALIGN), (dict(tokens=2 ** 31), CAPACITY), (dict(tokens=0), OK)]


@pytest.mark.parametrize("bad,code", ROWS)
def test_quant_arguments(bad, code):
    d = dict(x=0x1000, x_ld=128, dtype=0, tokens=4, dim=128, out=0x3000, out_ld=128, scale=0x4000, st=1, sb=4, stream=None)
    assert _lib.lib().zkv_quant_fp8(*{**d, **bad}.values()) == code


@pytest.mark.parametrize("bad,code", ROWS + [
    (dict(w=None), ARG), (dict(res=None), ARG), (dict(to=None), ARG), (dict(eps=-1.0), ARG), (dict(eps=float("nan")), ARG),
    (dict(res_ld=64), ARG), (dict(to_ld=64), ARG), (dict(w=0x5008), ALIGN), (dict(res=0x6008), ALIGN),
    (dict(to_ld=132), ALIGN), (dict(dim=32784, x_ld=32784, out_ld=32784, res_ld=32784, to_ld=32784), CAPACITY)])
def test_norm_arguments(bad, code):
    d = dict(x=0x1000, x_ld=128, res=0x6000, res_ld=128, to=0x7000, to_ld=128, w=0x5000, dtype=0, tokens=4, dim=128,
             eps=1e-6, out=0x3000, out_ld=128, scale=0x4000, st=1, sb=4, stream=None)
    assert _lib.lib().zkv_rmsnorm_fp8(*{**d, **bad}.values()) == code


def test_tensors_of_the_wrong_kind_are_refused():
    x, w = torch.zeros(4, 256, dtype=torch.bfloat16), torch.zeros(128, 256).to(torch.float8_e4m3fn)
    with pytest.raises(ValueError, match="CUDA"):
        ops.quant_fp8(x)
    with pytest.raises(TypeError, match="bfloat16 or float16"):
        ops.quant_fp8(x.float())
    with pytest.raises(ValueError, match="CUDA"):
        ops.rmsnorm_fp8(x, x[0], 1e-6)
    with pytest.raises(TypeError, match="bfloat16 or float16"):
        ops.rmsnorm_fp8(w, x[0], 1e-6)
    with pytest.raises(ValueError, match="CUDA"):
        ops.Fp8Weight(w, torch.zeros(1, 2))


@pytest.mark.skipif(shutil.which("gcc") is None, reason="gcc not available")
def test_weight_struct_layout_matches_c(tmp_path):
    lines = ["#include <stdio.h>", "#include <stddef.h>", f'#include "{os.path.join(ROOT, "include", "zkv.h")}"',
             "int main(void){", 'printf("%zu\\n", sizeof(zkv_fp8_weight));']
    lines += [f'printf("%zu\\n", offsetof(zkv_fp8_weight, {f}));' for f, _ in _lib.ZkvFp8Weight._fields_]
    src = tmp_path / "w.c"
    src.write_text("\n".join(lines + ["return 0;}"]))
    exe = tmp_path / "w"
    subprocess.run(["gcc", "-o", str(exe), str(src)], check=True)
    got = [int(v) for v in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split()]
    want = [ctypes.sizeof(_lib.ZkvFp8Weight)] + [getattr(_lib.ZkvFp8Weight, f).offset for f, _ in _lib.ZkvFp8Weight._fields_]
    assert got == want
