"""CPU: argument checks of the pooled KV cache run before any launch and need
no GPU; the ctypes mirror of zkv_pool has the C compiler's layout."""
import ctypes
import os
import shutil
import subprocess

import pytest
import torch

from conftest import ROOT
from zoomkv_revision_b200 import _lib, ops

OK, ARG, ALIGN, CAPACITY, UNSUPPORTED = 0, 1, 2, 3, 5


def pool(**kw):
    d = dict(k=0x10000, v=0x20000, k_block=4096, k_token=128, k_head=2048, v_block=4096, v_token=128, v_head=2048,
             n_blocks=4, block_size=16, kv_heads=2, head_dim=128, dtype=0, k_scale=None, v_scale=None)
    d.update(kw)
    return _lib.ZkvPool(**d)


@pytest.mark.parametrize("bad,code", [
    (dict(k=None), ARG), (dict(v=None), ARG), (dict(n_blocks=0), ARG), (dict(kv_heads=0), ARG), (dict(dtype=3), ARG),
    (dict(dtype=-1), ARG), (dict(k_scale=0x3000), ARG), (dict(k_token=0), ARG), (dict(v_block=-8), ARG),
    (dict(head_dim=96), UNSUPPORTED), (dict(head_dim=512), UNSUPPORTED), (dict(block_size=8), UNSUPPORTED),
    (dict(block_size=48), UNSUPPORTED), (dict(block_size=2048), UNSUPPORTED), (dict(n_blocks=2 ** 31), CAPACITY),
    (dict(k=0x10008), ALIGN), (dict(k_token=132), ALIGN), (dict(v_head=2052), ALIGN),
    (dict(dtype=2, k_token=136), ALIGN),
])
def test_pool_fields(bad, code):
    lib = _lib.lib()
    p = pool(**bad)
    assert lib.zkv_pool_init(ctypes.addressof(p)) == code
    assert lib.zkv_pool_write(0x1000, 256, 128, 0x1000, 256, 128, 0, 0x1000, 4, ctypes.addressof(p), None, None) == code
    assert lib.zkv_pool_decode(0x1000, 1024, 128, 0, ctypes.addressof(p), 0x1000, 0x1000, 4, 4, 2, 8, 0.1, 0, 0.0, 0,
                               0x1000, None, None, 0x1000, 1 << 30, None) == code


def decode(p, q=0x1000, q_row=1024, q_head=128, dtype=0, lens=0x1000, table=0x1000, ld=4, width=4, batch=2, heads=8,
           window=0, softcap=0.0, max_len=0, out=0x1000, ws=0x1000, ws_bytes=1 << 30):
    return _lib.lib().zkv_pool_decode(q, q_row, q_head, dtype, ctypes.addressof(p), lens, table, ld, width, batch, heads,
                                      0.1, window, softcap, max_len, out, None, None, ws, ws_bytes, None)


@pytest.mark.parametrize("bad,code", [
    (dict(q=None), ARG), (dict(lens=None), ARG), (dict(out=None), ARG), (dict(table=None), ARG), (dict(ws=None), ARG),
    (dict(batch=-1), ARG), (dict(width=-1), ARG), (dict(ld=3), ARG), (dict(heads=7), ARG), (dict(heads=0), ARG),
    (dict(window=-1), ARG), (dict(softcap=-1.0), ARG), (dict(softcap=float("nan")), ARG), (dict(max_len=-1), ARG),
    (dict(dtype=1), ARG), (dict(dtype=2), ARG), (dict(q=0x1008), ALIGN), (dict(q_row=1020), ALIGN),
    (dict(q_head=132), ALIGN), (dict(ws=0x1010), ALIGN), (dict(width=10 ** 6, ld=10 ** 6, ws_bytes=8), CAPACITY),
    (dict(heads=2 * 5121), CAPACITY), (dict(batch=0), OK),
])
def test_decode_arguments(bad, code):
    assert decode(pool(), **bad) == code


def test_write_plan_release_arguments():
    lib = _lib.lib()
    p = ctypes.addressof(pool_kept := pool())
    assert pool_kept.n_blocks == 4
    w = lambda **k: lib.zkv_pool_write(*{**dict(k=0x1000, kt=256, kh=128, v=0x1000, vt=256, vh=128, dt=0, slots=0x1000,  # noqa: E731
                                               n=4, p=p, st=None, stream=None), **k}.values())
    assert w(k=None) == ARG and w(slots=None) == ARG and w(n=-1) == ARG and w(dt=1) == ARG and w(dt=2) == ARG
    assert w(k=0x1004) == ALIGN and w(vt=130) == ALIGN and w(n=2 ** 31) == CAPACITY and w(n=0) == OK
    plan = lambda **k: lib.zkv_pool_plan(*{**dict(lens=0x1000, new=None, batch=2, S=16, table=0x1000, ld=4, width=4,  # noqa: E731
                                                 free=0x1000, n_free=0x1000, n_blocks=8, slots=0x1000, pos=None, n_slots=2,
                                                 cu=None, lo=0x1000, no=0x1000, st=None, stream=None), **k}.values())
    assert plan(lens=None) == ARG and plan(batch=-1) == ARG and plan(ld=3) == ARG and plan(slots=None) == ARG
    assert plan(S=0) == UNSUPPORTED and plan(S=17) == UNSUPPORTED
    assert plan(batch=8193) == CAPACITY and plan(n_slots=2 ** 31) == CAPACITY and plan(n_blocks=2 ** 31) == CAPACITY
    rel = lambda **k: lib.zkv_pool_release(*{**dict(done=0x1000, lens=0x1000, batch=2, S=16, table=0x1000, ld=4, width=4,  # noqa: E731
                                                   free=0x1000, n_free=0x1000, n_blocks=8, lo=0x1000, no=0x1000, st=None,
                                                   stream=None), **k}.values())
    assert rel(done=None) == ARG and rel(free=None) == ARG and rel(S=12) == UNSUPPORTED and rel(batch=9000) == CAPACITY


def test_workspace_sizes():
    lib, p = _lib.lib(), pool()
    f = lambda *x: lib.zkv_pool_decode_ws_bytes(ctypes.addressof(p), *x)  # noqa: E731
    assert f(-1, 8, 0, 10 ** 6) == 0 and f(1, 7, 0, 10 ** 6) == 0 and f(1, 8, -1, 10 ** 6) == 0 and f(1, 8, 0, -1) == 0
    assert lib.zkv_pool_decode_ws_bytes(None, 1, 8, 0, 10 ** 6) == 0
    # short bounds need none; long ones a part's size for each CTA of the largest grid, whatever the batch
    assert f(1, 8, 0, 256) == 0 and f(4096, 8, 0, 256) == 0 and f(64, 8, 100, 10 ** 6) == 0
    assert 0 < f(1, 8, 0, 10 ** 6) <= f(64, 8, 0, 10 ** 6) == f(6400, 8, 0, 10 ** 6) < 16 << 20


def test_python_checks_need_no_gpu():
    x = torch.zeros(4, 16, 2, 128, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="CUDA"):
        ops.KVPool(x, x)
    n = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        ops.pool_plan(n, None, n.view(2, 1), n, n[:1], 16, torch.zeros(2, dtype=torch.int64))
    with pytest.raises(TypeError):
        ops.pool_release(n, n.long(), n.view(2, 1), n, n[:1], 16)


@pytest.mark.skipif(shutil.which("gcc") is None, reason="gcc not available")
def test_struct_layout_matches_c(tmp_path):
    lines = ["#include <stdio.h>", "#include <stddef.h>", f'#include "{os.path.join(ROOT, "include", "zkv.h")}"',
             'int main(void){printf("%zu\\n", sizeof(zkv_pool));']
    lines += [f'printf("%zu\\n", offsetof(zkv_pool, {f}));' for f, _ in _lib.ZkvPool._fields_] + ["return 0;}"]
    c, exe = tmp_path / "a.c", tmp_path / "a"
    c.write_text("\n".join(lines))
    subprocess.run(["gcc", "-o", str(exe), str(c)], check=True)
    got = [int(x) for x in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split()]
    assert got == [ctypes.sizeof(_lib.ZkvPool)] + [getattr(_lib.ZkvPool, f).offset for f, _ in _lib.ZkvPool._fields_]
