"""GPU: a launch that the runtime refuses is reported by its own call alone.

The refusal: a launch on the legacy stream while another stream is captured,
which the runtime turns down on the host.  In a process of its own, since the
capture is lost with it."""
import os
import subprocess
import sys

import pytest

from conftest import ROOT

pytestmark = pytest.mark.gpu

PROGRAM = r"""
import ctypes, sys
sys.path.insert(0, sys.argv[1])
import torch
from zoomkv_revision_b200 import _lib

lib = _lib.lib()
path = next(l.split()[-1] for l in open("/proc/self/maps") if "libcudart" in l)
rt = ctypes.CDLL(path)
B, S, H, D = 2, 16, 2, 128
i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")
lens, table, free, n_free, lens_out, n_out = i32(3, 4), i32(0, 1), i32(2, 3), i32(2), i32(0, 0), i32(0)
slots = torch.zeros(B, dtype=torch.int64, device="cuda")
done = torch.zeros(B, dtype=torch.bool, device="cuda")
k, v = (torch.zeros(4, S, H, D, dtype=torch.bfloat16, device="cuda") for _ in range(2))
rows, q = (torch.zeros(B, n, D, dtype=torch.bfloat16, device="cuda") for n in (H, 4 * H))
out, x, w = torch.zeros_like(q), torch.zeros(2, D, dtype=torch.bfloat16, device="cuda"), torch.ones(D, dtype=torch.bfloat16, device="cuda")
pool = _lib.ZkvPool(k.data_ptr(), v.data_ptr(), S * H * D, H * D, D, S * H * D, H * D, D, 4, S, H, D, 0, None, None)
p = ctypes.addressof(pool)
assert lib.zkv_pool_init(p) == 0
P = lambda t: t.data_ptr()
calls = dict(
    plan=lambda: lib.zkv_pool_plan(P(lens), None, B, S, P(table), 1, 1, P(free), P(n_free), 4, P(slots), None, B, None,
                                   P(lens_out), P(n_out), None, None),
    release=lambda: lib.zkv_pool_release(P(done), P(lens), B, S, P(table), 1, 1, P(free), P(n_free), 4, P(lens_out), P(n_out),
                                         None, None),
    write=lambda: lib.zkv_pool_write(P(rows), H * D, D, P(rows), H * D, D, 0, P(slots), B, p, None, None),
    decode=lambda: lib.zkv_pool_decode(P(q), 4 * H * D, D, 0, p, P(lens), P(table), 1, 1, B, 4 * H, 0.1, 0, 0.0, 0, P(out),
                                       None, None, None, 0, None),
    rmsnorm=lambda: lib.zkv_rmsnorm(P(x), P(w), P(x), 2, D, 1e-6, None),
)
torch.cuda.synchronize()
for name, call in calls.items():
    assert call() == 0, name                       # loads the kernels
    torch.cuda.synchronize()
    stream, graph = ctypes.c_void_p(), ctypes.c_void_p()
    assert rt.cudaStreamCreate(ctypes.byref(stream)) == 0
    assert rt.cudaStreamBeginCapture(stream, 2) == 0
    assert call() == 4, name                       # refused
    left = rt.cudaPeekAtLastError()
    rt.cudaStreamEndCapture(stream, ctypes.byref(graph))
    rt.cudaGetLastError()
    assert rt.cudaStreamDestroy(stream) == 0
    assert left == 0, (name, left)
    assert call() == 0, name                       # the next one is judged by itself
torch.cuda.synchronize()
print("ok")
"""


def test_a_refused_launch_leaves_no_error_behind():
    got = subprocess.run([sys.executable, "-c", PROGRAM, ROOT], capture_output=True, text=True, timeout=300,
                         env=dict(os.environ))
    assert got.returncode == 0 and got.stdout.strip().endswith("ok"), got.stdout + got.stderr
