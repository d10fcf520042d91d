"""CPU: an operator whose tensors lie on another device than the current one
makes theirs current for its launch.  A default stream's handle is 0 on every
device, so the launch would go to the current one with the other's addresses.
The library, the tensors and the current device are stand-ins."""
import contextlib

import pytest
import torch

from zoomkv_revision_b200 import ops


class Tensor:
    """What the operators ask of a CUDA tensor, on cuda:1."""
    is_cuda, device = True, torch.device("cuda", 1)

    def __init__(self, dtype, *shape):
        self.dtype, self.shape = dtype, shape

    def get_device(self):
        return 1

    def data_ptr(self):
        return 1 << 20

    def is_contiguous(self):
        return True

    def contiguous(self):
        return self

    def dim(self):
        return len(self.shape)

    def numel(self):
        n = 1
        for s in self.shape:
            n *= s
        return n

    def stride(self, i=None):
        s = [1]
        for n in self.shape[:0:-1]:
            s.insert(0, s[0] * n)
        return tuple(s) if i is None else s[i]


class Pool:
    kv_heads, head_dim, block_size, dtype, code, index, ref, ws_sizes = 2, 128, 16, torch.bfloat16, 0, 1, 0, {}
    status_at = 0


@pytest.fixture
def launches(monkeypatch):
    """Entry point and current device of each launch."""
    current, seen = [0], []

    class Lib:
        def __getattr__(self, name):
            def call(*args):
                if not name.endswith("_ws_bytes"):
                    seen.append((name, current[0]))
                return 0
            return call

    @contextlib.contextmanager
    def device(index):
        before, current[0] = current[0], index
        yield
        current[0] = before

    monkeypatch.setattr(ops, "lib", Lib)
    monkeypatch.setattr(ops, "_RAW_STREAM", lambda index: 0)   # the default stream of any device
    monkeypatch.setattr(ops, "_current_device", lambda: current[0], raising=False)
    monkeypatch.setattr(torch.cuda, "device", device)
    yield seen
    assert current == [0]


def ints(*shape):
    return Tensor(torch.int32, *shape)


def test_the_pool_s_operators_run_on_its_device(launches):
    bf = torch.bfloat16
    slots, free, table = Tensor(torch.int64, 2), ints(8), ints(2, 4)
    ops.pool_plan(ints(2), ints(2), table, free, ints(1), 16, slots)
    ops.pool_release(Tensor(torch.bool, 2), ints(2), table, free, ints(1), 16)
    ops.pool_write(Tensor(bf, 2, 2, 128), Tensor(bf, 2, 2, 128), slots, Pool)
    q = Tensor(bf, 2, 8, 128)
    out, lse = ops.pool_decode(q, Pool, ints(2), table, out=q, lse=Tensor(torch.float32, 2, 8), return_lse=True)
    assert out is q and lse.shape == (2, 8)
    assert launches == [("zkv_pool_plan", 1), ("zkv_pool_release", 1), ("zkv_pool_write", 1), ("zkv_pool_decode", 1)]


def test_the_other_operators_too(launches):
    bf = torch.bfloat16
    x, w = Tensor(bf, 2, 256), Tensor(bf, 256)
    ops.rmsnorm(x, w, 1e-6, out=x)
    ops.silu_mul(Tensor(bf, 2, 512), x)
    ops.lse_merge_n(Tensor(torch.float32, 3, 2, 128), Tensor(torch.float32, 3, 2), Tensor(bf, 2, 128))
    assert [d for _, d in launches] == [1, 1, 1]


def test_every_operator_that_asks_for_a_stream_is_covered():
    """Each is wrapped, or looks at the current device itself."""
    import inspect
    import re
    for name, op in vars(ops).items():
        if not inspect.isfunction(op) or op.__module__ != ops.__name__:
            continue
        text = inspect.getsource(inspect.unwrap(op))
        if re.search(r"(?<!def )_(raw_)?stream\(", text) and name not in ("_stream", "_raw_stream"):
            assert hasattr(op, "__wrapped__") or "_current_device() != dev" in text, name
