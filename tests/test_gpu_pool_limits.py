"""GPU: bounds, limits and reports of the pooled KV cache's operators."""
import threading

import pytest
import torch

from test_gpu_pool import (BF, DEV, ERR_RANGE, check_decode, gen, i32, make_pool, make_table, plan_inputs)
from zoomkv_revision_b200 import ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("spare", [0, 20000])
@pytest.mark.parametrize("max_len", [1, 64, 300, 100000])
def test_max_len_never_cuts(max_len, spare):
    """Requests that are longer than the host believes, on every path that the belief chooses."""
    for lens, H, G, D, window in (([300, 0, 2000, 17], 2, 4, 128, 0), ([37 * i % 201 for i in range(700)], 1, 4, 64, 0),
                                  ([4000], 1, 4, 128, 0), ([37 * i % 201 for i in range(700)], 1, 12, 128, 100)):
        n_blocks = sum(-(-n // 16) for n in lens)
        k, v, _, _ = make_pool(1, n_blocks, 16, H, D, BF, "hnd")
        table = make_table(2, lens, 16, n_blocks, -(-max(lens) // 16) + spare)
        q = torch.randn(len(lens), H * G, D, generator=gen(3), device=DEV).to(BF)
        status = i32([0])
        out, lse = ops.pool_decode(q, ops.KVPool(k, v), i32(lens), table, window=window, max_len=max_len, return_lse=True,
                                   status=status)
        assert int(status) == 0
        check_decode(q, k, v, None, None, lens, table, out, lse, D ** -0.5, window)


def test_max_len_never_cuts_split_rows():
    """A belief that has the rows cut by units (over 128 MiB of K and V), and twice the tokens."""
    lens = [3000 - 17 * i for i in range(32)]
    n_blocks = sum(-(-n // 16) for n in lens)
    k, v, _, _ = make_pool(4, n_blocks, 16, 8, 128, BF, "hnd")
    table = make_table(5, lens, 16, n_blocks, 200)
    pool = ops.KVPool(k, v)
    assert ops.pool_decode_ws_bytes(32, 32, pool, 200, 1500) > 0
    q = torch.randn(32, 32, 128, generator=gen(6), device=DEV).to(BF)
    status = i32([0])
    out, lse = ops.pool_decode(q, pool, i32(lens), table, max_len=1500, return_lse=True, status=status)
    assert int(status) == 0
    check_decode(q, k, v, None, None, lens, table, out, lse, 128 ** -0.5)


def run_plan_and_release(batch):
    """One token for each of `batch` empty requests, and their release."""
    lens, n_free = i32([0] * batch), i32([batch])
    table = torch.full((batch, 1), -1, dtype=torch.int32, device=DEV)
    free = torch.arange(batch, device=DEV).int()
    slots = torch.empty(batch, dtype=torch.int64, device=DEV)
    ops.pool_plan(lens, None, table, free, n_free, 16, slots)
    assert sorted(slots.tolist()) == [16 * i for i in range(batch)]
    ops.pool_release(torch.ones(batch, dtype=torch.bool, device=DEV), lens, table, free, n_free, 16)
    assert int(n_free) == batch and not bool(lens.any())


def test_batches_of_every_size_from_several_threads():
    """A small batch of one thread does not lower what a large one of another needs."""
    failed = []

    def work(batch):
        try:
            run_plan_and_release(batch)
        except Exception as e:  # noqa: BLE001
            failed.append(e)

    run_plan_and_release(8192)
    for batch in (8, 8192, 3):
        t = threading.Thread(target=work, args=(batch,))
        t.start()
        t.join()
        run_plan_and_release(8192)
    assert not failed


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("B,ctx", [(1, 100), (5, 200), (3, 20000), (1300, 90)])
def test_release_leaves_bad_ids_out(B, ctx, in_place):
    """An id outside the pool goes on no stack: the next plan would give its request a place that is none."""
    import random
    S, r = 16, random.Random(B)
    lens, _, table, free, n_free = plan_inputs(B, B, S, ctx, 1)
    lens = [max(n, 1) for n in lens]
    n_blocks = len(free)
    done = [r.random() < 0.8 or b == 0 for b in range(B)]
    for b in range(B):
        for j in range(-(-lens[b] // S)):
            if table[b][j] < 0 or r.random() < 0.1 or (b, j) == (0, 0):
                table[b][j] = r.choice([-1, n_blocks, 2 ** 31 - 1, -2 ** 31])
    want = free[:n_free]
    for b in range(B):
        if done[b]:
            want += [i for i in table[b][: -(-lens[b] // S)] if 0 <= i < n_blocks]
    t_lens, t_free, t_n, status = i32(lens), i32(free), i32([n_free]), i32([0])
    lo, no = (None, None) if in_place else (torch.empty_like(t_lens), torch.empty_like(t_n))
    ops.pool_release(torch.tensor(done, device=DEV), t_lens, i32(table), t_free, t_n, S, lens_out=lo, n_free_out=no,
                     status=status)
    assert int(status) == ERR_RANGE
    assert (t_lens if in_place else lo).tolist() == [0 if d else n for d, n in zip(done, lens)]
    assert int(t_n if in_place else no) == len(want)
    assert t_free[: len(want)].tolist() == want


def test_failures_reach_the_pool_s_own_status():
    """A call without a status word of its own reports to the pool's."""
    k, v, _, _ = make_pool(7, 4, 16, 2, 64, BF, "hnd")
    pool = ops.KVPool(k, v)
    q = torch.randn(1, 8, 64, generator=gen(8), device=DEV).to(BF)
    ops.pool_decode(q, pool, i32([20]), i32([[0, 1]]))
    pool.check()
    ops.pool_decode(q, pool, i32([20]), i32([[0, 4]]))
    with pytest.raises(RuntimeError, match="range"):
        pool.check()
    pool.check()                                   # the report is given once
    rows = torch.zeros(1, 2, 64, dtype=BF, device=DEV)
    ops.pool_write(rows, rows, torch.tensor([64], device=DEV), pool)
    with pytest.raises(RuntimeError, match="range"):
        pool.check()
    status = i32([0])                              # a caller's own word: the pool's stays as it is
    ops.pool_write(rows, rows, torch.tensor([64], device=DEV), pool, status=status)
    assert int(status) == ERR_RANGE
    pool.check()
