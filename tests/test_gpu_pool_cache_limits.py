"""GPU: the pooled cache at its bounds: prompts without a bound, replayed
plans, and a decode loop that runs out of room."""
import pytest
import torch

from zoomkv_revision_b200 import decode_loop as DL
from zoomkv_revision_b200.pool_cache import PoolCache

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF = torch.bfloat16
SMALL = DL.Shape(hidden=256, layers=2, heads=6, kv_heads=2, head_dim=128, ffn=512, vocab=1000)


def rows(seed, *shape):
    return torch.randn(shape, generator=torch.Generator(device=DEV).manual_seed(seed), device=DEV).to(BF)


def dense(q, kv):
    """q [heads, dim] over kv [tokens, dim] as K and V, one kv head."""
    x = kv.double()
    return torch.softmax(q.double() @ x.T * q.shape[-1] ** -0.5, -1) @ x


def near(got, want, kv):
    """Rounding of the output, and of probabilities and scores as 2^-10 of the largest value."""
    return bool(((got.double() - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -10 * kv.double().abs().max()).all())


def test_prompts_planned_without_a_bound_are_attended_whole():
    cache = PoolCache(1, 2, 1, 64, 640)
    n = [600, 17]
    kv = rows(1, sum(n), 1, 64)
    slots = cache.plan(torch.tensor(n, dtype=torch.int32, device=DEV), sum(n))
    assert cache.bound >= max(n)
    cache.write(0, kv, kv, slots)
    q = rows(2, 2, 4, 64)
    out = cache.attend(0, q)
    cache.check()
    for b, part in enumerate((kv[:600, 0], kv[600:, 0])):
        assert near(out[b], dense(q[b], part), part)
    cache.plan(None, 2)                                # one token each
    assert cache.lens.tolist() == [601, 18] and cache.bound >= 601


def test_a_replayed_plan_is_attended_whole():
    """A captured plan and write move the lengths at every replay, and the host's bound only once."""
    cache = PoolCache(1, 1, 1, 64, 512)
    kv = torch.zeros(1, 1, 64, dtype=BF, device=DEV)
    all_rows = rows(3, 200, 1, 64)
    cache.write(0, kv, kv, cache.plan(None, 1))
    cache.release(torch.tensor([True], device=DEV), bound=0)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cache.write(0, kv, kv, cache.plan(None, 1))
    for t in range(200):
        kv.copy_(all_rows[t: t + 1])
        graph.replay()
    assert cache.lens.tolist() == [200]
    q = rows(4, 1, 4, 64)
    out = cache.attend(0, q)
    cache.check()
    assert near(out[0], dense(q[0], all_rows[:, 0]), all_rows)


@pytest.mark.parametrize("n_blocks", [None, 8])
def test_a_decode_loop_that_runs_out_of_room_is_told(n_blocks):
    """3 requests of 20 tokens: 64 tokens fit the table, 32 tokens each fit 8 blocks (two each, then 6 + 3 > 8)."""
    B, prompt, s = 3, 20, SMALL
    w = DL.Weights(s, DEV, seed=1, std=0.05)
    cache = PoolCache(s.layers, B, s.kv_heads, s.head_dim, 64, n_blocks=n_blocks)
    loop = DL.DecodeLoop(s, w, cache, B, 200, DEV, use_graphs=False, temperature=0.0)
    tok = loop.prefill(torch.randint(0, s.vocab, (B, prompt), generator=torch.Generator().manual_seed(7)).to(DEV))
    room = 64 if n_blocks is None else 32
    for _ in range(room - prompt):
        tok = loop.step(tok)
    cache.check()
    with pytest.raises(RuntimeError, match="outside the cache"):
        loop.step(tok)
    assert cache.lens.tolist() == [room] * B           # nothing was appended
    cache.check()


def test_a_prompt_that_does_not_fit_is_refused():
    cache = PoolCache(1, 2, 1, 64, 64)
    x = rows(5, 2, 65, 1, 64)
    with pytest.raises(RuntimeError, match="outside the cache"):
        cache.prefill_update_kv_cache(None, x, x, 0, 0)
    assert cache.lens.tolist() == [0, 0]
    cache.prefill_update_kv_cache(None, x[:, :64], x[:, :64], 0, 0)
    cache.check()
    assert cache.lens.tolist() == [64, 64]


def test_released_places_serve_the_hooks_again():
    """A release that leaves the host without a bound: the hooks ask the GPU instead of refusing."""
    cache = PoolCache(1, 2, 1, 64, 64)
    x = rows(6, 2, 60, 1, 64)
    for _ in range(4):
        cache.prefill_update_kv_cache(None, x, x, 0, 0)
        cache.decode_update_kv_cache(x[:, :1], x[:, :1], 0)
        assert cache.lens.tolist() == [61, 61]
        cache.release(torch.tensor([True, True], device=DEV))
    cache.check()
    assert cache.lens.tolist() == [0, 0] and int(cache.n_free) == cache.n_blocks


def test_the_hooks_know_of_replayed_plans():
    """Replays fill the cache without the host: the next hook has to look, not to trust its bound."""
    cache = PoolCache(1, 1, 1, 64, 64)
    x = rows(7, 1, 1, 1, 64)
    cache.decode_update_kv_cache(x, x, 0)
    cache.release(torch.tensor([True], device=DEV), bound=0)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cache.decode_update_kv_cache(x, x, 0)
    for _ in range(63):
        graph.replay()
    cache.decode_update_kv_cache(x, x, 0)              # the last place
    assert cache.lens.tolist() == [64]
    with pytest.raises(RuntimeError, match="outside the cache"):
        cache.decode_update_kv_cache(x, x, 0)
    cache.check()
