"""GPU: KVPool.check and PoolCache.check see what calls on other streams
report.  (The report stands behind a wait of some 50 ms on its stream.)"""
import pytest
import torch

from zoomkv_revision_b200 import ops
from zoomkv_revision_b200.pool_cache import PoolCache

pytestmark = pytest.mark.gpu
DEV = "cuda"


def reported_late(owner, call, own):
    """`call` on a stream of its own, then owner.check() on another."""
    work, mine = torch.cuda.Stream(), torch.cuda.Stream() if own else torch.cuda.current_stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(work):
        torch.cuda._sleep(100_000_000)
        call()
    with torch.cuda.stream(mine):
        with pytest.raises(RuntimeError, match="range"):
            owner.check()
    with torch.cuda.stream(work):
        seen = owner.status.clone()
    owner.check()
    assert int(seen.cpu()) == 0


@pytest.mark.parametrize("own", [False, True])
def test_pool(own):
    k, v = (torch.zeros(4, 16, 2, 64, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    pool = ops.KVPool(k, v)
    rows, slots = torch.zeros(1, 2, 64, dtype=torch.bfloat16, device=DEV), torch.tensor([64], device=DEV)
    reported_late(pool, lambda: ops.pool_write(rows, rows, slots, pool), own)


@pytest.mark.parametrize("own", [False, True])
def test_cache(own):
    cache = PoolCache(1, 1, 2, 64, 32)
    rows, slots = torch.zeros(1, 2, 64, dtype=torch.bfloat16, device=DEV), torch.tensor([1 << 20], device=DEV)
    reported_late(cache, lambda: cache.write(0, rows, rows, slots), own)
