"""CPU: workspace sizes of the pooled attention for a length that is not given."""
import ctypes

import pytest

from test_pool_cpu import CAPACITY, decode, pool
from zoomkv_revision_b200 import _lib


@pytest.mark.parametrize("batch,heads,window", [(1, 8, 0), (2, 8, 0), (64, 2, 0), (1, 8, 5000), (3, 66, 0), (900, 8, 300)])
def test_a_workspace_for_max_len_0_does_for_every_table(batch, heads, window):
    p = pool()
    size = lambda n: _lib.lib().zkv_pool_decode_ws_bytes(ctypes.addressof(p), batch, heads, window, n)  # noqa: E731
    most = size(0)
    assert most == size(2 ** 31 - 513) and (most > 0 or window)   # short windows need none
    for n in [1, 16, 256, 257, 1000, 4096, 10 ** 4, 10 ** 5, 10 ** 6, 10 ** 9, 2 ** 33] + [2 ** i + 1 for i in range(4, 31)]:
        assert size(n) <= most, n
    # what decode asks for with max_len 0 and a table of `width` columns is within it: a byte less than its own is refused
    for width in (10 ** 6, 2 ** 27 - 1, 2 ** 31 - 1):
        need = size(min(width * 16, 2 ** 31 - 513))
        assert need <= most
        assert not need or decode(p, batch=batch, heads=heads, window=window, width=width, ld=width, ws_bytes=need - 1) == CAPACITY
