"""GPU: the 8-bit layers at the ends of their ranges and in ways of use that
test_gpu_fp8.py leaves out.  Tolerances are that file's."""
import pytest
import torch

from test_gpu_fp8 import BF, DEV, check_linear, check_swiglu, make_weight, rows
from zoomkv_revision_b200 import ops

pytestmark = pytest.mark.gpu


def test_more_tiles_of_tokens_than_a_grid_holds():
    """65535 tiles of 128 tokens and a few more: rows of the first and the last tiles, zeros between."""
    T, k = 65535 * 128 + 300, 16
    ends = rows(1, 700, k, BF) * 0.1
    x = torch.zeros(T, k, dtype=BF, device=DEV)
    x[:200], x[-500:] = ends[:200], ends[200:]
    q, s = ops.quant_fp8(x)
    one, two = make_weight(1, 16, k), make_weight(2, 16, k, 2)
    out, (act, scale) = ops.fp8_linear(q, s, one), ops.fp8_swiglu(q, s, two)
    for part in (slice(0, 200), slice(T - 500, T)):
        check_linear(out[part], q[part], s[part], one)
        check_swiglu(act[part], scale[part], q[part], s[part], two)
    assert bool((out[200: -500] == 0).all()) and bool((scale[200: -500] == 0).all())
    one.check()
    two.check()


@pytest.mark.parametrize("own", [False, True])
def test_check_waits_for_every_stream(own):
    """What a product on another stream reports is seen, by a check on the default stream or on one of its own, and the word
    is zero for every stream once check has raised.  (The report is a copy to the status word behind a wait of some 50 ms:
    no product's wait runs out here.)"""
    w = make_weight(1, 128, 128)
    q, s = ops.quant_fp8(rows(1, 4, 128, BF))
    work, mine = torch.cuda.Stream(), torch.cuda.Stream() if own else torch.cuda.current_stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(work):
        torch.cuda._sleep(100_000_000)
        ops.fp8_linear(q, s, w)
        w.status.fill_(6)
    with torch.cuda.stream(mine):
        with pytest.raises(RuntimeError, match="status 6"):
            w.check()
    with torch.cuda.stream(work):
        seen = w.status.clone()
    w.check()
    assert int(seen.cpu()) == 0
