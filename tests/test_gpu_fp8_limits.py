"""GPU: the 8-bit layers at the ends of their ranges and in ways of use that
test_gpu_fp8.py leaves out.  Tolerances are that file's."""
import pytest
import torch

from test_gpu_fp8 import BF, DEV, F8, blocks, check_linear, check_stored, check_swiglu, gen, make_weight, rows, spread, value
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


def one_product(xs, f, gate_scale, up_scale, seed):
    """Rows of a single element 1 with the scales xs, and weights whose gate is -gate_scale for every feature and whose up part
    has random codes times up_scale: (q, s, weight, g [tokens, 1], u [tokens, f]), g and u in 64 bits."""
    T, k = xs.numel(), 16
    q = torch.zeros(T, k, device=DEV)
    q[:, 3] = 1
    w = torch.zeros(2 * f, k, device=DEV)
    w[:f, 3] = -448
    w[f:, 3] = torch.randint(-448, 449, (f,), generator=gen(seed), device=DEV)
    w = w.to(F8)
    scale = torch.empty(2 * blocks(f), 1, device=DEV)
    scale[:blocks(f)], scale[blocks(f):] = gate_scale / 448, up_scale
    s = xs[:, None].contiguous()
    u = s.double() * spread(scale[blocks(f):].double(), f, 0)[:, 0] * w[f:, 3].double()
    return q.to(F8), s, ops.Fp8Weight(w, scale, 2), -448 * s.double() * scale[0].double(), u


@pytest.mark.parametrize("T", [8, 40, 100, 700])
def test_swiglu_of_gates_far_below_zero(T):
    """silu(g) u where exp(-g) is past fp32's range or near its end (g < -87) and u is large: as good as elsewhere.  Here g and u
    are one product each, off by three roundings, 1.5 2^-23 of themselves, which the exponential makes (|g| + 1) 1.5 2^-23 of
    the result; exp(g / 2), twice over, is off by |g| 2^-24 for its argument's roundings and 2^-22 of its own, the reciprocal
    by 2^-23 and five operations by 2^-24 each: d = (2.5 |g| + 10) 2^-23 of the result."""
    f = 1040
    xs = torch.linspace(60, 140, T, device=DEV)
    q, s, w, g, u = one_product(xs, f, 1.0, 2.0 ** 100, T)
    a = g * torch.sigmoid(g) * u
    assert bool((a.abs().amax(-1) > 1e-30).all())
    check_stored(*ops.fp8_swiglu(q, s, w), a, (2.5 * g.abs() + 10) * 2.0 ** -23 * a.abs(), (2.5 * 140 + 10) * 2.0 ** -23)
    # and between, where it matters to every model: small gates of both signs
    q, s, w, g, u = one_product(torch.cat([xs / 100, -xs / 100]), f, 1.0, 1.0, T)
    a = g * torch.sigmoid(g) * u
    check_stored(*ops.fp8_swiglu(q, s, w), a, (2.5 * g.abs() + 10) * 2.0 ** -23 * a.abs(), (2.5 * 2 + 10) * 2.0 ** -23)
