"""GPU: the 8-bit layers at the ends of their ranges and in ways of use that
test_gpu_fp8.py leaves out.  Tolerances are that file's."""
import pytest
import torch

from test_gpu_fp8 import BF, DEV, F8, FL, HF, blocks, check_linear, check_stored, check_swiglu, gen, make_weight, rows, spread, value
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


@pytest.mark.parametrize("T", [8, 12, 30, 50, 700])
@pytest.mark.parametrize("power", [-126, -90, 90, 110])
def test_swiglu_of_scales_far_from_one(T, power):
    """Blocks of the output whose scale is below 1e-20, subnormal ones among them, or above 1e20 (their quotients are lifted by
    a power of two).  The bound is that of test_swiglu_of_gates_far_below_zero; a subnormal scale has a step of 2^-149, at
    most 2^-22 of the scales here."""
    f = 1040
    xs = torch.linspace(1, 2, T, device=DEV)
    q, s, w, g, u = one_product(torch.cat([xs, -xs]), f, 1.0, 2.0 ** power, T)
    a = g * torch.sigmoid(g) * u
    out, scale = ops.fp8_swiglu(q, s, w)
    full = scale[:, :-1]
    assert bool(((full < 1e-20) | (full > 1e20)).all()) and bool((full > 2.0 ** -128).all())
    check_stored(out, scale, a, (2.5 * g.abs() + 10) * 2.0 ** -23 * a.abs(), 15 * 2.0 ** -23)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("n", [256, 528, 4112, 16400])
def test_norm_of_rows_that_are_not_finite(dtype, n):
    """An infinity: the sum of squares is one, so the row's other elements are zeros and the infinity's block reads back as NaN;
    a NaN makes the row NaN.  So too where the sum with the residual overflows.  Other rows are as without them."""
    big = torch.finfo(dtype).max
    x, res, w = rows(n, 9, n, dtype), rows(n + 1, 9, n, dtype), torch.ones(n, dtype=dtype, device=DEV)
    clean = ops.rmsnorm_fp8(x, w, 1e-6, residual=res.clone())
    x[1, n - 20], x[3, 5], res[4, 130], res[6, n // 2] = float("inf"), float("nan"), float("-inf"), float("nan")
    x[7, 200] = res[7, 200] = big
    q, s = ops.rmsnorm_fp8(x, w, 1e-6, residual=res)
    r = res.double()     # the kept sum
    assert bool(torch.isinf(r[7, 200])) and bool(torch.isnan(r[3, 5])) and bool(torch.isinf(r[1, n - 20]))
    y = r * torch.rsqrt((r * r).mean(-1, keepdim=True) + 1e-6)
    bad, got = torch.isnan(y), value(q, s)
    for i in (1, 3, 4, 6, 7):
        for b in range(blocks(n)):
            part = slice(128 * b, min(n, 128 * b + 128))
            if bool(bad[i, part].any()):
                assert bool(torch.isnan(got[i, part]).all()), (i, b)
            else:
                assert bool((got[i, part] == 0).all()), (i, b)
    for i in (0, 2, 5, 8):
        assert torch.equal(q[i].view(torch.uint8), clean[0][i].view(torch.uint8)) and torch.equal(s[i], clean[1][i])


PAIRS = [(2048, 4096, 1024, BF), (1500, 4001, 1040, FL), (1600, 4096, 1040, HF), (1500, 4001, 1040, BF)]


def test_pairs_of_several_products_at_once_and_in_a_graph():
    """Products that pairs of CTAs take (test_fp8_launch_cpu.py: test_the_pairs_sizes), with outputs of each type whose rows start
    on 16 bytes and ones whose rows do not: on streams at the same time, with small products between, and captured and replayed
    with other inputs.  Every result is, bit for bit, that of a call alone."""
    ins = [[ops.quant_fp8(rows(T + i, T, k, BF)) for T, _, k, _ in PAIRS] for i in range(2)]
    ws = [make_weight(n, n, k) for _, n, k, _ in PAIRS]
    few, wf = ops.quant_fp8(rows(1, 30, 1040, BF)), make_weight(1, 500, 1040)

    def buffers():
        return [torch.zeros(T, n + 3 * (i == 3), dtype=dtype, device=DEV)[:, 2 * (i == 3):][:, :n]
                for i, (T, n, _, dtype) in enumerate(PAIRS)]

    want = []
    for one in ins:
        outs = buffers()
        for (q, s), w, out in zip(one, ws, outs):
            ops.fp8_linear(q, s, w, out=out)
            check_linear(out, q, s, w)
        want.append(outs)
    small = ops.fp8_linear(*few, wf)
    torch.cuda.synchronize()
    streams, got, smalls = [torch.cuda.Stream() for _ in PAIRS], buffers(), []
    for _ in range(10):
        for i, (q, s) in enumerate(ins[0]):
            with torch.cuda.stream(streams[i]):
                ops.fp8_linear(q, s, ws[i], out=got[i])
                smalls.append(ops.fp8_linear(*few, wf))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want[0])) and all(torch.equal(x, small) for x in smalls)
    held = [(q.clone(), s.clone()) for q, s in ins[0]]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for (q, s), w, out in zip(held, ws, got):
            ops.fp8_linear(q, s, w, out=out)
            between = ops.fp8_linear(*few, wf)
    for i in (1, 0):
        for (q, s), (nq, ns) in zip(held, ins[i]):
            q.view(torch.uint8).copy_(nq.view(torch.uint8))
            s.copy_(ns)
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(got, want[i])) and torch.equal(between, small)
    for w in ws:
        w.check()
