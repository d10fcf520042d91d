"""GPU: rows and products in e4m3 with block scales (zkv_quant_fp8,
zkv_rmsnorm_fp8, zkv_fp8_linear, zkv_fp8_swiglu) against plain restatements:
quantised rows bit for bit, the others against 64-bit arithmetic.

Tolerances, from the arithmetic.  A stored element is off by half a step,
2^-4 of itself, or below the smallest normal number by half the smallest
step, 2^-10 of the scale: h(y, s) = 2^-4 |y| + 2^-10 s.
norm: the sum of squares is off by (elements of a thread + 21 additions)
2^-24, rsqrt halves that and adds 2^-22, two products and the scale's
quotient 2^-24 each: e = (64 + 21) 2^-25 + 2^-22 + 3 2^-24; |stored - y| <=
h + 2 e |y|, |scale - s| <= e s.
linear: a block's 128 products are summed in fp32, 2^-23 of the running sum
for each (whichever way the tensor core rounds), the two scales' product and
its use 2^-23, a block's addition 2^-24: off by at most z = (blocks + 130)
2^-23 sum |x w|, and half a unit of the output's type (2^-8 of the value for
bf16, 2^-11 fp16, 2^-24 fp32; fp16 below its normal numbers 2^-25).
swiglu: a = silu(g) u, |silu'| <= 1.1, so d = 1.1 z_g |u| + |silu(g)| z_u +
z_g z_u + (|g| + 16) 2^-23 |a| (the exponential's argument and the five
operations); |scale - s| <= max d / 448 + 2^-23 s; |stored - a| <= h + 2 d."""
import pytest
import torch

from zoomkv_revision_b200 import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, HF, FL, F8 = torch.bfloat16, torch.float16, torch.float32, torch.float8_e4m3fn
U = {BF: 2.0 ** -8, HF: 2.0 ** -11, FL: 2.0 ** -24}


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def blocks(n):
    return -(-n // 128)


def spread(s, n, dim=1):
    return s.repeat_interleave(128, dim).narrow(dim, 0, n)


def plain_quant(x):
    """On the CPU, in 32 bits: bytes and scales."""
    x = x.detach().cpu().float()
    T, n = x.shape
    pad = torch.zeros(T, blocks(n) * 128)
    pad[:, :n] = x
    pad = pad.view(T, -1, 128)
    scale = pad.abs().amax(-1) / torch.full((T, blocks(n)), 448.0)
    q = pad / scale[..., None]
    q = torch.where((scale == 0)[..., None], torch.zeros_like(q), q)
    return q.view(T, -1)[:, :n].to(F8).contiguous(), scale


def rows(seed, T, n, dtype=FL):
    g = gen(seed)
    x = torch.randn(T, n, generator=g, device=DEV) * torch.exp(torch.randn(T, 1, generator=g, device=DEV))
    x[:, n // 3] *= 30.0
    return x.to(dtype)


def value(q, s):
    return q.double() * spread(s.double(), q.shape[1])


def check_stored(q, s, y, d, e=0.0):
    """q, s against y [rows, n] in 64 bits, off by at most d before it is stored."""
    T, n = y.shape
    pad = torch.zeros(T, blocks(n) * 128, dtype=torch.float64, device=DEV)
    pad[:, :n] = y
    dp = torch.zeros_like(pad)
    dp[:, :n] = d
    want = pad.view(T, -1, 128).abs().amax(-1) / 448
    assert bool(((s.double() - want).abs() <= dp.view(T, -1, 128).amax(-1) / 448 + (2.0 ** -23 + e) * want).all())
    assert bool(((value(q, s) - y).abs() <= 2.0 ** -4 * y.abs() + 2.0 ** -10 * spread(s.double(), n) + 2 * d).all())


# ------------------------------------------------------------------ rows
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("T,n", [(1, 16), (1, 128), (3, 144), (7, 4096), (129, 272), (1000, 1040), (33, 12288)])
def test_quant_is_bit_exact(dtype, T, n):
    x = rows(T + n, T, n, dtype)
    x[T // 2] = 0
    if n > 128:
        x[T - 1, 128: 256] = 0
    q, s = ops.quant_fp8(x)
    pq, ps = plain_quant(x)
    assert q.dtype == F8 and q.shape == x.shape and s.shape == (T, blocks(n))
    assert torch.equal(s.cpu(), ps)
    assert torch.equal(q.cpu().view(torch.uint8), pq.view(torch.uint8))


def test_quant_of_all_16_bit_numbers():
    """Every finite bf16 and fp16 number, beside ones of its own size and far larger ones; ties and subnormal scales among them."""
    for dtype in (BF, HF):
        every = torch.arange(65536, device=DEV, dtype=torch.int32).to(torch.int16).view(dtype)
        every = every[torch.isfinite(every)]
        every = every[torch.argsort(every.abs().float(), stable=True)]
        every = torch.cat([every, every.new_zeros(-every.numel() % 2048)]).view(-1, 2048)
        mixed = every.t().contiguous().view(-1, 2048)
        for x in (every, mixed):
            q, s = ops.quant_fp8(x)
            pq, ps = plain_quant(x)
            assert torch.equal(s.cpu(), ps)
            assert torch.equal(q.cpu().view(torch.uint8), pq.view(torch.uint8))


def test_quant_blocks_that_are_not_finite_read_back_as_nan():
    x = rows(5, 4, 512, BF)
    x[0, 3], x[1, 200], x[2, 400] = float("inf"), float("-inf"), float("nan")
    q, s = ops.quant_fp8(x)
    got = value(q, s).view(4, 4, 128)
    bad = torch.zeros(4, 4, dtype=torch.bool, device=DEV)
    bad[0, 0] = bad[1, 1] = bad[2, 3] = True
    assert bool(torch.isnan(got[bad]).all()) and bool(torch.isfinite(got[~bad]).all())


def test_quant_strides():
    wide = rows(6, 40, 1024, BF)
    x = wide[:, 256: 768]
    buf = torch.full((40, 640), 7, dtype=torch.uint8, device=DEV)
    out, scale = buf.view(F8)[:, 64: 576], torch.full((40, 9), -1.0, device=DEV)[:, 2: 6]
    ops.quant_fp8(x, out=out, scale=scale)
    pq, ps = plain_quant(x)
    assert torch.equal(out.cpu().view(torch.uint8), pq.view(torch.uint8)) and torch.equal(scale.cpu(), ps)
    assert bool((buf[:, :64] == 7).all()) and bool((buf[:, 576:] == 7).all())
    # rows that do not start on 16 bytes, and other orders, are copied
    for y in (wide[:, 3: 515], wide[:, :512].t().contiguous().t(), wide.view(8, 5, 1024)[:, :, :512]):
        q, s = ops.quant_fp8(y)
        pq, ps = plain_quant(y.reshape(-1, 512))
        assert q.shape == y.shape and torch.equal(q.cpu().view(torch.uint8).view(-1, 512), pq.view(torch.uint8))
        assert torch.equal(s.cpu(), ps)


NORM_E = (64 + 21) * 2.0 ** -25 + 2.0 ** -22 + 3 * 2.0 ** -24


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("T,n", [(1, 16), (5, 128), (9, 512), (6, 528), (3, 1040), (7, 2064), (130, 4096), (4, 4112),
                                 (2, 8208), (3, 16400), (2, 32768)])
@pytest.mark.parametrize("residual", [False, True])
def test_norm(dtype, T, n, residual):
    x, w = rows(n, T, n, dtype), (1 + 0.3 * torch.randn(n, generator=gen(1), device=DEV)).to(dtype)
    x[T // 2] = 0
    res = rows(n + 1, T, n, dtype) if residual else None
    kept = None if res is None else res.clone()
    r = x if res is None else (x.float() + res.float()).to(dtype)
    q, s = ops.rmsnorm_fp8(x, w, 1e-6, residual=kept)
    if residual:
        assert torch.equal(kept.view(torch.int16), r.view(torch.int16))
    r64 = r.double()
    y = r64 * torch.rsqrt((r64 * r64).mean(-1, keepdim=True) + 1e-6) * w.double()
    check_stored(q, s, y, NORM_E * y.abs(), NORM_E)


def test_norm_residual_elsewhere_and_strided():
    x, res = rows(1, 33, 2048, BF)[:, 512: 1552], rows(2, 33, 1040, BF)
    keep, to, w = res.clone(), torch.empty(33, 1056, dtype=BF, device=DEV)[:, 16:], torch.ones(1040, dtype=BF, device=DEV)
    q, s = ops.rmsnorm_fp8(x, w, 1e-5, residual=res, residual_out=to)
    r = (x.float() + keep.float()).to(BF)
    assert torch.equal(res, keep) and torch.equal(to, r)
    q2, s2 = ops.rmsnorm_fp8(r, w, 1e-5)
    assert torch.equal(q.view(torch.uint8), q2.view(torch.uint8)) and torch.equal(s, s2)
    ops.rmsnorm_fp8(x, w, 1e-5, residual=keep, residual_out=x)   # over x itself
    assert torch.equal(x, r)


# ------------------------------------------------------------------ products
def make_weight(seed, n, k, parts=1, ld=None):
    g = gen(seed)
    ws, scales = [], []
    for _ in range(parts):
        w = torch.randn(n, k, generator=g, device=DEV) * 60.0
        w[n // 2, k // 2] = 448.0
        ws.append(w.clamp(-448, 448).to(F8))
        scales.append(torch.rand(blocks(n), blocks(k), generator=g, device=DEV) * 1e-3 + 1e-5)
    w = torch.cat([x.view(torch.uint8) for x in ws])
    if ld:
        wide = torch.full((parts * n, ld), 0x7f, dtype=torch.uint8, device=DEV)
        wide[:, :k] = w
        w = wide[:, :k]
    return ops.Fp8Weight(w.view(F8), torch.cat(scales), parts)


def product64(q, s, w, part=0):
    """(y, sum |x w|) of a product in 64 bits."""
    n, nb = w.rows, blocks(w.rows)
    x = value(q, s)
    scale = w.scale[part * nb: (part + 1) * nb].double()
    ww = w.w[part * n: (part + 1) * n].double() * spread(spread(scale, n, 0), w.k)
    return x @ ww.t(), x.abs() @ ww.abs().t()


def check_linear(out, q, s, w):
    y, size = product64(q, s, w)
    z = (blocks(w.k) + 130) * 2.0 ** -23 * size
    tiny = 2.0 ** -25 if out.dtype == HF else 0.0
    off = (out.double().view(y.shape) - y).abs()
    assert bool((off <= z + U[out.dtype] * (y.abs() + z) + tiny).all()), float((off / (z + U[out.dtype] * y.abs() + 1e-300)).max())


TOKENS = [1, 2, 15, 16, 17, 32, 33, 64, 65, 128, 129, 257, 300]


@pytest.mark.parametrize("T", TOKENS)
@pytest.mark.parametrize("n,k", [(128, 128), (200, 272), (1, 16), (384, 1040), (1000, 4096)])
def test_linear(T, n, k):
    q, s = ops.quant_fp8(rows(T, T, k, BF))
    w = make_weight(n + k, n, k)
    for dtype in (BF, HF, FL):
        check_linear(ops.fp8_linear(q, s, w, dtype=dtype), q, s, w)
    w.check()


@pytest.mark.parametrize("T,n,k", [(1, 6144, 4096), (8, 4096, 12288), (32, 19000, 512), (100, 130, 16384), (777, 1536, 2048),
                                   (1025, 640, 1296), (2048, 4096, 1024)])
def test_linear_larger(T, n, k):
    q, s = ops.quant_fp8(rows(T, T, k, BF))
    w = make_weight(7, n, k)
    check_linear(ops.fp8_linear(q, s, w, dtype=FL), q, s, w)
    w.check()


@pytest.mark.parametrize("T", [3, 40, 150, 600])
def test_linear_strides(T):
    n, k = 200, 400
    full, fs = ops.quant_fp8(rows(T, T, 1024, BF))
    q = full[:, 128: 528]
    for s in (fs[:, 1: 5], fs[:, 1: 5].contiguous(), fs[:1, 1: 2].expand(T, 4)):
        w = make_weight(3, n, k, ld=448)
        buf = torch.full((T, 232), 5.0, dtype=FL, device=DEV)
        ops.fp8_linear(q, s, w, out=buf[:, 16: 216])
        check_linear(buf[:, 16: 216], q, s, w)
        assert bool((buf[:, :16] == 5).all()) and bool((buf[:, 216:] == 5).all())
        odd = torch.full((T, 203), 5.0, dtype=BF, device=DEV)
        ops.fp8_linear(q, s, w, out=odd[:, 1: 201])
        check_linear(odd[:, 1: 201], q, s, w)
        assert bool((odd[:, :1] == 5).all()) and bool((odd[:, 201:] == 5).all())
    q3 = q.contiguous().view(1, T, k)
    out = ops.fp8_linear(q3, fs[:, 1: 5], w)
    assert out.shape == (1, T, n) and torch.equal(out[0], ops.fp8_linear(q, fs[:, 1: 5], w))


@pytest.mark.parametrize("T", [5, 100, 400])
def test_linear_rows_do_not_touch_one_another(T):
    """A row of NaN or of huge scales changes no other row, and each row is what it is alone in a call of that size."""
    q, s = ops.quant_fp8(rows(T, T, 512, BF))
    w = make_weight(1, 300, 512)
    out = ops.fp8_linear(q, s, w)
    q2, s2 = q.clone(), s.clone()
    q2.view(torch.uint8)[2] = 0x7f
    s2[3] = float("inf")
    got = ops.fp8_linear(q2, s2, w)
    keep = [i for i in range(T) if i not in (2, 3)]
    assert torch.equal(got[keep], out[keep]) and bool(torch.isnan(got[2]).all()) and not bool(torch.isfinite(got[3]).any())


def check_swiglu(q2, s2, q, s, w):
    (g, sg), (u, su) = product64(q, s, w, 0), product64(q, s, w, 1)
    c = (blocks(w.k) + 130) * 2.0 ** -23
    silu = g * torch.sigmoid(g)
    a = silu * u
    d = 1.1 * c * sg * u.abs() + silu.abs() * c * su + c * c * sg * su + (g.abs() + 16) * 2.0 ** -23 * a.abs()
    check_stored(q2, s2, a, d)


@pytest.mark.parametrize("T", TOKENS)
@pytest.mark.parametrize("f,k", [(128, 128), (208, 272), (16, 16), (512, 1040), (1008, 2048)])
def test_swiglu(T, f, k):
    q, s = ops.quant_fp8(rows(T, T, k, BF) * 0.1)
    w = make_weight(f + k, f, k, 2)
    check_swiglu(*ops.fp8_swiglu(q, s, w), q, s, w)
    w.check()


@pytest.mark.parametrize("T,f,k", [(1, 12288, 4096), (8, 4096, 4096), (100, 2048, 4096), (777, 1536, 2048), (1025, 640, 1296)])
def test_swiglu_larger(T, f, k):
    q, s = ops.quant_fp8(rows(T, T, k, BF) * 0.05)
    w = make_weight(9, f, k, 2)
    check_swiglu(*ops.fp8_swiglu(q, s, w), q, s, w)
    w.check()


def test_swiglu_extremes():
    """Gates far below zero give zeros, not NaN; a token of zeros has scales of 0; strided outputs."""
    T, f, k = 20, 208, 256
    q, s = ops.quant_fp8(rows(2, T, k, BF) * 40.0)
    s[4] = 0
    w = make_weight(4, f, k, 2)
    buf = torch.full((T, 256), 9, dtype=torch.uint8, device=DEV)
    out, scale = buf.view(F8)[:, 32: 240], torch.full((T, 5), -1.0, device=DEV)[:, 1: 3]
    ops.fp8_swiglu(q, s, w, out=out, scale=scale)
    check_swiglu(out, scale, q, s, w)
    assert bool((scale[4] == 0).all()) and bool((buf[4, 32: 240] == 0).all())
    assert bool((buf[:, :32] == 9).all()) and bool((buf[:, 240:] == 9).all())


def test_empty_batches():
    x = torch.empty(0, 256, dtype=BF, device=DEV)
    w = torch.ones(256, dtype=BF, device=DEV)
    q, s = ops.quant_fp8(x)
    q2, s2 = ops.rmsnorm_fp8(x, w, 1e-6, residual=x.clone())
    assert q.shape == q2.shape == (0, 256) and s.shape == s2.shape == (0, 2)
    assert ops.fp8_linear(q, s, make_weight(1, 130, 256)).shape == (0, 130)
    q3, s3 = ops.fp8_swiglu(q, s, make_weight(1, 144, 256, 2))
    assert q3.shape == (0, 144) and s3.shape == (0, 2)


def test_quantize_weights():
    w16 = (torch.randn(2 * 208, 272, generator=gen(1), device=DEV) * 0.02).to(BF)
    w16[128: 208, :128] = 0      # a block of zeros (and of the second part, none)
    w = ops.Fp8Weight.quantize(w16, 2)
    back = w.dequantize()
    s = torch.cat([spread(spread(w.scale[p * 2: p * 2 + 2], 208, 0), 272) for p in range(2)])
    assert bool(((back - w16.float()).abs() <= 2.0 ** -4 * w16.float().abs() + 2.0 ** -10 * s).all())
    assert bool((back[128: 208, :128] == 0).all())
    for p in range(2):
        for i in range(2):
            for j in range(3):
                part = w16[p * 208: (p + 1) * 208][i * 128: (i + 1) * 128, j * 128: (j + 1) * 128].float()
                assert float(w.scale[p * 2 + i, j]) == float(part.abs().max().cpu() / torch.tensor(448.0))


# ------------------------------------------------------------------ refusals
def test_refusals():
    x = torch.randn(4, 256, device=DEV).to(BF)
    w = torch.ones(256, dtype=BF, device=DEV)
    q, s = ops.quant_fp8(x)
    one, two = make_weight(1, 144, 256), make_weight(1, 144, 256, 2)
    bad = [
        (ValueError, lambda: ops.quant_fp8(x[:, :250])),
        (ValueError, lambda: ops.quant_fp8(x.cpu())),
        (TypeError, lambda: ops.quant_fp8(x.float())),
        (TypeError, lambda: ops.quant_fp8(x, out=torch.empty_like(x))),
        (ValueError, lambda: ops.quant_fp8(x, out=q[:3])),
        (ValueError, lambda: ops.quant_fp8(x, out=torch.empty(4, 257, device=DEV).to(F8)[:, 1:])),
        (TypeError, lambda: ops.quant_fp8(x, scale=s.half())),
        (ValueError, lambda: ops.quant_fp8(x, scale=s[:, :1])),
        (ValueError, lambda: ops.quant_fp8(x, scale=s[:1].expand(4, 2))),
        (TypeError, lambda: ops.rmsnorm_fp8(x, w.half(), 1e-6)),
        (ValueError, lambda: ops.rmsnorm_fp8(x, w[:128], 1e-6)),
        (TypeError, lambda: ops.rmsnorm_fp8(x, w, 1e-6, residual=x.half())),
        (ValueError, lambda: ops.rmsnorm_fp8(x, w, 1e-6, residual=x[:2])),
        (ValueError, lambda: ops.rmsnorm_fp8(x, w, 1e-6, residual_out=x)),
        (ValueError, lambda: ops.rmsnorm_fp8(x, w, 1e-6, residual=x[:1].expand(4, 256))),
        (RuntimeError, lambda: ops.rmsnorm_fp8(x, w, -1.0)),
        (RuntimeError, lambda: ops.rmsnorm_fp8(torch.ones(1, 32784, device=DEV).to(BF), torch.ones(32784, device=DEV).to(BF), 1e-6)),
        (TypeError, lambda: ops.Fp8Weight(x, s)),
        (ValueError, lambda: ops.Fp8Weight(q, s)),
        (ValueError, lambda: ops.Fp8Weight(one.w, one.scale, 3)),
        (ValueError, lambda: ops.Fp8Weight(one.w, one.scale, 2)),
        (ValueError, lambda: ops.Fp8Weight(one.w[:, :250], one.scale)),
        (ValueError, lambda: ops.Fp8Weight(one.w.t(), one.scale.t().contiguous())),
        (TypeError, lambda: ops.fp8_linear(x, s, one)),
        (ValueError, lambda: ops.fp8_linear(q, s, two)),
        (ValueError, lambda: ops.fp8_swiglu(q, s, one)),
        (ValueError, lambda: ops.fp8_linear(q[:, :128], s[:, :1], one)),
        (ValueError, lambda: ops.fp8_linear(q, s[:, :1], one)),
        (TypeError, lambda: ops.fp8_linear(q, s.half(), one)),
        (TypeError, lambda: ops.fp8_linear(q, s, one, dtype=F8)),
        (ValueError, lambda: ops.fp8_linear(q, s, one, out=x)),
        (TypeError, lambda: ops.fp8_swiglu(q, s, two, out=torch.empty(4, 144, dtype=BF, device=DEV))),
        (ValueError, lambda: ops.fp8_swiglu(q, s, two, scale=s[:, :1])),
    ]
    for i, (kind, call) in enumerate(bad):
        with pytest.raises(kind):
            call()
            pytest.fail(f"call {i} was not refused")
    check_linear(ops.fp8_linear(q, s, one), q, s, one)   # and the next call is as ever


# ------------------------------------------------------------------ as they are used
def layer(x, attn, p):
    """One layer's dense half, as the decode loop runs it; x is updated."""
    q, s = ops.quant_fp8(attn)
    proj = ops.fp8_linear(q, s, p["wo"])
    q, s = ops.rmsnorm_fp8(proj, p["norm"], 1e-6, residual=x)
    q, s = ops.fp8_swiglu(q, s, p["gate_up"])
    return ops.fp8_linear(q, s, p["down"])


def layer_parts():
    return dict(wo=make_weight(1, 512, 256), norm=(1 + 0.1 * torch.randn(512, generator=gen(2), device=DEV)).to(BF),
                gate_up=make_weight(3, 400, 512, 2), down=make_weight(4, 512, 400))


@pytest.mark.parametrize("T", [1, 8, 70, 300])
def test_chain_streams_and_graphs(T):
    """A layer's calls one after another: on another stream, in a captured graph replayed with new inputs, twice at once on
    two streams, all bit for bit the same."""
    p = layer_parts()
    xs, attns = [rows(10 + i, T, 512, BF) * 0.3 for i in range(2)], [rows(20 + i, T, 256, BF) * 0.1 for i in range(2)]
    want = []
    for i in range(2):
        x = xs[i].clone()
        want.append((layer(x, attns[i], p), x))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for i in range(2):
        with torch.cuda.stream(streams[i]):
            x = xs[i].clone()
            got.append((layer(x, attns[i], p), x))
            for _ in range(20):
                layer(xs[i].clone(), attns[i], p)
    torch.cuda.synchronize()
    for a, b in zip(want, got):
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    x, attn = xs[0].clone(), attns[0].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = layer(x, attn, p)
    for i in (1, 0):
        x.copy_(xs[i])
        attn.copy_(attns[i])
        graph.replay()
        assert torch.equal(y, want[i][0]) and torch.equal(x, want[i][1])
    for w in ("wo", "gate_up", "down"):
        p[w].check()


def test_chain_against_64_bits():
    """The chain with each stage's stored values as the next one's inputs."""
    T, p = 33, layer_parts()
    x, attn = rows(1, T, 512, BF) * 0.3, rows(2, T, 256, BF) * 0.1
    q, s = ops.quant_fp8(attn)
    proj = ops.fp8_linear(q, s, p["wo"])
    check_linear(proj, q, s, p["wo"])
    r = (x.float() + proj.float()).to(BF)
    q, s = ops.rmsnorm_fp8(proj, p["norm"], 1e-6, residual=x)
    assert torch.equal(x, r)
    y = r.double() * torch.rsqrt((r.double() ** 2).mean(-1, keepdim=True) + 1e-6) * p["norm"].double()
    check_stored(q, s, y, NORM_E * y.abs(), NORM_E)
    q2, s2 = ops.fp8_swiglu(q, s, p["gate_up"])
    check_swiglu(q2, s2, q, s, p["gate_up"])
    check_linear(ops.fp8_linear(q2, s2, p["down"]), q2, s2, p["down"])


def test_products_of_all_kinds_at_once():
    """Clusters, single CTAs and pairs on three streams, over and over: every result as when it runs alone."""
    p = layer_parts()
    sizes = (5, 40, 100, 700)
    ins = [ops.quant_fp8(rows(T, T, 512, BF)) for T in sizes]
    wide = make_weight(5, 2000, 512)
    want = [(ops.fp8_linear(q, s, wide), *ops.fp8_swiglu(q, s, p["gate_up"])) for q, s in ins]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sizes]
    got = [None] * len(sizes)
    for _ in range(30):
        for i, (q, s) in enumerate(ins):
            with torch.cuda.stream(streams[i]):
                got[i] = (ops.fp8_linear(q, s, wide), *ops.fp8_swiglu(q, s, p["gate_up"]))
    torch.cuda.synchronize()
    for a, b in zip(want, got):
        assert torch.equal(a[0], b[0]) and torch.equal(a[1].view(torch.uint8), b[1].view(torch.uint8)) and torch.equal(a[2], b[2])
    wide.check()
    p["gate_up"].check()


def test_weights_written_just_before_they_are_read():
    """The products ask for their first weights early; what a call before them wrote is what they multiply."""
    q, s = ops.quant_fp8(rows(1, 8, 2048, BF))
    a, b = make_weight(1, 3000, 2048), make_weight(2, 3000, 2048)
    w = ops.Fp8Weight(a.w.clone(), a.scale.clone())
    want = [ops.fp8_linear(q, s, x) for x in (a, b)]
    for i in range(40):
        src = (a, b)[i % 2]
        w.w.view(torch.uint8).copy_(src.w.view(torch.uint8))
        w.scale.copy_(src.scale)
        ops.quant_fp8(rows(1, 8, 2048, BF))   # a launch between them that lets the next begin early
        assert torch.equal(ops.fp8_linear(q, s, w), want[i % 2]), i


def test_offsets_past_32_bits():
    """Rows whose first element is past 2^31 elements, of inputs and outputs."""
    T, n = 540000, 4096
    x = torch.zeros(T, n, dtype=BF, device=DEV)
    tail = rows(1, 300, n, BF)
    x[-300:] = tail
    q, s = ops.quant_fp8(x)
    pq, ps = plain_quant(tail)
    assert torch.equal(q[-300:].cpu().view(torch.uint8), pq.view(torch.uint8)) and torch.equal(s[-300:].cpu(), ps)
    assert bool((s[:-300] == 0).all())
    w = torch.ones(n, dtype=BF, device=DEV)
    q2, s2 = ops.rmsnorm_fp8(x, w, 1e-6, residual=x)
    r64 = (tail.float() * 2).to(BF).double()
    y = r64 * torch.rsqrt((r64 * r64).mean(-1, keepdim=True) + 1e-6)
    check_stored(q2[-300:], s2[-300:], y, NORM_E * y.abs(), NORM_E)
    assert torch.equal(x[-300:].double(), r64)
    del x, q2, s2
    wt = make_weight(1, 4200, n)
    out = ops.fp8_linear(q, s, wt)
    check_linear(out[-300:], q[-300:], s[-300:], wt)
    assert bool((out[:1000] == 0).all())
    wt.check()


def test_first_call_of_a_kernel_may_be_captured():
    """In a process of its own: nothing has been launched before the capture."""
    import subprocess
    import sys
    code = ("import torch\nfrom zoomkv_revision_b200 import ops\n"
            "q = torch.zeros(90, 256, device='cuda').to(torch.float8_e4m3fn); s = torch.ones(90, 2, device='cuda')\n"
            "w = ops.Fp8Weight(torch.ones(300, 256, device='cuda').to(torch.float8_e4m3fn), torch.ones(3, 2, device='cuda'))\n"
            "q.view(torch.uint8).fill_(0x38)\ng = torch.cuda.CUDAGraph()\ntorch.cuda.synchronize()\n"
            "with torch.cuda.graph(g):\n    a = ops.fp8_linear(q, s, w); b = ops.fp8_linear(q[:7], s[:7], w)\n"
            "g.replay(); torch.cuda.synchronize()\n"
            "assert bool((a == 256).all()) and bool((b == 256).all())\nprint('captured')\n")
    got = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=120)
    assert got.returncode == 0 and "captured" in got.stdout, got.stderr[-2000:]


# ------------------------------------------------------------------ long prompts (pairs of CTAs)
@pytest.mark.parametrize("T", [1500, 2049])
@pytest.mark.parametrize("dtype", [BF, HF, FL])
def test_linear_long(T, dtype):
    """A last tile of tokens and of features that is not full, a last block of the inner dimension of 16; rows of the output
    that start on 16 bytes and rows that do not; scales in any order."""
    n, k = 4001, 1040
    q, s = ops.quant_fp8(rows(T, T, k, BF))
    w = make_weight(n, n, k, ld=1088)
    check_linear(ops.fp8_linear(q, s, w, dtype=dtype), q, s, w)
    buf = torch.full((T, 4016), 5.0, dtype=dtype, device=DEV)
    ops.fp8_linear(q, s.contiguous(), w, out=buf[:, :n])
    check_linear(buf[:, :n], q, s, w)
    assert bool((buf[:, n:] == 5).all())
    one = s[:1].expand(T, blocks(k))
    check_linear(ops.fp8_linear(q, one, w, out=buf[:, :n]), q, one, w)
    w.check()


@pytest.mark.parametrize("T,f,k", [(1500, 4000, 1040), (2049, 4112, 256), (700, 12288, 512)])
def test_swiglu_long(T, f, k):
    q, s = ops.quant_fp8(rows(T, T, k, BF) * 0.05)
    w = make_weight(f, f, k, 2)
    out, scale = torch.full((T, f + 32), 9, dtype=torch.uint8, device=DEV), torch.full((T, blocks(f) + 1), -1.0, device=DEV)
    ops.fp8_swiglu(q, s, w, out=out.view(F8)[:, 16: 16 + f], scale=scale[:, :-1])
    check_swiglu(out.view(F8)[:, 16: 16 + f], scale[:, :-1], q, s, w)
    assert bool((out[:, :16] == 9).all()) and bool((out[:, 16 + f:] == 9).all()) and bool((scale[:, -1] == -1).all())
    w.check()


def test_long_rows_do_not_touch_one_another():
    T = 1500
    q, s = ops.quant_fp8(rows(T, T, 512, BF) * 0.1)
    w, w2 = make_weight(1, 4001, 512), make_weight(2, 4000, 512, 2)
    out, gated = ops.fp8_linear(q, s, w), ops.fp8_swiglu(q, s, w2)
    q2, s2 = q.clone(), s.clone()
    q2.view(torch.uint8)[200] = 0x7f
    s2[1301] = float("inf")
    got, g2 = ops.fp8_linear(q2, s2, w), ops.fp8_swiglu(q2, s2, w2)
    keep = torch.ones(T, dtype=torch.bool, device=DEV)
    keep[200] = keep[1301] = False
    assert torch.equal(got[keep], out[keep]) and torch.equal(g2[0].view(torch.uint8)[keep], gated[0].view(torch.uint8)[keep])
    assert torch.equal(g2[1][keep], gated[1][keep])
    assert bool(torch.isnan(got[200]).all()) and not bool(torch.isfinite(got[1301]).any())
    assert bool(torch.isnan(value(*g2)[~keep]).all())


def test_long_chain_in_a_graph():
    """Prompts of 1500 tokens through a layer, captured and replayed, on another stream too."""
    T, p = 1500, layer_parts()
    x, attn = rows(1, T, 512, BF) * 0.3, rows(2, T, 256, BF) * 0.1
    start = x.clone()
    want = layer(x, attn, p)
    kept = x.clone()
    x.copy_(start)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = layer(x, attn, p)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(5):
            x.copy_(start)
            graph.replay()
    side.synchronize()
    assert torch.equal(y, want) and torch.equal(x, kept)
