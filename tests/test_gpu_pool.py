"""GPU: the pooled KV cache (zkv_pool_plan, zkv_pool_write, zkv_pool_decode,
zkv_pool_release) against plain restatements: whole numbers and stored rows
bit for bit, attention against 64-bit arithmetic.

Tolerance of an attention output, from the arithmetic: the result is rounded
once to its type (u_out |o|, u_out = 2^-8 bf16, 2^-11 fp16: the half unit,
doubled for what is rounded being off itself), a probability carries at most
2^-11 of relative rounding, and a score is a sum of D products in fp32, off by
at most e = (D + 2) 2^-23 max_t sum_d |scale q_d k_td| + 2^-20, which moves
every probability by 2 e at most.  So |out - o| <= u_out |o| +
(2 e + 2^-11) sum_t p_t |v_t|, and |lse - l| <= e + 2^-20 + 2^-22 |l|; a soft
cap adds its tanh's rounding, softcap 2^-21, to e."""
import math

import pytest
import torch

from zoomkv_revision_b200 import _lib, ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, HF, F8 = torch.bfloat16, torch.float16, torch.float8_e4m3fn
ERR_CAPACITY, ERR_RANGE = 3, 7


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


# ------------------------------------------------------------------ attention
def make_pool(seed, n_blocks, S, H, D, dtype, layout, junk=None):
    g = gen(seed)
    made, scales = [], []
    for which in range(2):
        x = torch.randn((n_blocks, H, S, D) if layout == "hnd" else (n_blocks, S, H, D), generator=g, device=DEV)
        if which == 0:
            x[..., 1:3] *= 8.0
        scale = None
        if dtype == F8:
            scale = torch.rand(H, generator=g, device=DEV) * 0.05 + 0.02
            x = (x / (scale.view(1, H, 1, 1) if layout == "hnd" else scale.view(1, 1, H, 1))).clamp(-448, 448)
        x = x.to(dtype)
        made.append(x.transpose(1, 2) if layout == "hnd" else x)
        scales.append(scale)
    return made[0], made[1], scales[0], scales[1]


def make_table(seed, lens, S, n_blocks, width):
    g = gen(seed)
    perm = torch.randperm(n_blocks, generator=g, device=DEV).int()
    table = torch.full((len(lens), width), -1, dtype=torch.int32, device=DEV)
    at = 0
    for b, n in enumerate(lens):
        c = (n + S - 1) // S
        table[b, :c] = perm[at: at + c]
        at += c
    return table


def spoil(pool_k, pool_v, table, lens, S, lo=None):
    """NaN and infinities in every row of the pool that no request may see."""
    seen = torch.zeros(pool_k.shape[0], S, dtype=torch.bool, device=DEV)
    for b, n in enumerate(lens):
        first = 0 if lo is None else lo[b]
        t = torch.arange(first, n, device=DEV)
        seen[table[b].long()[t // S], t % S] = True
    for x in (pool_k, pool_v):
        if x.dtype == F8:
            x.view(torch.uint8)[~seen] = 0x7f
        else:
            x[~seen] = math.nan
            odd = ~seen
            odd[::2] = False
            x[odd] = -math.inf


def rows64(pool, ids, scale):
    x = pool.view(torch.uint8)[ids].view(pool.dtype) if pool.dtype == F8 else pool[ids]
    x = x.double().reshape(-1, pool.shape[2], pool.shape[3])
    return x if scale is None else x * scale.double().view(1, -1, 1)


def check_decode(q, k, v, ks, vs, lens, table, out, lse, scale, window=0, softcap=0.0):
    B, Hq, D = q.shape
    S, H = k.shape[1], k.shape[2]
    G = Hq // H
    u_out = 2.0 ** -8 if q.dtype == BF else 2.0 ** -11
    assert out.dtype == q.dtype
    for b, n in enumerate(lens):
        lo = max(0, n - window) if window else 0
        if n == 0:
            assert torch.equal(out[b], torch.zeros_like(out[b]))
            assert bool((lse[b] == -math.inf).all())
            continue
        ids = table[b, lo // S: (n + S - 1) // S].long()
        cut = slice(lo - lo // S * S, n - lo // S * S)
        kk, vv = rows64(k, ids, ks)[cut].permute(1, 2, 0), rows64(v, ids, vs)[cut].transpose(0, 1)
        qq = q[b].double().view(H, G, D)
        x = torch.matmul(qq, kk) * scale
        size = torch.matmul(qq.abs(), kk.abs()).amax(-1, keepdim=True) * abs(scale)
        if softcap:
            x = softcap * torch.tanh(x / softcap)
        ref_l = torch.logsumexp(x, -1, keepdim=True)
        p = torch.exp(x - ref_l)
        ref = torch.matmul(p, vv)
        e = (D + 2) * 2.0 ** -23 * size + 2.0 ** -20 + softcap * 2.0 ** -21
        tol = u_out * ref.abs() + (2 * e + 2.0 ** -11) * torch.matmul(p, vv.abs())
        err = (out[b].double().view(H, G, D) - ref).abs()
        assert bool((err <= tol).all()), f"request {b} of {n} tokens: {float((err / tol).max()):.2f} of the tolerance"
        le = (lse[b].double().view(H, G, 1) - ref_l).abs()
        lt = e + 2.0 ** -20 + 2.0 ** -22 * ref_l.abs()
        assert bool((le <= lt).all()), f"lse of request {b}: {float((le / lt).max()):.2f} of the tolerance"


def run_decode(seed, lens, S, H, G, D, qt, pt, layout, window=0, softcap=0.0, scale=None, max_len=0, spare=3, wide=None,
               **kw):
    """wide: a table of so many more columns that the bound of the lengths lets the rows be cut by units (None: both ways)."""
    if wide is None:
        run_decode(seed, lens, S, H, G, D, qt, pt, layout, window, softcap, scale, max_len, spare, True, **kw)
    need = sum((n + S - 1) // S for n in lens)
    n_blocks = need + spare
    width = max(1, max((n + S - 1) // S for n in lens)) + 1
    if wide and not 0 < window < 10000:
        width += (160 << 20) // (2 * len(lens) * H * D * S * (1 if pt == F8 else 2))
    k, v, ks, vs = make_pool(seed, n_blocks, S, H, D, pt, layout)
    table = make_table(seed + 1, lens, S, n_blocks, width)
    lo = [max(0, n - window) if window else 0 for n in lens]
    spoil(k, v, table, lens, S, lo)
    B = len(lens)
    q = torch.randn(B, H * G, D, generator=gen(seed + 2), device=DEV).to(qt)
    scale = D ** -0.5 if scale is None else scale
    status = i32([0])
    out, lse = ops.pool_decode(q, ops.KVPool(k, v, ks, vs), i32(lens), table, scale=scale, window=window, softcap=softcap,
                               max_len=max_len, return_lse=True, status=status, **kw)
    torch.cuda.synchronize()
    assert int(status) == 0
    check_decode(q, k, v, ks, vs, lens, table, out, lse, scale, window, softcap)
    return out, lse


EDGES = [0, 1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 100, 127, 128, 129, 255, 257]


@pytest.mark.parametrize("layout", ["hnd", "nhd"])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("qt,pt", [(BF, BF), (HF, HF), (BF, F8), (HF, F8)])
def test_decode_types_and_edges(qt, pt, D, layout):
    run_decode(1, EDGES, 16, 2, 4, D, qt, pt, layout)


@pytest.mark.parametrize("G", [1, 2, 3, 5, 7, 8, 9, 12, 15, 16, 17, 24, 33])
def test_decode_head_groups(G):
    run_decode(20 + G, [70, 0, 1, 333], 16, 2, G, 128, BF, BF, "hnd")
    run_decode(60 + G, [40, 513], 32, 1, G, 64, HF, F8, "nhd")
    run_decode(90 + G, [40, 213], 16, 1, G, 256, BF, BF, "nhd")


@pytest.mark.parametrize("S", [16, 32, 64, 128, 256, 1024])
@pytest.mark.parametrize("pt", [BF, F8])
def test_decode_block_sizes(S, pt):
    run_decode(200 + S, [S - 1, S, S + 1, 3 * S + 5, 1], S, 3, 4, 128, BF, pt, "hnd")
    run_decode(300 + S, [S - 1, S, S + 1, 2 * S + 9, 0], S, 1, 2, 64, BF, pt, "nhd")


@pytest.mark.parametrize("window", [1, 2, 16, 63, 64, 65, 100, 5000])
def test_decode_window(window):
    run_decode(400 + window, [0, 1, 64, 65, 100, 128, 1000, 1023, 2049], 16, 2, 4, 128, BF, BF, "hnd", window=window)
    run_decode(500 + window, [7, 300, 999], 64, 2, 3, 128, HF, F8, "nhd", window=window)


@pytest.mark.parametrize("softcap", [0.5, 30.0])
def test_decode_softcap_and_scale(softcap):
    run_decode(600, [5, 64, 700], 16, 2, 4, 128, BF, BF, "hnd", softcap=softcap, scale=0.3)
    run_decode(601, [5, 64, 700], 16, 2, 4, 128, BF, F8, "hnd", softcap=softcap, scale=0.3)
    run_decode(602, [5, 64, 700], 16, 2, 4, 128, BF, BF, "hnd", scale=0.0)
    run_decode(603, [5, 64, 700], 16, 2, 4, 128, HF, HF, "hnd", scale=-0.1)


@pytest.mark.parametrize("pt", [BF, F8])
def test_decode_wide_softcap(pt):
    """A cap far above the scores leaves them: c tanh(x / c) is off by x^3 / 3 c^2, under 2^-20 for |x| < 16 and c = 1e5,
    so the tolerance is the one without a cap."""
    lens, S, H, G, D = [1, 64, 700], 16, 2, 4, 128
    k, v, ks, vs = make_pool(610, 60, S, H, D, pt, "hnd")
    table = make_table(611, lens, S, 60, 44)
    q = torch.randn(3, H * G, D, generator=gen(612), device=DEV).to(BF)
    out, lse = ops.pool_decode(q, ops.KVPool(k, v, ks, vs), i32(lens), table, scale=0.03, softcap=1e5, return_lse=True)
    check_decode(q, k, v, ks, vs, lens, table, out, lse, 0.03)


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("qt,pt", [(BF, BF), (HF, HF), (BF, F8), (HF, F8)])
def test_decode_few_rows(qt, pt, D):
    """One to three rows: every CTA of the largest cluster has a part, or some have none."""
    run_decode(650, [2100], 16, 1, 4, D, qt, pt, "hnd", wide=False)
    run_decode(651, [1025, 7, 0], 32, 1, 12, D, qt, pt, "nhd", wide=False)
    run_decode(652, [513], 64, 1, 33, D, qt, pt, "hnd", window=500, wide=False)
    run_decode(653, [3000, 2999], 128, 1, 1, D, qt, pt, "nhd", wide=False)


def test_decode_long_and_uneven():
    run_decode(700, [40001], 16, 2, 4, 128, BF, BF, "hnd")
    run_decode(701, [1, 20000, 3, 0, 9999, 64, 64, 12345], 16, 2, 4, 128, BF, BF, "nhd")
    run_decode(702, [30011, 5], 128, 1, 16, 128, BF, F8, "hnd")
    run_decode(703, [17001, 16999], 32, 1, 8, 256, HF, HF, "nhd")


def test_decode_many_requests():
    lens = [(37 * i) % 301 for i in range(700)]
    run_decode(710, lens, 16, 1, 4, 64, BF, BF, "hnd")
    run_decode(711, [(91 * i) % 40 for i in range(1500)], 16, 1, 2, 64, BF, F8, "nhd")


def test_decode_empty_batch_and_endless_window():
    k, v, _, _ = make_pool(725, 4, 16, 2, 128, BF, "hnd")
    pool = ops.KVPool(k, v)
    out, lse = ops.pool_decode(torch.empty(0, 8, 128, dtype=BF, device=DEV), pool, i32([]),
                               torch.empty(0, 4, dtype=torch.int32, device=DEV), return_lse=True)
    assert out.shape == (0, 8, 128) and lse.shape == (0, 8)
    q, table = torch.randn(1, 8, 128, generator=gen(726), device=DEV).to(BF), make_table(727, [50], 16, 4, 4)
    for window in (2 ** 31 - 1, 2 ** 31, 2 ** 40):
        out, lse = ops.pool_decode(q, pool, i32([50]), table, window=window, return_lse=True)
        check_decode(q, k, v, None, None, [50], table, out, lse, 128 ** -0.5)


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("qt,pt", [(BF, BF), (HF, HF), (BF, F8), (HF, F8)])
def test_decode_many_short_rows(qt, pt, D):
    """Rows of a tile at most, few and more than the GPU's places: a warp's own."""
    run_decode(740, [0, 1, 5, 15, 16], 16, 2, 4, D, qt, pt, "hnd", wide=False)
    run_decode(741, [i % 14 for i in range(700)], 16, 2, 4, D, qt, pt, "nhd", wide=False)
    run_decode(742, [(7 * i) % 49 for i in range(700)], 16, 1, 16, D, qt, pt, "hnd", wide=False, softcap=20.0)
    run_decode(743, [i % 65 for i in range(350)], 64, 2, 17, D, qt, pt, "nhd", wide=False, max_len=64)
    run_decode(744, [i % 30 for i in range(300)], 32, 4, 1, D, qt, pt, "hnd", wide=False)
    run_decode(745, [200 - i % 200 for i in range(610)], 256, 1, 9, D, qt, pt, "hnd", wide=False, max_len=200)


@pytest.mark.parametrize("D,G", [(256, 4), (256, 16), (128, 16)])
@pytest.mark.parametrize("qt,pt", [(BF, BF), (HF, HF), (BF, F8), (HF, F8)])
@pytest.mark.parametrize("B", [297, 1100])
def test_decode_rows_of_a_tile(B, qt, pt, D, G):
    """Room for two or three rows in a CTA: as many warps work, each on rows of its own."""
    run_decode(750, [(11 * i) % 65 for i in range(B)], 16, 1, G, D, qt, pt, "nhd", wide=False, max_len=64)


@pytest.mark.parametrize("D,qt,pt,G", [(64, BF, F8, 8), (64, HF, HF, 16), (128, BF, BF, 4), (128, BF, F8, 20),
                                       (256, HF, HF, 4), (256, BF, F8, 12)])
@pytest.mark.parametrize("S,window", [(16, 0), (16, 7), (32, 100), (128, 0), (128, 65)])
def test_decode_many_rows_of_several_loads(S, window, D, qt, pt, G):
    """More rows than warps, up to 200 tokens or a window at any offset in a block; lengths 0 and 1 among them."""
    lens = [(37 * i) % 201 for i in range(500)] + [0, 1, 200]
    run_decode(760, lens, S, 2, G, D, qt, pt, "hnd" if S == 32 else "nhd", window=window, softcap=10.0 if S == 32 else 0.0,
               wide=False, max_len=200)


def test_decode_rows_of_several_loads_report_bad_ids():
    lens = [100] * 700
    k, v, _, _ = make_pool(770, 700 * 7, 16, 2, 64, BF, "hnd")
    table = make_table(771, lens, 16, 700 * 7, 7)
    q = torch.randn(700, 8, 64, generator=gen(772), device=DEV).to(BF)
    pool, status = ops.KVPool(k, v), i32([0])
    good = ops.pool_decode(q, pool, i32(lens), table, status=status)
    assert int(status) == 0
    table[5, 6] = 700 * 7
    table[9, 0] = -1
    cut = lens.copy()
    cut[5] = 96                                    # the tokens of a bad id at the end do not count
    out = ops.pool_decode(q, pool, i32(lens), table, status=status)
    assert int(status) == ERR_RANGE
    want = ops.pool_decode(q, pool, i32(cut), table)
    same = [b for b in range(700) if b not in (5, 9)]
    assert torch.equal(out[same], good[same]) and torch.equal(out[5], want[5]) and not torch.equal(out[9], good[9])
    status.zero_()
    ops.pool_decode(q, pool, i32([-1] + lens[1:]), table[:, :7], status=status)
    assert int(status) == ERR_RANGE


def test_decode_all_empty():
    run_decode(720, [0, 0, 0], 16, 2, 4, 128, BF, BF, "hnd")
    run_decode(721, [0], 16, 1, 1, 64, HF, F8, "hnd")


def test_decode_max_len_bounds_only_the_work():
    lens = [100, 0, 257, 64]
    a = run_decode(730, lens, 16, 2, 4, 128, BF, BF, "hnd")
    b = run_decode(730, lens, 16, 2, 4, 128, BF, BF, "hnd", max_len=257)
    assert all(torch.allclose(x.float(), y.float(), atol=1e-2) for x, y in zip(a, b))


def test_decode_is_deterministic_and_takes_dirty_workspaces():
    lens = [9000, 1, 0, 4097]
    k, v, ks, vs = make_pool(1, 900, 16, 2, 128, BF, "hnd")
    table = make_table(2, lens, 16, 900, 600)
    q = torch.randn(4, 8, 128, generator=gen(3), device=DEV).to(BF)
    pool = ops.KVPool(k, v)
    first = None
    wide = torch.full((4, 20000), -1, dtype=torch.int32, device=DEV)   # a bound of the lengths that cuts the rows by units
    wide[:, :600] = table
    short = [3900, 1, 0, 257]                                        # one that does not: no workspace
    assert ops.pool_decode_ws_bytes(4, 8, pool, 244) == 0
    for _ in range(3):
        got = ops.pool_decode(q, pool, i32(short), table[:, :244], return_lse=True)
        first = first or got
        assert all(torch.equal(x, y) for x, y in zip(first, got))
    check_decode(q, k, v, ks, vs, short, table, *first, 128 ** -0.5)
    first = None
    for fill in (0, 255, 127, 1):
        ws = torch.full((ops.pool_decode_ws_bytes(4, 8, pool, 20000),), fill, dtype=torch.uint8, device=DEV)
        assert ws.numel() > 0
        got = ops.pool_decode(q, pool, i32(lens), wide, return_lse=True, workspace=ws)
        first = first or got
        assert all(torch.equal(x, y) for x, y in zip(first, got))
    check_decode(q, k, v, ks, vs, lens, wide, *first, 128 ** -0.5)


def test_decode_strides_and_out():
    """q cut out of a projection output, out and lse given, [B, 1, heads, dim] queries."""
    lens = [33, 500]
    k, v, _, _ = make_pool(5, 40, 16, 2, 128, BF, "hnd")
    table = make_table(6, lens, 16, 40, 40)[:, :35]   # rows of a wider table
    qkv = torch.randn(2, 12, 128, generator=gen(7), device=DEV).to(BF)
    q = qkv[:, 2:10]
    out, lse = torch.empty(2, 1, 8, 128, dtype=BF, device=DEV), torch.empty(2, 8, device=DEV)
    got = ops.pool_decode(q.unsqueeze(1), ops.KVPool(k, v), i32(lens), table, out=out, lse=lse)
    assert got is out
    check_decode(q, k, v, None, None, lens, table, out[:, 0], lse, 128 ** -0.5)
    # rows that are not whole 16-byte words are laid out anew
    odd = torch.randn(2 * 8 * 128 + 4, generator=gen(8), device=DEV).to(BF)[4:].view(2, 8, 128)
    out, lse = ops.pool_decode(odd, ops.KVPool(k, v), i32(lens), table, return_lse=True)
    check_decode(odd, k, v, None, None, lens, table, out, lse, 128 ** -0.5)


def test_decode_pool_strides():
    """K and V as the two halves of one allocation, and a pool with room between its rows."""
    lens = [100, 17]
    both = torch.randn(12, 2, 16, 2, 128, generator=gen(9), device=DEV).to(BF)
    table = make_table(10, lens, 16, 12, 8)
    q = torch.randn(2, 6, 128, generator=gen(11), device=DEV).to(BF)
    k, v = both[:, 0], both[:, 1]
    out, lse = ops.pool_decode(q, ops.KVPool(k, v), i32(lens), table, return_lse=True)
    check_decode(q, k, v, None, None, lens, table, out, lse, 128 ** -0.5)
    wide = torch.randn(12, 16, 2, 200, generator=gen(12), device=DEV).to(BF)
    k, v = wide[..., :128], torch.randn(12, 16, 3, 136, generator=gen(13), device=DEV).to(BF)[:, :, 1:, :128]
    out, lse = ops.pool_decode(q, ops.KVPool(k, v), i32(lens), table, return_lse=True)
    check_decode(q, k, v, None, None, lens, table, out, lse, 128 ** -0.5)


def test_decode_offsets_past_32_bits():
    """Blocks whose element offsets pass 2^31 (and byte offsets 2^32)."""
    S, H, D = 16, 8, 128
    n_blocks = 2 ** 31 // (S * H * D) + 300     # 2.2e9 elements
    lens = [1000]
    k = torch.empty(n_blocks, H, S, D, dtype=BF, device=DEV).transpose(1, 2)
    v = torch.empty(n_blocks, H, S, D, dtype=BF, device=DEV).transpose(1, 2)
    c = (lens[0] + S - 1) // S
    table = (n_blocks - 1 - 4 * torch.arange(c, device=DEV)).int().view(1, c).contiguous()
    k[table[0].long()] = torch.randn(c, S, H, D, generator=gen(14), device=DEV).to(BF)
    v[table[0].long()] = torch.randn(c, S, H, D, generator=gen(15), device=DEV).to(BF)
    q = torch.randn(1, 32, D, generator=gen(16), device=DEV).to(BF)
    pool = ops.KVPool(k, v)
    out, lse = ops.pool_decode(q, pool, i32(lens), table, return_lse=True)
    check_decode(q, k, v, None, None, lens, table, out, lse, D ** -0.5)
    new = torch.randn(2, H, D, generator=gen(17), device=DEV).to(BF)
    slots = torch.tensor([n_blocks * S - 1, n_blocks * S - 2], device=DEV)
    ops.pool_write(new, new, slots, pool)
    assert torch.equal(k[n_blocks - 1, S - 1], new[0]) and torch.equal(v[n_blocks - 1, S - 2], new[1])


def test_decode_reports_bad_ids_and_lengths():
    """Ids outside the pool leave their tokens out; lengths past the table are cut; both are reported."""
    S, D = 16, 128
    k, v, _, _ = make_pool(21, 10, S, 2, D, BF, "hnd")
    q = torch.randn(3, 8, D, generator=gen(22), device=DEV).to(BF)
    table = i32([[0, 1, 2, 3], [4, 99, 5, -1], [6, 7, 8, 9]])
    status = i32([0])
    pool = ops.KVPool(k, v)
    out, lse = ops.pool_decode(q, pool, i32([64, 64, 500]), table, return_lse=True, status=status)
    assert int(status) == ERR_RANGE
    check_decode(q[:1], k, v, None, None, [64], table[:1], out[:1], lse[:1], D ** -0.5)
    check_decode(q[1:2], k, v, None, None, [32], i32([[4, 5]]), out[1:2], lse[1:2], D ** -0.5)
    check_decode(q[2:], k, v, None, None, [64], table[2:], out[2:], lse[2:], D ** -0.5)
    status.zero_()
    out, lse = ops.pool_decode(q, pool, i32([-5, 1, 0]), table, return_lse=True, status=status)
    assert int(status) == ERR_RANGE
    check_decode(q, k, v, None, None, [0, 1, 0], table, out, lse, D ** -0.5)


def test_decode_extreme_scores():
    """Scores far apart, all alike, and every score -inf (a row that is empty but for its length)."""
    S, D = 16, 64
    k, v, _, _ = make_pool(31, 20, S, 1, D, BF, "hnd")
    table = make_table(32, [300], S, 20, 20)
    q = torch.randn(1, 4, D, generator=gen(33), device=DEV).to(BF) * 50
    out, lse = ops.pool_decode(q, ops.KVPool(k, v), i32([300]), table, return_lse=True)
    check_decode(q, k, v, None, None, [300], table, out, lse, D ** -0.5)
    q = torch.zeros_like(q)
    out, lse = ops.pool_decode(q, ops.KVPool(k, v), i32([300]), table, return_lse=True)
    check_decode(q, k, v, None, None, [300], table, out, lse, D ** -0.5)
    big = torch.full_like(k, torch.finfo(BF).max)
    q = torch.full_like(q, -1e30)
    out, lse = ops.pool_decode(q, ops.KVPool(big, v), i32([300]), table, return_lse=True)
    assert torch.equal(out, torch.zeros_like(out)) and bool((lse == -math.inf).all())


@pytest.mark.parametrize("mag", [1e-30, 1e-4, 1e4, 1e30])
def test_decode_query_range_over_fp8(mag):
    """bf16 queries far outside fp16's range over e4m3 blocks."""
    S, D = 32, 128
    k, v, ks, vs = make_pool(41, 12, S, 2, D, F8, "hnd")
    table = make_table(42, [200, 77], S, 12, 12)
    q = (torch.randn(2, 8, D, generator=gen(43), device=DEV) * mag).to(BF)
    q[:, ::3] *= 0.01
    out, lse = ops.pool_decode(q, ops.KVPool(k, v, ks, vs), i32([200, 77]), table, scale=0.1 / mag, return_lse=True)
    check_decode(q, k, v, ks, vs, [200, 77], table, out, lse, 0.1 / mag)


@pytest.mark.parametrize("width", [80, 20000])
def test_decode_on_another_stream_and_in_a_graph(width):
    lens = [1000, 17, 0, 640]
    k, v, _, _ = make_pool(51, 120, 16, 2, 128, BF, "hnd")
    table = make_table(52, lens, 16, 120, width)
    q = torch.randn(4, 8, 128, generator=gen(53), device=DEV).to(BF)
    pool, n = ops.KVPool(k, v), i32(lens)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        out, lse = ops.pool_decode(q, pool, n, table, return_lse=True)
    side.synchronize()
    check_decode(q, k, v, None, None, lens, table, out, lse, 128 ** -0.5)
    ws = torch.empty(ops.pool_decode_ws_bytes(4, 8, pool, width), dtype=torch.uint8, device=DEV)
    g_out, g_lse = torch.empty_like(out), torch.empty_like(lse)
    with torch.cuda.stream(side):
        ops.pool_decode(q, pool, n, table, out=g_out, lse=g_lse, workspace=ws)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.pool_decode(q, pool, n, table, out=g_out, lse=g_lse, workspace=ws)
    lens2 = [999, 40, 3, 700]     # the lengths are read on the GPU: a replay sees the new ones
    table.copy_(make_table(54, lens2, 16, 120, width))
    n.copy_(i32(lens2))
    graph.replay()
    torch.cuda.synchronize()
    check_decode(q, k, v, None, None, lens2, table, g_out, g_lse, 128 ** -0.5)


# ------------------------------------------------------------------ write
@pytest.mark.parametrize("layout", ["hnd", "nhd"])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("st,pt", [(BF, BF), (HF, HF), (BF, F8), (HF, F8)])
@pytest.mark.parametrize("T,H", [(1, 1), (7, 3), (1000, 2)])
def test_write(T, H, st, pt, D, layout):
    S, n_blocks = 16, T // 8 + 2
    k, v, ks, vs = make_pool(61, n_blocks, S, H, D, pt, layout)
    x = (torch.randn(T, 4 * H, D, generator=gen(62), device=DEV) * 20).to(st)
    x[0, :, :6] = torch.tensor([0.0, -0.0, math.inf, -math.inf, math.nan, 1e-4], device=DEV).to(st)
    kk, vv = x[:, H: 2 * H], x[:, 3 * H:]
    slots = torch.randperm(n_blocks * S, generator=gen(63), device=DEV)[:T]
    slots[T // 2] = -1 if T > 1 else slots[0]
    want = []
    for src, pool, scale in ((kk, k, ks), (vv, v, vs)):
        w = pool.clone()
        live = slots >= 0
        at = slots[live]
        if pt == F8:
            y = (src[live].float() / scale[:, None]).clamp(-448, 448).to(F8)
            w.view(torch.uint8)[at // S, at % S] = y.view(torch.uint8)
        else:
            w[at // S, at % S] = src[live]
        want.append(w)
    status = i32([0])
    ops.pool_write(kk, vv, slots, ops.KVPool(k, v, ks, vs), status=status)
    bits = torch.uint8 if pt == F8 else torch.int16
    for got, w in zip((k, v), want):
        nan = w.float().isnan()
        assert torch.equal(got.float().isnan(), nan)
        assert torch.equal(got.view(bits)[~nan], w.view(bits)[~nan])
    assert int(status) == 0


def test_write_skips_and_reports_slots_outside_the_pool():
    k, v, _, _ = make_pool(71, 3, 16, 2, 64, BF, "hnd")
    before = k.clone(), v.clone()
    x = torch.randn(5, 2, 64, generator=gen(72), device=DEV).to(BF)
    status = i32([0])
    ops.pool_write(x, x, torch.tensor([-1, 48, -7, 2 ** 40, -1], device=DEV), ops.KVPool(k, v), status=status)
    assert int(status) == ERR_RANGE
    assert torch.equal(k, before[0]) and torch.equal(v, before[1])
    ops.pool_write(x[:0], x[:0], torch.empty(0, dtype=torch.int64, device=DEV), ops.KVPool(k, v))
    assert torch.equal(k, before[0])


# ------------------------------------------------------------------ plan and release
def plain_plan(lens, new, table, free, n_free, S, n_slots):
    """Request by request."""
    width = len(table[0]) if table else 0
    table, lens = [list(r) for r in table], list(lens)
    slots, positions, cu, used, failed = [-1] * n_slots, [-1] * n_slots, [0], 0, False
    taken = 0
    for b, (c, n) in enumerate(zip(lens, new)):
        start, cu_next = cu[-1], cu[-1] + max(n, 0)
        cu.append(cu_next)
        have, need = -(-c // S), -(-(c + n) // S)
        fits = c >= 0 and n >= 0 and need <= width and cu_next <= n_slots
        take = need - have if fits else 0
        served = fits and (take == 0 or taken + take <= n_free)
        if served:
            for j in range(take):
                table[b][have + j] = free[n_free - 1 - taken - j]
            for j in range(n):
                p = c + j
                slots[start + j], positions[start + j] = table[b][p // S] * S + p % S, p
            lens[b] = c + n
            used += take
        else:
            failed = True
        taken += take
    return table, slots, positions, cu, lens, n_free - used, ERR_CAPACITY if failed else 0


def run_plan(lens, new, table, free, n_free, S, n_slots, in_place=False):
    B = len(lens)
    t_lens, t_new, t_free, t_n = i32(lens), i32(new), i32(free), i32([n_free])
    t_table = i32(table).view(B, -1)
    slots = torch.full((n_slots,), 77, dtype=torch.int64, device=DEV)
    positions, cu = torch.full((n_slots,), 77, dtype=torch.int32, device=DEV), torch.full((B + 1,), 77, dtype=torch.int32,
                                                                                        device=DEV)
    status = i32([0])
    lens_out, n_out = (t_lens, t_n) if in_place else (torch.empty_like(t_lens), torch.empty_like(t_n))
    ops.pool_plan(t_lens, t_new, t_table, t_free, t_n, S, slots, positions=positions, cu_new=cu,
                  lens_out=None if in_place else lens_out, n_free_out=None if in_place else n_out, status=status)
    got = (t_table.tolist(), slots.tolist(), positions.tolist(), cu.tolist(), lens_out.tolist(), int(n_out), int(status))
    want = plain_plan(lens, new, table, free, n_free, S, n_slots)
    for name, x, y in zip(("table", "slots", "positions", "cu", "lens", "n_free", "status"), got, want):
        assert x == y, name
    if not in_place:
        assert t_lens.tolist() == list(lens) and int(t_n) == n_free
    assert t_free.tolist() == list(free)


def plan_inputs(seed, B, S, ctx_hi, new_hi, short=0):
    import random
    r = random.Random(seed)
    lens = [r.randint(0, ctx_hi) for _ in range(B)]
    new = [r.choice([0, 1, r.randint(0, new_hi)]) for _ in range(B)]
    width = (ctx_hi + new_hi) // S + 2
    ids = list(range(B * width))
    r.shuffle(ids)
    table, at = [], 0
    for c in lens:
        h = -(-c // S)
        table.append(ids[at: at + h] + [-1] * (width - h))
        at += h
    need = sum(-(-(c + n) // S) - -(-c // S) for c, n in zip(lens, new))
    rest = ids[at:]
    n_free = max(0, min(len(rest), need - short)) if short else len(rest)
    return lens, new, table, rest + [0] * (len(ids) - len(rest)), n_free


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("B,S,ctx,new", [(1, 16, 0, 1), (1, 16, 100, 5000), (3, 32, 64, 40), (33, 16, 200, 70),
                                         (1025, 16, 50, 9), (2500, 64, 300, 3)])
def test_plan(B, S, ctx, new, in_place):
    lens, add, table, free, n_free = plan_inputs(B + S, B, S, ctx, new)
    total = sum(add)
    for n_slots in (total, total + 5):
        run_plan(lens, add, table, free, n_free, S, n_slots, in_place)


def test_plan_block_edges():
    S = 16
    lens = [0, 15, 16, 17, 31, 32, 0, 48, 5]
    new = [16, 1, 1, 15, 1, 0, 33, 16, 0]
    ids = list(range(100, 200))
    table, at = [], 0
    for c in lens:
        h = -(-c // S)
        table.append(ids[at: at + h] + [-1] * (5 - h))
        at += h
    run_plan(lens, new, table, list(range(200)), 90, S, sum(new))


@pytest.mark.parametrize("short", [1, 2, 7, 1000000])
@pytest.mark.parametrize("B", [5, 700])
def test_plan_without_enough_blocks(B, short):
    lens, add, table, free, n_free = plan_inputs(B, B, 16, 100, 50, short)
    run_plan(lens, add, table, free, n_free, 16, sum(add), in_place=True)


def test_plan_refuses_what_does_not_fit():
    S = 16
    free = list(range(50))
    # past the table's width; negative counts; past the slot map
    run_plan([60, 3, 10, 3], [5, 2, -4, 1], [[0, 1, 2, 3], [4, -1, -1, -1], [5, -1, -1, -1], [6, -1, -1, -1]], free, 40, S, 12)
    run_plan([3, 3, 3], [4, 4, 4], [[0], [1], [2]], free, 40, S, 8)
    run_plan([2 ** 31 - 1, 0], [5, 1], [[0], [-1]], free, 40, S, 8)


def test_plan_default_is_one_token_each_and_bad_ids_are_reported():
    lens, table = i32([3, 16]), i32([[7, -1], [9, -1]])
    free, n_free, slots, status = i32(list(range(12))), i32([5]), torch.empty(2, dtype=torch.int64, device=DEV), i32([0])
    ops.pool_plan(lens, None, table, free, n_free, 16, slots, status=status)
    assert slots.tolist() == [7 * 16 + 3, 4 * 16] and lens.tolist() == [4, 17] and int(n_free) == 4 and int(status) == 0
    assert table.tolist() == [[7, -1], [9, 4]]
    table[0, 0] = 12
    ops.pool_plan(lens, None, table, free, n_free, 16, slots, status=status)
    assert slots.tolist() == [-1, 4 * 16 + 1] and int(status) == ERR_RANGE


def test_plan_empty_batch():
    slots, n_free = torch.full((3,), 5, dtype=torch.int64, device=DEV), i32([2])
    ops.pool_plan(i32([]), i32([]), torch.empty(0, 4, dtype=torch.int32, device=DEV), i32([1, 2]), n_free, 16, slots)
    assert slots.tolist() == [-1, -1, -1] and int(n_free) == 2


def plain_release(done, lens, table, free, n_free, S):
    free, lens = list(free), list(lens)
    for b, d in enumerate(done):
        if d:
            for j in range(-(-lens[b] // S)):
                if n_free < len(free):
                    free[n_free] = table[b][j]
                    n_free += 1
            lens[b] = 0
    return free, lens, n_free


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("B,S,ctx,p", [(1, 16, 40, 1.0), (4, 16, 100, 0.5), (3, 16, 20000, 0.7), (1300, 32, 90, 0.9),
                                       (50, 16, 300, 0.0)])
def test_release(B, S, ctx, p, in_place):
    import random
    lens, _, table, free, n_free = plan_inputs(B, B, S, ctx, 1)
    r = random.Random(B)
    done = [r.random() < p for _ in range(B)]
    t_lens, t_free, t_n, status = i32(lens), i32(free), i32([n_free]), i32([0])
    lo, no = (None, None) if in_place else (torch.empty_like(t_lens), torch.empty_like(t_n))
    ops.pool_release(torch.tensor(done, device=DEV), t_lens, i32(table), t_free, t_n, S, lens_out=lo, n_free_out=no,
                     status=status)
    want = plain_release(done, lens, table, free, n_free, S)
    got = (t_free.tolist(), (t_lens if in_place else lo).tolist(), int(t_n if in_place else no))
    assert got == want and int(status) == 0


def test_release_does_not_push_past_the_stack():
    free, n_free, status = i32([0, 1, 2, 3]), i32([3]), i32([0])
    lens = i32([40, 20])
    ops.pool_release(torch.tensor([True, True], device=DEV), lens, i32([[0, 1, 2], [3, 1, -1]]), free, n_free, 16,
                     status=status)
    assert int(status) == ERR_CAPACITY and int(n_free) == 4 and free.tolist() == [0, 1, 2, 0] and lens.tolist() == [0, 0]


def test_requests_come_and_go():
    """Random admissions, decode steps and releases: no block is owned twice, none is lost, and the attention of every
    step equals attention over rows kept on the side."""
    import random
    r = random.Random(0)
    B, S, H, G, D, n_blocks, width = 6, 16, 2, 2, 64, 64, 20
    k, v, _, _ = make_pool(80, n_blocks, S, H, D, BF, "hnd")
    pool = ops.KVPool(k, v)
    lens, table = i32([0] * B), torch.full((B, width), -1, dtype=torch.int32, device=DEV)
    free, n_free, status = torch.arange(n_blocks, device=DEV).int(), i32([n_blocks]), i32([0])
    held = [([], []) for _ in range(B)]
    g = gen(81)
    for step in range(60):
        if step % 7 == 6:
            done = torch.tensor([r.random() < 0.4 for _ in range(B)], device=DEV)
            ops.pool_release(done, lens, table, free, n_free, S, status=status)
            for b in range(B):
                if bool(done[b]):
                    held[b] = ([], [])
        host = lens.tolist()
        new = [r.randint(20, 60) if host[b] == 0 and r.random() < 0.5 else int(host[b] > 0) for b in range(B)]
        slots = torch.empty(sum(new) + 2, dtype=torch.int64, device=DEV)
        cu = torch.empty(B + 1, dtype=torch.int32, device=DEV)
        ops.pool_plan(lens, i32(new), table, free, n_free, S, slots, cu_new=cu, status=status)
        kv = torch.randn(2, sum(new) + 2, H, D, generator=g, device=DEV).to(BF)
        ops.pool_write(kv[0], kv[1], slots, pool, status=status)
        now, at = lens.tolist(), cu.tolist()
        for b in range(B):
            if now[b] == host[b] + new[b]:
                held[b][0].append(kv[0, at[b]: at[b + 1]])
                held[b][1].append(kv[1, at[b]: at[b + 1]])
        owned = [i for b in range(B) for i in table[b, : -(-now[b] // S)].tolist()] + free[: int(n_free)].tolist()
        assert sorted(owned) == list(range(n_blocks))
        q = torch.randn(B, H * G, D, generator=g, device=DEV).to(BF)
        out, lse = ops.pool_decode(q, pool, lens, table, return_lse=True, status=status)
        for b in range(B):
            if now[b] == 0:
                assert not bool(out[b].any())
                continue
            kk, vv = torch.cat(held[b][0]), torch.cat(held[b][1])
            assert kk.shape[0] == now[b]
            check_decode(q[b: b + 1], kk[None], vv[None], None, None, [now[b]], i32([[0]]), out[b: b + 1], lse[b: b + 1],
                         D ** -0.5)
    assert int(status) in (0, ERR_CAPACITY)


# ------------------------------------------------------------------ refusals
def test_refusals():
    k, v, _, _ = make_pool(91, 4, 16, 2, 128, BF, "hnd")
    pool = ops.KVPool(k, v)
    q, lens, table = torch.zeros(2, 8, 128, dtype=BF, device=DEV), i32([1, 1]), i32([[0], [1]])
    for bad in (q.float(), q.half()):
        with pytest.raises(TypeError):
            ops.pool_decode(bad, pool, lens, table)
    with pytest.raises(ValueError):
        ops.pool_decode(q[:, :7], pool, lens, table)
    with pytest.raises(ValueError):
        ops.pool_decode(q[..., :64], pool, lens, table)
    with pytest.raises(TypeError):
        ops.pool_decode(q, pool, lens.long(), table)
    with pytest.raises(TypeError):
        ops.pool_decode(q, pool, lens, table.long())
    with pytest.raises(ValueError):
        ops.pool_decode(q, pool, lens[:1], table)
    with pytest.raises(ValueError):
        ops.pool_decode(q, pool, lens, table.t())
    with pytest.raises(ValueError):
        ops.pool_decode(q, pool, lens, table, out=torch.empty(2, 8, 64, dtype=BF, device=DEV))
    with pytest.raises(ValueError):
        ops.pool_decode(q, pool, lens, table, lse=torch.empty(2, 8, dtype=BF, device=DEV))
    for kw in (dict(window=-1), dict(softcap=-1.0), dict(softcap=math.nan), dict(max_len=-1)):
        with pytest.raises(RuntimeError):
            ops.pool_decode(q, pool, lens, table, **kw)
    wide = torch.zeros(2, 10 ** 5, dtype=torch.int32, device=DEV)
    with pytest.raises(RuntimeError, match="limit"):
        ops.pool_decode(q, pool, lens, wide, workspace=torch.empty(256, dtype=torch.uint8, device=DEV))
    with pytest.raises(TypeError):
        ops.KVPool(k, v.half())
    with pytest.raises(ValueError):
        ops.KVPool(k, v[:2])
    with pytest.raises(ValueError):
        ops.KVPool(k, v, torch.ones(2, device=DEV))
    with pytest.raises(RuntimeError, match="unsupported"):
        ops.KVPool(k[..., :32], v[..., :32])
    with pytest.raises(RuntimeError, match="unsupported"):
        ops.KVPool(k[:, :12], v[:, :12])
    with pytest.raises(RuntimeError, match="align"):
        x = torch.zeros(4, 16, 2, 132, dtype=BF, device=DEV)[..., :128]
        ops.KVPool(x, x)
    rows = torch.zeros(3, 2, 128, dtype=BF, device=DEV)
    slots = torch.zeros(3, dtype=torch.int64, device=DEV)
    with pytest.raises(TypeError):
        ops.pool_write(rows.half(), rows.half(), slots, pool)
    with pytest.raises(TypeError):
        ops.pool_write(rows, rows, slots.int(), pool)
    with pytest.raises(ValueError):
        ops.pool_write(rows, rows, slots[:2], pool)
    with pytest.raises(ValueError):
        ops.pool_write(rows[:, :1], rows[:, :1], slots, pool)
    free, n = i32([0, 1]), i32([2])
    with pytest.raises(RuntimeError, match="unsupported"):
        ops.pool_plan(lens, None, table, free, n, 24, slots)
    with pytest.raises(ValueError):
        ops.pool_plan(lens, i32([1]), table, free, n, 16, slots)
    with pytest.raises(TypeError):
        ops.pool_plan(lens.long(), None, table, free, n, 16, slots)
    with pytest.raises(RuntimeError, match="limit"):
        big = torch.zeros(9000, dtype=torch.int32, device=DEV)
        ops.pool_plan(big, None, big.view(9000, 1), big, n, 16, slots)
    with pytest.raises(TypeError):
        ops.pool_release(i32([1, 0]), lens, table, free, n, 16)


def test_refusals_of_host_memory():
    """What the kernels would write lies on the pool's device."""
    k, v, _, _ = make_pool(92, 4, 16, 2, 128, BF, "hnd")
    pool = ops.KVPool(k, v)
    q, lens, table = torch.zeros(2, 8, 128, dtype=BF, device=DEV), i32([1, 1]), i32([[0], [1]])
    rows, slots = torch.zeros(2, 2, 128, dtype=BF, device=DEV), torch.zeros(2, dtype=torch.int64, device=DEV)
    host = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(ValueError):
        ops.pool_decode(q, pool, lens, table, status=host)
    with pytest.raises(TypeError):
        ops.pool_decode(q, pool, lens, table, status=host.to(DEV).long())
    with pytest.raises(ValueError):
        ops.pool_write(rows, rows, slots, pool, status=host)
    with pytest.raises(TypeError):
        ops.pool_write(rows, rows, slots, pool, status=host.to(DEV).float())
    n = ops.pool_decode_ws_bytes(2, 8, pool, 10 ** 5)
    assert n > 0
    for ws in (torch.empty(n, dtype=torch.uint8), torch.empty(n, dtype=torch.int8, device=DEV),
               torch.empty(2 * n, dtype=torch.uint8, device=DEV)[::2]):
        with pytest.raises(ValueError):
            ops.pool_decode(q, pool, lens, torch.zeros(2, 10 ** 5, dtype=torch.int32, device=DEV), workspace=ws)
