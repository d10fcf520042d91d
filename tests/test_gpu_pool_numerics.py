"""GPU: attention over the pool where the 16-bit products have least room:
probabilities far below the largest one, and query elements far below theirs.
The tolerance is test_gpu_pool's, derived there."""
import pytest
import torch

from test_gpu_pool import BF, DEV, F8, HF, check_decode, gen, i32, make_table
from zoomkv_revision_b200 import ops

pytestmark = pytest.mark.gpu


def narrow(x, dtype):
    return x.clamp(-448, 448).to(dtype) if dtype == F8 else x.to(dtype)


# name, lengths, columns of the table beyond the longest request, bound of the lengths
SHAPES = {
    "a_warp_a_row": ([100 + 37 * i % 101 for i in range(700)], 0, 200),
    "four_warps_a_row": ([150 + 37 * i % 101 for i in range(160)], 0, 250),
    "a_cluster_a_row": ([2100], 0, 0),
    "split_and_joined": ([3000, 150, 9000], 20000, 0),
}


@pytest.mark.parametrize("D,G", [(64, 4), (128, 4), (128, 12), (256, 4)])
@pytest.mark.parametrize("qt,pt", [(BF, BF), (HF, HF), (BF, F8), (HF, F8)])
@pytest.mark.parametrize("shape", list(SHAPES))
def test_tokens_far_below_a_sink(shape, qt, pt, D, G):
    """The first token's score is 14 to 18.5 above the others' (2^-20 to 2^-27 of its probability) and its V is zero, so the
    output is the others' alone: 100 or more times 9e-9 of values near 200, a normal number in every type."""
    lens, spare, bound = SHAPES[shape]
    S = 16
    n_blocks = sum(-(-n // S) for n in lens)
    g = gen(1)
    k = torch.randn(n_blocks, S, 1, D, generator=g, device=DEV) * 0.01
    v = 200 + 20 * torch.randn(n_blocks, S, 1, D, generator=g, device=DEV)
    table = make_table(2, lens, S, n_blocks, -(-max(lens) // S) + spare)
    first = table[:, 0].long()
    k[first, 0], v[first, 0] = 1.0, 0.0
    k, v = narrow(k, pt), narrow(v, pt)
    gap = torch.linspace(14.0, 18.5, G, device=DEV)
    q = (gap / D ** 0.5).view(1, G, 1).expand(len(lens), G, D).to(qt).contiguous()
    status = i32([0])
    out, lse = ops.pool_decode(q, ops.KVPool(k, v), i32(lens), table, max_len=bound, return_lse=True, status=status)
    assert int(status) == 0
    check_decode(q, k, v, None, None, lens, table, out, lse, D ** -0.5)


@pytest.mark.parametrize("small", [2.0 ** -16, 2.0 ** -20, 2.0 ** -27])
@pytest.mark.parametrize("G", [4, 12])
@pytest.mark.parametrize("lens", [[300, 77], [i % 60 for i in range(700)]])
def test_small_query_elements_over_fp8(lens, G, small):
    """A bf16 query's largest element meets zeros, the others are `small` of it and make the scores."""
    S, D = 16, 128
    n_blocks = sum(-(-n // S) for n in lens) + 1
    g = gen(3)
    k = torch.randn(n_blocks, S, 1, D, generator=g, device=DEV) * 100
    k[..., 0] = 0
    k = narrow(k, F8)
    v = narrow(torch.randn(n_blocks, S, 1, D, generator=g, device=DEV), F8)
    table = make_table(4, lens, S, n_blocks, -(-max(lens) // S))
    q = torch.randn(len(lens), G, D, generator=g, device=DEV) * small
    q[..., 0] = 1.3
    q = q.to(BF)
    scale = 0.004 / small
    out, lse = ops.pool_decode(q, ops.KVPool(k, v), i32(lens), table, scale=scale, return_lse=True)
    check_decode(q, k, v, None, None, lens, table, out, lse, scale)


@pytest.mark.parametrize("qt,pt", [(BF, BF), (HF, HF), (BF, F8), (HF, F8)])
@pytest.mark.parametrize("shape", list(SHAPES))
def test_scores_of_any_size(shape, qt, pt):
    """One token a request scores 2^20 to 2^30, the others 0, or as much below 0: its V row is the output, bit for bit, and
    its score, a power of two, the lse (1.4427 times which rounds by 2^-24, and back)."""
    lens, spare, bound = SHAPES[shape]
    S, D, G = 16, 128, 4
    n_blocks = sum(-(-n // S) for n in lens)
    g = gen(5)
    k = torch.zeros(n_blocks, S, 1, D, device=DEV)
    v = narrow(torch.randn(n_blocks, S, 1, D, generator=g, device=DEV), pt)
    table = make_table(6, lens, S, n_blocks, -(-max(lens) // S) + spare)
    at = torch.tensor([n * 2 // 3 for n in lens], device=DEV)
    block = table[torch.arange(len(lens), device=DEV), at // S].long()
    for sign in (1.0, -1.0):
        if sign > 0:
            k[block, at % S] = 8.0
        else:
            k.fill_(-8.0)
            k[block, at % S] = 0.0
        q = torch.full((len(lens), G, D), 1024.0, device=DEV).to(qt)     # scale times 2^(10 + 3 + 7)
        pool = ops.KVPool(narrow(k, pt), v)
        want = v.float()[block, at % S].to(qt).expand(len(lens), G, D)
        for power in range(11):
            out, lse = ops.pool_decode(q, pool, i32(lens), table, scale=2.0 ** power, max_len=bound, return_lse=True)
            assert torch.equal(out, want), (sign, power)
            score = 2.0 ** (20 + power) if sign > 0 else 0.0
            assert bool(((lse - score).abs() <= 2.0 ** -22 * score).all()), (sign, power)
