"""GPU: the pooled cache under the decode loop and as a server uses it."""
import pytest
import torch
import torch.nn.functional as F

from zoomkv_revision_b200 import decode_loop as DL
from zoomkv_revision_b200.pool_cache import PoolCache, serve

pytestmark = pytest.mark.gpu
DEV = "cuda"
SMALL = DL.Shape(hidden=256, layers=2, heads=6, kv_heads=2, head_dim=128, ffn=512, vocab=1000)


@pytest.mark.parametrize("graphs", [False, True])
def test_decode_loop_over_the_pool_follows_a_dense_forward(graphs):
    """The loop's logits against a PyTorch forward over every token (the bar of the loop's own test over polar_cache)."""
    B, prompt, steps, s = 3, 45, 20, SMALL
    w = DL.Weights(s, DEV, seed=1, std=0.05)
    cache = PoolCache(s.layers, B, s.kv_heads, s.head_dim, prompt + steps + 1)
    loop = DL.DecodeLoop(s, w, cache, B, prompt + steps + 16, DEV, use_graphs=graphs, temperature=0.0)
    ids = torch.randint(0, s.vocab, (B, prompt), generator=torch.Generator().manual_seed(7)).to(DEV)
    tok = loop.prefill(ids)
    toks, logits = [tok], []
    for _ in range(steps):
        tok = loop.step(tok)
        toks.append(tok)
        logits.append(loop.logits.clone())
    cache.check()
    assert cache.lens.tolist() == [prompt + steps] * B
    assert int(cache.n_free) == cache.n_blocks - B * -(-(prompt + steps) // 16)
    seq = torch.cat([ids, torch.stack(toks, 1)[:, :steps]], 1)
    x = F.embedding(seq, w.embed)
    cos, sin = loop.cos[:seq.shape[1]], loop.sin[:seq.shape[1]]
    for L in w.layers:
        q, k, v = loop._qkv(x, L, cos, sin)
        o = F.scaled_dot_product_attention(q.transpose(1, 2).float(), k.transpose(1, 2).float(), v.transpose(1, 2).float(),
                                           is_causal=True, enable_gqa=True).to(torch.bfloat16)
        x = loop._post_attn(x, o.transpose(1, 2), L)
    ref = loop._lm(x)
    for i in range(steps):
        got, want = logits[i], ref[:, prompt + i]
        assert (got - want).abs().max().item() <= 0.05 * want.abs().max().item(), i


def test_a_request_may_fill_its_last_block():
    cache = PoolCache(1, 1, 1, 64, 20)             # two blocks of 16
    rows = torch.randn(30, 1, 64, generator=torch.Generator(device=DEV).manual_seed(3), device=DEV).to(torch.bfloat16)
    cache.write(0, rows, rows, cache.plan(torch.tensor([30], dtype=torch.int32, device=DEV), 30, 30))
    q = torch.randn(1, 2, 64, generator=torch.Generator(device=DEV).manual_seed(4), device=DEV).to(torch.bfloat16)
    out, wide = cache.attend(0, q), cache.attend(0, q, max_len=0)
    cache.check()
    x = rows[:, 0].double()
    want = torch.softmax(q[0].double() @ x.T / 8, -1) @ x
    for got in (out, wide):  # rounding of the output, and of probabilities and scores as 2^-10 of the largest value
        assert bool(((got[0].double() - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -10 * x.abs().max()).all())


def test_too_few_blocks_are_reported():
    cache = PoolCache(1, 2, 1, 64, 64, n_blocks=5)
    slots = cache.plan(torch.tensor([40, 40], dtype=torch.int32, device=DEV), 80, 40)
    assert (slots[:40] >= 0).all() and (slots[40:] == -1).all()
    with pytest.raises(RuntimeError, match="limit"):
        cache.check()
    cache.check()                                  # the report is given once
    rows = torch.randn(80, 1, 64, device=DEV).to(torch.bfloat16)
    cache.write(0, rows, rows, slots)              # the rows of the request that found no room go nowhere
    out = cache.attend(0, torch.randn(2, 4, 64, device=DEV).to(torch.bfloat16))
    assert bool(out[0].any()) and not bool(out[1].any())
    cache.release(torch.tensor([True, False], device=DEV), bound=0)
    cache.plan(torch.tensor([0, 40], dtype=torch.int32, device=DEV), 40, 40)
    cache.check()
    assert cache.lens.tolist() == [0, 40] and int(cache.n_free) == 2


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float8_e4m3fn])
def test_serving_run(dtype):
    got = serve(40, 8, layers=2, kv_heads=2, max_length=256, dtype=dtype)
    assert got["tokens"] > 8 * 16 and 0 < got["free_blocks"] <= got["blocks"]


def test_prompts_come_for_the_whole_batch():
    cache = PoolCache(1, 2, 1, 64, 64)
    rows = torch.zeros(1, 4, 1, 64, dtype=torch.bfloat16, device=DEV)
    with pytest.raises(ValueError):
        cache.prefill_update_kv_cache(None, rows, rows, 0, 0)


def test_sliding_window_through_the_cache():
    cache = PoolCache(1, 2, 2, 128, 512, block_size=32)
    g = torch.Generator(device=DEV).manual_seed(3)
    kv = torch.randn(2, 2, 300, 2, 128, generator=g, device=DEV).to(torch.bfloat16)
    cache.prefill_update_kv_cache(None, kv[0], kv[1], 0, 0)
    q = torch.randn(2, 1, 8, 128, generator=g, device=DEV).to(torch.bfloat16)
    out = cache.attend(0, q, window=100)
    k, v = (x[:, -100:].transpose(1, 2).double() for x in kv)
    ref = F.scaled_dot_product_attention(q.transpose(1, 2).double(), k, v, enable_gqa=True).transpose(1, 2)
    assert torch.allclose(out.double(), ref, atol=2e-2, rtol=2e-2)
