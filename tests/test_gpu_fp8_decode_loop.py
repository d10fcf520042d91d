"""GPU: the decode loop with 8-bit weights (decode_loop.Fp8Weights) over the
pooled cache, on a small Qwen3-shaped model."""
import pytest
import torch
import torch.nn.functional as F

from zoomkv_revision_b200 import decode_loop as DL
from zoomkv_revision_b200 import ops
from zoomkv_revision_b200.pool_cache import PoolCache

pytestmark = pytest.mark.gpu
DEV = "cuda"
SMALL = DL.Shape(hidden=256, layers=2, heads=2, kv_heads=1, head_dim=128, ffn=528, vocab=1000)


def run(graphs, steps, B=2, prompt=48):
    s = SMALL
    w = DL.Fp8Weights(DL.Weights(s, DEV, seed=1, std=0.05))
    cache = PoolCache(s.layers, B, s.kv_heads, s.head_dim, prompt + steps + 1)
    loop = DL.DecodeLoop(s, w, cache, B, prompt + steps + 1, DEV, use_graphs=graphs, temperature=0.0)
    ids = torch.randint(0, s.vocab, (B, prompt), generator=torch.Generator().manual_seed(7)).to(DEV)
    tok = loop.prefill(ids)
    toks, logits = [tok], []
    for _ in range(steps):
        tok = loop.step(tok)
        toks.append(tok)
        logits.append(loop.logits.clone())
    cache.check()
    w.check()
    return ids, torch.stack(toks, 1), logits, loop


def test_graphs_equal_eager():
    _, t1, l1, _ = run(True, 24)
    _, t2, l2, _ = run(False, 24)
    assert torch.equal(t1, t2)
    for a, b in zip(l1, l2):
        assert torch.equal(a, b)


def test_loop_follows_a_forward_over_all_tokens():
    """The steps' logits against the prompt's form over the loop's own tokens.  The two round q, k and the attention's outputs
    to bf16 in different places, and a quantiser makes a step of its own of any difference that crosses the middle of two
    codes; what the steps' and the prompt's quantisers do to a product is at most independent.  An element of a product's
    rows is off by up to 2^-4 of itself, evenly spread: 2^-4 / sqrt(3) rms, sqrt(2) of that for the difference of two, and
    as much of the product's output, a sum of such errors.  Nine products, added in squares: 3 * 0.051 = 0.153 of the
    logits, in norm.  (The first bound written here, 0.05 of the largest logit for every one of them, took the
    difference at each quantiser to be bf16's rounding, where it is what the quantisers before have made of that: the
    largest of 2000 logits was 0.076 off.)"""
    steps = 24
    ids, toks, logits, loop = run(True, steps)
    w = loop.w
    seq = torch.cat([ids, toks[:, :steps]], 1)
    T = seq.shape[1]
    x = F.embedding(seq, w.embed)
    for L in w.layers:
        q, k, v = loop._qkv(x, L, loop.cos[:T], loop.sin[:T])
        o = F.scaled_dot_product_attention(q.transpose(1, 2).float(), k.transpose(1, 2).float(), v.transpose(1, 2).float(),
                                           is_causal=True, enable_gqa=True).to(torch.bfloat16)
        x = loop._post_attn(x, o.transpose(1, 2), L)
    ref = loop._lm(x).view(*seq.shape, -1)
    for i in range(steps):
        want = ref[:, ids.shape[1] + i]
        assert (logits[i] - want).norm().item() <= 0.153 * want.norm().item(), i


def test_a_layer_is_its_operators():
    """_segment's 8-bit form against the same quantities from dequantised tensors in 64 bits, stage by stage on the loop's own
    buffers: 2^-8 of the sum of magnitudes covers bf16's half step and the fp32 sums."""
    _, _, _, loop = run(False, 2)
    s, L = SMALL, loop.w.layers[1]
    loop._segment(2)     # layer 1's second half, final norm and head, once more on the buffers as they are

    def value(rows8):
        q, scale = rows8
        return q.double() * scale.double().repeat_interleave(128, 1)[:, : q.shape[1]]

    act, h = value(loop.act8), value(loop.h8)
    down, head = L["down"].dequantize().double(), loop.w.lm_head.dequantize().double()
    assert ((loop.h.double() - act @ down.t()).abs() <= 2.0 ** -8 * (act.abs() @ down.abs().t())).all()
    assert ((loop.logits.double() - h @ head.t()).abs() <= 2.0 ** -16 * (h.abs() @ head.abs().t())).all()
    x = loop.hidden.view(-1, s.hidden).double()
    y = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + s.rms_eps)
    assert ((h - y).abs() <= 2.0 ** -4 * y.abs() * (1 + 2.0 ** -15) + 2.0 ** -10 * loop.h8[1].double().repeat_interleave(128, 1)[:, : s.hidden]).all()


def test_weights_in_8_bits_stand_for_the_weights():
    w = DL.Weights(SMALL, DEV, seed=3)
    q = DL.Fp8Weights(w)
    for L, Q in zip(w.layers, q.layers):
        for name in ("wqkv", "wo", "gate_up", "down"):
            got, want = Q[name].dequantize(), L[name].float()
            assert isinstance(Q[name], ops.Fp8Weight)
            # half a step of the element, or of the smallest step of its block (whose largest is at most the matrix's)
            assert ((got - want).abs() <= 2.0 ** -4 * want.abs() + 2.0 ** -10 * want.abs().max() / 448).all()


def test_the_command(capsys):
    DL.main(["--layers", "1", "--batch", "2", "--prompt", "16", "--steps", "3", "--fp8"])
    assert "e4m3 weights, batch 2" in capsys.readouterr().out
