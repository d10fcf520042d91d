"""GPU: a decode step's segment with 8-bit weights, stage by stage against
64-bit arithmetic on what the stage before it stored.  Tolerances are those of
test_gpu_fp8.py; its bound for the products takes any order of the sums."""
import pytest
import torch

from test_gpu_fp8 import BF, DEV, NORM_E, check_linear, check_stored, check_swiglu, gen, rows
from zoomkv_revision_b200 import decode_loop as DL
from zoomkv_revision_b200 import ops
from zoomkv_revision_b200.pool_cache import PoolCache

pytestmark = pytest.mark.gpu
SHAPE = DL.Shape(hidden=528, layers=3, heads=6, kv_heads=2, head_dim=128, ffn=1040, vocab=1000)


def norm64(x, w, eps):
    x = x.double()
    return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + eps) * w.double()


def equal8(a, b):
    return torch.equal(a[0].view(torch.uint8), b[0].view(torch.uint8)) and torch.equal(a[1], b[1])


@pytest.mark.parametrize("B", [1, 5, 40, 70])
@pytest.mark.parametrize("graphs", [False, True])
def test_a_segment(B, graphs):
    s = SHAPE
    w = DL.Weights(s, DEV, seed=5, std=0.05)
    for L in w.layers:   # norms that are not all ones
        for name in ("in_norm", "post_norm"):
            L[name].copy_((1 + 0.3 * torch.randn(s.hidden, generator=gen(6), device=DEV)).to(BF))
    w = DL.Fp8Weights(w)
    loop = DL.DecodeLoop(s, w, PoolCache(s.layers, B, s.kv_heads, s.head_dim, 64), B, 64, DEV, use_graphs=graphs)
    if graphs:
        loop._build_graphs()
    for l in range(s.layers + 1):
        x0, attn = rows(10 + l, B, s.hidden, BF), rows(20 + l, B, s.heads * s.head_dim, BF) * 0.3
        loop.hidden.copy_(x0.view_as(loop.hidden))
        loop.attn.copy_(attn.view_as(loop.attn))
        loop.graphs[l].replay() if graphs else loop._segment(l)
        x = x0
        if l > 0:
            L = w.layers[l - 1]
            a8 = ops.quant_fp8(attn)
            assert equal8(loop.attn8, a8)
            proj = ops.fp8_linear(*a8, L["wo"])
            check_linear(proj, *a8, L["wo"])
            x = (x.float() + proj.float()).to(BF)            # the residual stream after the attention
            kept = x0.clone()
            h8 = ops.rmsnorm_fp8(proj, L["post_norm"], s.rms_eps, residual=kept)
            assert torch.equal(kept, x)
            y = norm64(x, L["post_norm"], s.rms_eps)
            check_stored(*h8, y, NORM_E * y.abs(), NORM_E)
            check_swiglu(*loop.act8, *h8, L["gate_up"])
            check_linear(loop.h, *loop.act8, L["down"])
            x = (x.float() + loop.h.float()).to(BF)          # and after the layer, in the norm that follows
        assert torch.equal(loop.hidden.view(B, -1), x)
        y = norm64(x, w.layers[l]["in_norm"] if l < s.layers else w.norm, s.rms_eps)
        check_stored(*loop.h8, y, NORM_E * y.abs(), NORM_E)
        if l < s.layers:
            check_linear(loop.qkv, *loop.h8, w.layers[l]["wqkv"])
            assert torch.equal(loop.v.view(B, -1), loop.qkv[:, (s.heads + s.kv_heads) * s.head_dim:])
        else:
            check_linear(loop.logits, *loop.h8, w.lm_head)
    w.check()
