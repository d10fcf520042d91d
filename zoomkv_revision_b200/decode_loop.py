"""Decode-loop caller of the sparse attention path (the benchmark's config 4).

The reference's loop is a Qwen3 decoder whose attention is the polar_cache
plugin: model_hub/LLM.py:208-294 (layer_decode, prefill/decode_forward),
:398-446 (inference_cot), :63-110 (sample_next_token) and model_hub/qwen.py:
429-612 (embedding, fused QKV with per-head q/k RMSNorm, neox RoPE, o_proj,
SwiGLU MLP, LM head).  This module is that caller around this package's
drop-in cache:

  * weights of the Qwen3-8B shape are random-initialised (no checkpoint is
    available), bf16; projections are library GEMMs (torch / cuBLAS);
  * per layer and step: RMSNorm -> QKV -> q/k RMSNorm -> RoPE ->
    cache.decode_update_kv_cache(k, v, layer) -> cache.compute(q, layer) ->
    o_proj + residual -> RMSNorm -> MLP + residual, as layer_decode does;
  * the dense segments between two attention calls (o_proj, MLP, the next
    layer's norm, QKV and RoPE) are replayed as one CUDA graph per layer, the
    RoPE position read from a device counter, so a step issues 36 graph
    launches plus the attention calls, whose arguments change every step;
  * with Fp8Weights the dense half runs in 8 bits (e4m3, scales for blocks of
    128), which halves the weights that a step reads; the reference has no
    such mode (python -m zoomkv_revision_b200.decode_loop --fp8 times it);
  * sampling: temperature, top-k, top-p (nucleus), as sample_next_token,
    with a seeded generator.
"""
from __future__ import annotations

import argparse
from dataclasses import dataclass
from typing import Optional

import torch
import torch.nn.functional as F

from . import ops


@dataclass
class Shape:
    hidden: int = 4096
    layers: int = 36
    heads: int = 32
    kv_heads: int = 8
    head_dim: int = 128
    ffn: int = 12288
    vocab: int = 151936
    rms_eps: float = 1e-6
    rope_theta: float = 1_000_000.0


QWEN3_8B = Shape()


def rmsnorm(x: torch.Tensor, w: torch.Tensor, eps: float) -> torch.Tensor:
    """RMSNorm in fp32, result in x's dtype (as flashinfer.rmsnorm)."""
    xf = x.float()
    return (xf * torch.rsqrt(xf.pow(2).mean(-1, keepdim=True) + eps) * w.float()).to(x.dtype)


def rope_tables(shape: Shape, max_pos: int, device) -> tuple[torch.Tensor, torch.Tensor]:
    """cos / sin [max_pos, head_dim/2] of the neox rotation (qwen.py:131-140)."""
    half = shape.head_dim // 2
    inv = 1.0 / (shape.rope_theta ** (torch.arange(0, half, device=device, dtype=torch.float32) / half))
    t = torch.arange(max_pos, device=device, dtype=torch.float32)
    f = torch.outer(t, inv)
    return f.cos(), f.sin()


def apply_rope(x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor) -> torch.Tensor:
    """x [..., seq, heads, head_dim]; cos/sin [seq, head_dim/2]: rotate_half
    form (qwen.py:579-592), computed in fp32."""
    half = x.shape[-1] // 2
    xf = x.float()
    x1, x2 = xf[..., :half], xf[..., half:]
    c = cos[:, None, :]
    s = sin[:, None, :]
    return torch.cat((x1 * c - x2 * s, x2 * c + x1 * s), dim=-1).to(x.dtype)


def sample_next_token(logits: torch.Tensor, temperature: float, top_p: float, top_k: int,
                      generator: Optional[torch.Generator] = None) -> torch.Tensor:
    """LLM.py:63-110: greedy below temperature 1e-5, else temperature, top-k
    mask, nucleus mask (tokens whose preceding cumulative probability already
    exceeds top_p are removed; the first is always kept), multinomial over
    the survivors."""
    if logits.dim() == 3:
        logits = logits.squeeze(1)
    if temperature < 1e-5:
        return logits.argmax(dim=-1)
    logits = logits / temperature
    if top_k > 0:
        # the top-k survivors, sorted; the nucleus mask over them equals the
        # mask over the whole row (masked tokens have probability 0), apart
        # from exact ties at the k-th logit
        vals, idx = torch.topk(logits, min(top_k, logits.size(-1)), dim=-1)
    else:
        vals, idx = torch.sort(logits, descending=True, dim=-1)
    if 0.0 < top_p < 1.0:
        cum = torch.cumsum(F.softmax(vals, dim=-1), dim=-1)
        remove = cum > top_p
        remove[..., 1:] = remove[..., :-1].clone()
        remove[..., 0] = False
        vals = vals.masked_fill(remove, float("-inf"))
    pick = torch.multinomial(F.softmax(vals, dim=-1), 1, generator=generator)
    return idx.gather(-1, pick).squeeze(-1)


class Weights:
    """Random-initialised Qwen3 weights (N(0, std), norms at 1), bf16."""

    def __init__(self, shape: Shape, device, seed: int = 0, std: float = 0.02):
        g = torch.Generator(device=device).manual_seed(seed)
        bf = torch.bfloat16
        H, D, KV = shape.hidden, shape.head_dim, shape.kv_heads

        def w(*s):
            return (torch.randn(*s, generator=g, device=device, dtype=torch.float32) * std).to(bf)

        self.embed = w(shape.vocab, H)
        self.lm_head = w(shape.vocab, H)
        self.norm = torch.ones(H, device=device, dtype=bf)
        self.layers = []
        for _ in range(shape.layers):
            self.layers.append(dict(
                in_norm=torch.ones(H, device=device, dtype=bf),
                post_norm=torch.ones(H, device=device, dtype=bf),
                q_norm=torch.ones(D, device=device, dtype=bf),
                k_norm=torch.ones(D, device=device, dtype=bf),
                wqkv=w((shape.heads + 2 * KV) * D, H),
                wo=w(H, shape.heads * D),
                gate_up=w(2 * shape.ffn, H),
                down=w(H, shape.ffn),
            ))


class Fp8Weights:
    """The same weights in 8 bits: every product's matrix e4m3 with a scale for each block of 128 x 128 (ops.Fp8Weight), the
    embedding and the norms as they are.  `of`: any Weights, whose matrices are let go layer by layer where `consume` is
    true."""

    def __init__(self, of: Weights, consume: bool = False):
        self.embed, self.norm = of.embed, of.norm
        self.lm_head = ops.Fp8Weight.quantize(of.lm_head)
        self.layers = []
        for L in of.layers:
            self.layers.append(dict(
                in_norm=L["in_norm"], post_norm=L["post_norm"], q_norm=L["q_norm"], k_norm=L["k_norm"],
                wqkv=ops.Fp8Weight.quantize(L["wqkv"]), wo=ops.Fp8Weight.quantize(L["wo"]),
                gate_up=ops.Fp8Weight.quantize(L["gate_up"], 2), down=ops.Fp8Weight.quantize(L["down"])))
            if consume:
                L.clear()

    def check(self) -> None:
        """Raises if a wait inside a product ran out (waits for the GPU, all streams)."""
        for L in self.layers:
            for name in ("wqkv", "wo", "gate_up", "down"):
                L[name].check()
        self.lm_head.check()


class DecodeLoop:
    """A Qwen3-shape decoder over `cache` (the polar_cache drop-in, built
    with the same layer count, batch and heads).  prefill(prompt) then
    step() per generated token; `use_graphs` replays the dense segments as
    CUDA graphs.  With Fp8Weights the dense segments run in 8 bits: the norms
    (with the residual's addition) and the attention's output are quantised in
    blocks of 128 and multiplied with e4m3 weights, and the gate and up
    products, SiLU and their product are one kernel; the residual stream, q, k,
    v and the attention stay 16-bit, the logits fp32."""

    def __init__(self, shape: Shape, weights: Weights, cache, batch: int, max_pos: int, device,
                 use_graphs: bool = True, temperature: float = 0.6, top_p: float = 0.95, top_k: int = 20,
                 seed: int = 42):
        self.s, self.w, self.cache, self.B = shape, weights, cache, batch
        self.dev = torch.device(device)
        self.cos, self.sin = rope_tables(shape, max_pos, self.dev)
        self.temperature, self.top_p, self.top_k = temperature, top_p, top_k
        self.gen = torch.Generator(device=self.dev).manual_seed(seed)
        self.use_graphs = use_graphs
        bf = torch.bfloat16
        H, D = shape.hidden, shape.head_dim
        # static buffers of the decode step
        self.pos = torch.zeros(1, dtype=torch.long, device=self.dev)        # RoPE position of the new token
        self.hidden = torch.zeros(batch, 1, H, dtype=bf, device=self.dev)   # residual stream
        self.q = torch.zeros(batch, 1, shape.heads, D, dtype=bf, device=self.dev)
        self.k = torch.zeros(batch, 1, shape.kv_heads, D, dtype=bf, device=self.dev)
        self.v = torch.zeros_like(self.k)
        self.attn = torch.zeros(batch, 1, shape.heads, D, dtype=bf, device=self.dev)
        self.logits = torch.zeros(batch, shape.vocab, dtype=torch.float32, device=self.dev)
        self.h = torch.zeros(batch, H, dtype=bf, device=self.dev)                  # normed activations
        self.qkv = torch.zeros(batch, (shape.heads + 2 * shape.kv_heads) * D, dtype=bf, device=self.dev)
        self.gu = torch.zeros(batch, 2 * shape.ffn, dtype=bf, device=self.dev)
        self.act = torch.zeros(batch, shape.ffn, dtype=bf, device=self.dev)
        self.lg = torch.zeros(batch, shape.vocab, dtype=bf, device=self.dev)
        self.fp8 = isinstance(weights, Fp8Weights)
        if self.fp8:
            def rows8(n):   # e4m3 rows and their scales
                return (torch.zeros(batch, n, dtype=torch.float8_e4m3fn, device=self.dev),
                        torch.zeros(-(-n // 128), batch, device=self.dev).t())
            self.attn8, self.h8, self.act8 = rows8(shape.heads * D), rows8(H), rows8(shape.ffn)
        self.graphs: list = []
        self.position = 0

    # ------------------------------------------------------------------ pieces
    def _qkv(self, x: torch.Tensor, L: dict, pos_cos: torch.Tensor, pos_sin: torch.Tensor):
        """x [B, T, H] -> q [B, T, heads, D], k / v [B, T, kv, D] (qwen.py:439-453, :550-612)."""
        s = self.s
        B, T, _ = x.shape
        if self.fp8:
            qkv = ops.fp8_linear(*ops.rmsnorm_fp8(x, L["in_norm"], s.rms_eps), L["wqkv"])
        else:
            qkv = F.linear(rmsnorm(x, L["in_norm"], s.rms_eps), L["wqkv"])
        q, k, v = qkv.split([s.heads * s.head_dim, s.kv_heads * s.head_dim, s.kv_heads * s.head_dim], dim=-1)
        q = rmsnorm(q.reshape(B, T, s.heads, s.head_dim), L["q_norm"], s.rms_eps)
        k = rmsnorm(k.reshape(B, T, s.kv_heads, s.head_dim), L["k_norm"], s.rms_eps)
        v = v.reshape(B, T, s.kv_heads, s.head_dim)
        return apply_rope(q, pos_cos, pos_sin), apply_rope(k, pos_cos, pos_sin), v

    def _post_attn(self, x: torch.Tensor, attn: torch.Tensor, L: dict) -> torch.Tensor:
        """o_proj + residual, RMSNorm, SwiGLU MLP + residual (LLM.py:240-249)."""
        s = self.s
        B, T = attn.shape[:2]
        if self.fp8:
            x = x.clone()
            proj = ops.fp8_linear(*ops.quant_fp8(attn.reshape(B, T, s.heads * s.head_dim)), L["wo"])
            h = ops.rmsnorm_fp8(proj, L["post_norm"], s.rms_eps, residual=x)
            act, scale = ops.fp8_swiglu(*h, L["gate_up"])
            return x + ops.fp8_linear(act, scale, L["down"])
        x = x + F.linear(attn.reshape(B, T, s.heads * s.head_dim), L["wo"])
        h = rmsnorm(x, L["post_norm"], s.rms_eps)
        gu = F.linear(h, L["gate_up"])
        g, u = gu.split(s.ffn, dim=-1)
        return x + F.linear(F.silu(g) * u, L["down"])

    def _lm(self, x: torch.Tensor) -> torch.Tensor:
        if self.fp8:
            return ops.fp8_linear(*ops.rmsnorm_fp8(x, self.w.norm, self.s.rms_eps), self.w.lm_head, dtype=torch.float32)
        return F.linear(rmsnorm(x, self.w.norm, self.s.rms_eps), self.w.lm_head).float()

    # ------------------------------------------------------------------ prefill
    @torch.no_grad()
    def prefill(self, prompt: torch.Tensor) -> torch.Tensor:
        """prompt [B, T] token ids -> the first generated token [B]
        (prefill_forward, LLM.py:252-276, with causal attention over the
        prompt; the K/V go to the cache by prefill_update_kv_cache)."""
        s = self.s
        B, T = prompt.shape
        x = F.embedding(prompt, self.w.embed)
        cos, sin = self.cos[:T], self.sin[:T]
        for l, L in enumerate(self.w.layers):
            q, k, v = self._qkv(x, L, cos, sin)
            self.cache.prefill_update_kv_cache(None, k, v, l, 0)
            rep = s.heads // s.kv_heads
            o = F.scaled_dot_product_attention(q.transpose(1, 2), k.transpose(1, 2).repeat_interleave(rep, 1),
                                               v.transpose(1, 2).repeat_interleave(rep, 1), is_causal=True)
            x = self._post_attn(x, o.transpose(1, 2), L)
        logits = self._lm(x[:, -1:])
        self.position = T
        self.pos.fill_(T)
        return sample_next_token(logits, self.temperature, self.top_p, self.top_k, self.gen)

    # ------------------------------------------------------------------ decode
    def _segment(self, l: int) -> None:
        """Dense work between attention calls: layer l-1's post-attention
        part (l > 0) and layer l's pre-attention part (l < layers); with
        l == layers the final norm and LM head.  Library GEMMs (the residual
        adds in their epilogues) and this package's fused element-wise
        kernels; every tensor is a preallocated buffer."""
        s = self.s
        x = self.hidden.view(self.B, s.hidden)
        if self.fp8:
            return self._segment8(l, x)
        if l > 0:
            L = self.w.layers[l - 1]
            x.addmm_(self.attn.view(self.B, s.heads * s.head_dim), L["wo"].t())
            ops.rmsnorm(x, L["post_norm"], s.rms_eps, out=self.h)
            torch.matmul(self.h, L["gate_up"].t(), out=self.gu)
            ops.silu_mul(self.gu, self.act)
            x.addmm_(self.act, L["down"].t())
        if l < s.layers:
            L = self.w.layers[l]
            ops.rmsnorm(x, L["in_norm"], s.rms_eps, out=self.h)
            torch.matmul(self.h, L["wqkv"].t(), out=self.qkv)
            ops.qk_norm_rope(self.qkv, L["q_norm"], L["k_norm"], self.cos, self.sin, self.pos, s.heads, s.kv_heads,
                             s.rms_eps, self.q, self.k, self.v)
        else:
            ops.rmsnorm(x, self.w.norm, s.rms_eps, out=self.h)
            torch.matmul(self.h, self.w.lm_head.t(), out=self.lg)
            self.logits.copy_(self.lg)

    def _segment8(self, l: int, x: torch.Tensor) -> None:
        """The same in 8 bits.  A product's output is added to the residual stream by the norm that follows it."""
        s, proj = self.s, None
        if l > 0:
            L = self.w.layers[l - 1]
            ops.quant_fp8(self.attn.view(self.B, s.heads * s.head_dim), out=self.attn8[0], scale=self.attn8[1])
            ops.fp8_linear(*self.attn8, L["wo"], out=self.h)
            ops.rmsnorm_fp8(self.h, L["post_norm"], s.rms_eps, residual=x, out=self.h8[0], scale=self.h8[1])
            ops.fp8_swiglu(*self.h8, L["gate_up"], out=self.act8[0], scale=self.act8[1])
            proj = ops.fp8_linear(*self.act8, L["down"], out=self.h)
        w = self.w.layers[l]["in_norm"] if l < s.layers else self.w.norm
        ops.rmsnorm_fp8(x if proj is None else proj, w, s.rms_eps, residual=None if proj is None else x, out=self.h8[0],
                        scale=self.h8[1])
        if l < s.layers:
            L = self.w.layers[l]
            ops.fp8_linear(*self.h8, L["wqkv"], out=self.qkv)
            ops.qk_norm_rope(self.qkv, L["q_norm"], L["k_norm"], self.cos, self.sin, self.pos, s.heads, s.kv_heads,
                             s.rms_eps, self.q, self.k, self.v)
        else:
            ops.fp8_linear(*self.h8, self.w.lm_head, out=self.logits)

    def _build_graphs(self) -> None:
        side = torch.cuda.Stream(device=self.dev)
        side.wait_stream(torch.cuda.current_stream(self.dev))
        with torch.cuda.stream(side):
            for l in range(self.s.layers + 1):   # warm-up on the capture stream
                self._segment(l)
        torch.cuda.current_stream(self.dev).wait_stream(side)
        torch.cuda.synchronize(self.dev)
        pool = None
        for l in range(self.s.layers + 1):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, pool=pool):
                self._segment(l)
            pool = g.pool()
            self.graphs.append(g)

    @torch.no_grad()
    def step(self, token: torch.Tensor) -> torch.Tensor:
        """One decode step (decode_forward, LLM.py:279-294): token [B] -> next [B]."""
        s = self.s
        if self.use_graphs and not self.graphs:
            self._build_graphs()   # its warm-up pass writes the step buffers: before the embedding
        self.hidden.copy_(F.embedding(token.view(-1, 1), self.w.embed))
        run = (lambda l: self.graphs[l].replay()) if self.use_graphs else self._segment
        for l in range(s.layers):
            run(l)
            self.cache.decode_update_kv_cache(self.k, self.v, l)
            self.attn.copy_(self.cache.compute(self.q, l))
        run(s.layers)
        self.position += 1
        self.pos.add_(1)
        return sample_next_token(self.logits, self.temperature, self.top_p, self.top_k, self.gen)


def config4_cache_kwargs(shape: Shape, batch: int, prompt: int, max_new: int, device) -> dict:
    """polar_cache keywords of the benchmark's config 4: refresh every 512
    steps, dense below 2048 tokens, the reference run's sink 64 / local 256
    (run/eval_math_aime.py:202-206)."""
    return dict(valid_start=[0] * batch, layer_num=shape.layers, batch_size=batch, max_length=prompt + max_new,
                num_key_value_heads=shape.kv_heads, num_heads=shape.heads, head_dim=shape.head_dim,
                dtype=torch.bfloat16, layer_mapping={str(l): str(device) for l in range(shape.layers)},
                max_new_length=max_new, sink_size=64, local_size=256, final_topk=100,
                dynamic_update_interval=512, full_attention_threshold=2048, enable_offload=True)


def generate(shape: Shape, batch: int, prompt: int, steps: int, fp8: bool, device="cuda", seed: int = 0) -> dict:
    """`steps` decode steps after a random prompt, dense attention over the pooled cache: ms of the prompt and of a step."""
    from .pool_cache import PoolCache
    w = Weights(shape, device, seed)
    if fp8:
        w = Fp8Weights(w, consume=True)
    cache = PoolCache(shape.layers, batch, shape.kv_heads, shape.head_dim, prompt + steps + 1, device=device)
    loop = DecodeLoop(shape, w, cache, batch, prompt + steps + 1, device, seed=seed)
    ids = torch.randint(0, shape.vocab, (batch, prompt), generator=torch.Generator().manual_seed(seed)).to(device)
    ev = [torch.cuda.Event(enable_timing=True) for _ in range(4)]
    ev[0].record()
    tok = loop.prefill(ids)
    ev[1].record()
    for i in range(steps):
        if i == 1:           # the first step captures the graphs
            ev[2].record()
        tok = loop.step(tok)
    ev[3].record()
    torch.cuda.synchronize()
    cache.check()
    if fp8:
        w.check()
    return dict(prefill_ms=ev[0].elapsed_time(ev[1]), step_ms=ev[2].elapsed_time(ev[3]) / (steps - 1), tokens=tok.tolist())


def main(argv=None) -> None:
    ap = argparse.ArgumentParser(description="decode steps of a random-init Qwen3-8B over the pooled cache")
    ap.add_argument("--layers", type=int, default=QWEN3_8B.layers)
    ap.add_argument("--batch", type=int, default=32)
    ap.add_argument("--prompt", type=int, default=512)
    ap.add_argument("--steps", type=int, default=64)
    ap.add_argument("--fp8", action="store_true", help="8-bit weights and products")
    a = ap.parse_args(argv)
    if a.steps < 2:
        ap.error("--steps: two at least, the first one captures the graphs")
    got = generate(Shape(layers=a.layers), a.batch, a.prompt, a.steps, a.fp8)
    print(f"{a.layers} layers, {'e4m3' if a.fp8 else 'bf16'} weights, batch {a.batch}: prompt of {a.prompt} in "
          f"{got['prefill_ms']:.1f} ms, {got['step_ms']:.3f} ms per decode step = {a.batch / got['step_ms'] * 1e3:.0f} tokens/s")


if __name__ == "__main__":
    main()
