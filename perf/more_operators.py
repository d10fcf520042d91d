"""Measured cases of a decoder layer's dense half in 8 bits: e4m3 elements with an fp32 scale for each block of 128.

Four operators, in the order in which a layer runs them (a block is 128 consecutive elements of a row, the last perhaps
shorter; a row of K elements has ceil(K / 128) scales):

  norm     the residual's addition (rounded to its type), the root-mean-square norm of the sum, and its output in e4m3
  quant    16-bit rows (an attention's output) to e4m3: scale = largest magnitude / 448, element = e4m3(x / scale)
  linear   x w^T of e4m3 rows and e4m3 weights, the weights' scales for blocks of 128 x 128; 16-bit or fp32 out
  swiglu   both halves g, u of a gated block's first product, silu(g) * u, and its output in e4m3

`run` computes them from elementary torch operations in 32 bits, or (where `own` is true) by the calls a user makes.  Row
scales [tokens, blocks] lie block-major in memory, as the operators write them ("rows": row-major, as other programs may).
"""
import math

import torch

own = False

DEV = "cuda"
F8 = torch.float8_e4m3fn
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
FP8_MAX = 448.0
BLOCK = 128
EPS = 1e-6


def listed():
    return [
        # the attention's output of a decode step of 8 requests: all latency
        dict(name="quant_step", op="quant", tokens=8, dim=4096, dtype="bf16"),
        # the same of a long prompt, an odd count
        dict(name="quant_prompt", op="quant", tokens=16383, dim=4096, dtype="bf16"),
        # a decode step of 32 requests between two products
        dict(name="norm_step", op="norm", tokens=32, dim=4096, dtype="bf16", residual=True),
        # a chunk of prompts
        dict(name="norm_prompt", op="norm", tokens=16384, dim=4096, dtype="bf16", residual=True),
        # one request's token through the fused QKV projection
        dict(name="linear_one", op="linear", tokens=1, out=6144, dim=4096, dtype="bf16", rows=False),
        # a decode step of 32 requests through the down projection
        dict(name="linear_step", op="linear", tokens=32, out=4096, dim=12288, dtype="bf16", rows=False),
        # the same step's logits over the vocabulary, fp32
        dict(name="linear_logits", op="linear", tokens=32, out=151936, dim=4096, dtype="fp32", rows=False),
        # a short prompt of an odd length, scales row-major
        dict(name="linear_short", op="linear", tokens=333, out=4096, dim=4096, dtype="bf16", rows=True),
        # a chunk of prompts through the fused QKV projection
        dict(name="linear_prompt", op="linear", tokens=4096, out=6144, dim=4096, dtype="bf16", rows=False),
        # a decode step of 8 requests through the gated block's first half
        dict(name="swiglu_step", op="swiglu", tokens=8, ffn=12288, dim=4096, rows=False),
        # a batch of 100 requests
        dict(name="swiglu_batch", op="swiglu", tokens=100, ffn=12288, dim=4096, rows=False),
        # a long prompt of an odd length, the largest
        dict(name="swiglu_prompt", op="swiglu", tokens=8191, ffn=12288, dim=4096, rows=False),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(["quant", "norm", "linear", "linear", "linear", "swiglu", "swiglu"])
    # whole 16-byte rows; a half of the sizes in whole blocks, as most models have them
    dim = 16 * _log_int(rng, 8, 768)
    if rng.random() < 0.5:
        dim = BLOCK * max(1, dim // BLOCK)
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    if op in ("quant", "norm"):
        tokens = _log_int(rng, 1, 16384 * 4096 // dim)
        got = dict(op=op, tokens=tokens, dim=dim, dtype=dtype)
        return got if op == "quant" else dict(got, residual=rng.random() < 0.7)
    most = 8191 * 2 * 12288 * 4096  # tokens * out * dim of the largest listed case
    rows = rng.random() < 0.25
    if op == "linear":
        out = _log_int(rng, 1, 32768)
        if rng.random() < 0.6:
            out = 64 * max(1, out // 64)
        tokens = _log_int(rng, 1, min(16384, most // (out * dim)))
        return dict(op=op, tokens=tokens, out=out, dim=dim, dtype=rng.choice([dtype, dtype, "fp32"]), rows=rows)
    ffn = 16 * _log_int(rng, 2, 1024)
    return dict(op=op, tokens=_log_int(rng, 1, min(16384, most // (2 * ffn * dim))), ffn=ffn, dim=dim, rows=rows)


def _blocks(n):
    return (n + BLOCK - 1) // BLOCK


def _rows(gen, tokens, dim):
    """Activations: normal, a few channels some twenty times as large, tokens of different sizes, one in 50 a padded zero."""
    x = torch.randn(tokens, dim, generator=gen, device=DEV)
    x[:, torch.randint(0, dim, (max(1, dim // 512),), generator=gen, device=DEV)] *= 20.0
    x *= torch.exp(torch.randn(tokens, 1, generator=gen, device=DEV) * 0.7)
    return x * (torch.rand(tokens, 1, generator=gen, device=DEV) > 0.02)


def _weights(gen, out, dim):
    """e4m3 [out, dim] and fp32 scales [blocks of out, blocks of dim] of normal weights whose size varies with the row."""
    w = torch.randn(out, dim, generator=gen, device=DEV) * 0.02
    w *= torch.exp(torch.randn(out, 1, generator=gen, device=DEV) * 0.3)
    pad = torch.zeros(_blocks(out) * BLOCK, _blocks(dim) * BLOCK, device=DEV)
    pad[:out, :dim] = w
    del w
    tile = pad.view(_blocks(out), BLOCK, _blocks(dim), BLOCK)
    scale = tile.abs().amax(dim=(1, 3)) / FP8_MAX
    q = (tile / scale[:, None, :, None].clamp(min=1e-30)).view_as(pad)[:out, :dim].to(F8).contiguous()
    return q, scale.contiguous()


def _scale_buffer(tokens, dim, rows):
    n = _blocks(dim)
    if rows:
        return torch.empty(tokens, n, device=DEV)
    return torch.empty(n, tokens, device=DEV).t()


def _handle(st, parts):
    """The weights' handle, made once when they are loaded and kept with them, as a serving program does (it holds
    addresses and sizes, nothing of the data)."""
    if own:
        from zoomkv_revision_b200 import ops
        st["weight"] = ops.Fp8Weight(st["w"], st["w_scale"], parts=parts)
    return st


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    op, T, D = case["op"], case["tokens"], case["dim"]
    if op in ("quant", "norm"):
        dt = DTYPES[case["dtype"]]
        # the buffers of a program that replays its steps
        st = dict(op=op, x=_rows(gen, T, D).to(dt), q=torch.empty(T, D, dtype=F8, device=DEV), scale=_scale_buffer(T, D, False))
        if op == "norm":
            st["w"] = (1.0 + 0.2 * torch.randn(D, generator=gen, device=DEV)).to(dt)
            st["residual"] = (_rows(gen, T, D) * 3.0).to(dt) if case["residual"] else None
            st["sum"] = torch.empty(T, D, dtype=dt, device=DEV) if case["residual"] else None
        return st
    q, scale = _plain_quant(_rows(gen, T, D))
    x_scale = _scale_buffer(T, D, case["rows"])
    x_scale.copy_(scale)
    st = dict(op=op, x=q, x_scale=x_scale)
    if op == "linear":
        st["w"], st["w_scale"] = _weights(gen, case["out"], D)
        st["out"] = torch.empty(T, case["out"], dtype=DTYPES[case["dtype"]], device=DEV)
        return _handle(st, 1)
    F = case["ffn"]
    gate, up = _weights(gen, F, D), _weights(gen, F, D)
    # one tensor, gate rows before up rows; each half has blocks of its own
    st["w"], st["w_scale"] = torch.cat([gate[0].view(torch.uint8), up[0].view(torch.uint8)]).view(F8), torch.cat([gate[1], up[1]])
    st["q"], st["scale"] = torch.empty(T, F, dtype=F8, device=DEV), _scale_buffer(T, F, False)
    return _handle(st, 2)


# ---------------------------------------------------------------- plain forms
def _plain_quant(x):
    """e4m3 [tokens, n] and scales [tokens, blocks] of fp32 rows."""
    T, n = x.shape
    nb = _blocks(n)
    if n % BLOCK:
        x = torch.cat([x, x.new_zeros(T, nb * BLOCK - n)], 1)
    x = x.view(T, nb, BLOCK)
    amax = x.abs().amax(-1)
    scale = amax / torch.full_like(amax, FP8_MAX)
    q = x / scale[..., None]
    q = torch.where(scale[..., None] == 0, torch.zeros_like(q), q).clamp(-FP8_MAX, FP8_MAX)
    return q.view(T, nb * BLOCK)[:, :n].to(F8).contiguous(), scale


def _plain_norm(s):
    x = s["x"].float()
    if s["residual"] is not None:
        s["sum"].copy_(x + s["residual"].float())
        x = s["sum"].float()
    y = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * s["w"].float()
    return _plain_quant(y)


def _spread(scale, n, dim):
    return scale.repeat_interleave(BLOCK, dim).narrow(dim, 0, n)


def _plain_product(x, x_scale, w, w_scale):
    N, K = w.shape
    wide = w.float()
    wide *= _spread(_spread(w_scale, N, 0), K, 1)
    return torch.matmul(x.float() * _spread(x_scale, K, 1), wide.t())


def _own(s):
    """The calls a user makes."""
    from zoomkv_revision_b200 import ops
    if s["op"] == "quant":
        ops.quant_fp8(s["x"], out=s["q"], scale=s["scale"])
        return dict(q=s["q"], scale=s["scale"])
    if s["op"] == "norm":
        ops.rmsnorm_fp8(s["x"], s["w"], EPS, residual=s["residual"], residual_out=s["sum"], out=s["q"], scale=s["scale"])
        return dict(q=s["q"], scale=s["scale"], sum=s["sum"])
    if s["op"] == "linear":
        return ops.fp8_linear(s["x"], s["x_scale"], s["weight"], out=s["out"])
    ops.fp8_swiglu(s["x"], s["x_scale"], s["weight"], out=s["q"], scale=s["scale"])
    return dict(q=s["q"], scale=s["scale"])


def run(state):
    if own:
        return _own(state)
    s = state
    if s["op"] == "quant":
        q, scale = _plain_quant(s["x"].float())
        return dict(q=q, scale=scale)
    if s["op"] == "norm":
        q, scale = _plain_norm(s)
        return dict(q=q, scale=scale, sum=s["sum"])
    if s["op"] == "linear":
        return _plain_product(s["x"], s["x_scale"], s["w"], s["w_scale"]).to(s["out"].dtype)
    F, nb = s["w"].shape[0] // 2, s["w_scale"].shape[0] // 2
    g = _plain_product(s["x"], s["x_scale"], s["w"][:F], s["w_scale"][:nb])
    u = _plain_product(s["x"], s["x_scale"], s["w"][F:], s["w_scale"][nb:])
    q, scale = _plain_quant(g / (1.0 + torch.exp(-g)) * u)
    return dict(q=q, scale=scale)


# ---------------------------------------------------------------- work and the definitions in 64 bits
def work(case):
    T, D = case["tokens"], case["dim"]
    row = D + 4 * _blocks(D)
    if case["op"] == "quant":
        return dict(bytes=T * (2 * D + row), flops=0)
    if case["op"] == "norm":
        return dict(bytes=T * (2 * D + row) + (4 * T * D if case["residual"] else 0) + 2 * D, flops=0)
    if case["op"] == "linear":
        N = case["out"]
        return dict(bytes=T * row + N * D + 4 * _blocks(N) * _blocks(D) + T * N * (4 if case["dtype"] == "fp32" else 2),
                    flops=2 * T * N * D)
    F = case["ffn"]
    return dict(bytes=T * row + 2 * F * D + 8 * _blocks(F) * _blocks(D) + T * (F + 4 * _blocks(F)), flops=4 * T * F * D)


def _exact_quant(y):
    """Elements before their rounding, and scales, of 64-bit rows."""
    T, n = y.shape
    q, scales = torch.zeros_like(y), y.new_zeros(T, _blocks(n))
    for b in range(_blocks(n)):
        part = slice(b * BLOCK, min(n, (b + 1) * BLOCK))
        scales[:, b] = torch.amax(torch.abs(y[:, part]), -1) / FP8_MAX
        q[:, part] = torch.nan_to_num(y[:, part] / scales[:, b, None], nan=0.0)
    return dict(q=q, scale=scales)


def exact(case, seed):
    """From the definitions in 64 bits; None for products that would take too long."""
    T, D = case["tokens"], case["dim"]
    if case["op"] in ("linear", "swiglu") and T * D * (case["out"] if case["op"] == "linear" else 2 * case["ffn"]) > 1.2e11:
        return None
    s = prepare(case, seed)
    if case["op"] == "quant":
        return _exact_quant(s["x"].to(torch.float64))
    if case["op"] == "norm":
        r = s["x"].to(torch.float64)
        if s["residual"] is not None:  # the sum is kept in its type, and the norm is that of the sum as it is kept
            r = (r + s["residual"].to(torch.float64)).to(s["x"].dtype).to(torch.float64)
        got = _exact_quant(r / torch.sqrt(torch.sum(r * r, -1, keepdim=True) / D + EPS) * s["w"].to(torch.float64))
        return dict(got, sum=None if s["residual"] is None else r)

    def product(rows, blocks):
        """Block by block of the inner dimension."""
        w, w_scale = s["w"][rows], s["w_scale"][blocks]
        y = torch.zeros(T, w.shape[0], dtype=torch.float64, device=DEV)
        of_row = torch.arange(w.shape[0], device=DEV) // BLOCK
        for b in range(_blocks(D)):
            part = slice(b * BLOCK, min(D, (b + 1) * BLOCK))
            y.addmm_(s["x"][:, part].to(torch.float64) * s["x_scale"][:, b, None].to(torch.float64),
                     (w[:, part].to(torch.float64) * w_scale[of_row, b, None].to(torch.float64)).t())
        return y

    if case["op"] == "linear":
        return product(slice(None), slice(None))
    F, nb = case["ffn"], _blocks(case["ffn"])
    g, u = product(slice(0, F), slice(0, nb)), product(slice(F, None), slice(nb, None))
    return _exact_quant(g * torch.sigmoid(g) * u)
