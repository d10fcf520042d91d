"""Measured cases of the pooled KV cache: requests of their own lengths share one pool of fixed-size blocks.

Four operators, in the order in which a serving step runs them:

  plan     lengths and new tokens per request -> new blocks from the free stack into the block table, one slot and one
           position per new token, the new lengths (whole numbers only)
  write    the new tokens' K/V rows into their slots of the pool (bf16, fp16, or e4m3 with a scale per head)
  decode   attention of one new token per request over its blocks: softmax(scale q.k) v, grouped heads, optional
           sliding window and soft cap, with the log-sum-exp of each row
  release  the blocks of finished requests back on the free stack

`run` computes them from elementary torch operations, or (where `own` is true) by the calls a user makes.  A pool is
indexed [block][token in block][kv head][dim]; "hnd" pools are laid out head before token in memory, "nhd" ones as indexed.
"""
import math

import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp8": torch.float8_e4m3fn}
FP8_MAX = 448.0


def listed():
    return [
        # one decode step of 8 requests of 32768 tokens: the smallest plan, all latency
        dict(name="plan_step", op="plan", batch=8, ctx_lo=32768, ctx_hi=32768, new_lo=1, new_hi=1, block=16),
        # admission: prompts of uneven lengths in a batch with running requests, 12 % of them idle in this step
        dict(name="plan_admit", op="plan", batch=256, ctx_lo=0, ctx_hi=8704, new_lo=0, new_hi=1024, block=16),
        # a few short requests end
        dict(name="release_few", op="release", batch=32, ctx_lo=1, ctx_hi=2048, done=0.2, block=16),
        # a long batch is cancelled
        dict(name="release_many", op="release", batch=512, ctx_lo=512, ctx_hi=8704, done=0.9, block=16),
        # the 8 new tokens of a decode step, one layer
        dict(name="write_step", op="write", tokens=8, kv_heads=8, dim=128, block=16, layout="hnd", src="bf16", pool="bf16",
             idle=0.0),
        # a chunk of prompts, one layer, K and V cut out of one projection output
        dict(name="write_prompt", op="write", tokens=16384, kv_heads=8, dim=128, block=16, layout="hnd", src="bf16",
             pool="bf16", idle=0.01),
        # the same into 8-bit blocks, token-major, an odd count
        dict(name="write_prompt_fp8", op="write", tokens=8191, kv_heads=8, dim=128, block=32, layout="nhd", src="bf16",
             pool="fp8", idle=0.01),
        # one short request: latency
        dict(name="decode_one", op="decode", batch=1, len_lo=4096, len_hi=4096, kv_heads=8, group=4, dim=128, block=16,
             layout="hnd", q="bf16", pool="bf16", window=0, softcap=0.0),
        # a serving batch of uneven requests, a few of them empty
        dict(name="decode_ragged", op="decode", batch=32, len_lo=0, len_hi=8704, kv_heads=8, group=4, dim=128, block=16,
             layout="hnd", q="bf16", pool="bf16", window=0, softcap=0.0),
        # one request of 131072 tokens: all of the GPU on 8 rows
        dict(name="decode_long", op="decode", batch=1, len_lo=131071, len_hi=131071, kv_heads=8, group=4, dim=128, block=16,
             layout="hnd", q="bf16", pool="bf16", window=0, softcap=0.0),
        # 8 requests of 32768 tokens, the largest
        dict(name="decode_32k", op="decode", batch=8, len_lo=32768, len_hi=32768, kv_heads=8, group=4, dim=128, block=16,
             layout="hnd", q="bf16", pool="bf16", window=0, softcap=0.0),
        # 8-bit blocks, token-major, uneven long requests
        dict(name="decode_fp8", op="decode", batch=32, len_lo=1000, len_hi=32768, kv_heads=8, group=4, dim=128, block=32,
             layout="nhd", q="bf16", pool="fp8", window=0, softcap=0.0),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(["plan", "release", "write", "decode", "decode", "decode"])
    block = rng.choice([16, 16, 32, 64, 128])
    if op == "plan":
        batch = _log_int(rng, 1, 512)
        new_hi = _log_int(rng, 1, 131072 // batch)
        return dict(op=op, batch=batch, ctx_lo=0, ctx_hi=_log_int(rng, 1, 32768), new_lo=rng.choice([0, 1]),
                    new_hi=new_hi, block=block)
    if op == "release":
        return dict(op=op, batch=_log_int(rng, 1, 512), ctx_lo=0, ctx_hi=_log_int(rng, 1, 8704),
                    done=rng.choice([0.1, 0.5, 1.0]), block=block)
    kv_heads = rng.choice([1, 2, 4, 8, 8, 16])
    dim = rng.choice([64, 128, 128, 128, 256])
    layout = rng.choice(["hnd", "nhd"])
    src = rng.choice(["bf16", "bf16", "fp16"])
    pool = rng.choice([src, src, "fp8"])
    if op == "write":
        return dict(op=op, tokens=_log_int(rng, 1, 16384 * 1024 // (kv_heads * dim)), kv_heads=kv_heads, dim=dim,
                    block=block, layout=layout, src=src, pool=pool, idle=rng.choice([0.0, 0.1]))
    batch = _log_int(rng, 1, 256)
    group = rng.choice([1, 2, 4, 4, 5, 7, 8, 12, 16])
    # tokens such that K and V take at most a half of the largest listed case's bytes
    most = 2 ** 28 // (batch * kv_heads * dim * 2)
    hi = _log_int(rng, 1, max(1, min(131072, most)))
    lo = rng.choice([0, hi // 2, hi])
    window = _log_int(rng, 1, hi) if rng.random() < 0.25 else 0
    return dict(op=op, batch=batch, len_lo=lo, len_hi=hi, kv_heads=kv_heads, group=group, dim=dim, block=block,
                layout=layout, q=src, pool=pool, window=window, softcap=rng.choice([0.0, 0.0, 0.0, 30.0]))


def _ints(gen, lo, hi, n):
    return torch.randint(lo, hi + 1, (n,), generator=gen, device=DEV, dtype=torch.int32)


def _table(gen, lens, block, width, n_blocks):
    """Block ids of a pool in random order, dealt to the requests; -1 past a request's last block."""
    perm = torch.randperm(n_blocks, generator=gen, device=DEV, dtype=torch.int32)
    have = (lens.long() + block - 1) // block
    start = torch.cumsum(have, 0) - have
    col = torch.arange(width, device=DEV)
    at = (start[:, None] + col).clamp(max=n_blocks - 1)
    table = torch.where(col < have[:, None], perm[at], torch.full_like(perm[at], -1))
    return table.contiguous(), perm, int(have.sum())


def _pool_pair(gen, case, n_blocks):
    """K with a few channels ten times as large (as rotated keys have), V normal; e4m3 pools with the scale of their head."""
    H, D, S, dt = case["kv_heads"], case["dim"], case["block"], DTYPES[case["pool"]]
    made = []
    for which in range(2):
        shape = (n_blocks, H, S, D) if case["layout"] == "hnd" else (n_blocks, S, H, D)
        x = torch.randn(shape, generator=gen, device=DEV)
        if which == 0:
            x[..., :4] *= 10.0
        scale = None
        if case["pool"] == "fp8":
            amax = x.abs().amax(dim=(0, 2, 3) if case["layout"] == "hnd" else (0, 1, 3)).float()
            scale = (amax / FP8_MAX).contiguous()
            x = x / (scale[:, None, None] if case["layout"] == "hnd" else scale[:, None])
        x = x.to(dt)
        made.append((x.transpose(1, 2) if case["layout"] == "hnd" else x, scale))
    return made


def _handle(st):
    """The pool's handle, made once when the pool is allocated and kept for its life, as a serving program does (it holds
    addresses and strides, nothing of the data)."""
    if own:
        from zoomkv_revision_b200 import ops
        st["pool"] = ops.KVPool(st["pool_k"], st["pool_v"], st["k_scale"], st["v_scale"])
    return st


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    op, S = case["op"], case["block"]
    if op in ("plan", "release"):
        B = case["batch"]
        lens = _ints(gen, case["ctx_lo"], case["ctx_hi"], B)
        if op == "plan":
            new = _ints(gen, case["new_lo"], case["new_hi"], B)
            new = torch.where(_ints(gen, 0, 7, B) == 0, torch.full_like(new, case["new_lo"]), new)
        else:
            new = torch.zeros_like(lens)
        # room for every request at its longest; the host knows these bounds without asking the GPU
        width = (case["ctx_hi"] + case.get("new_hi", 0)) // S + 2
        n_blocks = B * width
        table, perm, used = _table(gen, lens, S, width, n_blocks)
        free = torch.zeros(n_blocks, dtype=torch.int32, device=DEV)
        free[: n_blocks - used] = perm[used:]
        st = dict(op=op, lens=lens, table=table, free=free, block=S,
                  n_free=torch.full((1,), n_blocks - used, dtype=torch.int32, device=DEV),
                  lens_out=torch.empty_like(lens), n_free_out=torch.empty(1, dtype=torch.int32, device=DEV))
        if op == "plan":
            n_slots = B * max(1, case["new_hi"])
            st.update(new=new, slots=torch.empty(n_slots, dtype=torch.int64, device=DEV),
                      positions=torch.empty(n_slots, dtype=torch.int32, device=DEV),
                      cu=torch.empty(B + 1, dtype=torch.int32, device=DEV))
        else:
            st.update(done=torch.rand(B, generator=gen, device=DEV) < case["done"])
        return st
    H, D = case["kv_heads"], case["dim"]
    if op == "write":
        T = case["tokens"]
        n_blocks = (2 * T + S - 1) // S + 1
        (pk, ks), (pv, vs) = _pool_pair(gen, case, n_blocks)
        dt = DTYPES[case["src"]]
        # K and V are column ranges of one projection output [tokens, (q heads + 2 kv heads) * dim]
        qkv = torch.randn(T, 6 * H * D, generator=gen, device=DEV).to(dt)
        slots = torch.randperm(n_blocks * S, generator=gen, device=DEV)[:T]
        if T >= S:  # whole runs of tokens inside a block, blocks in any order
            blocks = torch.randperm(n_blocks, generator=gen, device=DEV)[: (T + S - 1) // S]
            slots = (blocks[:, None] * S + torch.arange(S, device=DEV)).reshape(-1)[:T]
        if case["idle"]:
            slots = torch.where(torch.rand(T, generator=gen, device=DEV) < case["idle"], torch.full_like(slots, -1), slots)
        return _handle(dict(op=op, k=qkv[:, 4 * H * D: 5 * H * D].unflatten(1, (H, D)),
                            v=qkv[:, 5 * H * D:].unflatten(1, (H, D)), slots=slots.contiguous(), pool_k=pk, pool_v=pv,
                            k_scale=ks, v_scale=vs))
    B, G = case["batch"], case["group"]
    lens = _ints(gen, case["len_lo"], case["len_hi"], B)
    width = (case["len_hi"] + S - 1) // S
    n_blocks = int(((lens.long() + S - 1) // S).sum()) + 8
    table, _, _ = _table(gen, lens, S, width, n_blocks)
    (pk, ks), (pv, vs) = _pool_pair(gen, case, n_blocks)
    q = torch.randn(B, H * G, D, generator=gen, device=DEV).to(DTYPES[case["q"]])
    return _handle(dict(op=op, q=q, pool_k=pk, pool_v=pv, k_scale=ks, v_scale=vs, lens=lens, table=table,
                        window=case["window"], softcap=case["softcap"], scale=1.0 / math.sqrt(D)))


# ---------------------------------------------------------------- plain forms
def _plain_plan(s):
    lens, new, table, free, S = s["lens"].long(), s["new"].long(), s["table"], s["free"], s["block"]
    n_slots, width = s["slots"].numel(), table.shape[1]
    n_free = s["n_free"].long()
    have, need = (lens + S - 1) // S, (lens + new + S - 1) // S
    cu = torch.cumsum(new, 0)
    fits = (need <= width) & (cu <= n_slots)
    take = torch.where(fits, need - have, torch.zeros_like(need))
    base = torch.cumsum(take, 0) - take
    served = fits & ((take == 0) | (base + take <= n_free))
    col = torch.arange(width, device=DEV)
    fresh = (col >= have[:, None]) & (col < need[:, None]) & served[:, None]
    at = (n_free - 1 - base[:, None] - (col - have[:, None])).clamp(0, free.numel() - 1)
    table.copy_(torch.where(fresh, free[at], table))
    i = torch.arange(n_slots, device=DEV)
    b = torch.searchsorted(cu, i, right=True).clamp(max=lens.numel() - 1)
    pos = lens[b] + i - (cu - new)[b]
    ok = (i < cu[-1]) & served[b]
    block = table[b, (pos // S).clamp(0, width - 1)].long()
    slots = torch.where(ok, block * S + pos % S, torch.full_like(pos, -1))
    positions = torch.where(ok, pos, torch.full_like(pos, -1)).int()
    lens_out = torch.where(served, lens + new, lens).int()
    n_free_out = (n_free - torch.where(served, take, torch.zeros_like(take)).sum()).int()
    return dict(table=table, slots=slots, positions=positions, cu=torch.cat([cu.new_zeros(1), cu]).int(), lens=lens_out,
                n_free=n_free_out)


def _plain_release(s):
    lens, table, free, S, done = s["lens"].long(), s["table"], s["free"], s["block"], s["done"]
    count = torch.where(done, (lens + S - 1) // S, torch.zeros_like(lens))
    base = s["n_free"].long() + torch.cumsum(count, 0) - count
    col = torch.arange(table.shape[1], device=DEV)
    back = col < count[:, None]
    free[(base[:, None] + col)[back]] = table[back]
    return dict(free=free, lens=torch.where(done, torch.zeros_like(lens), lens).int(), n_free=(s["n_free"] + count.sum()).int())


def _plain_store(x, pool, scale, slots):
    S = pool.shape[1]
    live = slots >= 0
    at, y = slots[live], x[live].float()
    if scale is None:
        pool[at // S, at % S] = y.to(pool.dtype)
    else:  # indexing is not defined on e4m3: its bytes are stored
        y = (y / scale[:, None]).clamp(-FP8_MAX, FP8_MAX)
        pool.view(torch.uint8)[at // S, at % S] = y.to(pool.dtype).view(torch.uint8)
    return pool


def _plain_write(s):
    return dict(k=_plain_store(s["k"], s["pool_k"], s["k_scale"], s["slots"]),
                v=_plain_store(s["v"], s["pool_v"], s["v_scale"], s["slots"]))


def _plain_rows(pool, table):
    """The requests' rows [batch, table width * block, kv heads, dim] in 32 bits."""
    if pool.dtype == torch.float8_e4m3fn:
        rows = pool.view(torch.uint8)[table].view(pool.dtype)
    else:
        rows = pool[table]
    return rows.float().flatten(1, 2)


def _plain_decode(s):
    q, table, lens = s["q"].float(), s["table"].long().clamp(min=0), s["lens"].long()
    B, Hq, D = q.shape
    S, H = s["pool_k"].shape[1], s["pool_k"].shape[2]
    L = table.shape[1] * S
    x = torch.einsum("bhgd,blhd->bhgl", q.view(B, H, Hq // H, D), _plain_rows(s["pool_k"], table)) * s["scale"]
    if s["k_scale"] is not None:
        x = x * s["k_scale"][:, None, None]
    if s["softcap"]:
        x = s["softcap"] * torch.tanh(x / s["softcap"])
    t = torch.arange(L, device=DEV)
    seen = t < lens[:, None]
    if s["window"]:
        seen = seen & (t >= lens[:, None] - s["window"])
    x = x.masked_fill(~seen[:, None, None], -math.inf)
    m = x.amax(-1, keepdim=True)
    p = torch.exp(x - torch.where(m == -math.inf, torch.zeros_like(m), m))
    total = p.sum(-1, keepdim=True)
    o = torch.einsum("bhgl,blhd->bhgd", p, _plain_rows(s["pool_v"], table))
    o = o / torch.where(total == 0, torch.ones_like(total), total)
    if s["v_scale"] is not None:
        o = o * s["v_scale"][:, None, None]
    return dict(out=o.reshape(B, Hq, D).to(s["q"].dtype), lse=(m + torch.log(total)).reshape(B, Hq))


def _own(s):
    """The calls a user makes."""
    from zoomkv_revision_b200 import ops
    if s["op"] == "plan":
        ops.pool_plan(s["lens"], s["new"], s["table"], s["free"], s["n_free"], s["block"], s["slots"],
                      positions=s["positions"], cu_new=s["cu"], lens_out=s["lens_out"], n_free_out=s["n_free_out"])
        return dict(table=s["table"], slots=s["slots"], positions=s["positions"], cu=s["cu"], lens=s["lens_out"],
                    n_free=s["n_free_out"])
    if s["op"] == "release":
        ops.pool_release(s["done"], s["lens"], s["table"], s["free"], s["n_free"], s["block"], lens_out=s["lens_out"],
                         n_free_out=s["n_free_out"])
        return dict(free=s["free"], lens=s["lens_out"], n_free=s["n_free_out"])
    if s["op"] == "write":
        ops.pool_write(s["k"], s["v"], s["slots"], s["pool"])
        return dict(k=s["pool_k"], v=s["pool_v"])
    out, lse = ops.pool_decode(s["q"], s["pool"], s["lens"], s["table"], scale=s["scale"], window=s["window"],
                               softcap=s["softcap"], return_lse=True)
    return dict(out=out, lse=lse)


def run(state):
    if own:
        return _own(state)
    if state["op"] == "plan":
        return _plain_plan(state)
    if state["op"] == "release":
        return _plain_release(state)
    if state["op"] == "write":
        return _plain_write(state)
    return _plain_decode(state)


# ---------------------------------------------------------------- work and the definitions in 64 bits
def work(case):
    S = case["block"]
    if case["op"] == "plan":
        B = case["batch"]
        new = (case["new_lo"] + 7 * (case["new_lo"] + case["new_hi"]) / 2) / 8 * B
        return dict(bytes=B * 16 + B * max(1, case["new_hi"]) * 12 + 8 * new / S, flops=0)
    if case["op"] == "release":
        blocks = case["batch"] * case["done"] * ((case["ctx_lo"] + case["ctx_hi"]) / 2 / S + 0.5)
        return dict(bytes=case["batch"] * 9 + 8 * blocks, flops=0)
    H, D = case["kv_heads"], case["dim"]
    el = 1 if case["pool"] == "fp8" else 2
    if case["op"] == "write":
        T = case["tokens"]
        return dict(bytes=8 * T + 2 * T * (1 - case["idle"]) * H * D * (2 + el), flops=0)
    B, Hq = case["batch"], case["kv_heads"] * case["group"]
    lo, hi, w = case["len_lo"], case["len_hi"], case["window"]
    if w and w < hi:  # the mean of min(len, w)
        kept = ((w - lo) * (lo + w) / 2 + (hi - w) * w) / (hi - lo) if lo < w else w
    else:
        kept = (lo + hi) / 2
    tokens = B * kept
    return dict(bytes=2 * tokens * H * D * el + 4 * tokens / S + 4 * B + 4 * B * Hq * D + 4 * B * Hq,
                flops=4 * tokens * Hq * D)


def exact(case, seed):
    """From the definitions, request by request, in 64 bits; None in the place of whole numbers."""
    s = prepare(case, seed)
    if s["op"] in ("plan", "release"):
        return None
    if s["op"] == "write":
        got = {}
        for name in ("k", "v"):
            pool, scale = s["pool_" + name], s[name + "_scale"]
            S = pool.shape[1]
            y = pool.to(torch.float64)
            x = s[name].to(torch.float64)
            if scale is not None:
                x = torch.clamp(x / scale.to(torch.float64).view(1, -1, 1), -FP8_MAX, FP8_MAX)
            rows = torch.nonzero(s["slots"] >= 0).squeeze(1)
            to = s["slots"][rows]
            y[torch.div(to, S, rounding_mode="floor"), to.remainder(S)] = x[rows]
            got[name] = y
        return got
    B, Hq, D = s["q"].shape
    S, H = s["pool_k"].shape[1:3]
    out = torch.zeros(B, Hq, D, dtype=torch.float64, device=DEV)
    lse = torch.full((B, Hq), -math.inf, dtype=torch.float64, device=DEV)

    def rows(name, ids, scale):
        got = s[name][ids] if scale is None else s[name].view(torch.uint8)[ids].view(s[name].dtype)
        got = got.to(torch.float64).reshape(-1, H, D)
        return got if scale is None else got * scale.to(torch.float64).view(1, H, 1)

    for b, n in enumerate(s["lens"].tolist()):
        first = max(0, n - s["window"]) if s["window"] else 0
        if n == first:
            continue
        ids = s["table"][b, first // S: (n + S - 1) // S].long()
        cut = slice(first - first // S * S, n - first // S * S)
        kk, vv = rows("pool_k", ids, s["k_scale"])[cut], rows("pool_v", ids, s["v_scale"])[cut]
        x = torch.matmul(s["q"][b].to(torch.float64).view(H, Hq // H, D), kk.permute(1, 2, 0)) * s["scale"]
        if s["softcap"]:
            x = torch.tanh(x / s["softcap"]) * s["softcap"]
        total = torch.logsumexp(x, -1)
        lse[b] = total.reshape(Hq)
        out[b] = torch.matmul(torch.exp(x - total[..., None]), vv.transpose(0, 1)).reshape(Hq, D)
    return dict(out=out, lse=lse)
