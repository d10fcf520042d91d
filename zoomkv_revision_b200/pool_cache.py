"""A pooled KV cache for requests of their own lengths, over the pool operators.

`polar_cache` keeps one dense buffer per row and one length for the whole
batch.  `PoolCache` keeps fixed-size blocks that the requests own through a
block table on the GPU: a request is admitted by appending its prompt, grows
by a token per step and gives its blocks back when it ends, and no step asks
the GPU for a length.  Attention is dense over each request's own tokens, as
the runtime attends below its full-attention threshold.

A serving step:

    slots = cache.plan(new_lens, n_slots, max_new)     # once per step
    for l in range(layers):
        cache.write(l, k, v, slots)                    # k, v [n_slots, kv_heads, head_dim]
        out = cache.attend(l, q)                       # q [batch, q_heads, head_dim], one token each
    cache.release(done)                                # requests that ended

The cache hooks of the decode loop (prefill_update_kv_cache, sync,
decode_update_kv_cache, compute; model_hub/LLM.py:208-294 of the reference's
runtime calls them) are there too, so that decode_loop.DecodeLoop runs over
it with a batch of equal prompts; they raise when a token has no room, where a
server's own steps find out by `check`.  The reference has no pooled cache.

    python -m zoomkv_revision_b200.pool_cache          # a small serving run
"""
from __future__ import annotations

import argparse

import torch

from . import ops


class PoolCache:
    """layers x pools of n_blocks blocks of block_size tokens for up to
    `batch` requests of up to max_length tokens, in whole blocks (n_blocks:
    room for all of them by default; fewer blocks serve more, shorter
    requests).  dtype bfloat16, float16 or float8_e4m3fn, for which
    k_scale / v_scale [layers, kv_heads] fp32 give what a stored 1.0 stands
    for (None: 1)."""

    def __init__(self, layers: int, batch: int, kv_heads: int, head_dim: int, max_length: int, *, n_blocks=None,
                 block_size: int = 16, dtype=torch.bfloat16, k_scale=None, v_scale=None, device="cuda"):
        self.width = -(-max_length // block_size)
        self.n_blocks = batch * self.width if n_blocks is None else int(n_blocks)
        self.layers, self.batch, self.block_size, self.max_length = layers, batch, block_size, max_length
        shape = (layers, self.n_blocks, kv_heads, block_size, head_dim)   # head before token: a block's rows of a head together
        self.k = torch.empty(shape, dtype=dtype, device=device)           # (an unwritten row is never read)
        self.v = torch.empty(shape, dtype=dtype, device=device)
        self.pools = [ops.KVPool(self.k[l].transpose(1, 2), self.v[l].transpose(1, 2),
                                 None if k_scale is None else k_scale[l], None if v_scale is None else v_scale[l])
                      for l in range(layers)]
        ints = dict(dtype=torch.int32, device=self.k.device)
        self.lens = torch.zeros(batch, **ints)
        self.table = torch.full((batch, self.width), -1, **ints)
        self.free = torch.arange(self.n_blocks, **ints)
        self.n_free = torch.full((1,), self.n_blocks, **ints)
        self.status = torch.zeros(1, **ints)
        self.bound = 0                       # no request is longer, as far as the host knows (a replayed plan does not tell it)
        self.captured = False                # a plan was: replays may have moved the lengths
        self.slots = None                    # of the step that is being written

    # ------------------------------------------------------------------ a serving step
    def plan(self, new_lens, n_slots: int, max_new=None):
        """Blocks and slots for the step's new tokens: new_lens [batch] int32 on the GPU (None: one each), at most
        n_slots in all and max_new for one request (None: what n_slots allows; a step of single tokens from new_lens
        gives 1).  Returns the slot map [n_slots]."""
        slots = torch.empty(n_slots, dtype=torch.int64, device=self.k.device)
        ops.pool_plan(self.lens, new_lens, self.table, self.free, self.n_free, self.block_size, slots, status=self.status)
        if max_new is None:
            max_new = 1 if new_lens is None else n_slots
        self.bound = min(self.bound + max_new, self.width * self.block_size)
        self.captured |= torch.cuda.is_current_stream_capturing()
        self.slots = slots
        return slots

    def write(self, layer: int, k, v, slots) -> None:
        """K and V of the new tokens [n, kv_heads, head_dim] into one layer's pool."""
        ops.pool_write(k, v, slots, self.pools[layer], status=self.status)

    def attend(self, layer: int, q, **kw):
        """Attention of q [batch, (1,) q_heads, head_dim] over each request's tokens (keywords of ops.pool_decode;
        max_len, which chooses how the work is cut, is the bound that plan keeps; a call that is captured in a graph for
        longer requests gives its own, 0 for all of the table's room)."""
        kw.setdefault("max_len", self.bound)
        return ops.pool_decode(q, self.pools[layer], self.lens, self.table, status=self.status, **kw)

    def release(self, done, bound=None) -> None:
        """Ends the requests with done[b] ([batch] bool on the GPU).  bound: the longest that is left, where the host
        knows it."""
        ops.pool_release(done, self.lens, self.table, self.free, self.n_free, self.block_size, status=self.status)
        if bound is not None:
            self.bound = int(bound)

    def check(self) -> None:
        """Raises if a step found no room for a request or met an index outside the pool (waits for the GPU)."""
        code = int(self.status.item())
        if code:
            self.status.zero_()
            raise RuntimeError(f"pool cache: {ops.lib().zkv_status_string(code).decode()}")

    # ------------------------------------------------------------------ hooks of the decode loop
    def _make_room(self, new: int) -> None:
        """Raises if `new` more tokens of every request do not fit: the loop's caller has no status to look at.  Where the
        host's bound leaves a doubt, or a captured plan may have been replayed, the GPU is asked, and the bound is what it
        says; not in a graph capture, whose replays only `check` can judge."""
        def blocks(n):
            return -(-n // self.block_size)

        if not self.captured and blocks(self.bound + new) <= min(self.width, self.n_blocks // self.batch):
            return
        if torch.cuda.is_current_stream_capturing():
            return
        lens, n_free = self.lens.tolist(), int(self.n_free.item())
        self.bound = max(lens)
        if blocks(self.bound + new) > self.width or sum(blocks(n + new) - blocks(n) for n in lens) > n_free:
            raise RuntimeError(f"KV write is outside the cache: {new} more tokens for requests of up to {self.bound}, of "
                               f"{self.width * self.block_size} each; {n_free} of {self.n_blocks} blocks are free")

    def prefill_update_kv_cache(self, query_states, key_states, value_states, layer_idx: int, batch_idx: int):
        """Appends a prompt to every request: key_states, value_states [batch, T, kv_heads, head_dim]."""
        del query_states
        B, T = key_states.shape[:2]
        if B != self.batch or batch_idx != 0:
            raise ValueError(f"prompts come for the whole batch of {self.batch} at once; got {B} from {batch_idx} on")
        if layer_idx == 0:
            self._make_room(T)
            self.plan(torch.full((B,), T, dtype=torch.int32, device=self.k.device), B * T, T)
        self.write(layer_idx, key_states.reshape(B * T, *key_states.shape[2:]),
                   value_states.reshape(B * T, *value_states.shape[2:]), self.slots)
        return key_states, value_states

    def sync(self, layer_idx: int, batch_idx: int) -> None:
        """Nothing to wait for: every step runs on the caller's stream."""

    def decode_update_kv_cache(self, key_states, value_states, layer_idx: int):
        """Appends one token to every request: [batch, 1, kv_heads, head_dim]."""
        if layer_idx == 0:
            self._make_room(1)
            self.plan(None, self.batch, 1)
        self.write(layer_idx, key_states[:, 0], value_states[:, 0], self.slots)

    def compute(self, queries, layer_idx: int):
        """[batch, 1, q_heads, head_dim] -> the same, over the tokens appended so far."""
        return self.attend(layer_idx, queries)


def serve(steps: int, batch: int, layers: int = 4, kv_heads: int = 8, group: int = 4, head_dim: int = 128,
          max_length: int = 2048, dtype=torch.bfloat16, seed: int = 0) -> dict:
    """Requests come with prompts of 16 to max_length / 2 tokens, grow by a token per step, end at random and make room
    for others; K, V and Q are random rows.  Returns what was served and how long a decode step of all layers took."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    cache = PoolCache(layers, batch, kv_heads, head_dim, max_length, dtype=dtype)
    qkv = torch.randn(batch * max_length // 2, kv_heads * 3, head_dim, generator=g, device="cuda").to(torch.bfloat16)
    q = torch.randn(batch, kv_heads * group, head_dim, generator=g, device="cuda").to(torch.bfloat16)
    prompt = torch.randint(16, max_length // 2 + 1, (batch,), generator=g, device="cuda", dtype=torch.int32)
    total = torch.zeros((), dtype=torch.int64, device="cuda")
    times = []
    for step in range(steps):
        live = cache.lens > 0
        if step % 16 == 0:    # a step that admits: prompts for the empty places, one token for the others
            new, n = torch.where(live, torch.ones_like(prompt), prompt), qkv.shape[0]
            slots = cache.plan(new, n, max_length // 2)
        else:
            new, n = live.int(), batch
            slots = cache.plan(new, n, 1)
        total += new.sum()
        begin, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        begin.record()
        for l in range(layers):
            cache.write(l, qkv[:n, :kv_heads], qkv[:n, kv_heads: 2 * kv_heads], slots)
            cache.attend(l, q)
        end.record()
        times.append((step % 16 == 0, begin, end))
        over = cache.lens >= max_length - 1
        cache.release(over | (torch.rand(batch, generator=g, device="cuda") < 0.01))
    torch.cuda.synchronize()
    cache.check()
    us = sorted(b.elapsed_time(e) * 1e3 for admits, b, e in times if not admits)
    return dict(steps=steps, tokens=int(total), free_blocks=int(cache.n_free), blocks=cache.n_blocks,
                decode_step_us=us[len(us) // 2] if us else 0.0)


def main(argv=None) -> None:
    ap = argparse.ArgumentParser(description="a small serving run over the pooled cache")
    ap.add_argument("--steps", type=int, default=200)
    ap.add_argument("--batch", type=int, default=64)
    ap.add_argument("--layers", type=int, default=4)
    ap.add_argument("--max-length", type=int, default=2048)
    ap.add_argument("--fp8", action="store_true", help="e4m3 blocks")
    a = ap.parse_args(argv)
    got = serve(a.steps, a.batch, a.layers, max_length=a.max_length,
                dtype=torch.float8_e4m3fn if a.fp8 else torch.bfloat16)
    print(f"{got['steps']} steps, {got['tokens']} tokens appended, {got['free_blocks']} of {got['blocks']} blocks free, "
          f"{got['decode_step_us']:.1f} us per decode step of {a.layers} layers (median)")


if __name__ == "__main__":
    main()
