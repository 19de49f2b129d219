"""Self attention of a decoder layer over a prefix that all requests share and each request's own
tokens in a paged cache: what stands before a ConditionedBlock's cross attention where tokens are
generated one by one.

    q, k, v = W_q x, W_k x, W_v x (one product), q and k rotated, k and v written to the pages
    y = x + W_o prefix_attention(q, prefix, own tokens)

ops.cache_plan finds the pages, ops.rope_append fills them and ops.prefix_attention reads them; the
low-rank adapters of each request's fine-tune stand beside both projections (ops.adapter_gemm).
The reference has no counterpart.

    python -m msst_b200.conditioned          # with a conditioned block behind it, on random data
"""
from __future__ import annotations

from typing import NamedTuple

from . import _need, _torch, ops


class Step(NamedTuple):
    """A plan's rows: first row of each request, slot and position of each row, lengths after it.

    It stays as it is while the next step is planned ahead; its layers have to be launched before the
    next step's, and before the plan behind that (which may fill an ended request's row of the block table)."""
    q_starts: object
    slots: object
    positions: object
    lens: object


class TokenCache:
    """Pages of keys and values for up to `requests` requests at a time, on one GPU.

    `layers` layers share the block table and slots; `blocks` pages of page_size tokens are the most
    that a request may hold, `pages` the most of all together (None: enough for all).  A plan is
    made once a step, for all layers, on the current stream; the cache's lengths, table and free pages
    are updated in place, so a captured step may be replayed."""

    def __init__(self, requests, blocks, kv_heads, head_dim, layers=1, page_size=64, pages=None, dtype=None, device=None):
        torch = _torch()
        pages = requests * blocks if pages is None else pages
        _need(requests > 0 and blocks > 0 and pages > 0 and layers > 0, "requests, blocks, pages and layers must be above 0")
        device = torch.device("cuda", torch.cuda.current_device()) if device is None else device
        self.page_size = page_size
        self.kv = torch.zeros(layers, 2, pages, page_size, kv_heads, head_dim, dtype=dtype or torch.bfloat16, device=device)

        def ints(n, fill):
            return torch.full((n,), fill, dtype=torch.int32, device=device)

        self.lens, self.block_table = ints(requests, 0), ints(requests * blocks, 0).view(requests, blocks)
        self.free_pages = torch.arange(pages - 1, -1, -1, dtype=torch.int32, device=device)
        self.free_count = ints(1, pages)

    def plan(self, new_tokens, tokens, start=0) -> Step:
        """Room for new_tokens[r] more tokens of each request (int32 [requests]; -1: the request has
        ended and its pages are free), `tokens` rows in all, positions from `start` (the prefix's length)."""
        q_starts, slots, positions, lens, _ = ops.cache_plan(
            new_tokens, self.lens, self.block_table, self.free_pages, self.free_count, self.page_size, tokens, start=start,
            out_free_count=self.free_count)
        self.lens.copy_(lens)  # (the step keeps its own)
        return Step(q_starts, slots, positions, lens)


class CachedBlock:
    """One block on the GPU of its weights, inference only.

    w_qkv [(Hq + 2 Hk) d, dim] (queries, keys, values), w_o [dim, Hq d], 16-bit; inv_freq / amplitude as
    rope_frequencies gives them; `adapters` maps "qkv" or "o" to (lora_a [n, rank, in], lora_b
    [n, out, rank], scales [n] or None)."""

    def __init__(self, w_qkv, w_o, q_heads, kv_heads, head_dim, inv_freq, amplitude=1.0, adapters=None, pairing="halves"):
        _need(w_qkv.shape[0] == (q_heads + 2 * kv_heads) * head_dim and w_o.shape == (w_qkv.shape[1], q_heads * head_dim),
              "weights do not fit the heads")
        _need(set(adapters or ()) <= {"qkv", "o"}, "adapters may stand beside qkv and o")
        self.w = {"qkv": w_qkv, "o": w_o}
        self.q_heads, self.kv_heads, self.head_dim = q_heads, kv_heads, head_dim
        self.inv_freq, self.amplitude, self.pairing = inv_freq, amplitude, pairing
        self.adapters = dict(adapters or {})

    def _project(self, name, x, row_adapter):
        w = self.w[name]
        if name in self.adapters:
            return ops.adapter_gemm(x, w, *self.adapters[name][:2], row_adapter, scales=self.adapters[name][2])
        none = w.new_empty((0, 8, w.shape[1])), w.new_empty((0, w.shape[0], 8))
        return ops.adapter_gemm(x, w, *none, row_adapter.new_full(row_adapter.shape, -1))

    def _heads(self, x, row_adapter):
        qkv = self._project("qkv", x, row_adapter).view(x.shape[0], self.q_heads + 2 * self.kv_heads, self.head_dim)
        return qkv[:, :self.q_heads], qkv[:, self.q_heads:-self.kv_heads], qkv[:, -self.kv_heads:]

    def _append(self, x, positions, slots, row_adapter, k_cache, v_cache):
        q, k, v = self._heads(x, row_adapter)
        return ops.rope_append(q, k, v, positions, slots, self.inv_freq, k_cache, v_cache, amplitude=self.amplitude,
                               pairing=self.pairing, out_q=q)

    def prefill(self, x):
        """The shared prefix [P, dim], once: (y [P, dim], its keys and values [P, Hk, d]), without adapters."""
        torch = _torch()
        P = x.shape[0]
        page = 256
        room = x.new_zeros(2, max(1, -(-P // page)), page, self.kv_heads, self.head_dim)
        at = torch.arange(P, dtype=torch.int32, device=x.device)
        q = self._append(x, at, at, at.new_full((P,), -1), room[0], room[1])
        pages = at[:-(-P // page)].view(1, -(-P // page))
        o = ops.prefix_attention(q, None, None, room[0], room[1], pages, at.new_full((1,), P),
                                 q_starts=P * torch.arange(2, dtype=torch.int32, device=x.device))
        y = x + self._project("o", o.flatten(1), at.new_full((P,), -1))
        return y, room[0].view(-1, self.kv_heads, self.head_dim)[:P], room[1].view(-1, self.kv_heads, self.head_dim)[:P]

    def __call__(self, x, prefix_k, prefix_v, cache: TokenCache, step: Step, row_adapter, layer=0, single=False):
        """x [rows, dim], the step's rows in their order -> [rows, dim].  row_adapter int32 [rows], -1 for
        none.  single: every request of the cache has exactly one row."""
        k_cache, v_cache = cache.kv[layer, 0], cache.kv[layer, 1]
        q = self._append(x, step.positions, step.slots, row_adapter, k_cache, v_cache)
        o = ops.prefix_attention(q, prefix_k, prefix_v, k_cache, v_cache, cache.block_table, step.lens,
                                 q_starts=None if single else step.q_starts)
        return x + self._project("o", o.flatten(1), row_adapter)


def random_cached_block(dim=512, q_heads=8, kv_heads=2, head_dim=64, count=3, rank=16, dtype=None, seed=0, **scaling):
    """A block with seeded random weights (synthetic, for the example and its test)."""
    from . import rope_frequencies

    torch = _torch()
    dtype = dtype or torch.bfloat16
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)

    def normal(*shape, scale):
        return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)

    sizes = {"qkv": (dim, (q_heads + 2 * kv_heads) * head_dim), "o": (q_heads * head_dim, dim)}
    w = {n: normal(o, i, scale=i ** -0.5) for n, (i, o) in sizes.items()}
    adapters = {n: (normal(count, rank, i, scale=i ** -0.5), normal(count, o, rank, scale=0.5 * rank ** -0.5),
                    0.5 + torch.rand(count, generator=g, device="cuda")) for n, (i, o) in sizes.items()}
    inv_freq, amplitude = rope_frequencies(head_dim, device="cuda", **scaling)
    return CachedBlock(w["qkv"], w["o"], q_heads, kv_heads, head_dim, inv_freq, amplitude, adapters)
