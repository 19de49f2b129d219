"""A conditioned block: residual cross attention from a sequence to an encoder's states, with the
low-rank adapters of many requests beside every projection.

    q = W_q x + adapters,  (k, v) = W_kv enc + adapters
    q, k normed per head, both rotated (the encoder's states by their own positions)
    y = x + W_o cross_attention(q, k, v) + adapters

The three operators behind it are ops.adapter_gemm, ops.qk_norm_rope and
ops.cross_attention.  The reference has no counterpart; its closest relative is HTDemucs'
cross transformer (src/model_htdemucs.cu:600-664), whose cross attention has neither
grouped heads, ragged encoder lengths nor adapters.

    python -m msst_b200.conditioned          # one block on random data, prompt and single-token form, then tokens
                                             # one by one behind a shared prefix (msst_b200.cached)
"""
from __future__ import annotations

from . import _need, _torch, ops


class ConditionedBlock:
    """One block on the GPU of its weights, inference only.

    w_q [Hq*d, dim], w_kv [2*Hk*d, enc_dim] (keys, then values), w_o [dim, Hq*d], 16-bit; q_gamma /
    k_gamma float32 [d]; cos / sin float32 [positions, rot/2].  `adapters` maps any of "q", "kv",
    "o" to (lora_a [n, rank, in], lora_b [n, out, rank], scales [n] or None); all share the
    numbering of the requests' adapters."""

    def __init__(self, w_q, w_kv, w_o, q_heads: int, kv_heads: int, head_dim: int, q_gamma, k_gamma, cos, sin,
                 adapters=None, eps: float = 1e-6, pairing: str = "halves"):
        _need(w_q.shape[0] == q_heads * head_dim and w_kv.shape[0] == 2 * kv_heads * head_dim and
              w_o.shape[1] == q_heads * head_dim and w_o.shape[0] == w_q.shape[1], "weights do not fit the heads")
        _need(set(adapters or ()) <= {"q", "kv", "o"}, "adapters may stand beside q, kv and o")
        self.w = {"q": w_q, "kv": w_kv, "o": w_o}
        self.q_heads, self.kv_heads, self.head_dim = q_heads, kv_heads, head_dim
        self.q_gamma, self.k_gamma, self.cos, self.sin = q_gamma, k_gamma, cos, sin
        self.adapters = dict(adapters or {})
        self.eps, self.pairing = eps, pairing

    def _project(self, name, x, row_adapter):
        """x [B, N, in] through weight `name` with the rows' adapters -> [B, N, out]."""
        w = self.w[name]
        if name in self.adapters:
            a, b, scales = self.adapters[name]
        else:  # no adapter stands beside this weight
            a, b, scales = w.new_empty((0, 8, w.shape[1])), w.new_empty((0, w.shape[0], 8)), None
            row_adapter = row_adapter.new_full(row_adapter.shape, -1)
        return ops.adapter_gemm(x, w, a, b, row_adapter, scales=scales)

    def encode(self, states, request_adapter):
        """Keys and values of the encoder's states [B, Nk, enc_dim], once per prompt: (k, v), each
        [B, Nk, Hk, d].  request_adapter int32 [B], -1 for none."""
        B, Nk = states.shape[:2]
        kv = self._project("kv", states, request_adapter.repeat_interleave(Nk))
        kv = kv.view(B, Nk, 2, self.kv_heads, self.head_dim)
        k, v = kv[:, :, 0], kv[:, :, 1]
        # the keys are normed and rotated where they lie, beside the values
        ops.qk_norm_rope(k, None, self.k_gamma, None, self.cos, self.sin, eps=self.eps, pairing=self.pairing, out_q=k)
        return k, v

    def __call__(self, x, k, v, request_adapter, positions=None, key_lens=None, key_mask=None):
        """x [B, Nq, dim] (Nq = 1: one new token per request) attending to encode()'s keys and
        values -> [B, Nq, dim].  positions int32 [B, Nq]."""
        B, Nq = x.shape[:2]
        rows = request_adapter.repeat_interleave(Nq)
        q = self._project("q", x, rows).view(B, Nq, self.q_heads, self.head_dim)
        ops.qk_norm_rope(q, None, self.q_gamma, None, self.cos, self.sin, positions=positions, eps=self.eps,
                         pairing=self.pairing, out_q=q)
        o = ops.cross_attention(q, k, v, key_lens=key_lens, key_mask=key_mask)
        return x + self._project("o", o.view(B, Nq, -1), rows)


def random_block(dim=512, enc_dim=384, q_heads=8, kv_heads=2, head_dim=64, count=3, rank=16, positions=4096,
                 dtype=None, seed=0):
    """A block with seeded random weights (synthetic, for the example and its test)."""
    torch = _torch()
    dtype = dtype or torch.bfloat16
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)

    def normal(*shape, scale):
        return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)

    sizes = {"q": (dim, q_heads * head_dim), "kv": (enc_dim, 2 * kv_heads * head_dim), "o": (q_heads * head_dim, dim)}
    w = {n: normal(o, i, scale=i ** -0.5) for n, (i, o) in sizes.items()}
    adapters = {n: (normal(count, rank, i, scale=i ** -0.5), normal(count, o, rank, scale=0.5 * rank ** -0.5),
                    0.5 + torch.rand(count, generator=g, device="cuda")) for n, (i, o) in sizes.items()}
    half = head_dim // 2
    angle = torch.arange(positions, device="cuda", dtype=torch.float64)[:, None] * \
        10000.0 ** (-torch.arange(half, device="cuda", dtype=torch.float64) / half)
    gammas = [1 + 0.1 * torch.randn(head_dim, generator=g, device="cuda") for _ in range(2)]
    return ConditionedBlock(w["q"], w["kv"], w["o"], q_heads, kv_heads, head_dim, *gammas, angle.cos().float(),
                            angle.sin().float(), adapters)


def main():
    torch = _torch()
    block = random_block()
    B, Nq, Nk = 4, 100, 801
    dt = block.w["q"].dtype
    x = torch.randn(B, Nq, 512, device="cuda").to(dt)
    states = torch.randn(B, Nk, 384, device="cuda").to(dt)
    lens = torch.tensor([801, 640, 333, 1], dtype=torch.int32, device="cuda")
    who = torch.tensor([0, 2, -1, 1], dtype=torch.int32, device="cuda")
    k, v = block.encode(states, who)
    y = block(x, k, v, who, key_lens=lens)
    last = torch.full((B, 1), Nq - 1, dtype=torch.int32, device="cuda")
    token = block(x[:, -1:], k, v, who, positions=last, key_lens=lens)
    torch.cuda.synchronize()
    print(f"prompt {tuple(y.shape)}, its last token alone differs by at most "
          f"{float((token - y[:, -1:]).abs().max()):.2g} (one bf16 step at the output's size: "
          f"{float(2.0 ** -8 * y[:, -1:].abs().max()):.2g})")
    generate(block, k, v, who, lens)


def generate(block, k, v, who, key_lens, prefix=300, steps=20):
    """Rows one by one through a layer of both blocks: a CachedBlock over a shared prefix and each request's own
    rows, then `block` over the encoder's states, each row the next one's input."""
    from .cached import TokenCache, random_cached_block

    torch = _torch()
    layer = random_cached_block(dim=block.w["q"].shape[1], dtype=block.w["q"].dtype)
    R = who.numel()
    _, prefix_k, prefix_v = layer.prefill(torch.randn(prefix, block.w["q"].shape[1], device="cuda").to(block.w["q"].dtype))
    cache = TokenCache(R, -(-steps // 16), layer.kv_heads, layer.head_dim, page_size=16, dtype=block.w["q"].dtype)
    x = torch.randn(R, block.w["q"].shape[1], device="cuda").to(block.w["q"].dtype)
    one = torch.ones_like(who)
    for _ in range(steps):
        step = cache.plan(one, R, start=prefix)
        h = layer(x, prefix_k, prefix_v, cache, step, who, single=True)
        y = block(h[:, None], k, v, who, positions=step.positions[:, None], key_lens=key_lens)[:, 0]
        x = y / y.float().square().mean(-1, keepdim=True).sqrt().to(y.dtype)
    cache.plan(-one, 0)  # all requests have ended
    torch.cuda.synchronize()
    print(f"{steps} tokens of {R} requests behind a prefix of {prefix}; {int(cache.free_count)} of "
          f"{cache.free_pages.numel()} pages free at the end")
    return x


if __name__ == "__main__":
    main()
