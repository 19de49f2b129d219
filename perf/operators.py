"""Cases, plain forms and 64-bit forms of the framework's operators for conditioned Roformer blocks:
per-head norms of queries and keys with the position rotation, cross attention to an encoder's
states, and a shared projection with the low-rank adapters of many requests beside it."""
from __future__ import annotations

import os
import sys

import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


# ------------------------------------------------------------------------------------- cases
def listed():
    return [
        # one new token for each of 64 requests, grouped heads: launch latency is all there is
        dict(name="qk_token", op="qk", batch=64, seq=1, q_heads=32, k_heads=8, dim=128, rot=128, pairing="halves",
             layout="plain", dtype="bf16"),
        # the time axis of one 801-frame, 60-band Roformer chunk, read from its packed QKV rows
        dict(name="qk_time_axis", op="qk", batch=60, seq=801, q_heads=8, k_heads=8, dim=64, rot=64,
             pairing="interleaved", layout="time", dtype="fp16"),
        # four long prompts with grouped heads
        dict(name="qk_prompt", op="qk", batch=4, seq=4096, q_heads=32, k_heads=8, dim=128, rot=128, pairing="halves",
             layout="plain", dtype="bf16"),
        # HTDemucs' time branch: 48 columns a head, an odd length, part of each head rotated
        dict(name="qk_part", op="qk", batch=3, seq=1895, q_heads=8, k_heads=8, dim=48, rot=32, pairing="interleaved",
             layout="plain", dtype="fp16"),
        # one new token for each of 16 requests over encoder states of ragged lengths
        dict(name="cross_token", op="cross", batch=16, q_len=1, k_len=4096, q_heads=32, kv_heads=8, dim=128,
             mask="lens", dtype="bf16"),
        # one request, one token, very long encoder states: the keys have to be shared out
        dict(name="cross_token_long", op="cross", batch=1, q_len=1, k_len=131072, q_heads=8, kv_heads=8, dim=64,
             mask="none", dtype="fp16"),
        # HTDemucs' cross transformer, time branch to frequency branch, 4 segments
        dict(name="cross_branches", op="cross", batch=4, q_len=1895, k_len=3792, q_heads=8, kv_heads=8, dim=64,
             mask="none", dtype="fp16"),
        # long prompts to long encoder states of ragged lengths, grouped heads
        dict(name="cross_prompt", op="cross", batch=4, q_len=4096, k_len=4096, q_heads=32, kv_heads=8, dim=128,
             mask="lens", dtype="bf16"),
        # odd everything, keys masked one by one, one batch entry with no key left
        dict(name="cross_masked", op="cross", batch=5, q_len=77, k_len=1501, q_heads=12, kv_heads=4, dim=80,
             mask="keys", dtype="fp16"),
        # one new token for each of 32 requests with adapters of their own: the shared weight is what is read
        dict(name="adapters_token", op="adapters", rows=32, requests=32, k=4096, n=4096, adapters=16, rank=16,
             bias=False, dtype="bf16"),
        # prompts of six requests
        dict(name="adapters_prompt", op="adapters", rows=8192, requests=6, k=4096, n=4096, adapters=6, rank=32,
             bias=False, dtype="bf16"),
        # the QKV projection of one Roformer chunk (801 frames, 60 bands), chunks of four users' fine-tunes
        dict(name="adapters_roformer", op="adapters", rows=48060, requests=5, k=384, n=1536, adapters=4, rank=8,
             bias=True, dtype="fp16"),
    ]


def _spread(rng, lo, hi, never=3072):
    """A whole number between lo and hi other than `never`, spread over its logarithm."""
    n = int(round(lo * (hi / lo) ** rng.random()))
    n = min(max(n, lo), hi)
    return n - 1 if n == never else n


def draw(rng):
    op = rng.choice(["qk", "cross", "adapters"])
    dtype = rng.choice(["fp16", "bf16"])
    if op == "qk":
        dim = rng.choice([32, 48, 64, 80, 96, 128, 256])
        group = rng.choice([1, 2, 4])
        k_heads = rng.choice([1, 4, 5, 8])
        seq = _spread(rng, 1, 8192)
        if 3072 in (k_heads * group * dim, k_heads * (group + 2) * dim):
            dim = 80
        most = 80_000_000 // (seq * k_heads * (group + 1) * dim)  # queries and keys together stay below 160 MB
        return dict(op=op, batch=_spread(rng, 1, max(1, min(64, most))), seq=seq, q_heads=k_heads * group,
                    k_heads=k_heads, dim=dim, rot=rng.choice([dim, dim, dim // 2]),
                    pairing=rng.choice(["interleaved", "halves"]), layout=rng.choice(["plain", "plain", "time"]),
                    dtype=dtype)
    if op == "cross":
        dim = rng.choice([32, 48, 64, 64, 80, 96, 128, 128])
        q_len = rng.choice([1, 1, _spread(rng, 2, 64), _spread(rng, 2, 4096)])
        group = rng.choice([1, 1, 2, 3, 4, 8 if q_len <= 64 else 4])
        kv_heads = rng.choice([1, 2, 4, 8])
        if kv_heads * group * dim == 3072:
            dim = 80
        batch = rng.choice([1, 2, 3, 4, 4, 16 if q_len <= 64 else 2])
        most = 80_000_000 // (batch * kv_heads * dim)  # keys and values together stay below 320 MB
        k_len = _spread(rng, 1, min(131072 if q_len <= 64 else 4096, most))
        return dict(op=op, batch=batch, q_len=q_len, k_len=k_len,
                    q_heads=kv_heads * group, kv_heads=kv_heads, dim=dim,
                    mask=rng.choice(["none", "lens", "lens", "keys"]), dtype=dtype)
    rows = _spread(rng, 1, 8192)
    return dict(op=op, rows=rows, requests=_spread(rng, 1, min(rows, 64)), k=8 * _spread(rng, 8, 512, 384),
                n=8 * _spread(rng, 8, 512, 384), adapters=rng.choice([1, 3, 8, 16]), rank=rng.choice([8, 16, 16, 24, 32, 64]),
                bias=rng.random() < 0.5, dtype=dtype)


def _lens(case):
    """Encoder lengths of a ragged batch: from all of k_len down to about half of it."""
    b = case["batch"]
    return [max(1, case["k_len"] - (i * case["k_len"]) // (2 * b)) for i in range(b)]


def _rows_of(case):
    """Row counts of the requests, about as uneven as 1 : 2."""
    r = case["requests"]
    weights = [2 * r + (7 * i) % (2 * r) for i in range(r)]
    spare, total = case["rows"] - r, sum(weights)
    counts = [1 + spare * w // total for w in weights]
    counts[-1] += case["rows"] - sum(counts)
    return counts


def work(case):
    if case["op"] == "qk":
        tokens = case["batch"] * case["seq"]
        values = tokens * (case["q_heads"] + case["k_heads"]) * case["dim"]
        # each value is read and written once; the rotation's factors once for each position
        return {"bytes": 4 * values + 4 * tokens + 4 * case["seq"] * case["rot"], "flops": 7 * values}
    if case["op"] == "cross":
        if case["mask"] == "lens":
            keys = sum(_lens(case))
        else:
            keys = case["batch"] * case["k_len"]
        q = case["batch"] * case["q_len"] * case["q_heads"] * case["dim"]
        kv = 2 * keys * case["kv_heads"] * case["dim"]
        extra = case["batch"] * case["k_len"] if case["mask"] == "keys" else 4 * case["batch"]
        return {"bytes": 2 * (2 * q + kv) + extra, "flops": 4 * keys * case["q_len"] * case["q_heads"] * case["dim"]}
    m, k, n, r = case["rows"], case["k"], case["n"], case["rank"]
    used = min(case["adapters"], case["requests"])
    return {"bytes": 2 * (m * k + n * k + m * n + used * r * (k + n)) + 4 * m, "flops": 2 * m * (k * n + r * (k + n))}


# ------------------------------------------------------------------------------------- inputs
def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def normal(*shape, scale=1.0, dtype=dt):
        return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)

    s = dict(case)
    if case["op"] == "qk":
        b, n, hq, hk, d = (case[x] for x in ("batch", "seq", "q_heads", "k_heads", "dim"))
        if case["layout"] == "time":  # packed [n, b, (q k v) heads d] rows, as a QKV projection leaves them
            packed = normal(n, b, (hq + 2 * hk) * d)
            heads = packed.view(n, b, hq + 2 * hk, d).transpose(0, 1)
            s["q"], s["k"], s["positions"] = heads[:, :, :hq], heads[:, :, hq:hq + hk], None
            table = n
        else:
            s["q"], s["k"] = normal(b, n, hq, d), normal(b, n, hk, d)
            table = 8192 + n
            start = torch.randint(0, 8192, (b, 1), generator=g, device="cuda", dtype=torch.int32)
            s["positions"] = start + torch.arange(n, device="cuda", dtype=torch.int32)
        s["q_gamma"] = 1 + normal(d, scale=0.1, dtype=torch.float32)
        s["k_gamma"] = 1 + normal(d, scale=0.1, dtype=torch.float32)
        half = case["rot"] // 2
        freq = 10000.0 ** (-torch.arange(half, device="cuda", dtype=torch.float64) / half)
        angle = torch.arange(table, device="cuda", dtype=torch.float64)[:, None] * freq
        s["cos"], s["sin"] = angle.cos().float(), angle.sin().float()
    elif case["op"] == "cross":
        b, nq, nk, hq, hk, d = (case[x] for x in ("batch", "q_len", "k_len", "q_heads", "kv_heads", "dim"))
        s["q"] = normal(b, nq, hq, d)
        kv = normal(b, nk, 2, hk, d)  # one projection writes keys and values side by side
        s["k"], s["v"] = kv[:, :, 0], kv[:, :, 1]
        s["key_lens"] = s["key_mask"] = None
        if case["mask"] == "lens":
            s["key_lens"] = torch.tensor(_lens(case), dtype=torch.int32, device="cuda")
        elif case["mask"] == "keys":
            s["key_mask"] = torch.rand(b, nk, generator=g, device="cuda") < 0.75
            if b > 1:
                s["key_mask"][b - 1] = False  # an empty encoder
    else:
        m, k, n, r = case["rows"], case["k"], case["n"], case["rank"]
        s["x"] = normal(m, k)
        s["w"] = normal(n, k, scale=k ** -0.5)
        s["bias"] = normal(n, scale=0.1, dtype=torch.float32) if case["bias"] else None
        s["lora_a"] = normal(case["adapters"], r, k, scale=k ** -0.5)
        s["lora_b"] = normal(case["adapters"], n, r, scale=0.5 * r ** -0.5)
        s["scales"] = 0.5 + torch.rand(case["adapters"], generator=g, device="cuda")
        # request i takes adapter i modulo their number; every fifth runs the shared weight alone
        ids = torch.tensor([-1 if i % 5 == 4 else i % case["adapters"] for i in range(case["requests"])],
                           dtype=torch.int32, device="cuda")
        s["row_adapter"] = ids.repeat_interleave(torch.tensor(_rows_of(case), device="cuda"))
    return s


# ------------------------------------------------------------------------------------- one pass
def run(s):
    return _run_own(s) if own else {"qk": _plain_qk, "cross": _plain_cross, "adapters": _plain_adapters}[s["op"]](s)


def _run_own(s):
    package = os.path.abspath("cuda-msst-infer_b200")
    if package not in sys.path:
        sys.path.insert(0, package)
    from msst_b200 import ops

    if s["op"] == "qk":
        return ops.qk_norm_rope(s["q"], s["k"], s["q_gamma"], s["k_gamma"], s["cos"], s["sin"],
                                positions=s["positions"], eps=1e-6, pairing=s["pairing"])
    if s["op"] == "cross":
        return ops.cross_attention(s["q"], s["k"], s["v"], key_lens=s["key_lens"], key_mask=s["key_mask"])
    return ops.adapter_gemm(s["x"], s["w"], s["lora_a"], s["lora_b"], s["row_adapter"], scales=s["scales"],
                            bias=s["bias"])


def _plain_rotate(x, gamma, cos, sin, pairing):
    y = x.float()
    y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + 1e-6) * gamma
    half = cos.shape[-1]
    turn, rest = y[..., :2 * half], y[..., 2 * half:]
    if pairing == "halves":
        a, b = turn[..., :half], turn[..., half:]
        out = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    else:
        a, b = turn[..., 0::2], turn[..., 1::2]
        out = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    return torch.cat((out, rest), -1).to(x.dtype)


def _plain_qk(s):
    if s["positions"] is None:
        cos, sin = s["cos"][None, :, None], s["sin"][None, :, None]
    else:
        at = s["positions"].long()
        cos, sin = s["cos"][at][:, :, None], s["sin"][at][:, :, None]
    return (_plain_rotate(s["q"], s["q_gamma"], cos, sin, s["pairing"]),
            _plain_rotate(s["k"], s["k_gamma"], cos, sin, s["pairing"]))


def _plain_cross(s):
    q, k, v = s["q"].float(), s["k"].float(), s["v"].float()
    b, nq, hq, d = q.shape
    nk, hk = k.shape[1:3]
    q = q.view(b, nq, hk, hq // hk, d).permute(0, 2, 3, 1, 4).reshape(b, hk, -1, d)
    score = q @ k.permute(0, 2, 3, 1)
    score *= d ** -0.5
    keep = s["key_mask"]
    if s["key_lens"] is not None:
        keep = torch.arange(nk, device=q.device) < s["key_lens"][:, None]
    if keep is not None:
        score.masked_fill_(~keep[:, None, None], -torch.inf)
    top = score.amax(-1, keepdim=True)
    score -= torch.where(top == -torch.inf, 0.0, top)
    score.exp_()
    total = score.sum(-1, keepdim=True)
    out = (score @ v.transpose(1, 2)) / torch.where(total == 0, 1.0, total)
    return out.view(b, hk, hq // hk, nq, d).permute(0, 3, 1, 2, 4).reshape(b, nq, hq, d).to(s["q"].dtype)


def _plain_adapters(s):
    x = s["x"].float()
    y = x @ s["w"].float().t()
    if s["bias"] is not None:
        y += s["bias"]
    count, rank, k = s["lora_a"].shape
    u = (x @ s["lora_a"].float().view(-1, k).t()).view(-1, count, rank)
    mine = s["row_adapter"][:, None] == torch.arange(count, device=x.device)
    u *= (mine * s["scales"])[:, :, None]
    y += u.view(-1, count * rank) @ s["lora_b"].float().permute(0, 2, 1).reshape(count * rank, -1)
    return y.to(s["x"].dtype)


# ------------------------------------------------------------------------------------- 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "qk":
        return tuple(_exact_qk(s[x].double(), s[x + "_gamma"].double(), s) for x in ("q", "k"))
    if case["op"] == "cross":
        return _exact_cross(s)
    return _exact_adapters(s)


def _exact_qk(x, gamma, s):
    """Each pair as a complex number times exp(i angle)."""
    b, n, h, d = x.shape
    y = x / (torch.linalg.vector_norm(x, dim=-1, keepdim=True).pow(2) / d + 1e-6).sqrt() * gamma
    at = torch.arange(n, device=x.device).expand(b, n) if s["positions"] is None else s["positions"].long()
    turn = torch.complex(s["cos"].double(), s["sin"].double())[at].unsqueeze(2)
    half = turn.shape[-1]
    first = torch.arange(half, device=x.device) * (2 if s["pairing"] == "interleaved" else 1)
    second = first + (1 if s["pairing"] == "interleaved" else half)
    z = torch.complex(y[..., first], y[..., second]) * turn
    y[..., first], y[..., second] = z.real, z.imag
    return y


def _exact_cross(s):
    """Head by head over the keys that are left, through the logarithm of the sum."""
    b, nq, hq, d = s["q"].shape
    hk = s["k"].shape[2]
    out = torch.zeros(b, nq, hq, d, dtype=torch.float64, device=s["q"].device)
    for i in range(b):
        if s["key_lens"] is not None:
            left = torch.arange(int(s["key_lens"][i]), device=out.device)
        elif s["key_mask"] is not None:
            left = s["key_mask"][i].nonzero().flatten()
        else:
            left = torch.arange(s["k"].shape[1], device=out.device)
        if not left.numel():
            continue
        for h in range(hq):
            k, v = s["k"][i, left, h * hk // hq].double(), s["v"][i, left, h * hk // hq].double()
            score = torch.einsum("nd,md->nm", s["q"][i, :, h].double(), k) / d ** 0.5
            out[i, :, h] = torch.exp(score - torch.logsumexp(score, 1, keepdim=True)) @ v
    return out


def _exact_adapters(s):
    """Adapter by adapter over the rows that have it."""
    out = s["x"].double() @ s["w"].double().T
    if s["bias"] is not None:
        out = out + s["bias"].double()
    for a in range(s["lora_a"].shape[0]):
        rows = (s["row_adapter"] == a).nonzero().flatten()
        delta = s["x"][rows].double() @ s["lora_a"][a].double().T @ s["lora_b"][a].double().T
        out[rows] += float(s["scales"][a]) * delta
    return out
