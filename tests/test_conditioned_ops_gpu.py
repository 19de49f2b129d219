"""GPU tests of the operators of conditioned blocks (msst_qk_norm_rope,
msst_cross_attention, msst_adapter_gemm) against plain 64-bit forms of the same
16-bit inputs, element by element.

Tolerances, with u = 2^-11 (fp16) or 2^-8 (bf16) the unit roundoff of the 16-bit type
and e = 2^-24 that of fp32:
* qk_norm_rope: one rounding of the result, u |y|; inside, fp32: the sum of squares,
  rsqrt and four products, bounded by 16 e (|a| + |b|) of the pair; half of fp16's
  smallest subnormal, 2^-25.
* cross_attention: the result's rounding, u |y|; the weights of P V are rounded to 16
  bits, u A with A = softmax(s) |v|; the scores carry d fp32 roundings, which move a
  weight by 2 d e max_j sum|q k_j| scale (numerator and sum), and an exponential
  good to 2^-21, each on A; the fp32 sum of P V over the keys, 2 Nk e A; fp16 weights
  below 2^-14 of the largest lose relative precision: Nk 2^-25 max|v|.
* adapter_gemm: the result's rounding, u |y|; fp32 sums (K + rank + 8) e (sum|w x| +
  |bias| + sum|B| |A x|-sums); the low-rank values are rounded to 16 bits once, u sum|s u B|,
  plus 2^-25 sum|B| where fp16 is subnormal.
"""
from __future__ import annotations

import math

import pytest

pytestmark = pytest.mark.gpu

U = {"fp16": 2.0 ** -11, "bf16": 2.0 ** -8}
E = 2.0 ** -24
TINY = {"fp16": 2.0 ** -25, "bf16": 0.0}


def _dt(torch, prec):
    return torch.float16 if prec == "fp16" else torch.bfloat16


def _gen(torch, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _within(y, ref, bound, what):
    err = (y.double() - ref).abs()
    assert bool((err <= bound).all()), f"{what}: {float((err - bound).max()):.3g} over, worst ratio " \
                                       f"{float((err / bound.clamp_min(1e-300)).max()):.3g}"


# ------------------------------------------------------------------ norms + rotation
def _qk_ref(torch, x, gamma, cos, sin, at, eps, pairing):
    """(y, bound on the fp32 arithmetic) of one tensor [B, N, H, d] in 64 bits."""
    y = x.double()
    d = y.shape[-1]
    y = y / (y.pow(2).sum(-1, keepdim=True) / d + eps).sqrt()
    if gamma is not None:
        y = y * gamma.double()
    mag = y.abs()
    if cos is not None:
        half = cos.shape[1]
        i = torch.arange(half, device=y.device)
        first, second = (2 * i, 2 * i + 1) if pairing == "interleaved" else (i, i + half)
        c, s = cos.double()[at].unsqueeze(-2), sin.double()[at].unsqueeze(-2)
        a, b = y[..., first], y[..., second]
        mag[..., first] = mag[..., second] = a.abs() + b.abs()
        y[..., first], y[..., second] = a * c - b * s, b * c + a * s
    return y, 16 * E * mag


def _tables(torch, n, half):
    ang = torch.arange(n, device="cuda", dtype=torch.float64)[:, None] * \
        100.0 ** (-torch.arange(half, device="cuda", dtype=torch.float64) / max(half, 1))
    return ang.cos().float(), ang.sin().float()


QK_CASES = [
    # B, N, Hq, Hk, d, rot, layout
    (1, 1, 1, 1, 64, 64, "bnhd"),
    (2, 33, 8, 8, 64, 64, "packed"),
    (3, 17, 8, 2, 128, 128, "bnhd"),
    (2, 5, 6, 3, 128, 64, "bhnd"),
    (1, 70, 5, 1, 48, 32, "bnhd"),
    (1, 9, 3, 1, 48, 24, "packed"),
    (2, 7, 4, 4, 80, 80, "bhnd"),
    (2, 40, 9, 5, 96, 96, "packed"),
    (1, 13, 2, 1, 256, 256, "bnhd"),
    (2, 3, 3, 2, 256, 128, "bhnd"),
    (2, 6, 3, 1, 10, 6, "bnhd"),       # no 8-column loads
    (1, 11, 2, 2, 2, 2, "bnhd"),
    (1, 4, 3, 2, 64, 62, "packed"),    # rotation ends inside a group of columns
    (1, 4, 3, 2, 64, 0, "bnhd"),       # norm alone
    (4, 257, 16, 2, 8, 8, "bnhd"),
    (1, 5, 1, 1, 72, 16, "odd"),       # rows that start off 16 bytes
]


@pytest.mark.parametrize("prec", ["fp16", "bf16"])
@pytest.mark.parametrize("pairing", ["interleaved", "halves"])
@pytest.mark.parametrize("case", QK_CASES, ids=lambda c: "-".join(map(str, c)))
def test_qk_norm_rope(cuda, case, pairing, prec):
    torch = cuda
    from msst_b200 import device_error, ops

    B, N, Hq, Hk, d, rot, layout = case
    g, dt = _gen(torch, B * 100 + N + d), _dt(torch, prec)

    def make(h):
        if layout == "bhnd":
            return torch.randn(B, h, N, d, generator=g, device="cuda").to(dt).transpose(1, 2)
        if layout == "odd":
            return torch.randn(B, N, h * d + 3, generator=g, device="cuda").to(dt)[..., 1:1 + h * d].unflatten(-1, (h, d))
        return torch.randn(B, N, h, d, generator=g, device="cuda").to(dt)

    if layout == "packed":  # [N, B, (q k v) heads, d] rows
        allh = torch.randn(N, B, Hq + 2 * Hk, d, generator=g, device="cuda").to(dt).transpose(0, 1)
        q, k = allh[:, :, :Hq], allh[:, :, Hq:Hq + Hk]
    else:
        q, k = make(Hq), make(Hk)
    q[0, 0, 0] = 0  # an all-zero vector: eps alone under the root
    qg = 1 + 0.3 * torch.randn(d, generator=g, device="cuda")
    kg = None if B == 2 else 1 + 0.3 * torch.randn(d, generator=g, device="cuda")
    cos, sin = _tables(torch, N + 50, rot // 2) if rot else (None, None)
    pos = None if N % 2 else torch.randint(0, N + 50, (B, N), generator=g, device="cuda", dtype=torch.int32)
    at = torch.arange(N, device="cuda").expand(B, N) if pos is None else pos.long()
    yq, yk = ops.qk_norm_rope(q, k, qg, kg, cos, sin, positions=pos, eps=1e-5, pairing=pairing)
    for y, x, gm in ((yq, q, qg), (yk, k, kg)):
        ref, arith = _qk_ref(torch, x, gm, cos, sin, at, 1e-5, pairing)
        _within(y, ref, U[prec] * ref.abs() + arith * (1 + U[prec]) + TINY[prec] + 1e-30, "qk_norm_rope")
    one, none = ops.qk_norm_rope(q, None, qg, None, cos, sin, positions=pos, eps=1e-5, pairing=pairing)
    assert none is None and torch.equal(one, yq)
    # in place, in the operands' own layout
    q2, k2 = q.clone(), k.clone()
    if layout == "packed":
        buf = allh.transpose(0, 1).clone().transpose(0, 1)
        q2, k2 = buf[:, :, :Hq], buf[:, :, Hq:Hq + Hk]
    elif layout == "odd":
        q2, k2 = make(Hq).copy_(q), make(Hk).copy_(k)
    iq, ik = ops.qk_norm_rope(q2, k2, qg, kg, cos, sin, positions=pos, eps=1e-5, pairing=pairing, out_q=q2, out_k=k2)
    assert iq is q2 and ik is k2 and torch.equal(q2, yq) and torch.equal(k2, yk)
    if layout == "packed":
        assert torch.equal(buf[:, :, Hq + Hk:], allh[:, :, Hq + Hk:])
    assert device_error(True) == 0


def test_qk_norm_rope_extremes(cuda):
    """Large values whose squares pass fp16 (not fp32), infinities and NaN stay in their head vector."""
    torch = cuda
    from msst_b200 import ops

    g = _gen(torch, 5)
    q = torch.randn(1, 4, 8, 64, generator=g, device="cuda").half()
    q[0, 0] *= 30000 / q[0, 0].abs().max()
    clean = q.clone()
    q[0, 1, 3, 5] = float("inf")
    q[0, 2, 4, 6] = float("nan")
    cos, sin = _tables(torch, 4, 32)
    y, _ = ops.qk_norm_rope(q, None, None, None, cos, sin, pairing="halves")
    z, _ = ops.qk_norm_rope(clean, None, None, None, cos, sin, pairing="halves")
    hurt = torch.zeros(1, 4, 8, dtype=torch.bool, device="cuda")
    hurt[0, 1, 3] = hurt[0, 2, 4] = True
    assert torch.equal(y[~hurt], z[~hurt]) and bool(z.isfinite().all())
    assert bool(y[0, 1, 3].isnan().any()) and bool(y[0, 2, 4].isnan().all())


def test_qk_norm_rope_position_outside(cuda):
    """A position outside the tables leaves its token unrotated and is reported."""
    torch = cuda
    from msst_b200 import device_error, ops

    g = _gen(torch, 6)
    for d in (64, 10):
        q = torch.randn(1, 3, 2, d, generator=g, device="cuda").half()
        cos, sin = _tables(torch, 4, d // 2)
        pos = torch.tensor([[1, 4, -1]], dtype=torch.int32, device="cuda")
        y, _ = ops.qk_norm_rope(q, None, None, None, cos, sin, positions=pos)
        assert device_error(True) == 14 and device_error(True) == 0
        plain, _ = ops.qk_norm_rope(q)
        assert torch.equal(y[:, 1:], plain[:, 1:]) and not torch.equal(y[:, :1], plain[:, :1])


# ------------------------------------------------------------------ cross attention
def _cross_check(torch, y, q, k, v, keep, scale, prec):
    """keep [B, Nk] bool; one batch entry and head at a time."""
    B, Nq, Hq, d = q.shape
    Nk, Hk = k.shape[1:3]
    u = U[prec]
    for b in range(B):
        left = keep[b].nonzero().flatten()
        if left.numel() == 0:
            assert bool((y[b] == 0).all())
            continue
        for h in range(Hq):
            qq, kk, vv = q[b, :, h].double(), k[b, left, h * Hk // Hq].double(), v[b, left, h * Hk // Hq].double()
            s = qq @ kk.T * scale
            p = torch.softmax(s, -1)
            ref, A = p @ vv, p @ vv.abs()
            move = 2 * d * E * (qq.abs() @ kk.abs().T).amax(-1, keepdim=True) * abs(scale) + 2.0 ** -20
            n = left.numel()
            bound = u * ref.abs() + (1 + u) * A * (u + move + 2 * n * E) + n * TINY[prec] * vv.abs().amax(0) + 1e-30
            _within(y[b, :, h], ref, bound + TINY[prec], f"batch {b} head {h}")


def _cross_inputs(torch, B, Nq, Nk, Hq, Hk, d, prec, seed, layout="kv"):
    g, dt = _gen(torch, seed), _dt(torch, prec)

    def r(*s):
        return torch.randn(*s, generator=g, device="cuda").to(dt)

    if layout == "bhnd":
        return r(B, Hq, Nq, d).transpose(1, 2), r(B, Hk, Nk, d).transpose(1, 2), r(B, Hk, Nk, d).transpose(1, 2)
    q, kv = r(B, Nq, Hq, d), r(B, Nk, 2, Hk, d)
    return q, kv[:, :, 0], kv[:, :, 1]


CROSS_CASES = [
    # B, Nq, Nk, Hq, Hk, d, mask, layout
    (1, 1, 1, 1, 1, 64, "none", "kv"),
    (2, 1, 129, 8, 2, 128, "lens", "kv"),
    (3, 1, 1000, 4, 4, 64, "keys", "kv"),
    (1, 1, 4097, 8, 1, 128, "none", "bhnd"),
    (1, 1, 20011, 2, 2, 64, "lens", "kv"),
    (2, 1, 700, 6, 2, 80, "keys", "bhnd"),
    (1, 1, 300, 32, 1, 64, "none", "kv"),      # 32 rows share a key head
    (2, 3, 515, 15, 3, 48, "lens", "kv"),      # 5 query heads a key head
    (1, 7, 33, 3, 1, 8, "keys", "kv"),
    (2, 16, 64, 4, 4, 128, "none", "bhnd"),
    (2, 17, 65, 4, 4, 128, "lens", "kv"),
    (1, 40, 2000, 3, 1, 40, "lens", "kv"),
    (1, 33, 9001, 2, 2, 128, "keys", "kv"),
    (2, 127, 128, 4, 2, 64, "none", "kv"),
    (2, 128, 127, 4, 2, 64, "lens", "bhnd"),
    (1, 129, 257, 3, 3, 64, "keys", "kv"),
    (5, 77, 1501, 12, 4, 80, "keys", "kv"),
    (2, 255, 384, 6, 2, 128, "lens", "kv"),
    (1, 300, 300, 7, 1, 128, "none", "kv"),    # 7 query heads a key head
    (3, 513, 640, 2, 1, 16, "both", "kv"),
    (2, 700, 1025, 8, 8, 64, "lens", "kv"),
    (1, 260, 130, 130, 1, 32, "none", "kv"),   # more query heads a key head than a tile has rows
]


def _keep(torch, B, Nk, mask, seed):
    g = _gen(torch, seed + 1)
    lens = km = None
    keep = torch.ones(B, Nk, dtype=torch.bool, device="cuda")
    if mask in ("lens", "both"):
        lens = torch.randint(0, Nk + 1, (B,), generator=g, device="cuda", dtype=torch.int32)
        lens[0] = Nk
        if B > 1:
            lens[1] = max(1, Nk // 3)
        if B > 2:
            lens[2] = 0
        keep &= torch.arange(Nk, device="cuda") < lens[:, None]
    if mask in ("keys", "both"):
        km = torch.rand(B, Nk, generator=g, device="cuda") < 0.6
        if B > 1:
            km[1] = False
        if Nk > 200:
            km[0, : Nk // 2] = False  # whole tiles without a kept key, the first among them
        keep &= km
    return keep, lens, km


@pytest.mark.parametrize("prec", ["fp16", "bf16"])
@pytest.mark.parametrize("case", CROSS_CASES, ids=lambda c: "-".join(map(str, c)))
def test_cross_attention(cuda, case, prec):
    torch = cuda
    from msst_b200 import device_error, ops

    B, Nq, Nk, Hq, Hk, d, mask, layout = case
    seed = B * 7 + Nq * 3 + Nk + Hq
    q, k, v = _cross_inputs(torch, B, Nq, Nk, Hq, Hk, d, prec, seed, layout)
    keep, lens, km = _keep(torch, B, Nk, mask, seed)
    y = ops.cross_attention(q, k, v, key_lens=lens, key_mask=km)
    assert device_error(True) == 0
    _cross_check(torch, y, q, k, v, keep, d ** -0.5, prec)
    # what is not kept may hold anything
    if mask != "none":
        bad_k, bad_v = k.clone(), v.clone()
        fill = torch.tensor([float("nan"), float("inf"), -float("inf"), torch.finfo(k.dtype).min], device="cuda")
        pick = torch.arange(Nk, device="cuda") % 4
        junk = fill[pick].to(k.dtype)[None, :, None, None].expand_as(k)
        out = ~keep[:, :, None, None].expand_as(k)
        bad_k[out], bad_v[out] = junk[out], junk[out]
        z = ops.cross_attention(q, bad_k, bad_v, key_lens=lens, key_mask=km)
        assert torch.equal(y, z)
    # the same call gives the same bits
    assert torch.equal(y, ops.cross_attention(q, k, v, key_lens=lens, key_mask=km))


@pytest.mark.parametrize("Nq", [1, 20, 200])
@pytest.mark.parametrize("prec", ["fp16", "bf16"])
def test_cross_attention_large_scores(cuda, Nq, prec):
    """Scores of several hundred, growing along the keys: the running maximum moves in every tile."""
    torch = cuda
    from msst_b200 import ops

    for d in (64, 128):
        q, k, v = _cross_inputs(torch, 2, Nq, 777, 4, 2, d, prec, 11 + d)
        q = q.abs() * 4
        k = (k.float().abs() * torch.linspace(0, 4, 777, device="cuda")[None, :, None, None]).to(k.dtype)
        keep, lens, _ = _keep(torch, 2, 777, "lens", 3)
        y = ops.cross_attention(q, k, v, key_lens=lens)
        _cross_check(torch, y, q, k, v, keep, d ** -0.5, prec)
        y = ops.cross_attention(q, k, v, key_lens=lens, scale=-0.25)  # and falls with a negative scale
        _cross_check(torch, y, q, k, v, keep, -0.25, prec)


@pytest.mark.parametrize("Nq", [1, 150])
def test_cross_attention_shared_states_and_out(cuda, Nq):
    """One encoder's states for the whole batch (stride 0), lengths outside [0, Nk], a strided out."""
    torch = cuda
    from msst_b200 import ops

    q, k, v = _cross_inputs(torch, 4, Nq, 333, 4, 2, 64, "fp16", 21)
    k, v = k[:1].expand(4, -1, -1, -1), v[:1].expand(4, -1, -1, -1)
    lens = torch.tensor([1000, -5, 333, 100], dtype=torch.int32, device="cuda")
    keep = torch.arange(333, device="cuda") < lens[:, None]
    big = torch.full((4, 4, Nq, 2, 64), 7.0, dtype=torch.float16, device="cuda")
    out = big[:, :, :, 0].transpose(1, 2)
    y = ops.cross_attention(q, k, v, key_lens=lens, out=out)
    assert y is out and bool((big[:, :, :, 1] == 7).all())
    _cross_check(torch, y, q, k, v, keep, 0.125, "fp16")
    # heads that share one key head through stride 0
    z = ops.cross_attention(q, k[:, :, :1].expand(-1, -1, 4, -1), v[:, :, :1].expand(-1, -1, 4, -1), key_lens=lens)
    w = ops.cross_attention(q, k[:, :, :1], v[:, :, :1], key_lens=lens)
    assert float((z.float() - w.float()).abs().max()) <= 4e-3


def test_cross_attention_unaligned_and_empty(cuda):
    torch = cuda
    from msst_b200 import ops

    q, k, v = _cross_inputs(torch, 1, 5, 50, 2, 1, 64, "fp16", 31)
    pad = torch.zeros(1, 5, 2, 67, dtype=torch.float16, device="cuda")
    pad[..., 1:65] = q
    y = ops.cross_attention(q, k, v)
    assert torch.equal(ops.cross_attention(pad[..., 1:65], k, v), y)
    flat = torch.zeros(5 * 2 * 64 + 1, dtype=torch.float16, device="cuda")[1:].view(1, 5, 2, 64).copy_(q)
    assert torch.equal(ops.cross_attention(flat, k, v), y)
    assert bool((ops.cross_attention(q, k[:, :0], v[:, :0]) == 0).all())
    assert ops.cross_attention(q[:, :0], k, v).shape == (1, 0, 2, 64)
    assert ops.cross_attention(q[:0], k[:0], v[:0]).shape == (0, 5, 2, 64)


# ------------------------------------------------------------------ adapters
def _adapter_inputs(torch, rows, K, N, count, rank, prec, seed):
    g, dt = _gen(torch, seed), _dt(torch, prec)

    def r(*s, scale=1.0):
        return (torch.randn(*s, generator=g, device="cuda") * scale).to(dt)

    x, w = r(rows, K), r(N, K, scale=K ** -0.5)
    la, lb = r(count, rank, K, scale=K ** -0.5), r(count, N, rank, scale=rank ** -0.5)
    ids = torch.randint(-1, count, (rows,), generator=g, device="cuda", dtype=torch.int32)
    scales = 0.5 + torch.rand(count, generator=g, device="cuda")
    bias = torch.randn(N, generator=g, device="cuda")
    return x, w, la, lb, ids, scales, bias


def _adapter_check(torch, y, x, w, la, lb, ids, scales, bias, prec):
    K, N, rank = x.shape[1], w.shape[0], la.shape[1]
    xd, wd = x.double(), w.double()
    ref, mass = xd @ wd.T, xd.abs() @ wd.abs().T
    if bias is not None:
        ref, mass = ref + bias.double(), mass + bias.double().abs()
    low = torch.zeros_like(ref)
    for a in range(la.shape[0]):
        t = (ids == a).nonzero().flatten()
        if not t.numel():
            continue
        s = float(scales[a]) if scales is not None else 1.0
        A, Bm = la[a].double(), lb[a].double()
        uu = s * (xd[t] @ A.T)
        ref[t] += uu @ Bm.T
        mass[t] += s * (xd[t].abs() @ A.abs().T) @ Bm.abs().T
        low[t] += U[prec] * uu.abs() @ Bm.abs().T + TINY[prec] * Bm.abs().sum(1)
    _within(y, ref, (U[prec] * ref.abs() + low + (K + rank + 8) * E * mass) * (1 + U[prec]) + TINY[prec], "adapter_gemm")


ADAPTER_CASES = [
    # rows, K, N, adapters, rank, order
    (1, 64, 64, 1, 8, "mixed"),
    (3, 512, 384, 5, 16, "mixed"),
    (16, 1000, 1032, 16, 16, "mixed"),
    (17, 8, 8, 2, 8, "mixed"),
    (33, 520, 264, 33, 24, "mixed"),
    (64, 2048, 512, 3, 64, "mixed"),
    (100, 384, 1536, 40, 32, "mixed"),
    (128, 384, 1536, 128, 16, "each"),
    (129, 256, 200, 2, 256, "sorted"),
    (300, 1024, 1024, 4, 40, "sorted"),
    (517, 384, 392, 7, 8, "mixed"),
    (1000, 640, 2056, 3, 128, "sorted"),
    (2500, 384, 1536, 5, 8, "sorted"),
    (700, 264, 136, 1, 16, "none"),
]


@pytest.mark.parametrize("prec", ["fp16", "bf16"])
@pytest.mark.parametrize("case", ADAPTER_CASES, ids=lambda c: "-".join(map(str, c)))
def test_adapter_gemm(cuda, case, prec):
    torch = cuda
    from msst_b200 import device_error, ops

    rows, K, N, count, rank, order = case
    x, w, la, lb, ids, scales, bias = _adapter_inputs(torch, rows, K, N, count, rank, prec, rows + K)
    if order == "sorted":
        ids = ids.sort().values
    elif order == "each":
        ids = torch.randperm(count, device="cuda")[:rows].int()
    elif order == "none":
        ids = torch.full_like(ids, -1)
    if rows % 2:
        scales = None
    if rows % 3 == 0:
        bias = None
    y = ops.adapter_gemm(x, w, la, lb, ids, scales=scales, bias=bias)
    assert device_error(True) == 0
    _adapter_check(torch, y, x, w, la, lb, ids, scales, bias, prec)
    assert torch.equal(y, ops.adapter_gemm(x, w, la, lb, ids, scales=scales, bias=bias))
    # a request's rows do not take in what other requests' rows or adapters hold
    if count > 1 and rows > 2:
        bad = ids == 0
        x2, la2, lb2 = x.clone(), la.clone(), lb.clone()
        la2[0], lb2[0] = float("nan"), float("inf")
        z = ops.adapter_gemm(x2, w, la2, lb2, ids, scales=scales, bias=bias)
        assert torch.equal(z[~bad], y[~bad])


def test_adapter_gemm_strides_and_ids(cuda):
    torch = cuda
    from msst_b200 import device_error, ops

    x, w, la, lb, ids, scales, bias = _adapter_inputs(torch, 50, 128, 64, 3, 16, "fp16", 77)
    y = ops.adapter_gemm(x, w, la, lb, ids, scales=scales, bias=bias)
    wide = torch.zeros(50, 200, dtype=torch.float16, device="cuda")
    wide[:, 8:136] = x
    big = torch.full((50, 80), 3.0, dtype=torch.float16, device="cuda")
    z = ops.adapter_gemm(wide[:, 8:136], w, la, lb, ids, scales=scales, bias=bias, out=big[:, 8:72])
    assert torch.equal(z, y) and bool((big[:, :8] == 3).all()) and bool((big[:, 72:] == 3).all())
    assert torch.equal(ops.adapter_gemm(x.view(5, 10, 128), w, la, lb, ids.view(5, 10), scales=scales, bias=bias),
                       y.view(5, 10, 64))
    off = ids.clone()
    off[::2] = 3 + torch.arange(25, device="cuda", dtype=torch.int32)
    off[1] = -7
    z = ops.adapter_gemm(x, w, la, lb, off, scales=scales, bias=bias)
    assert device_error(True) == 15
    none = torch.where((off < 0) | (off >= 3), -1, off).int()
    assert torch.equal(z, ops.adapter_gemm(x, w, la, lb, none, scales=scales, bias=bias))
    assert device_error(True) == 0
    assert ops.adapter_gemm(x[:0], w, la, lb, ids[:0]).shape == (0, 64)
    plain = ops.adapter_gemm(x, w, la[:0], lb[:0], torch.full_like(ids, -1), bias=bias)
    _adapter_check(torch, plain, x, w, la, lb, torch.full_like(ids, -1), None, bias, "fp16")


# ------------------------------------------------------------------ streams
def test_operators_on_a_side_stream(cuda):
    """Launched on the current stream: results are ordered after work queued there."""
    torch = cuda
    from msst_b200 import ops

    q, k, v = _cross_inputs(torch, 2, 1, 5000, 8, 2, 64, "fp16", 41)
    want = ops.cross_attention(q, k, v)
    x, w, la, lb, ids, _, _ = _adapter_inputs(torch, 40, 512, 256, 3, 16, "fp16", 42)
    want2 = ops.adapter_gemm(x, w, la, lb, ids)
    qn, _ = ops.qk_norm_rope(q)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        big = torch.randn(4096, 4096, device="cuda")
        for _ in range(20):
            big = big @ big * 1e-3
        late_q, late_x = torch.empty_like(q), torch.empty_like(x)
        late_q.copy_(q)
        late_x.copy_(x)
        got, got2 = ops.cross_attention(late_q, k, v), ops.adapter_gemm(late_x, w, la, lb, ids)
        gotn, _ = ops.qk_norm_rope(late_q)
    s.synchronize()
    assert torch.equal(got, want) and torch.equal(got2, want2) and torch.equal(gotn, qn)


@pytest.mark.parametrize("op", ["masked", "pairs", "token", "adapters"])
def test_calls_back_to_back(cuda, op):
    """Many calls queued without a host wait between them give the first call's bits, and no kernel
    wait gives up (a wait that runs out takes two seconds and is recorded)."""
    torch = cuda
    from msst_b200 import device_error, ops

    if op == "adapters":
        x, w, la, lb, ids, scales, bias = _adapter_inputs(torch, 300, 640, 520, 9, 24, "bf16", 51)
        call = lambda: ops.adapter_gemm(x, w, la, lb, ids, scales=scales, bias=bias)  # noqa: E731
    else:
        B, Nq, Nk, Hq, Hk, d = dict(masked=(5, 77, 1501, 12, 4, 80), pairs=(2, 600, 1000, 4, 4, 64),
                                    token=(6, 1, 900, 8, 2, 128))[op]
        q, k, v = _cross_inputs(torch, B, Nq, Nk, Hq, Hk, d, "fp16", 52)
        _, lens, km = _keep(torch, B, Nk, "keys" if op == "masked" else "lens", 53)
        call = lambda: ops.cross_attention(q, k, v, key_lens=lens, key_mask=km)  # noqa: E731
    want = call()
    for _ in range(8):
        got = [call() for _ in range(40)]
        torch.cuda.synchronize()
        assert all(torch.equal(y, want) for y in got)
    assert device_error(True) == 0


def test_cross_attention_far_reference(cuda):
    """The first kept scores far below the later ones and far above them, in turns along the keys:
    the exponentials' reference has to move in the middle of a sequence, more than once."""
    torch = cuda
    from msst_b200 import ops

    for d, prec in ((64, "fp16"), (128, "bf16"), (96, "fp16")):
        q, k, v = _cross_inputs(torch, 1, 300, 1100, 2, 2, d, prec, 61)
        q = q.abs()
        level = torch.zeros(1100, device="cuda")
        level[100:130] = 3.0
        level[400:430] = 6.0
        level[900:910] = 9.0
        k = (k.float() * 0.2 + level[None, :, None, None]).to(k.dtype)
        keep = torch.ones(1, 1100, dtype=torch.bool, device="cuda")
        _cross_check(torch, ops.cross_attention(q, k, v), q, k, v, keep, d ** -0.5, prec)
        _cross_check(torch, ops.cross_attention(q[:, :1], k, v), q[:, :1], k, v, keep, d ** -0.5, prec)


# ------------------------------------------------------------------ the block they form
@pytest.mark.parametrize("prec", ["fp16", "bf16"])
def test_conditioned_block(cuda, prec):
    """ConditionedBlock against the same block in 64 bits.  Each of its four 16-bit intermediate
    results (q, k, attention, projection) is rounded once, u relative each, and a rounding of
    q or k moves a score by up to 2 u |q||k| scale <= 2 u sqrt(d) for normed vectors (gammas
    about 1); with the weights' rounding of the attention that is below
    u (4 + 2 * 2 * sqrt(64)) = 36 u of the attention's and the projections' size in the 2-norm."""
    torch = cuda
    from msst_b200 import device_error
    from msst_b200.conditioned import random_block

    blk = random_block(dtype=_dt(torch, prec), seed=3)
    g = _gen(torch, 8)
    B, Nq, Nk, d = 3, 70, 333, 64
    x = torch.randn(B, Nq, 512, generator=g, device="cuda").to(_dt(torch, prec))
    enc = torch.randn(B, Nk, 384, generator=g, device="cuda").to(_dt(torch, prec))
    lens = torch.tensor([333, 100, 0], dtype=torch.int32, device="cuda")
    who = torch.tensor([1, -1, 2], dtype=torch.int32, device="cuda")
    k, v = blk.encode(enc, who)
    y = blk(x, k, v, who, key_lens=lens)
    pos = torch.full((B, 1), Nq - 1, dtype=torch.int32, device="cuda")
    tok = blk(x[:, -1:], k, v, who, positions=pos, key_lens=lens)
    assert device_error(True) == 0

    def project(name, t):
        a, b, s = blk.adapters[name]
        out = t @ blk.w[name].double().T
        for i in range(B):
            if who[i] >= 0:
                out[i] += float(s[who[i]]) * (t[i] @ a[who[i]].double().T) @ b[who[i]].double().T
        return out

    q64 = project("q", x.double()).view(B, Nq, 8, d)
    kv = project("kv", enc.double()).view(B, Nk, 2, 2, d)
    q64, _ = _qk_ref(torch, q64, blk.q_gamma, blk.cos, blk.sin, torch.arange(Nq, device="cuda").expand(B, Nq), 1e-6, "halves")
    k64, _ = _qk_ref(torch, kv[:, :, 0], blk.k_gamma, blk.cos, blk.sin, torch.arange(Nk, device="cuda").expand(B, Nk), 1e-6, "halves")
    att = torch.zeros(B, Nq, 8, d, dtype=torch.float64, device="cuda")
    for i in range(B):
        n = int(lens[i])
        for h in range(8):
            if n:
                p = torch.softmax(q64[i, :, h] @ k64[i, :n, h // 4].T / math.sqrt(d), -1)
                att[i, :, h] = p @ kv[i, :n, 1, h // 4]
    delta = project("o", att.reshape(B, Nq, -1))
    ref = x.double() + delta
    bar = 36 * U[prec] * float(delta.norm()) + U[prec] * float(ref.norm())
    assert float((y.double() - ref).norm()) <= bar
    assert float((tok.double() - ref[:, -1:]).norm()) <= 36 * U[prec] * float(delta[:, -1:].norm()) + \
        U[prec] * float(ref[:, -1:].norm())


# many tiles (rows on the MMA's M side: more 128 x 128 tiles than SMs), several tiles of rows beside
# the weights, and each width of the split along K (2, 4 and 8 CTAs)
ADAPTER_PLANS = [
    (2501, 264, 1032, 6, 24, "mixed"),
    (3333, 72, 776, 9, 8, "sorted"),
    (1290, 136, 2056, 3, 128, "mixed"),
    (130, 2048, 1032, 4, 16, "mixed"),
    (385, 2056, 1544, 2, 40, "sorted"),
    (40, 4096, 648, 40, 16, "each"),
    (257, 4104, 520, 5, 16, "mixed"),
    (5, 8200, 264, 5, 16, "mixed"),
    (150, 8192, 136, 3, 72, "mixed"),
]


@pytest.mark.parametrize("prec", ["fp16", "bf16"])
@pytest.mark.parametrize("case", ADAPTER_PLANS, ids=lambda c: "-".join(map(str, c)))
def test_adapter_gemm_plans(cuda, case, prec):
    test_adapter_gemm(cuda, case, prec)


# runs that end with the items (one item, several, a key head's pairs and lone tile) or cut them evenly
CROSS_RUNS = [
    (8, 100, 600, 8, 8, 64, "none", "kv"),
    (16, 32, 300, 8, 8, 64, "keys", "kv"),
    (30, 16, 300, 32, 16, 64, "none", "kv"),
    (4, 257, 256, 16, 16, 64, "keys", "bhnd"),
    (2, 77, 1501, 12, 12, 64, "none", "kv"),
    (1, 300, 2000, 16, 4, 128, "keys", "kv"),
    (4, 257, 1024, 16, 16, 64, "none", "kv"),
    (2, 300, 77, 8, 8, 128, "keys", "kv"),      # items of one unit
    (1, 1, 4096, 32, 8, 128, "none", "kv"),
    (4, 1, 1500, 8, 8, 64, "keys", "kv"),
    (64, 1, 200, 8, 8, 64, "none", "bhnd"),
]


@pytest.mark.parametrize("prec", ["fp16", "bf16"])
@pytest.mark.parametrize("case", CROSS_RUNS, ids=lambda c: "-".join(map(str, c)))
def test_cross_attention_runs(cuda, case, prec):
    test_cross_attention(cuda, case, prec)
