"""GPU tests of the conditioned-block operators at the edges of their ranges: values that do not
fit 16 bits, infinities, many keys of tiny weight, codes of several errors, graphs and threads.
Reference forms and tolerances as in test_conditioned_ops_gpu.py, unless a test derives its own."""
from __future__ import annotations

import math
import threading

import pytest

from test_conditioned_ops_gpu import (U, _adapter_check, _adapter_inputs, _cross_check, _cross_inputs, _dt, _gen, _qk_ref,
                                      _tables, _within)

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------ norms: very many tokens
@pytest.mark.parametrize("d, tokens", [(136, 2 ** 27 + 5), (72, 2 ** 28 + 5)])
def test_qk_norm_rope_past_32_bits_of_threads(cuda, d, tokens):
    """In place over 36 to 39 GB of one-head tokens, more than 2^32 threads: the first and the last
    tokens are normed, once."""
    torch = cuda
    from msst_b200 import device_error, ops

    if torch.cuda.mem_get_info()[0] < 45e9:
        pytest.skip("needs 45 GB of device memory")
    x = torch.empty(1, tokens, 1, d, dtype=torch.bfloat16, device="cuda")
    some = torch.tensor([0, 1, 2, 3, 4, 5, tokens // 2, tokens - 6, tokens - 5, tokens - 4, tokens - 1], device="cuda")
    before = (3 * torch.randn(1, some.numel(), 1, d, generator=_gen(torch, 2), device="cuda")).bfloat16()
    x[:, some] = before
    ops.qk_norm_rope(x, out_q=x)
    got = x[:, some]
    del x
    torch.cuda.empty_cache()
    ref, arith = _qk_ref(torch, before, None, None, None, None, 1e-6, "halves")
    _within(got, ref, U["bf16"] * ref.abs() + arith * 2 + 1e-30, "qk_norm_rope")
    assert device_error(True) == 0


# ------------------------------------------------------------------ norms: infinities
@pytest.mark.parametrize("prec", ["fp16", "bf16"])
@pytest.mark.parametrize("pairing", ["interleaved", "halves"])
@pytest.mark.parametrize("d, rot", [(64, 32), (48, 0), (10, 6)])
def test_qk_norm_rope_infinity_beside_the_rotation(cuda, d, rot, pairing, prec):
    """An infinite column that is not rotated, in the tail or for a position outside the tables, is NaN
    after its norm (inf / inf); its neighbour is x / inf = 0, since nothing turns it."""
    torch = cuda
    from msst_b200 import device_error, ops

    q = torch.randn(1, 4, 3, d, generator=_gen(torch, 9), device="cuda").to(_dt(torch, prec))
    col = d - 2
    q[0, 1, 1, col] = float("inf")
    q[0, 2, 2, col + 1] = -float("inf")
    q[0, 3, 0, 0] = float("inf")
    cos, sin = _tables(torch, 4, rot // 2) if rot else (None, None)
    pos = torch.tensor([[0, 1, 2, 4]], dtype=torch.int32, device="cuda")
    y, _ = ops.qk_norm_rope(q, None, None, None, cos, sin, positions=pos, pairing=pairing)
    assert device_error(True) == (14 if rot else 0)
    want = torch.zeros(1, 4, 3, d, dtype=torch.bool, device="cuda")
    want[0, 1, 1, col] = want[0, 2, 2, col + 1] = want[0, 3, 0, 0] = True
    assert torch.equal(y.isnan(), want)
    hurt = want.any(-1, keepdim=True)
    assert bool((y[hurt.expand_as(y) & ~want] == 0).all()) and bool(y[~hurt.expand_as(y)].isfinite().all())


# ------------------------------------------------------------------ codes of several errors
def test_device_error_of_two_operators(cuda):
    """A position and an adapter index outside their ranges before the host asks: both are reported."""
    torch = cuda
    from msst_b200 import device_error, ops

    device_error(True)
    q = torch.randn(1, 3, 2, 64, generator=_gen(torch, 6), device="cuda").half()
    cos, sin = _tables(torch, 4, 32)
    x, w, la, lb, ids, _, _ = _adapter_inputs(torch, 10, 64, 64, 2, 8, "fp16", 7)
    ids[3] = 2
    ops.adapter_gemm(x, w, la, lb, ids)
    ops.qk_norm_rope(q, None, None, None, cos, sin, positions=torch.full((1, 3), 4, dtype=torch.int32, device="cuda"))
    assert device_error(False) == 14 and device_error(False) == 14
    assert device_error(True) == 14 and device_error(True) == 15 and device_error(True) == 0


# ------------------------------------------------------------------ adapters: values off fp16's range
# rows, K, N, adapters, rank: weights on the MMA's M side whole and split along K, rows on it
ADAPTER_SIDES = [(40, 264, 136, 3, 16), (5, 8200, 264, 5, 24), (2501, 264, 1032, 6, 24)]


@pytest.mark.parametrize("prec", ["fp16", "bf16"])
@pytest.mark.parametrize("order", ["mixed", "sorted"])
@pytest.mark.parametrize("case", ADAPTER_SIDES, ids=lambda c: "-".join(map(str, c)))
def test_adapter_gemm_large_low_rank_values(cuda, case, order, prec):
    """A_a x about 1e5 (above fp16's 65504 for about half the values) against a B_a about 1e-4."""
    torch = cuda
    from msst_b200 import device_error, ops

    x, w, la, lb, ids, scales, bias = _adapter_inputs(torch, *case, prec, 5 + case[0])
    ids[0], ids[1], ids[2] = 0, -1, 1
    if order == "sorted":
        ids = ids.sort().values
    la[0] *= 2.0 ** 17
    lb[0] *= 2.0 ** -14
    u = x[ids == 0].double() @ la[0].double().T
    assert bool((u.abs() > 65504).any()) and bool((u.abs() < 65504).any())
    y = ops.adapter_gemm(x, w, la, lb, ids, scales=scales, bias=bias)
    assert device_error(True) == 0
    _adapter_check(torch, y, x, w, la, lb, ids, scales, bias, prec)
    assert torch.equal(y, ops.adapter_gemm(x, w, la, lb, ids, scales=scales, bias=bias))
    # rows of the other adapters are as they are without those values
    la[0] *= 2.0 ** -17
    z = ops.adapter_gemm(x, w, la, lb, ids, scales=scales, bias=bias)
    assert torch.equal(z[ids != 0], y[ids != 0])


@pytest.mark.parametrize("rows", [3, 2501])
def test_adapter_gemm_large_values_cancel(cuda, rows):
    """-2.2 * 64992 + 1 * 150000: neither the first product nor the sum without the part above 65504
    fits fp16, the result does."""
    torch = cuda
    from msst_b200 import ops

    N = 1032
    x = torch.zeros(rows, 64, dtype=torch.float16, device="cuda")
    x[:, 0], x[:, 1] = 1, 2.5
    la = torch.zeros(2, 8, 64, dtype=torch.float16, device="cuda")
    la[1, 0, 0], la[1, 1, 1] = 64992, 60000
    lb = torch.zeros(2, N, 8, dtype=torch.float16, device="cuda")
    lb[1, :, 0], lb[1, :, 1] = -2.2, 1
    w = torch.zeros(N, 64, dtype=torch.float16, device="cuda")
    ids = torch.ones(rows, dtype=torch.int32, device="cuda")
    ids[1::2] = -1
    y = ops.adapter_gemm(x, w, la, lb, ids)
    _adapter_check(torch, y, x, w, la, lb, ids, None, None, "fp16")
    assert bool((y[::2] > 6000).all()) and bool((y[1::2] == 0).all())


# ------------------------------------------------------------------ adapters: infinities in a B_a
@pytest.mark.parametrize("prec", ["fp16", "bf16"])
@pytest.mark.parametrize("order", ["mixed", "sorted"])
@pytest.mark.parametrize("case", ADAPTER_SIDES, ids=lambda c: "-".join(map(str, c)))
def test_adapter_gemm_nonfinite_b(cuda, case, order, prec):
    """Single Inf, -Inf and NaN entries of one adapter's B_a reach that adapter's rows in their own
    columns, with the right sign, and nothing else."""
    torch = cuda
    from msst_b200 import device_error, ops

    x, w, la, lb, ids, scales, bias = _adapter_inputs(torch, *case, prec, 15 + case[0])
    ids[0], ids[1], ids[2] = 0, -1, 1
    if order == "sorted":
        ids = ids.sort().values
    y = ops.adapter_gemm(x, w, la, lb, ids, scales=scales, bias=bias)
    N, rank = lb.shape[1:]
    plus, minus, nan = (3, 2), (N // 2 + 1, rank - 1), (N - 1, 5)
    bad = lb.clone()
    bad[1][plus], bad[1][minus], bad[1][nan] = float("inf"), -float("inf"), float("nan")
    z = ops.adapter_gemm(x, w, la, bad, ids, scales=scales, bias=bias)
    assert device_error(True) == 0
    hit = torch.zeros_like(y, dtype=torch.bool)
    rows = ids == 1
    for col, _ in (plus, minus, nan):
        hit[rows, col] = True
    assert torch.equal(z[~hit], y[~hit])
    u = scales[1].double() * (x[rows].double() @ la[1].double().T)
    for (col, r), sign in ((plus, 1), (minus, -1)):
        sure = u[:, r].abs() > 1e-2  # far from where a sum in fp32 could turn the sign
        assert torch.equal(z[rows, col].double()[sure], sign * u[sure, r].sign() * float("inf"))
    assert bool(z[rows, nan[0]].isnan().all())


# ------------------------------------------------------------------ cross attention: many tiny weights
@pytest.mark.parametrize("form", ["token", "tiles"])
def test_cross_attention_many_small_weights(cuda, form):
    """fp16 weights just below 2^-25 of their reference, 2^18 of them for each large one: they are
    0.8 % of the sum.  Every v is 1, so every output is 1.

    Bound: the result's and the weights' roundings, 2^-11 each; the fp32 sums: 2^14 products of 16
    keys added to about 1, truncated, 2^-23 each; 2^14 additions of the row sum, 2^-24 each; the
    weights themselves on fp16's subnormal grid after their shift (2^4 at least), 2^18 2^-29."""
    torch = cuda
    from msst_b200 import ops

    items = torch.cuda.get_device_properties(0).multi_processor_count  # one a CTA, whole
    # a running maximum belongs to 16 keys of every second 64 (token form) or to every second 128
    Nk, every, heads, Nq = (2 ** 21, 16, 8, 1) if form == "token" else (2 ** 19, 128, 2, 32)
    q = torch.zeros(1, Nq, 1, 8, dtype=torch.float16, device="cuda")
    q[..., 0] = 1
    k = torch.zeros(1, Nk, 1, 8, dtype=torch.float16, device="cuda")
    k[..., 0] = -25.015625
    k[:, 0:every * heads:every, :, 0] = 0
    v = torch.ones_like(k)
    wide = (items, -1, -1, -1)
    y = ops.cross_attention(q.expand(wide), k.expand(wide), v.expand(wide), scale=math.log(2))
    bound = 2 * 2.0 ** -11 + 2.0 ** 14 * 2.0 ** -23 + 2.0 ** 14 * 2.0 ** -24 + 2.0 ** 18 * 2.0 ** -29
    assert float((y.double() - 1).abs().max()) <= bound


# ------------------------------------------------------------------ cross attention: scores of -inf
@pytest.mark.parametrize("Nq", [1, 40, 300])
@pytest.mark.parametrize("prec", ["fp16", "bf16"])
def test_cross_attention_infinitely_low_first(cuda, Nq, prec):
    """Kept keys whose scores are -inf have weight zero, wherever they lie; the others' scores are
    far below zero, so a reference of zero would leave nothing of them."""
    torch = cuda
    from msst_b200 import device_error, ops

    for d, dead in ((64, 33), (64, 130), (128, 300), (40, 128)):
        q, k, v = _cross_inputs(torch, 2, Nq, 500, 4, 2, d, prec, 91 + d)
        q, k = q.abs() + 0.5, -(k.abs() + 20)
        keep = torch.ones(2, 500, dtype=torch.bool, device="cuda")
        keep[0, :dead] = False
        keep[1, 1:dead:2] = False
        low = torch.where(keep[:, :, None, None], k, torch.full_like(k, -float("inf")))
        y = ops.cross_attention(q, low, v)
        _cross_check(torch, y, q, k, v, keep, d ** -0.5, prec)
    assert device_error(True) == 0


# ------------------------------------------------------------------ graphs and threads
def _three_operators(torch, ops, seed):
    """Calls of each operator, cross attention by tiles and by tokens, as functions of one input."""
    g = _gen(torch, seed)
    cos, sin = _tables(torch, 128, 32)
    _, k, v = _cross_inputs(torch, 2, 1, 900, 4, 2, 64, "fp16", seed + 1)
    lens = torch.tensor([900, 411], dtype=torch.int32, device="cuda")
    keep = torch.rand(2, 900, generator=g, device="cuda") < 0.5
    _, w, la, lb, ids, scales, bias = _adapter_inputs(torch, 200, 256, 264, 4, 16, "fp16", seed + 2)
    calls = [
        lambda x: ops.qk_norm_rope(x, None, None, None, cos, sin)[0],
        lambda x: ops.cross_attention(x, k, v, key_lens=lens),
        lambda x: ops.cross_attention(x[:, :1], k, v, key_mask=keep),
        lambda x: ops.adapter_gemm(x.reshape(200, 256), w, la, lb, ids, scales=scales, bias=bias),
    ]
    make = lambda: torch.randn(2, 100, 4, 64, generator=g, device="cuda").half()  # noqa: E731
    return calls, make


def test_operators_in_a_graph(cuda):
    """Captured once, replayed over new inputs: the same bits as the calls themselves."""
    torch = cuda
    from msst_b200 import device_error, ops

    calls, make = _three_operators(torch, ops, 71)
    x = make()
    for call in calls:
        call(x)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = [call(x) for call in calls]
    for _ in range(3):
        x.copy_(make())
        graph.replay()
        torch.cuda.synchronize()
        for call, y in zip(calls, outs):
            assert torch.equal(call(x), y)
    assert device_error(True) == 0


def test_operators_from_two_threads(cuda):
    """Two threads on streams of their own, calls interleaved as they come: each its own results."""
    torch = cuda
    from msst_b200 import device_error, ops

    work = [_three_operators(torch, ops, seed) for seed in (81, 82)]
    inputs = [[make() for _ in range(6)] for _, make in work]
    wants = [[[call(x) for call in calls] for x in xs] for (calls, _), xs in zip(work, inputs)]
    torch.cuda.synchronize()
    wrong = []

    def body(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(20):
                    got = [[call(x) for call in work[i][0]] for x in inputs[i]]
                    torch.cuda.current_stream().synchronize()
                    for a, b in zip(got, wants[i]):
                        if not all(torch.equal(y, z) for y, z in zip(a, b)):
                            wrong.append(i)
        except Exception as e:  # a thread's exception would be lost
            wrong.append(e)

    threads = [threading.Thread(target=body, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong and device_error(True) == 0


@pytest.mark.parametrize("Nq, Nk, dims", [(1, 1, dict(dim=64, enc_dim=72, q_heads=3, kv_heads=1, head_dim=24, rank=8)),
                                          (33, 515, dict(dim=320, enc_dim=200, q_heads=4, kv_heads=4, head_dim=80, rank=40)),
                                          (200, 130, dict(dim=1024, enc_dim=512, q_heads=8, kv_heads=2, head_dim=128))])
def test_conditioned_block_sizes(cuda, Nq, Nk, dims):
    """The block against its own operators' plain forms in 64 bits at other sizes: tolerance as in
    test_conditioned_block, 4 + 4 sqrt(head_dim) roundings of the sizes in the 2-norm."""
    torch = cuda
    from msst_b200 import device_error
    from msst_b200.conditioned import random_block

    blk = random_block(dtype=torch.float16, seed=5, **dims)
    g, d, hq, hk = _gen(torch, 4), dims["head_dim"], dims["q_heads"], dims["kv_heads"]
    B = 3
    x = torch.randn(B, Nq, dims["dim"], generator=g, device="cuda").half()
    enc = torch.randn(B, Nk, dims["enc_dim"], generator=g, device="cuda").half()
    keep = torch.rand(B, Nk, generator=g, device="cuda") < 0.7
    keep[1], keep[2] = True, False
    who = torch.tensor([1, -1, 2], dtype=torch.int32, device="cuda")
    y = blk(x, *blk.encode(enc, who), who, key_mask=keep)
    assert device_error(True) == 0

    def project(name, t):
        a, b, s = blk.adapters[name]
        out = t @ blk.w[name].double().T
        for i in range(B):
            if who[i] >= 0:
                out[i] += float(s[who[i]]) * (t[i] @ a[who[i]].double().T) @ b[who[i]].double().T
        return out

    at = lambda n: torch.arange(n, device="cuda").expand(B, n)  # noqa: E731
    q64, _ = _qk_ref(torch, project("q", x.double()).view(B, Nq, hq, d), blk.q_gamma, blk.cos, blk.sin, at(Nq), 1e-6, "halves")
    kv = project("kv", enc.double()).view(B, Nk, 2, hk, d)
    k64, _ = _qk_ref(torch, kv[:, :, 0], blk.k_gamma, blk.cos, blk.sin, at(Nk), 1e-6, "halves")
    att = torch.zeros(B, Nq, hq, d, dtype=torch.float64, device="cuda")
    for i in range(2):
        for h in range(hq):
            j = h * hk // hq
            p = torch.softmax(q64[i, :, h] @ k64[i, keep[i], j].T / math.sqrt(d), -1)
            att[i, :, h] = p @ kv[i, keep[i], 1, j]
    delta = project("o", att.reshape(B, Nq, -1))
    ref = x.double() + delta
    bar = (4 + 4 * math.sqrt(d)) * U["fp16"] * float(delta.norm()) + U["fp16"] * float(ref.norm())
    assert float((y.double() - ref).norm()) <= bar
    assert torch.equal(y[2], x[2])


@pytest.mark.parametrize("case", [(2501, 264, 1032, 6, 24), (40, 4104, 136, 3, 16)], ids=lambda c: "-".join(map(str, c)))
def test_adapter_gemm_writes_its_columns_alone(cuda, case):
    """x and out as columns of wider rows: the same bits, and nothing beside them."""
    torch = cuda
    from msst_b200 import ops

    x, w, la, lb, ids, scales, bias = _adapter_inputs(torch, *case, "bf16", 3)
    y = ops.adapter_gemm(x, w, la, lb, ids, scales=scales, bias=bias)
    wide = torch.full((case[0], case[1] + 24), float("nan"), dtype=x.dtype, device="cuda")
    wide[:, 8:8 + case[1]] = x
    big = torch.full((case[0], case[2] + 16), 3.0, dtype=x.dtype, device="cuda")
    ops.adapter_gemm(wide[:, 8:8 + case[1]], w, la, lb, ids, scales=scales, bias=bias, out=big[:, 8:8 + case[2]])
    assert torch.equal(big[:, 8:8 + case[2]], y)
    assert bool((big[:, :8] == 3).all()) and bool((big[:, 8 + case[2]:] == 3).all())
