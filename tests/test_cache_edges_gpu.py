"""GPU tests of the paged-cache operators at the edges of their ranges: many requests, odd numbers of
key heads, heads that share one, graphs, streams and threads, strides.  Forms and tolerances as in
test_cache_ops_gpu.py."""
from __future__ import annotations

import threading

import pytest

from test_cache_ops_gpu import U, _attend_check, _attend_inputs, _dt, _gen

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("counts, lens", [
    ([1] * 1000, [i * 37 % 60 for i in range(1000)]),                                     # more requests than threads
    ([1 + 39 * (i % 50 == 7) for i in range(700)], [40 + i * 11 % 90 for i in range(700)]),  # single tokens and prompts
    ([i % 3 for i in range(400)], [i * 7 % 50 for i in range(400)]),                       # some without a row
    ([0] * 500 + [30, 1], [5] * 500 + [30, 400]),                                          # rows of the last two alone
], ids=["single", "mixed", "ragged", "idle"])
def test_many_requests(cuda, counts, lens):
    torch = cuda
    from msst_b200 import device_error, ops

    lens = [max(a, b) for a, b in zip(counts, lens)]
    for prefix in (0, 100):
        args = _attend_inputs(torch, counts, lens, prefix, 4, 2, 64, 16, "bf16", 41)
        q, pk, pv, kc, vc, table, own, starts = args
        y = ops.prefix_attention(q, pk, pv, kc, vc, table, own, q_starts=starts)
        assert device_error(True) == 0
        _attend_check(torch, y, *args, 0.125, "bf16")


def test_most_requests(cuda):
    """8192 requests of one token, planned, appended and attended to; checked on some of them."""
    torch = cuda
    from msst_b200 import device_error, ops

    R, Hk, d, page = 8192, 2, 32, 16
    g = _gen(torch, 43)
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    lens, table = ints([0] * R), torch.zeros(R, 1, dtype=torch.int32, device="cuda")
    free, count = torch.randperm(R, generator=g, device="cuda").int(), ints([R])
    kc, vc = torch.full((2, R, page, Hk, d), float("nan"), device="cuda").half()
    tokens = []
    for i in range(3):
        q, k, v = (torch.randn(R, h, d, generator=g, device="cuda").half() for h in (4, Hk, Hk))
        tokens.append((k, v))
        starts, slots, positions, _, _ = ops.cache_plan(ints([1] * R), lens, table, free, count, page, R, out_lens=lens,
                                                        out_free_count=count)
        assert positions.tolist() == [i] * R
        ops.rope_append(q, k, v, positions, slots, None, kc, vc)
        y = ops.prefix_attention(q, None, None, kc, vc, table, lens)
        assert torch.equal(y, ops.prefix_attention(q, None, None, kc, vc, table, lens, q_starts=starts))
    assert device_error(True) == 0 and int(count) == 0 and sorted(table.flatten().tolist()) == list(range(R))
    k, v = (torch.stack(x, 1).double().repeat_interleave(2, 2) for x in zip(*tokens))  # [R, 3, 4, d]
    p = torch.softmax(torch.einsum("rhd,rnhd->rhn", q.double(), k) * d ** -0.5, -1)
    ref, A = torch.einsum("rhn,rnhd->rhd", p, v), torch.einsum("rhn,rnhd->rhd", p, v.abs())
    assert bool(((y.double() - ref).abs() <= U["fp16"] * (ref.abs() + 1.01 * A) + 2.0 ** -18 * A + 2.0 ** -22).all())


@pytest.mark.parametrize("Hq, Hk, d", [(11, 11, 64), (16, 16, 40), (27, 9, 128), (20, 5, 128), (14, 7, 72), (48, 24, 32),
                                       (34, 2, 64), (6, 6, 8)])
def test_key_heads(cuda, Hq, Hk, d):
    """Key heads of any number: items of up to eight that divide them."""
    torch = cuda
    from msst_b200 import ops

    for counts, lens, page in (([1] * 7, [3, 90, 33, 64, 1, 200, 31], 16), ([2] * 9, [2 + 40 * i for i in range(9)], 64),
                               ([1], [5000], 32)):
        for prefix in (0, 77, 1000):
            args = _attend_inputs(torch, counts, lens, prefix, Hq, Hk, d, page, "fp16", Hq + d)
            q, pk, pv, kc, vc, table, own, starts = args
            y = ops.prefix_attention(q, pk, pv, kc, vc, table, own, q_starts=starts)
            _attend_check(torch, y, *args, d ** -0.5, "fp16")


@pytest.mark.parametrize("counts", [[1] * 30, [50, 3], [2]], ids=str)
def test_heads_that_share_one(cuda, counts):
    """Caches whose heads are one expanded head (stride 0) give what that head alone gives."""
    torch = cuda
    from msst_b200 import ops

    lens = [n + 70 for n in counts]
    q, pk, pv, kc, vc, table, own, starts = _attend_inputs(torch, counts, lens, 200, 8, 1, 64, 16, "fp16", 47)
    y = ops.prefix_attention(q, pk.expand(-1, 4, -1), pv.expand(-1, 4, -1), kc.expand(-1, -1, 4, -1), vc.expand(-1, -1, 4, -1),
                             table, own, q_starts=starts)
    _attend_check(torch, y, q, pk.expand(-1, 4, -1), pv.expand(-1, 4, -1), kc.expand(-1, -1, 4, -1),
                  vc.expand(-1, -1, 4, -1), table, own, starts, 0.125, "fp16")


@pytest.mark.parametrize("prec", ["fp16", "bf16"])
@pytest.mark.parametrize("counts, lens, prefix", [
    ([40], [0], 0), ([40, 1], [0, 0], 30), ([300], [0], 0), ([1, 1], [0, 0], 0),  # no own token, no key at all
    ([1], [1], 70001), ([2], [70000], 3), ([1], [30000], 0),                       # one row's parts on every worker
    ([17, 16], [128, 256], 128), ([1, 1, 1], [32, 64, 16], 32),                    # ends on the edges of tiles and pages
    ([600, 600], [600, 600], 1),
], ids=str)
def test_lengths(cuda, counts, lens, prefix, prec):
    torch = cuda
    from msst_b200 import device_error, ops

    for Hq, Hk, d in ((2, 1, 64), (4, 2, 128)):
        args = _attend_inputs(torch, counts, lens, prefix, Hq, Hk, d, 32, prec, 53)
        q, pk, pv, kc, vc, table, own, starts = args
        y = ops.prefix_attention(q, pk, pv, kc, vc, table, own, q_starts=starts)
        assert device_error(True) == 0
        _attend_check(torch, y, *args, d ** -0.5, prec)


@pytest.mark.parametrize("prec", ["fp16", "bf16"])
@pytest.mark.parametrize("counts, lens, prefix", [
    ([4] * 20, [130 + 97 * i for i in range(20)], 127),         # lone tiles, the last keys with either half
    ([1, 9, 5, 16], [700, 2003, 129, 385], 0),
    ([600], [600], 32),
    ([250, 183, 260, 831], [250, 879, 287, 1526], 0),
], ids=["few", "ragged", "prompt", "prompts"])
def test_last_token_not_finite(cuda, counts, lens, prefix, prec):
    """The V row of a request's last token, which its last row alone sees, holds infinities and NaN."""
    torch = cuda
    from msst_b200 import ops

    for value in (float("nan"), -float("inf")):
        q, pk, pv, kc, vc, table, own, starts = _attend_inputs(torch, counts, lens, prefix, 16, 2, 64, 32, prec, 61)
        upto, keep, early = [0], [], own.clone()
        for r, (n, m) in enumerate(zip(counts, lens)):
            vc[table[r, (m - 1) // 32].long(), (m - 1) % 32] = value
            early[r] -= 1
            keep += range(int(starts[r]), int(starts[r + 1]) - 1)
            upto.append(len(keep))
        for _ in range(3):
            z = ops.prefix_attention(q, pk, pv, kc, vc, table, own, q_starts=starts)
            last = (starts[1:] - 1).long()
            assert not bool(z[last].isfinite().any())
            _attend_check(torch, z[keep], q[keep], pk, pv, kc, vc, table, early, torch.tensor(upto), 0.125, prec)


def test_lengths_outside_their_range(cuda):
    """Lengths below 0 count as 0, those past the table's row as the row's."""
    torch = cuda
    from msst_b200 import ops

    q, pk, pv, kc, vc, table, own, starts = _attend_inputs(torch, [1, 1, 1], [20, 32, 40], 50, 4, 2, 64, 16, "fp16", 59)
    table = table[:, :2].contiguous()
    odd = torch.tensor([-7, 0x7fffffff, 33], dtype=torch.int32, device="cuda")
    want = torch.tensor([0, 32, 32], dtype=torch.int32, device="cuda")
    assert torch.equal(ops.prefix_attention(q, pk, pv, kc, vc, table, odd), ops.prefix_attention(q, pk, pv, kc, vc, table, want))


def test_strides_and_alignment(cuda):
    """q and the prefix off 16 bytes (copied), rows of wider tensors, a table and an output that are views."""
    torch = cuda
    from msst_b200 import ops

    q, pk, pv, kc, vc, table, own, starts = _attend_inputs(torch, [3, 1], [60, 9], 90, 4, 2, 64, 16, "bf16", 61)
    y = ops.prefix_attention(q, pk, pv, kc, vc, table, own, q_starts=starts)

    def shifted(t):
        wide = torch.zeros(*t.shape[:-1], t.shape[-1] + 5, dtype=t.dtype, device="cuda")
        wide[..., 3:-2] = t
        return wide[..., 3:-2]

    wide = torch.zeros(table.shape[0], table.shape[1] + 3, dtype=torch.int32, device="cuda")
    wide[:, 1:1 + table.shape[1]] = table
    out = torch.zeros(4, 6, 80, dtype=q.dtype, device="cuda")
    z = ops.prefix_attention(shifted(q), shifted(pk), shifted(pv), kc, vc, wide[:, 1:1 + table.shape[1]], own, q_starts=starts,
                             out=out[:, 1:5, 8:72])
    assert torch.equal(z, y) and bool((out[:, 0] == 0).all()) and bool((out[..., :8] == 0).all()) and bool((out[..., 72:] == 0).all())
    args = (torch.randn(4, 2, 64, device="cuda").to(q.dtype), torch.arange(4, dtype=torch.int32, device="cuda"))
    a, b = kc.clone(), kc.clone()
    k1 = ops.rope_append(q, args[0], args[0], args[1], args[1], None, a, b)
    a2, b2 = kc.clone(), kc.clone()
    k2 = ops.rope_append(shifted(q), shifted(args[0]), shifted(args[0]), args[1], args[1], None, a2, b2)
    assert torch.equal(k1, k2) and torch.equal(a, a2) and torch.equal(b, b2)


def test_captured_calls_see_new_lengths(cuda):
    """A captured attention replayed after its lengths, starts and values have changed."""
    torch = cuda
    from msst_b200 import ops

    for counts in ([1] * 20, [30, 1, 9]):
        lens = [n + 100 for n in counts]
        q, pk, pv, kc, vc, table, own, starts = _attend_inputs(torch, counts, lens, 300, 8, 2, 64, 16, "fp16", 67)
        out = torch.zeros_like(q)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            ops.prefix_attention(q, pk, pv, kc, vc, table, own, q_starts=starts, out=out)
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            ops.prefix_attention(q, pk, pv, kc, vc, table, own, q_starts=starts, out=out)
        for new in (lens, [n - 60 for n in lens], counts, lens):
            own.copy_(torch.tensor(new, dtype=torch.int32))
            q.mul_(-1)
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, ops.prefix_attention(q, pk, pv, kc, vc, table, own, q_starts=starts))
        if len(counts) == 3:  # other rows of the same tensors
            starts.copy_(torch.tensor([0, 1, 31, 40], dtype=torch.int32))
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, ops.prefix_attention(q, pk, pv, kc, vc, table, own, q_starts=starts))
        del graph


def test_streams_and_threads(cuda):
    """Calls from several threads on streams of their own, at the same time."""
    torch = cuda
    from msst_b200 import device_error, ops

    cases = [([1] * 40, 500, 8, 2, 64), ([5] * 12, 200, 12, 4, 80), ([400, 3], 300, 4, 4, 128), ([1, 1], 1000, 8, 8, 128)]
    jobs = []
    for i, (counts, prefix, Hq, Hk, d) in enumerate(cases):
        args = _attend_inputs(torch, counts, [n + 60 for n in counts], prefix, Hq, Hk, d, 32, "bf16", 71 + i)
        jobs.append((args, ops.prefix_attention(*args[:7], q_starts=args[7])))
    torch.cuda.synchronize()
    wrong = []

    def work(args, want):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            for _ in range(25):
                y = ops.prefix_attention(*args[:7], q_starts=args[7])
                if not torch.equal(y, want):
                    wrong.append(1)

    threads = [threading.Thread(target=work, args=j) for j in jobs]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not wrong and device_error(True) == 0


def test_late_operands_on_a_stream(cuda):
    """Operands written on the same side stream just before the call."""
    torch = cuda
    from msst_b200 import ops

    args = _attend_inputs(torch, [2, 7], [80, 30], 200, 4, 2, 64, 16, "fp16", 79)
    want = ops.prefix_attention(*args[:7], q_starts=args[7])
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        late = [torch.zeros_like(a) for a in args]
        torch.cuda._sleep(20_000_000)
        for a, b in zip(late, args):
            a.copy_(b)
        got = ops.prefix_attention(*late[:7], q_starts=late[7])
    side.synchronize()
    assert torch.equal(got, want)
