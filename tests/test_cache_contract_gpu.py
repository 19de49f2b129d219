"""GPU tests of what the header promises of the paged-cache operators beyond the Python entry points' own use
of them.  Forms and tolerances as in test_cache_ops_gpu.py."""
from __future__ import annotations

import ctypes
import struct

import pytest

from test_cache_ops_gpu import _attend_check, _attend_inputs, _dt

pytestmark = pytest.mark.gpu


def _view(t):
    """The msst_heads of a [.., heads, head_dim] tensor of three or four dimensions."""
    st = t.stride()
    return struct.pack("Pi4xqqq", t.data_ptr(), t.shape[-2], st[0] if t.dim() == 4 else 0, st[-3], st[-2])


def _workspace_bytes(T, R, P, Hq, Hk, d):
    from msst_b200 import check, lib

    n = ctypes.c_longlong()
    check(lib().msst_prefix_attention_workspace(T, R, P, Hq, Hk, d, ctypes.byref(n)))
    return n.value


def _attend_c(torch, q, pk, pv, kc, vc, table, own, starts, out, rest, ws, ws_bytes):
    """msst_prefix_attention by its C signature."""
    from msst_b200 import check, lib

    check(lib().msst_prefix_attention(
        _view(q), q.shape[0], starts.data_ptr(), own.numel(), _view(pk), _view(pv), pk.shape[0], _view(kc), _view(vc),
        kc.shape[0], kc.shape[1], table.data_ptr(), table.shape[1], table.stride(0), own.data_ptr(), q.shape[2], 0.0,
        1 if q.dtype is torch.bfloat16 else 0, _view(out), rest, ws, ws_bytes, torch.cuda.current_stream().cuda_stream))


@pytest.mark.parametrize("counts, lens", [
    ([1] * 30, [5 * i for i in range(30)]),       # tile items of the prefix, whole and cut, token items of the requests
    ([40, 3], [90, 200]),
    ([700, 300], [700, 900]),                     # prefix and own keys as one sequence
    ([2], [70]),
], ids=["single", "few", "prompts", "one"])
@pytest.mark.parametrize("d, prec", [(64, "fp16"), (128, "bf16"), (40, "bf16")])
def test_workspace_on_any_16_bytes(cuda, counts, lens, d, prec):
    """A workspace of just the size asked for at any multiple of 16 bytes, and nothing written around it."""
    torch = cuda
    from msst_b200 import device_error

    args = _attend_inputs(torch, counts, lens, 900, 8, 2, d, 16, prec, 83)
    q, pk, pv, kc, vc, table, own, starts = args
    need = _workspace_bytes(q.shape[0], len(counts), 900, 8, 2, d)
    results = []
    for off in (0, 16, 32, 48, 112, 240):
        space = torch.full((need + 512,), 0x5a, dtype=torch.uint8, device="cuda")
        out = torch.zeros_like(q)
        assert space.data_ptr() % 256 == 0
        _attend_c(torch, q, pk, pv, kc, vc, table, own, starts, out, 0, space.data_ptr() + off, need)
        assert bool((space[:off] == 0x5a).all()) and bool((space[off + need:] == 0x5a).all())
        results.append(out)
    assert device_error(True) == 0
    _attend_check(torch, results[0], *args, d ** -0.5, prec)
    assert all(torch.equal(results[0], r) for r in results[1:])


@pytest.mark.parametrize("T, Hq, d", [(1, 1, 8), (7, 4, 64), (300, 6, 40), (20000, 32, 128)])
def test_rows_without_a_request(cuda, T, Hq, d):
    """No request at all: every row of `out` is zeroed with zero_rest, and left as it was without."""
    torch = cuda
    from msst_b200 import device_error, ops

    q, pk, pv, kc, vc, table, own, starts = _attend_inputs(torch, [T], [3], 5, Hq, 1, d, 16, "fp16", 89)
    table, own, starts = table[:0], own[:0], starts[:1]
    wide = torch.full((T, Hq + 2, d + 8), float("nan"), dtype=q.dtype, device="cuda")
    out = wide[:, 1:-1, :d]
    _attend_c(torch, q, pk, pv, kc, vc, table, own, starts, out, 0, None, 0)
    assert bool(wide.isnan().all())
    assert _workspace_bytes(T, 0, 5, Hq, 1, d) == 0
    _attend_c(torch, q, pk, pv, kc, vc, table, own, starts, out, 1, None, 0)
    assert bool((out == 0).all()) and int(wide.isnan().sum()) == wide.numel() - out.numel()
    y = ops.prefix_attention(q, pk, pv, kc, vc, table, own, q_starts=starts)
    assert y.shape == q.shape and bool((y == 0).all())
    left = torch.full_like(q, 3.0)
    assert ops.prefix_attention(q, pk, pv, kc, vc, table, own, q_starts=starts, out=left) is left and bool((left == 3).all())
    assert device_error(True) == 0


@pytest.mark.parametrize("tokens", [60, 5000])  # one CTA, a cluster
def test_positions_of_a_refused_request_end_at_the_largest(cuda, tokens):
    torch = cuda
    from msst_b200 import device_error, ops

    ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    start, n = 2 ** 31 - 1 - 32, tokens - 11
    starts, slots, positions, lens, count = ops.cache_plan(ints([3, n, 2]), ints([5, 30, 0]), ints([[4, 9], [7, 2], [0, 0]]),
                                                           ints([1, 3, 5]), ints([3]), 16, tokens, start=start)
    assert device_error(True) == 16 and starts.tolist() == [0, 3, 3 + n, 5 + n]
    assert lens.tolist() == [8, 30, 2] and count.tolist() == [2]
    assert slots.tolist() == [69, 70, 71] + [-1] * n + [80, 81] + [-1] * 6
    want = [start + 5 + i for i in range(3)] + [min(start + 30 + i, 2 ** 31 - 1) for i in range(n)] + [start, start + 1] + [0] * 6
    assert positions.tolist() == want


def test_a_run_that_lasts_longer_than_a_wait_may(cuda):
    """Items of seconds (a prefix of 2^28 tokens for 37 thousand rows) with short ones behind them: nothing gives up.

    All weights are 1 (q is 0) and all values too: a bf16 row's sums are whole numbers that fp32 holds, a multiple of 128
    up to 2^28, and the requests' own tokens behind them 2^-24 of the whole."""
    torch = cuda
    from msst_b200 import device_error, ops

    R, n, P = 1900, 5, 1 << 28
    if torch.cuda.mem_get_info()[0] < 12 << 30:
        pytest.skip("12 GB of GPU memory")
    ones = torch.ones(P, 1, 8, dtype=torch.bfloat16, device="cuda")
    q = torch.zeros(R * n, 4, 8, dtype=torch.bfloat16, device="cuda")
    cache = torch.ones(R, 16, 1, 8, dtype=torch.bfloat16, device="cuda")
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    y = ops.prefix_attention(q, ones, ones, cache, cache, ints([[r] for r in range(R)]), ints([n] * R),
                             q_starts=ints([n * r for r in range(R + 1)]))
    assert device_error(True) == 0
    assert float((y.double() - 1).abs().max()) <= 2.0 ** -8


@pytest.mark.parametrize("which", ["k", "v", "kv"])
@pytest.mark.parametrize("counts, lens, prefix", [
    ([1] * 30, [3 + 5 * i for i in range(30)], 900),   # tile items of the prefix beside token items
    ([1, 1], [40, 3], 1000),                           # token items of the prefix
    ([300, 2], [310, 90], 500),                        # one sequence: tile items and token items
], ids=["beside", "tokens", "one"])
@pytest.mark.parametrize("d, prec", [(64, "fp16"), (128, "bf16")])
def test_prefix_of_shared_heads(cuda, counts, lens, prefix, which, d, prec):
    """A prefix whose heads are one expanded head, with caches that have heads of their own."""
    torch = cuda
    from msst_b200 import device_error, ops

    q, pk, pv, kc, vc, table, own, starts = _attend_inputs(torch, counts, lens, prefix, 8, 4, d, 16, prec, 107)
    pk, pv = (x[:, 1:2].expand(-1, 4, -1) if name in which else x for name, x in (("k", pk), ("v", pv)))
    y = ops.prefix_attention(q, pk, pv, kc, vc, table, own, q_starts=starts)
    assert device_error(True) == 0
    _attend_check(torch, y, q, pk, pv, kc, vc, table, own, starts, d ** -0.5, prec)


def test_prefix_of_shared_heads_is_not_copied(cuda):
    torch = cuda
    from msst_b200 import ops

    q, _, _, kc, vc, table, own, starts = _attend_inputs(torch, [1] * 20, [9] * 20, 1, 16, 8, 128, 16, "bf16", 109)
    pk, pv = (torch.zeros(100000, 1, 128, dtype=torch.bfloat16, device="cuda").expand(-1, 8, -1) for _ in range(2))
    ops.prefix_attention(q, pk, pv, kc, vc, table, own)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    ops.prefix_attention(q, pk, pv, kc, vc, table, own)
    need = _workspace_bytes(20, 20, 100000, 16, 8, 128)
    assert torch.cuda.max_memory_allocated() - before < need + (1 << 24) < pk.numel() * 2
