"""GPU tests of TokenCache and CachedBlock beyond the steps of test_cache_ops_gpu.py."""
from __future__ import annotations

import pytest

pytestmark = pytest.mark.gpu


def _ints(torch, x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _steps(torch, ahead):
    """Outputs of a few steps, each planned just before its layer or one step ahead."""
    from msst_b200 import device_error
    from msst_b200.cached import TokenCache, random_cached_block

    block = random_cached_block(dim=128, q_heads=4, kv_heads=2, head_dim=64, seed=5)
    g = torch.Generator(device="cuda")
    g.manual_seed(7)
    rows = lambda n: torch.randn(n, 128, generator=g, device="cuda").bfloat16()  # noqa: E731
    P, new = 40, [[30, 3, 17, 1], [1, 1, 1, 1], [1, 16, -1, 1], [2, 1, 0, -1], [1, 1, 1, 5]]
    _, pk, pv = block.prefill(rows(P))
    cache = TokenCache(4, 6, 2, 64, page_size=16)
    plan = lambda i: cache.plan(_ints(torch, new[i]), sum(max(n, 0) for n in new[i]), start=P)  # noqa: E731
    out, step = [], plan(0)
    for i in range(len(new)):
        later = plan(i + 1) if ahead and i + 1 < len(new) else None
        x = rows(sum(max(n, 0) for n in new[i]))
        out.append(block(x, pk, pv, cache, step, _ints(torch, [-1] * x.shape[0])))
        if i + 1 < len(new):
            step = later if ahead else plan(i + 1)
    assert cache.lens.tolist() == [35, 22, 1, 5] and device_error(True) == 0
    return out


def test_steps_planned_ahead(cuda):
    """A step's lengths are its own: the next one's plan does not show its rows keys that are not there yet."""
    for a, b in zip(_steps(cuda, False), _steps(cuda, True)):
        assert cuda.equal(a, b)


def test_steps_without_a_row(cuda):
    """A prefix of no token, and a step in which no request has a new one."""
    torch = cuda
    from msst_b200 import device_error
    from msst_b200.cached import TokenCache, random_cached_block

    block = random_cached_block(dim=128, q_heads=4, kv_heads=2, head_dim=64, seed=5)
    nothing = torch.empty(0, 128, dtype=torch.bfloat16, device="cuda")
    y, pk, pv = block.prefill(nothing)
    assert y.shape == (0, 128) and pk.shape == pv.shape == (0, 2, 64)
    cache = TokenCache(3, 2, 2, 64, page_size=16)
    x = torch.randn(6, 128, device="cuda").bfloat16()
    who = _ints(torch, [0, -1, 2] * 2)
    outs = []
    for k, v in ((pk, pv), (None, None)):
        step = cache.plan(_ints(torch, [2, 3, 1]), 6)
        outs.append(block(x, k, v, cache, step, who))
        step = cache.plan(_ints(torch, [0, 0, 0]), 0)
        assert block(nothing, k, v, cache, step, who[:0]).shape == (0, 128) and step.lens.tolist() == [2, 3, 1]
        cache.plan(_ints(torch, [-1, -1, -1]), 0)
    assert torch.equal(*outs) and device_error(True) == 0


def test_prefill_in_a_graph(cuda):
    """The prefix may be computed in a captured step: nothing in it comes from the host."""
    torch = cuda
    from msst_b200 import device_error
    from msst_b200.cached import random_cached_block

    block = random_cached_block(dim=128, q_heads=4, kv_heads=2, head_dim=64, seed=5)
    x = torch.randn(300, 128, device="cuda").bfloat16()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        block.prefill(x)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        got = block.prefill(x)
    x.copy_(torch.randn(300, 128, device="cuda").bfloat16())
    graph.replay()
    torch.cuda.synchronize()
    for a, b in zip(got, block.prefill(x)):
        assert torch.equal(a, b)
    assert device_error(True) == 0
    del graph
