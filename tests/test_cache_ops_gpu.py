"""GPU tests of the operators of a paged cache behind a shared prefix (msst_cache_plan,
msst_rope_append, msst_prefix_attention) against plain 64-bit forms of the same 16-bit inputs,
element by element; whole numbers have to be equal.

Tolerances, with u = 2^-11 (fp16) or 2^-8 (bf16) the unit roundoff of the 16-bit type and
e = 2^-24 that of fp32:
* rope_append: one rounding of the result, u |y|.  Inside: the turns carry three roundings to 53
  bits, 4 2^-53 |angle| radians; what is left of them one to fp32, sine and cosine and the
  amplitude two or three e each, two products and a sum, bounded by 16 e of amplitude (|a| + |b|);
  half of fp16's smallest subnormal, 2^-25.
* prefix_attention: as a cross attention's.  The result's rounding, u |y|; the weights of P V are
  rounded to 16 bits, u A with A = softmax(s) |v|; the scores carry d fp32 roundings, which move a
  weight by 2 d e max_j sum|q k_j| scale (numerator and sum), and an exponential good to 2^-21,
  each on A; the fp32 sum of P V over n keys and at most 400 partial results, 2 (n + 400) e A; fp16
  weights below 2^-14 of the largest lose relative precision: n 2^-25 max|v|.
"""
from __future__ import annotations

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


# ------------------------------------------------------------------ block tables and slots
def _plan_ref(new, lens, table, free, count, page, tokens, start):
    """Request by request, with a list as the stack."""
    blocks = len(table[0]) if table else 0
    lens, table, free = list(lens), [list(t) for t in table], list(free)
    stack, refused = free[:count], False
    for r, n in enumerate(new):
        if n < 0:
            stack += table[r][:-(-lens[r] // page)]
            lens[r] = 0
    free[:len(stack)] = stack
    starts, slots, positions, short, row, upto = [0], [-1] * tokens, [0] * tokens, False, 0, len(stack)
    for r, n in enumerate(new):
        n = max(n, 0)
        have, want = -(-lens[r] // page), -(-(lens[r] + n) // page)
        good = want <= blocks and row + n <= tokens
        if good and want > have:
            short = short or want - have > upto
            good = not short
            if good:
                for b in range(have, want):
                    upto -= 1
                    table[r][b] = stack.pop()
        refused |= not good
        for i in range(n):
            if row + i < tokens:
                p = lens[r] + i
                positions[row + i] = start + p
                slots[row + i] = table[r][p // page] * page + p % page if good else -1
        row += n
        starts.append(min(row, tokens))
        lens[r] += n if good else 0
    return starts, slots, positions, lens, [len(stack)], table, free, refused


def _plan_state(torch, R, blocks, page, most, spare, seed):
    """Lengths up to `most`, a table of distinct pages in any order, `spare` free pages."""
    import random
    rng = random.Random(seed)
    lens = [rng.randint(0, most) for _ in range(R)]
    have = [-(-n // page) for n in lens]
    pages = list(range(sum(have) + spare))
    rng.shuffle(pages)
    table, taken = [], 0
    for n in have:
        table.append(pages[taken:taken + n] + [-7] * (blocks - n))
        taken += n
    return lens, table, pages[taken:] + [-9] * taken, spare


PLAN_CASES = [
    # requests, blocks, page, most tokens there, spare pages, new tokens, rows behind the last
    (1, 1, 16, 0, 1, lambda r: 1, 0),
    (1, 4, 16, 30, 3, lambda r: -1, 3),
    (64, 8, 64, 300, 64, lambda r: 1, 0),
    (64, 8, 64, 300, 64, lambda r: 1 - 2 * (r % 3 == 1), 5),       # a third has ended
    (37, 40, 16, 200, 2000, lambda r: 17 * r % 230, 11),           # prompts, some of no token
    (37, 40, 16, 200, 3, lambda r: (17 * r % 230) - 40 * (r % 4 == 0), 0),  # not enough pages
    (9, 3, 32, 90, 100, lambda r: 5 * r, 0),                       # rows of the table that end
    (1000, 12, 16, 100, 4000, lambda r: -1 if r % 9 == 8 else 1 + r % 3, 1),
    (8192, 2, 256, 200, 8192, lambda r: 1, 0),                     # the most requests
    (5, 700, 16, 100, 3000, lambda r: 2000 + r, 0),                # more rows than one CTA is given
    (48, 64, 128, 512, 3000, lambda r: 1001 - r, 100),
]


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("case", range(len(PLAN_CASES)))
def test_cache_plan(cuda, case, in_place):
    torch = cuda
    from msst_b200 import device_error, ops

    R, blocks, page, most, spare, rule, behind = PLAN_CASES[case]
    lens, table, free, count = _plan_state(torch, R, blocks, page, most, spare, case)
    new = [rule(r) for r in range(R)]
    tokens = sum(max(n, 0) for n in new) + behind
    want = _plan_ref(new, lens, table, free, count, page, tokens, 5000)
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    new_t, lens_t, table_t, free_t, count_t = ints(new), ints(lens), ints(table), ints(free), ints([count])
    out = dict(out_lens=lens_t, out_free_count=count_t) if in_place else {}
    for again in range(1 if in_place else 2):  # with outputs of their own a call may be repeated
        got = ops.cache_plan(new_t, lens_t, table_t, free_t, count_t, page, tokens, start=5000, **out)
        for name, g, w in zip(("q_starts", "slots", "positions", "lens", "count"), got, want):
            assert g.tolist() == w, name
        assert table_t.tolist() == want[5] and free_t.tolist() == want[6]
        assert device_error(True) == (16 if want[7] else 0)
    if not in_place:
        assert lens_t.tolist() == lens and count_t.tolist() == [count]


def test_cache_plan_few_rows_and_odd_values(cuda):
    """Fewer rows than new tokens, a table that is a view, lengths and a count outside their ranges."""
    torch = cuda
    from msst_b200 import device_error, ops

    ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    wide = torch.full((3, 9), 77, dtype=torch.int32, device="cuda")
    table = wide[:, 2:6]
    free = torch.arange(10, dtype=torch.int32, device="cuda")
    starts, slots, positions, lens, count = ops.cache_plan(ints([3, 4, 2]), ints([0, 0, 0]), table, free, ints([10]), 16, 8)
    assert starts.tolist() == [0, 3, 7, 8] and lens.tolist() == [3, 4, 0] and count.tolist() == [8]
    assert slots.tolist() == [144, 145, 146, 128, 129, 130, 131, -1] and positions.tolist() == [0, 1, 2, 0, 1, 2, 3, 0]
    assert device_error(True) == 16
    assert wide[:, :2].eq(77).all() and wide[:, 6:].eq(77).all() and wide[0, 2] == 9 and wide[1, 2] == 8
    # -5 counts as 0, 1000 as the row's 64, a count of 99 as the stack's 10
    got = ops.cache_plan(ints([1, 1, -3]), ints([-5, 1000, 16]), table, free, ints([99]), 16, 2)
    assert got[3].tolist() == [1, 64, 0] and got[1].tolist()[1] == -1 and device_error(True) == 16
    # no request and no row
    got = ops.cache_plan(ints([]), ints([]), table[:0], free, ints([4]), 16, 3)
    assert got[0].tolist() == [0] and got[1].tolist() == [-1] * 3 and got[4].tolist() == [4] and device_error(True) == 0


def test_cache_plan_over_many_steps(cuda):
    """A cache's life: no page is ever held twice or lost, and every token keeps its slot."""
    import random
    torch = cuda
    from msst_b200 import device_error, ops

    R, blocks, page, pages = 20, 6, 16, 90
    rng = random.Random(3)
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    lens, table = ints([0] * R), torch.full((R, blocks), -1, dtype=torch.int32, device="cuda")
    free, count = torch.arange(pages, dtype=torch.int32, device="cuda"), ints([pages])
    where = [[] for _ in range(R)]
    for step in range(120):
        new = [rng.choice([-1, 0, 1, 1, 1, 7, 40]) if rng.random() < 0.8 else 1 for _ in range(R)]
        tokens = sum(max(n, 0) for n in new)
        before = lens.tolist()
        starts, slots, positions, _, _ = ops.cache_plan(ints(new), lens, table, free, count, page, tokens, out_lens=lens,
                                                        out_free_count=count)
        starts, slots, after, held = starts.tolist(), slots.tolist(), lens.tolist(), table.tolist()
        for r in range(R):
            if new[r] < 0:
                where[r] = []
            elif after[r] != before[r]:
                where[r] += slots[starts[r]:starts[r + 1]]
            else:
                assert all(s == -1 for s in slots[starts[r]:starts[r + 1]])
            assert len(where[r]) == after[r]
            assert [held[r][i // page] * page + i % page for i in range(after[r])] == where[r]
        used = [p for r in range(R) for p in held[r][:-(-after[r] // page)]]
        assert sorted(used + free.tolist()[:int(count)]) == list(range(pages))
        device_error(True)


# ------------------------------------------------------------------ rotation and append
def _rotate_ref(torch, x, positions, freq, amplitude, pairing):
    """(y, bound on the arithmetic inside) of one tensor [T, H, d] in 64 bits."""
    y, half = x.double(), 0 if freq is None else freq.numel()
    slack = torch.zeros_like(y)
    if half:
        angle = (positions.double()[:, None] * freq)[:, None]
        i = torch.arange(half, device="cuda")
        first, second = (2 * i, 2 * i + 1) if pairing == "interleaved" else (i, i + half)
        a, b = y[..., first], y[..., second]
        bound = (16 * E + 4 * 2.0 ** -53 * angle.abs()) * abs(amplitude) * (a.abs() + b.abs())
        slack[..., first] = slack[..., second] = bound
        y[..., first] = amplitude * (a * angle.cos() - b * angle.sin())
        y[..., second] = amplitude * (b * angle.cos() + a * angle.sin())
    return y, slack


APPEND_CASES = [
    # T, Hq, Hk, d, rot, page, farthest position, layout
    (1, 1, 1, 64, 64, 16, 1, "plain"),
    (64, 32, 8, 128, 128, 64, 1 << 20, "packed"),
    (33, 8, 8, 48, 32, 16, 1 << 17, "packed"),
    (7, 3, 1, 8, 8, 32, 100, "heads first"),
    (200, 5, 5, 80, 80, 128, 1 << 31, "plain"),
    (19, 6, 2, 256, 128, 256, 5000, "packed"),
    (50, 4, 4, 256, 256, 16, 1 << 24, "heads first"),
    (21, 2, 1, 16, 0, 16, 1, "plain"),
    (40, 9, 3, 96, 24, 16, 9000, "odd"),
    (3000, 12, 4, 32, 16, 64, 1 << 20, "plain"),
]


@pytest.mark.parametrize("prec", ["fp16", "bf16"])
@pytest.mark.parametrize("pairing", ["interleaved", "halves"])
@pytest.mark.parametrize("case", APPEND_CASES, ids=lambda c: "-".join(map(str, c)))
def test_rope_append(cuda, case, pairing, prec):
    torch = cuda
    from msst_b200 import device_error, ops, rope_frequencies

    T, Hq, Hk, d, rot, page, far, layout = case
    g, dt = _gen(torch, T + d), _dt(torch, prec)

    def make(heads):
        if layout == "heads first":
            return torch.randn(heads, T, d, generator=g, device="cuda").to(dt).transpose(0, 1)
        if layout == "odd":
            return torch.randn(T, heads * d + 3, generator=g, device="cuda").to(dt)[:, 1:1 + heads * d].unflatten(-1, (heads, d))
        return torch.randn(T, heads, d, generator=g, device="cuda").to(dt)

    if layout == "packed":
        rows = torch.randn(T, Hq + 2 * Hk, d, generator=g, device="cuda").to(dt)
        q, k, v = rows[:, :Hq], rows[:, Hq:Hq + Hk], rows[:, Hq + Hk:]
    else:
        q, k, v = make(Hq), make(Hk), make(Hk)
    pages = T // page + 3
    both = torch.randn(pages, 2, page, Hk, d, generator=g, device="cuda").to(dt)  # keys and values page by page
    k_cache, v_cache = both[:, 0], both[:, 1]
    slots = torch.randperm(pages * page, generator=g, device="cuda")[:T].int()
    slots[T // 2] = -1 - T % 2 * 100
    positions = torch.randint(-far if far > 1000 else 0, far, (T,), generator=g, device="cuda", dtype=torch.int64).int()
    freq, amplitude = rope_frequencies(rot, 10000.0, device="cuda") if rot else (None, 1.0)
    amplitude *= 1.25
    want_k, want_v, before = k_cache.double(), v_cache.double(), both.clone()
    kr, k_slack = _rotate_ref(torch, k, positions, freq, amplitude, pairing)
    qr, q_slack = _rotate_ref(torch, q, positions, freq, amplitude, pairing)
    y = ops.rope_append(q, k, v, positions, slots, freq, k_cache, v_cache, amplitude=amplitude, pairing=pairing)
    assert device_error(True) == 0
    _within(y, qr, U[prec] * qr.abs() + (1 + U[prec]) * q_slack + TINY[prec], "q")
    there = slots >= 0
    at = slots[there].long()
    got_k, got_v = k_cache[at // page, at % page], v_cache[at // page, at % page]
    _within(got_k, kr[there], U[prec] * kr[there].abs() + (1 + U[prec]) * k_slack[there] + TINY[prec], "k")
    assert torch.equal(got_v, v[there])
    before[at // page, 0, at % page], before[at // page, 1, at % page] = got_k, got_v
    assert torch.equal(both, before)  # nothing else was written
    del want_k, want_v
    if layout != "odd":  # in place
        z = ops.rope_append(q, k, v, positions, slots, freq, k_cache, v_cache, amplitude=amplitude, pairing=pairing, out_q=q)
        assert z is q and torch.equal(z, y)


def test_rope_append_slots_outside(cuda):
    torch = cuda
    from msst_b200 import device_error, ops

    x = torch.randn(3, 2, 64, device="cuda").half()
    cache = torch.zeros(2, 2, 16, 2, 64, device="cuda", dtype=torch.float16)
    slots = torch.tensor([32, 31, 0x7fffffff], dtype=torch.int32, device="cuda")
    ops.rope_append(x, x, x, slots, slots, None, cache[0], cache[1])
    assert device_error(True) == 17 and device_error(True) == 0
    want = torch.zeros_like(cache)
    want[:, 1, 15] = x[1]
    assert torch.equal(cache, want)


def test_rope_append_keeps_values_that_nothing_turns(cuda):
    """Infinities and NaN outside the rotated columns and in v stay where they are."""
    torch = cuda
    from msst_b200 import ops, rope_frequencies

    x = torch.randn(4, 2, 64, device="cuda").half()
    x[..., 40], x[..., 41], x[..., 63] = float("inf"), float("nan"), -float("inf")
    freq, _ = rope_frequencies(32, device="cuda")
    cache = torch.zeros(2, 1, 16, 2, 64, device="cuda", dtype=torch.float16)
    at = torch.arange(4, device="cuda", dtype=torch.int32)
    for pairing in ("interleaved", "halves"):
        y = ops.rope_append(x, x, x, at, at, freq, cache[0], cache[1], pairing=pairing)
        assert torch.equal(y[..., 32:].nan_to_num(7.0), x[..., 32:].nan_to_num(7.0)) and bool(y[..., :32].isfinite().all())
        assert torch.equal(cache[1, 0, :4].nan_to_num(7.0), x.nan_to_num(7.0))


# ------------------------------------------------------------------ attention
def _attend_inputs(torch, counts, lens, prefix, Hq, Hk, d, page, prec, seed, layout="plain"):
    g, dt = _gen(torch, seed), _dt(torch, prec)

    def r(*s):
        return torch.randn(*s, generator=g, device="cuda").to(dt)

    T, R = sum(counts), len(counts)
    if layout == "strided":
        q = r(Hq, T, d).transpose(0, 1)
        pre = r(prefix, 2, Hk, d)
        pk, pv = pre[:, 0], pre[:, 1]
    else:
        q, pk, pv = r(T, Hq, d), r(prefix, Hk, d), r(prefix, Hk, d)
    have = [-(-n // page) for n in lens]
    pages, blocks = sum(have) + 3, max(have + [1]) + 1
    both = r(pages, 2, page, Hk, d) if layout == "strided" else r(2, pages, page, Hk, d)
    kc, vc = (both[:, 0], both[:, 1]) if layout == "strided" else (both[0], both[1])
    order = torch.randperm(pages, generator=g, device="cuda").int()
    table = torch.full((R, blocks), 1 << 30, dtype=torch.int32, device="cuda")  # never looked up past a request's pages
    taken = 0
    for i, n in enumerate(have):
        table[i, :n] = order[taken:taken + n]
        taken += n
    starts = [0]
    for n in counts:
        starts.append(starts[-1] + n)
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    return q, pk, pv, kc, vc, table, ints(lens), ints(starts)


def _own_keys(torch, cache, table, r, length):
    page = cache.shape[1]
    j = torch.arange(length, device="cuda")
    return cache[table[r].long()[j // page], j % page]


def _attend_check(torch, y, q, pk, pv, kc, vc, table, lens, starts, scale, prec):
    u, Hk, Hq, d = U[prec], kc.shape[2], q.shape[1], q.shape[2]
    lens, starts = lens.tolist(), starts.tolist()
    P = 0 if pk is None else pk.shape[0]
    for r, length in enumerate(lens):
        a, b = starts[r], starts[r + 1]
        if a == b:
            continue
        k, v = _own_keys(torch, kc, table, r, length), _own_keys(torch, vc, table, r, length)
        if P:
            k, v = torch.cat((pk, k)), torch.cat((pv, v))
        limit = P + (length - (b - a) + 1 + torch.arange(b - a, device="cuda")).clamp(0, length)
        late = torch.arange(P + length, device="cuda") >= limit[:, None]
        for h in range(Hq):
            qq, kk, vv = q[a:b, h].double(), k[:, h * Hk // Hq].double(), v[:, h * Hk // Hq].double()
            s = (qq @ kk.T * scale).masked_fill(late, -torch.inf)
            p = torch.softmax(s, -1).nan_to_num(0.0) if P + length else s  # rows without a key: zeros
            ref, A = p @ vv, p @ vv.abs()
            n = limit[:, None]
            reach = (qq.abs() @ kk.abs().T).amax(-1, keepdim=True) if P + length else 0.0
            move = 2 * d * E * reach * abs(scale) + 2.0 ** -20
            top = vv.abs().amax(0) if P + length else 0.0
            bound = u * ref.abs() + (1 + u) * A * (u + move + 2 * (n + 400) * E) + n * TINY[prec] * top + 1e-30
            _within(y[a:b, h], ref, bound + TINY[prec], f"request {r} head {h}")


ATTEND_CASES = [
    # new tokens, own tokens, prefix, Hq, Hk, d, page, layout
    ([1], [1], 0, 1, 1, 64, 16, "plain"),
    ([1], [1], 1, 1, 1, 8, 16, "plain"),
    ([1], [0], 0, 2, 1, 64, 16, "plain"),                       # no key at all: zeros
    ([1, 1], [0, 40], 0, 4, 2, 128, 16, "plain"),
    ([1] * 5, [1, 17, 0, 64, 65], 100, 8, 2, 128, 64, "strided"),
    ([1] * 3, [300, 5, 1000], 1895, 8, 8, 64, 16, "plain"),
    ([1] * 40, [i * 13 % 200 for i in range(40)], 777, 8, 2, 128, 32, "plain"),
    ([1] * 64, [i * 7 % 90 for i in range(64)], 2049, 6, 2, 80, 16, "strided"),
    ([1] * 9, [50] * 9, 0, 32, 1, 64, 128, "plain"),            # 32 rows a key head, no prefix
    ([1] * 2, [50, 700], 5001, 130, 1, 32, 256, "plain"),       # more heads a key head than a tile has rows
    ([3, 0, 1, 7, 2], [3, 9, 500, 30, 130], 333, 4, 2, 64, 16, "plain"),
    ([5] * 12, [5 + 31 * i for i in range(12)], 1000, 12, 4, 80, 32, "strided"),
    ([8] * 20, [8 + 40 * i for i in range(20)], 801, 8, 8, 64, 16, "plain"),
    ([200, 1, 1, 33, 1], [200, 300, 1, 64, 129], 500, 8, 2, 128, 64, "plain"),   # prompts among single tokens
    ([300], [300], 0, 7, 1, 128, 128, "plain"),
    ([129, 500], [1000, 500], 257, 4, 4, 64, 16, "strided"),
    ([700, 64, 257], [701, 64, 900], 130, 6, 2, 96, 32, "plain"),
    ([40, 3], [10, 2], 20, 2, 1, 48, 16, "plain"),              # fewer own tokens than new ones: the first rows see none
    ([1000], [1200], 1500, 8, 1, 40, 256, "plain"),
    ([900, 1, 1300, 3], [900, 70, 1500, 40], 600, 8, 4, 64, 32, "plain"),       # many rows, most of them of one worker
    ([2, 1, 1], [3000, 5000, 10], 0, 3, 3, 48, 16, "strided"),
]


@pytest.mark.parametrize("prec", ["fp16", "bf16"])
@pytest.mark.parametrize("case", range(len(ATTEND_CASES)))
def test_prefix_attention(cuda, case, prec):
    torch = cuda
    from msst_b200 import device_error, ops

    counts, lens, prefix, Hq, Hk, d, page, layout = ATTEND_CASES[case]
    args = _attend_inputs(torch, counts, lens, prefix, Hq, Hk, d, page, prec, case, layout)
    q, pk, pv, kc, vc, table, own, starts = args
    single = all(n == 1 for n in counts)
    call = lambda qs: ops.prefix_attention(q, pk, pv, kc, vc, table, own, q_starts=qs)  # noqa: E731
    y = call(None if single else starts)
    assert device_error(True) == 0
    _attend_check(torch, y, *args, d ** -0.5, prec)
    assert torch.equal(y, call(None if single else starts))
    if single:
        assert torch.equal(y, call(starts))
    if prefix == 0:
        assert torch.equal(y, ops.prefix_attention(q, None, None, kc, vc, table, own, q_starts=starts))
    # what no row sees may hold anything: the rest of the last pages, pages of nobody
    seen = torch.zeros(kc.shape[:2], dtype=torch.bool, device="cuda")
    for r, n in enumerate(lens):
        j = torch.arange(n, device="cuda")
        seen[table[r].long()[j // page], j % page] = True
    for value in (float("nan"), float("inf"), torch.finfo(q.dtype).min):
        kc[~seen], vc[~seen] = value, value
        assert torch.equal(y, call(None if single else starts))
    assert device_error(True) == 0


@pytest.mark.parametrize("prec", ["fp16", "bf16"])
@pytest.mark.parametrize("counts", [[4] * 6, [40, 9], [300, 5], [4200, 9]], ids=str)
def test_prefix_attention_values_of_later_tokens(cuda, counts, prec):
    """What a new token holds, infinities and NaN included, does not reach the rows before it."""
    torch = cuda
    from msst_b200 import ops

    lens = [n + 11 * i for i, n in enumerate(counts)]
    q, pk, pv, kc, vc, table, own, starts = _attend_inputs(torch, counts, lens, 150, 4, 2, 64, 16, prec, 5)
    at = starts.tolist()
    for r, n in enumerate(counts):
        j = lens[r] - n // 2  # a new token in the middle
        kc[table[r, j // 16].long(), j % 16] = float("nan")
        vc[table[r, j // 16].long(), j % 16, 0, 3] = float("inf")
        vc[table[r, j // 16].long(), j % 16, 1] = float("nan")
    z = ops.prefix_attention(q, pk, pv, kc, vc, table, own, q_starts=starts)
    before, upto, early = [], [0], own.clone()
    for r, n in enumerate(counts):
        first = at[r + 1] - n // 2
        assert bool(z[first:at[r + 1]].isnan().all())
        before += range(at[r], first)
        upto.append(len(before))
        early[r] -= n // 2
    # the rows before are those of a shorter call
    _attend_check(torch, z[before], q[before], pk, pv, kc, vc, table, early, torch.tensor(upto), 0.125, prec)


@pytest.mark.parametrize("prec", ["fp16", "bf16"])
def test_prefix_attention_large_scores(cuda, prec):
    """Scores of hundreds that grow along the keys, and fall with a negative scale."""
    torch = cuda
    from msst_b200 import ops

    for counts, lens in (([1] * 20, [30 * i for i in range(20)]), ([90, 200], [400, 200])):
        args = _attend_inputs(torch, counts, lens, 900, 8, 2, 64, 32, prec, 9)
        q, pk, pv, kc, vc, table, own, starts = args
        q.copy_(q.abs() * 3)
        pk.copy_((pk.abs() * torch.linspace(0.1, 3, 900, device="cuda")[:, None, None]).to(pk.dtype))
        kc.copy_(kc.abs() * 4)
        for scale in (0.0, -0.25):
            y = ops.prefix_attention(q, pk, pv, kc, vc, table, own, q_starts=starts, scale=scale)
            _attend_check(torch, y, *args, scale or 0.125, prec)


def test_prefix_attention_rows_of_nobody(cuda):
    """Rows behind the last request (and before the first) stay as they were; zeros without `out`."""
    torch = cuda
    from msst_b200 import ops

    for counts, Hq in (([1] * 30, 8), ([50, 90], 4), ([3, 2], 2), ([2500, 1700], 4)):
        lens = [n + 20 for n in counts]
        q, pk, pv, kc, vc, table, own, starts = _attend_inputs(torch, counts, lens, 200, Hq, 2, 64, 16, "fp16", 13)
        y = ops.prefix_attention(q, pk, pv, kc, vc, table, own, q_starts=starts)
        padded = torch.nn.functional.pad(q, (0, 0, 0, 0, 2, 37), value=float("nan"))
        wide = torch.full((padded.shape[0], Hq, 72), 5.0, dtype=q.dtype, device="cuda")
        out = wide[..., :64]
        ops.prefix_attention(padded, pk, pv, kc, vc, table, own, q_starts=starts + 2, out=out)
        assert bool((wide[:2] == 5).all()) and bool((wide[-37:] == 5).all()) and bool((wide[..., 64:] == 5).all())
        near = (out[2:-37].double() - y.double()).abs().max()  # other sums, the same precision
        assert float(near) <= 4 * U["fp16"] * float(y.abs().max())
        z = ops.prefix_attention(padded, pk, pv, kc, vc, table, own, q_starts=starts + 2)
        assert bool((z[:2] == 0).all()) and bool((z[-37:] == 0).all()) and torch.equal(z[2:-37], out[2:-37])


def test_prefix_attention_pages_outside(cuda):
    """A page outside the cache reads as zeros, and the other requests do not mind."""
    torch = cuda
    from msst_b200 import device_error, ops

    for counts in ([1, 1, 1], [20, 70, 1]):
        q, pk, pv, kc, vc, table, own, starts = _attend_inputs(torch, counts, [100, 100, 100], 50, 4, 2, 64, 16, "fp16", 17)
        for bad in (-1, kc.shape[0], 0x7fffffff):
            broken = table.clone()
            broken[1, 6] = bad  # its last four tokens
            y = ops.prefix_attention(q, pk, pv, kc, vc, broken, own, q_starts=starts)
            assert device_error(True) == 18 and device_error(True) == 0 and bool(y.isfinite().all())
        good = ops.prefix_attention(q, pk, pv, kc, vc, table, own, q_starts=starts)
        a, b = starts.tolist()[0:2]
        assert torch.equal(y[a:b], good[a:b])


def test_far_slots_of_a_large_cache(cuda):
    """Element offsets past 2^31 and byte offsets past 2^32 in a cache of 9 GB."""
    torch = cuda
    from msst_b200 import device_error, ops, rope_frequencies

    pages, page, Hk, d = 17000, 256, 8, 64
    both = torch.empty(2, pages, page, Hk, d, dtype=torch.bfloat16, device="cuda")
    kc, vc = both[0], both[1]
    lens, R = [300, 90], 2
    g = _gen(torch, 23)
    table = torch.tensor([[pages - 1, pages - 2], [16500, 3]], dtype=torch.int32, device="cuda")
    T = sum(lens)
    k, v, q = (torch.randn(T, h, d, generator=g, device="cuda").bfloat16() for h in (Hk, Hk, 16))
    at = torch.cat([torch.arange(n, device="cuda") for n in lens])
    r = torch.arange(R, device="cuda").repeat_interleave(torch.tensor(lens, device="cuda"))
    slots = (table[r, at // page] * page + at % page).int()
    freq, _ = rope_frequencies(d, device="cuda")
    positions = at.int()
    q2 = ops.rope_append(q, k, v, positions, slots, freq, kc, vc)
    own = torch.tensor(lens, dtype=torch.int32, device="cuda")
    starts = torch.tensor([0, 300, 390], dtype=torch.int32, device="cuda")
    pk = torch.randn(20, Hk, d, generator=g, device="cuda").bfloat16()
    args = (q2, pk, pk, kc, vc, table, own, starts)
    y = ops.prefix_attention(*args[:7], q_starts=starts)
    last = (starts[1:] - 1).long()
    z = ops.prefix_attention(q2[last], *args[1:7])
    assert device_error(True) == 0
    ref, _ = _rotate_ref(torch, k, positions, freq, 1.0, "interleaved")
    got = torch.cat([_own_keys(torch, kc, table, i, n) for i, n in enumerate(lens)])
    assert float((got.double() - ref).abs().max()) <= 2.0 ** -7 * 4 and torch.equal(
        torch.cat([_own_keys(torch, vc, table, i, n) for i, n in enumerate(lens)]), v)
    _attend_check(torch, y, *args, d ** -0.5, "bf16")
    _attend_check(torch, z, q2[last], *args[1:7], torch.arange(3), d ** -0.5, "bf16")


# ------------------------------------------------------------------ together
def _plain_block(torch, block, x, adapter):
    """64-bit form of a CachedBlock on one request's whole sequence [N, dim] (adapter None: none), with the
    16-bit roundings of what it stores: heads, rotated heads, attention, result."""
    dt, d, Hq, Hk = x.dtype, block.head_dim, block.q_heads, block.kv_heads

    def project(name, y):
        z = y.double() @ block.w[name].double().T
        if adapter is not None:
            for rows, a in adapter:
                if a >= 0:
                    la, lb, sc = block.adapters[name]
                    z[rows] += float(sc[a]) * (y[rows].double() @ la[a].double().T @ lb[a].double().T)
        return z.to(dt)

    qkv = project("qkv", x).view(x.shape[0], -1, d)
    at = torch.arange(x.shape[0], device="cuda")
    rot = [_rotate_ref(torch, y, at, block.inv_freq, block.amplitude, block.pairing)[0].to(dt).double()
           for y in (qkv[:, :Hq], qkv[:, Hq:Hq + Hk])]
    v = qkv[:, Hq + Hk:].double()
    o = torch.empty(x.shape[0], Hq, d, dtype=torch.float64, device="cuda")
    late = at > at[:, None]
    for h in range(Hq):
        s = (rot[0][:, h] @ rot[1][:, h * Hk // Hq].T * d ** -0.5).masked_fill(late, -torch.inf)
        o[:, h] = torch.softmax(s, -1) @ v[:, h * Hk // Hq]
    return x.double() + project("o", o.to(dt).view(x.shape[0], -1)).double()


@pytest.mark.parametrize("graph", [False, True])
@pytest.mark.parametrize("prec", ["fp16", "bf16"])
def test_blocks_over_many_steps(cuda, prec, graph):
    """A prefix, ragged prompts, single tokens (in a captured graph or not) and draft tokens through
    plan, append, attention and projections, against each request's whole sequence at once.

    The two sides round the same stored values to 16 bits and differ by fp32 sums before that, so a
    value is off by a rounding here and there: heads, weights, attention and result, four of at most one
    step of their size (2 u), which the next product averages; 8 u of the largest value covers them."""
    torch = cuda
    from msst_b200 import device_error
    from msst_b200.cached import TokenCache, random_cached_block

    block = random_cached_block(dim=256, q_heads=8, kv_heads=2, head_dim=64, dtype=_dt(torch, prec), seed=3,
                                scaling="parts", factor=4.0, original=64)
    P, prompts, singles, drafts = 150, [40, 1, 9, 17], 9, 3
    R = len(prompts)
    g = _gen(torch, 31)
    rows = lambda n: torch.randn(n, 256, generator=g, device="cuda").to(_dt(torch, prec))  # noqa: E731
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    prefix, own = rows(P), [rows(n + singles + drafts) for n in prompts]
    adapters = [0, -1, 2, 1]
    y0, pk, pv = block.prefill(prefix)
    u = U[prec]
    want = _plain_block(torch, block, prefix, None)
    _within(y0, want, 8 * u * want.abs().max() + 0 * want, "prefix")
    cache = TokenCache(R, 5, 2, 64, page_size=16, dtype=_dt(torch, prec))
    got = [[] for _ in range(R)]

    def feed(new, single=False):
        """The next new[r] rows of each request through the block."""
        x = torch.cat([own[r][sum(map(len, got[r])):][:n] for r, n in enumerate(new)])
        step = cache.plan(ints(new), sum(new), start=P)
        who = ints(adapters).repeat_interleave(ints(new))
        y = block(x, pk, pv, cache, step, who, single=single)
        for r, n in enumerate(new):
            got[r].append(y[sum(new[:r]):sum(new[:r + 1])])

    feed(prompts)
    if graph:
        x, one, who = torch.empty(R, 256, dtype=_dt(torch, prec), device="cuda"), ints([1] * R), ints(adapters)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        saved = [t.clone() for t in (cache.lens, cache.block_table, cache.free_pages, cache.free_count)]
        with torch.cuda.stream(side):
            block(x, pk, pv, cache, cache.plan(one, R, start=P), who, single=True)  # (warm up)
        side.synchronize()
        for t, old in zip((cache.lens, cache.block_table, cache.free_pages, cache.free_count), saved):
            t.copy_(old)
        torch.cuda.synchronize()
        captured = torch.cuda.CUDAGraph()
        with torch.cuda.graph(captured, stream=side):
            y = block(x, pk, pv, cache, cache.plan(one, R, start=P), who, single=True)
        for i in range(singles):
            x.copy_(torch.stack([own[r][prompts[r] + i] for r in range(R)]))
            captured.replay()
            for r in range(R):
                got[r].append(y[r:r + 1].clone())
    else:
        for _ in range(singles):
            feed([1] * R, single=True)
    feed([drafts] * R)
    assert device_error(True) == 0 and cache.lens.tolist() == [n + singles + drafts for n in prompts]
    for r in range(R):
        whole = torch.cat((prefix, own[r]))
        want = _plain_block(torch, block, whole, [(slice(P, None), adapters[r])])[P:]
        y = torch.cat(got[r])
        _within(y, want, 8 * u * want.abs().max() + 0 * want, f"request {r}")
    cache.plan(ints([-1] * R), 0)
    assert int(cache.free_count) == cache.free_pages.numel() and cache.lens.tolist() == [0] * R


def test_example_runs(cuda, capsys):
    from msst_b200 import conditioned, device_error

    conditioned.main()
    assert "8 of 8 pages free" in capsys.readouterr().out and device_error(True) == 0
