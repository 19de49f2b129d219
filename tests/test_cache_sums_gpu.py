"""GPU tests of attention sums over very many keys, with values of one sign, against 64 bits.

Tolerance, with u the 16-bit type's unit roundoff and e = 2^-24: as in test_cache_ops_gpu.py, but what it allows the
fp32 sums is told apart.  The product with V adds up to 2^14 keys (fp16) or 2^16 (bf16) where what is cut off is
below 2^-26 of the sum, c = 2^-12 or 2^-10; sums of these, of n keys' weights in tiles of 128 and of at most 400 partial
results are rounded to nearest: (n / 128 + n / 2^14 + 400) e."""
from __future__ import annotations

import pytest

from test_cache_ops_gpu import E, U, _dt, _gen, _own_keys, _within

pytestmark = pytest.mark.gpu

CUT = {"fp16": 2.0 ** -12, "bf16": 2.0 ** -10}


@pytest.mark.parametrize("grow", [False, True])
@pytest.mark.parametrize("prec", ["fp16", "bf16"])
@pytest.mark.parametrize("counts, lens, prefix, Hq, Hk, d", [
    ([256 * 148], [256 * 148 + 40], 2 ** 21 + 77, 1, 1, 16),    # an item a worker, one sequence
    ([400, 200], [400, 260], 1700000, 8, 2, 32),                # items that are cut
    ([60] * 12, [60 + i for i in range(12)], 700001, 8, 2, 32),  # the prefix for all requests
    ([128], [128], 140001, 148, 148, 16),                       # lone tiles
    ([30], [1700000], 5, 16, 8, 40),                            # own keys
], ids=["whole", "cut", "shared", "lone", "own"])
def test_many_keys_of_one_sign(cuda, counts, lens, prefix, Hq, Hk, d, prec, grow):
    torch = cuda
    from msst_b200 import device_error, ops

    g, dt, page, u, T = _gen(torch, 97), _dt(torch, prec), 256, U[prec], sum(counts)
    q = torch.randn(T, Hq, d, generator=g, device="cuda").to(dt)

    def keys(n):
        k = torch.randn(n, Hk, d, generator=g, device="cuda")
        if grow:  # the largest score moves on
            k *= torch.linspace(0.5, 2.5, n, device="cuda")[:, None, None]
        return k.to(dt), (1 + torch.rand(n, Hk, d, generator=g, device="cuda")).to(dt)

    pk, pv = keys(prefix)
    have = [-(-n // page) for n in lens]
    kc, vc = (x.view(-1, page, Hk, d) for x in keys(sum(have) * page))
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    order = torch.randperm(sum(have), generator=g, device="cuda").int()
    table = torch.zeros(len(lens), max(have), dtype=torch.int32, device="cuda")
    starts = [0]
    for r, n in enumerate(counts):
        table[r, :have[r]] = order[sum(have[:r]):sum(have[:r + 1])]
        starts.append(starts[-1] + n)
    y = ops.prefix_attention(q, pk, pv, kc, vc, table, ints(lens), q_starts=ints(starts))
    assert device_error(True) == 0 and bool(y.isfinite().all())
    for r in (0, len(lens) - 1):
        k = torch.cat((pk, _own_keys(torch, kc, table, r, lens[r])))
        v = torch.cat((pv, _own_keys(torch, vc, table, r, lens[r])))
        for i in sorted({0, counts[r] // 2, counts[r] - 1}):
            n = prefix + lens[r] - counts[r] + i + 1
            for h in {0, Hq // 2, Hq - 1}:
                qq, kk, vv = q[starts[r] + i, h].double(), k[:n, h * Hk // Hq].double(), v[:n, h * Hk // Hq].double()
                p = torch.softmax(kk @ qq * d ** -0.5, -1)
                ref = p @ vv  # (values above 0: the sum of magnitudes as well)
                move = 2 * d * E * float((kk.abs() @ qq.abs()).max()) * d ** -0.5 + 2.0 ** -20
                # fp16 weights below 2^-14 of 2^4 of the largest lose relative precision
                small = n * 2.0 ** -29 * float(vv.max()) * (prec == "fp16") if grow else 0.0
                bound = u * ref + (1 + u) * ref * (u + move + CUT[prec] + (n / 128 + n / 2.0 ** 14 + 400) * E) + small
                _within(y[starts[r] + i, h], ref, bound, f"request {r} row {i} head {h}")
