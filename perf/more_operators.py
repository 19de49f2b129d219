"""Cases, plain forms and 64-bit forms of the framework's operators for a cache of generated tokens
behind one shared prefix: block tables and slots from request lengths, rotated keys written to the
cache's pages, and attention to the shared prefix and each request's own tokens."""
from __future__ import annotations

import math
import os
import sys

import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


# ------------------------------------------------------------------------------------- cases
def listed():
    return [
        # the next token of each of 64 requests: launch latency is all there is
        dict(name="plan_token", op="plan", requests=64, tokens=64, ending=0, page=64, blocks=64),
        # a busy server's step: a thousand requests, small pages, every ninth request just finished
        dict(name="plan_turnover", op="plan", requests=1024, tokens=910, ending=9, page=16, blocks=256),
        # prompts of 48 requests at once: as many tokens as a Roformer chunk of 801 frames and 60 bands
        dict(name="plan_prompts", op="plan", requests=48, tokens=48060, ending=0, page=128, blocks=64),
        # the next token of each of 64 requests, grouped heads, frequencies scaled by parts
        dict(name="append_token", op="append", tokens=64, padding=0, q_heads=32, kv_heads=8, dim=128, rot=128,
             pairing="halves", scaling="parts", page=64, spread=True, dtype="bf16"),
        # long prompts with grouped heads, positions interpolated
        dict(name="append_prompts", op="append", tokens=16384, padding=0, q_heads=32, kv_heads=8, dim=128, rot=128,
             pairing="halves", scaling="linear", page=128, spread=False, dtype="bf16"),
        # HTDemucs' heads of 48 columns, three sequences of 1895, part of each head rotated, rows of padding behind
        dict(name="append_part", op="append", tokens=5685, padding=75, q_heads=8, kv_heads=8, dim=48, rot=32,
             pairing="interleaved", scaling="none", page=16, spread=False, dtype="fp16"),
        # two requests, one token each, behind a short prefix: latency
        dict(name="prefix_few", op="prefix", requests=2, tokens=2, prefix=1895, most=40, q_heads=8, kv_heads=8, dim=64,
             page=16, dtype="fp16"),
        # the next token of each of 64 requests behind a prompt of 8192, grouped heads
        dict(name="prefix_token", op="prefix", requests=64, tokens=64, prefix=8192, most=1024, q_heads=32, kv_heads=8,
             dim=128, page=64, dtype="bf16"),
        # 16 questions to one very long document
        dict(name="prefix_long", op="prefix", requests=16, tokens=16, prefix=131072, most=512, q_heads=32, kv_heads=8,
             dim=128, page=128, dtype="bf16"),
        # five draft tokens a request to be checked, odd everything
        dict(name="prefix_draft", op="prefix", requests=32, tokens=160, prefix=3791, most=801, q_heads=12, kv_heads=4,
             dim=80, page=32, dtype="fp16"),
        # a Roformer's 60 bands as sequences that share a prefix of 801 frames, eight new frames each
        dict(name="prefix_frames", op="prefix", requests=60, tokens=480, prefix=801, most=801, q_heads=8, kv_heads=8,
             dim=64, page=16, dtype="fp16"),
        # ragged prompts of six requests behind a shared one
        dict(name="prefix_prompts", op="prefix", requests=6, tokens=4096, prefix=4096, most=1600, q_heads=32, kv_heads=8,
             dim=128, page=128, dtype="bf16"),
    ]


def _spread(rng, lo, hi):
    """A whole number between lo and hi, spread over its logarithm."""
    return min(max(int(round(lo * (hi / lo) ** rng.random())), lo), hi)


def draw(rng):
    op = rng.choice(["plan", "append", "prefix", "prefix"])
    page = rng.choice([16, 32, 64, 128, 256])
    if op == "plan":
        requests = _spread(rng, 1, 1024)
        ending = rng.choice([0, 3, 9])
        alive = len(_alive(dict(requests=requests, ending=ending)))
        tokens = alive * rng.choice([1, 1, 3]) if rng.random() < 0.5 else _spread(rng, max(1, alive), 48060)
        # a request's row holds what it has (up to 16 pages) and the largest share of the new tokens
        return dict(op=op, requests=requests, tokens=tokens, ending=ending, page=page,
                    blocks=18 + 3 * tokens // (alive * page))
    dtype = rng.choice(["fp16", "bf16"])
    if op == "append":
        dim = rng.choice([32, 48, 64, 80, 96, 128, 256])
        group, kv_heads = rng.choice([1, 2, 3, 4]), rng.choice([1, 4, 5, 8])
        most = 80_000_000 // (kv_heads * (group + 2) * dim)  # queries, keys and values together stay below 160 MB
        return dict(op=op, tokens=_spread(rng, 1, min(16384, most)), padding=rng.choice([0, 0, 13]),
                    q_heads=kv_heads * group, kv_heads=kv_heads, dim=dim, rot=rng.choice([dim, dim, dim // 2]),
                    pairing=rng.choice(["halves", "interleaved"]), scaling=rng.choice(["none", "linear", "parts"]),
                    page=page, spread=rng.random() < 0.5, dtype=dtype)
    dim = rng.choice([32, 48, 64, 64, 80, 96, 128, 128])
    group, kv_heads = rng.choice([1, 2, 3, 4, 8]), rng.choice([1, 2, 4, 8])
    requests = _spread(rng, 1, 64)
    tokens = requests * rng.choice([1, 1, 1, 2, 5]) if rng.random() < 0.7 else _spread(rng, requests, 2048)
    # keys and values of all requests stay below 240 MB, as do the prefix's; the products below the listed prompts'
    room = 60_000_000 // (kv_heads * dim)
    most = _spread(rng, 1, min(2048, room // requests))
    prefix = rng.choice([0, 1, 1, 1, 1, 1])
    if prefix:
        flops = 30_000_000_000 // (tokens * kv_heads * group * dim)
        prefix = _spread(rng, 1, max(1, min(65536, room, flops)))
    return dict(op=op, requests=requests, tokens=tokens, prefix=prefix, most=max(most, *_counts(requests, tokens), 1),
                q_heads=kv_heads * group, kv_heads=kv_heads, dim=dim, page=page, dtype=dtype)


def _alive(case):
    """Requests that go on: all but every `ending`-th."""
    return [r for r in range(case["requests"]) if not (case["ending"] and r % case["ending"] == case["ending"] - 1)]


def _counts(requests, tokens):
    """New tokens of each request: equal where they divide, about as uneven as 1 : 2 : 3 otherwise, the last the most."""
    if tokens % requests == 0 and tokens // requests < 16:
        return [tokens // requests] * requests
    weights = [1 + (7 * i + 3) % 2 for i in range(requests - 1)] + [3]
    spare, total, upto, counts = tokens - requests, sum(weights), 0, []
    for w in weights:
        counts.append(1 + spare * (upto + w) // total - spare * upto // total)
        upto += w
    return counts


def _new_tokens(case):
    """A plan's new tokens: -1 for a request that has ended."""
    new = [-1] * case["requests"]
    alive = _alive(case)
    for r, n in zip(alive, _counts(len(alive), case["tokens"])):
        new[r] = n
    return new


def _own_lens(case, counts):
    """Own tokens of each request, its new ones included: from `most` down to the new ones alone."""
    n = case["requests"]
    return [max(c, case["most"] - (i * case["most"]) // max(1, n - 1)) for i, c in enumerate(counts)]


def _pages_held(case):
    """The most pages a plan's request holds before the call."""
    new = _new_tokens(case)
    return max(1, min(16, case["blocks"] - (max(new) + case["page"] - 1) // case["page"] - 1))


def work(case):
    if case["op"] == "plan":
        new, page = _new_tokens(case), case["page"]
        moved = sum((n + page - 1) // page if n > 0 else 8 for n in new)  # pages taken and given back, about
        # lengths, counts and starts; a page moved is read and written; a slot and a position a token
        return {"bytes": 20 * case["requests"] + 8 * moved + 8 * case["tokens"], "flops": 4 * case["tokens"]}
    if case["op"] == "append":
        real = case["tokens"] * case["dim"]
        rows = (case["tokens"] + case["padding"]) * case["dim"]
        return {"bytes": 4 * (rows * case["q_heads"] + 2 * real * case["kv_heads"]) + 8 * case["tokens"],
                "flops": 3 * (rows * case["q_heads"] + real * case["kv_heads"])}
    counts = _counts(case["requests"], case["tokens"])
    lens = _own_lens(case, counts)
    width = case["dim"] * case["q_heads"]
    pairs = sum(n * (case["prefix"] + length - n) + n * (n + 1) // 2 for n, length in zip(counts, lens))
    return {"bytes": 4 * (case["tokens"] * width + (case["prefix"] + sum(lens)) * case["kv_heads"] * case["dim"]),
            "flops": 4 * pairs * width}


# ------------------------------------------------------------------------------------- inputs
def _frequencies(case):
    """Radians a position for each pair, in 64 bits, and what cos and sin are multiplied by."""
    half = case["rot"] // 2
    freq = 500000.0 ** (-torch.arange(half, dtype=torch.float64) / half)
    if case["scaling"] == "linear":
        return freq / 4, 1.0
    if case["scaling"] == "parts":  # slow pairs interpolated, fast ones kept, a ramp between
        turns = freq * 8192 / (2 * math.pi)
        keep = ((turns - 1) / (32 - 1)).clamp(0, 1)
        return freq * keep + freq / 16 * (1 - keep), 0.1 * math.log(16.0) + 1.0
    return freq, 1.0


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    s = dict(case)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda").to(DTYPES[case["dtype"]])

    def ints(values):
        return torch.tensor(values, dtype=torch.int32, device="cuda")

    def shuffled(n):
        return torch.randperm(n, generator=g, device="cuda").int()

    page = case["page"]
    if case["op"] == "plan":
        requests, blocks, held = case["requests"], case["blocks"], _pages_held(case)
        new = _new_tokens(case)
        pages = requests * held + sum(max(n, 0) // page + 1 for n in new) + 5
        lens = torch.randint(0, held * page + 1, (requests,), generator=g, device="cuda", dtype=torch.int32)
        order = shuffled(pages)
        have = (lens + page - 1) // page
        at = torch.arange(blocks, device="cuda", dtype=torch.int32)
        before = have.cumsum(0) - have
        table = torch.where(at < have[:, None], order[(before[:, None] + at).clamp(max=pages - 1)], -1).int()
        taken = int(have.sum())
        s["new"], s["lens"], s["table"], s["start"] = ints(new), lens, table, 8192
        s["free"] = torch.cat((order[taken:], order.new_full((taken,), -1)))
        s["count"] = ints([pages - taken])
    elif case["op"] == "append":
        real, rows = case["tokens"], case["tokens"] + case["padding"]
        s["q"] = normal(rows, case["q_heads"], case["dim"])
        kv = normal(rows, 2, case["kv_heads"], case["dim"])  # one projection writes keys and values side by side
        s["k"], s["v"] = kv[:, 0], kv[:, 1]
        at = torch.arange(rows, device="cuda", dtype=torch.int32)
        if case["spread"]:  # a token in each of many requests' pages, at a place and a position of its own
            pages = real + 3
            inside = torch.randint(0, page, (rows,), generator=g, device="cuda", dtype=torch.int32)
            slots = torch.cat((shuffled(pages), shuffled(pages)))[at.clamp(max=real).long()] * page + inside
            s["positions"] = torch.randint(0, 1 << 20, (rows,), generator=g, device="cuda", dtype=torch.int32)
        else:  # a prompt's tokens one behind the other, through pages in any order
            pages = rows // page + 4
            slots = shuffled(pages)[(at // page).long()] * page + at % page
            s["positions"] = at + torch.randint(0, 1 << 17, (1,), generator=g, device="cuda", dtype=torch.int32)
        s["slots"] = torch.where(at < real, slots, -1).int()
        s["k_cache"], s["v_cache"] = normal(2, pages, page, case["kv_heads"], case["dim"])
        freq, s["amplitude"] = _frequencies(case)
        s["freq"] = freq.cuda()
    else:
        counts = _counts(case["requests"], case["tokens"])
        lens = _own_lens(case, counts)
        s["counts"], s["lens_host"], width = counts, lens, (case["kv_heads"], case["dim"])
        s["q"] = normal(case["tokens"], case["q_heads"], case["dim"])
        s["prefix_k"], s["prefix_v"] = normal(2, case["prefix"], *width)
        have = [(n + page - 1) // page for n in lens]
        pages = sum(have) + 3
        order, table, taken = shuffled(pages), [], 0
        for n in have:
            table.append(torch.nn.functional.pad(order[taken:taken + n], (0, max(have) - n)))
            taken += n
        s["k_cache"], s["v_cache"] = normal(2, pages, page, *width)
        s["table"], s["lens"] = torch.stack(table).contiguous(), ints(lens)
        starts = [0]
        for n in counts:
            starts.append(starts[-1] + n)
        s["starts"] = None if case["tokens"] == case["requests"] else ints(starts)
    return s


# ------------------------------------------------------------------------------------- one pass
def run(s):
    return _run_own(s) if own else {"plan": _plain_plan, "append": _plain_append, "prefix": _plain_prefix}[s["op"]](s)


def _run_own(s):
    package = os.path.abspath("cuda-msst-infer_b200")
    if package not in sys.path:
        sys.path.insert(0, package)
    from msst_b200 import ops

    if s["op"] == "plan":
        starts, slots, positions, lens, count = ops.cache_plan(
            s["new"], s["lens"], s["table"], s["free"], s["count"], page_size=s["page"], tokens=s["tokens"],
            start=s["start"])
        return starts, slots, positions, lens, count, s["table"], s["free"]
    if s["op"] == "append":
        q = ops.rope_append(s["q"], s["k"], s["v"], s["positions"], s["slots"], s["freq"], s["k_cache"], s["v_cache"],
                            amplitude=s["amplitude"], pairing=s["pairing"])
        return q, s["k_cache"], s["v_cache"]
    return ops.prefix_attention(s["q"], s["prefix_k"], s["prefix_v"], s["k_cache"], s["v_cache"], s["table"], s["lens"],
                                q_starts=s["starts"])


def _plain_plan(s):
    new, lens, table, free, count, page = s["new"], s["lens"], s["table"], s["free"], s["count"], s["page"]
    blocks, pages = table.shape[1], free.numel()
    at = torch.arange(blocks, device=new.device)
    # pages of ended requests go on top of the stack, request by request
    have = (lens + page - 1) // page
    back = torch.where(new < 0, have, 0)
    first = count + back.cumsum(0) - back
    target = torch.where(at < back[:, None], first[:, None] + at, pages).flatten()
    stack = torch.cat((free, free.new_zeros(1))).scatter(0, target.long(), table.flatten())[:pages]
    free.copy_(stack)
    top = count + back.sum()
    # pages that are wanted come off its top in the same order
    kept, more = torch.where(new < 0, 0, lens), new.clamp(min=0)
    ends = more.cumsum(0)
    have = (kept + page - 1) // page
    wide = ((kept + more + page - 1) // page > blocks) | (ends > s["tokens"])
    need = torch.where(wide, 0, (kept + more + page - 1) // page - have)
    upto = need.cumsum(0)
    fits = ~wide & ((need == 0) | (upto <= top))
    got = torch.where(fits, need, 0)
    source = top - 1 - (upto - need)[:, None] - (at - have[:, None])
    taken = (at >= have[:, None]) & (at < (have + got)[:, None])
    table.copy_(torch.where(taken, free[source.clamp(0, pages - 1).long()], table))
    # the place of each new token
    starts = torch.cat((ends.new_zeros(1), ends)).clamp(max=s["tokens"])
    t = torch.arange(s["tokens"], device=new.device)
    r = torch.searchsorted(starts[1:].contiguous(), t, right=True)
    there = r < new.numel()
    r = r.clamp(max=new.numel() - 1)
    position = kept[r] + t - starts[r]
    slot = table[r, (position // page).clamp(max=blocks - 1)] * page + position % page
    return (starts.int(), torch.where(there & fits[r], slot, -1).int(), torch.where(there, position + s["start"], 0).int(),
            torch.where(fits, kept + more, kept).int(), (top - got.sum()).int(), table, free)


def _plain_append(s):
    angle = s["positions"].double()[:, None, None] * s["freq"]
    cos, sin = (angle.cos() * s["amplitude"]).float(), (angle.sin() * s["amplitude"]).float()
    half, real = s["freq"].numel(), s["tokens"]

    def rotate(x):
        x = x.float()
        turn, rest = x[..., :2 * half], x[..., 2 * half:]
        if s["pairing"] == "halves":
            a, b = turn[..., :half], turn[..., half:]
            out = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
        else:
            a, b = turn[..., 0::2], turn[..., 1::2]
            out = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
        return torch.cat((out, rest), -1).to(s["q"].dtype)

    slots = s["slots"][:real].long()  # the rows of padding behind have none
    s["k_cache"].flatten(0, 1).index_copy_(0, slots, rotate(s["k"])[:real])
    s["v_cache"].flatten(0, 1).index_copy_(0, slots, s["v"][:real])
    return rotate(s["q"]), s["k_cache"], s["v_cache"]


def _plain_prefix(s):
    tokens, heads, dim = s["q"].shape
    kv_heads, page = s["k_cache"].shape[2], s["page"]
    group = heads // kv_heads
    out = torch.empty(tokens, heads, dim, device=s["q"].device)
    prefix_k, prefix_v = s["prefix_k"].float().permute(1, 2, 0), s["prefix_v"].float().transpose(0, 1)
    begin = 0
    for r, (n, length) in enumerate(zip(s["counts"], s["lens_host"])):
        pages = s["table"][r, :(length + page - 1) // page].long()
        k = s["k_cache"][pages].flatten(0, 1)[:length].float().permute(1, 2, 0)
        v = s["v_cache"][pages].flatten(0, 1)[:length].float().transpose(0, 1)
        q = s["q"][begin:begin + n].float().view(n, kv_heads, group, dim).permute(1, 2, 0, 3).reshape(kv_heads, -1, dim)
        # all of the prefix; of the request's own tokens those up to the row's
        late = torch.arange(length, device=q.device) > torch.arange(length - n, length, device=q.device)[:, None]
        score = torch.cat((q @ prefix_k, (q @ k).masked_fill_(late.repeat(group, 1), -torch.inf)), -1)
        score *= dim ** -0.5
        score -= score.amax(-1, keepdim=True)
        score.exp_()
        y = score[..., :s["prefix"]] @ prefix_v
        y += score[..., s["prefix"]:] @ v
        y /= score.sum(-1, keepdim=True)
        out[begin:begin + n] = y.view(kv_heads, group, n, dim).permute(2, 0, 1, 3).reshape(n, heads, dim)
        begin += n
    return out.to(s["q"].dtype)


# ------------------------------------------------------------------------------------- 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    return {"plan": _exact_plan, "append": _exact_append, "prefix": _exact_prefix}[case["op"]](s)


def _exact_plan(s):
    """Request by request, with a list as the stack."""
    new, lens, table = s["new"].tolist(), s["lens"].tolist(), s["table"].tolist()
    free, count, page = s["free"].tolist(), int(s["count"]), s["page"]
    stack = free[:count]
    for r, n in enumerate(new):
        if n < 0:
            stack += table[r][:-(-lens[r] // page)]
            lens[r] = 0
    free[:len(stack)] = stack
    starts, slots, positions, short = [0], [], [], False
    for r, n in enumerate(new):
        n = max(n, 0)
        have, want = -(-lens[r] // page), -(-(lens[r] + n) // page)
        good = want <= s["blocks"] and starts[-1] + n <= s["tokens"]
        if good and want > have:
            short = short or want - have > len(stack)
            good = not short
        if good:
            for b in range(have, want):
                table[r][b] = stack.pop()
        for p in range(lens[r], lens[r] + min(n, s["tokens"] - starts[-1])):
            slots.append(table[r][p // page] * page + p % page if good else -1)
            positions.append(p + s["start"])
        starts.append(min(starts[-1] + n, s["tokens"]))
        lens[r] += n if good else 0
    slots += [-1] * (s["tokens"] - len(slots))
    positions += [0] * (s["tokens"] - len(positions))
    return tuple(torch.tensor(x, dtype=torch.int32, device="cuda")
                 for x in (starts, slots, positions, lens, [len(stack)], table, free))


def _exact_append(s):
    """Each pair as a complex number times amplitude * exp(i angle)."""
    angle = s["positions"].double()[:, None] * s["freq"]
    turn = torch.polar(torch.full_like(angle, s["amplitude"]), angle).unsqueeze(1)
    half = s["freq"].numel()
    first = torch.arange(half, device="cuda") * (2 if s["pairing"] == "interleaved" else 1)
    second = first + (1 if s["pairing"] == "interleaved" else half)
    done = []
    for x in (s["q"].double(), s["k"].double()):
        z = torch.complex(x[..., first], x[..., second]) * turn
        x[..., first], x[..., second] = z.real, z.imag
        done.append(x)
    k_cache, v_cache = s["k_cache"].double(), s["v_cache"].double()
    where = s["slots"][:s["tokens"]].long()
    page, inside = where // s["page"], where % s["page"]
    k_cache[page, inside], v_cache[page, inside] = done[1][:s["tokens"]], s["v"][:s["tokens"]].double()
    return done[0], k_cache, v_cache


def _exact_prefix(s):
    """Head by head over a request's keys in one row, through the logarithm of the sum."""
    tokens, heads, dim = s["q"].shape
    out = torch.zeros(tokens, heads, dim, dtype=torch.float64, device="cuda")
    group = heads // s["k_cache"].shape[2]
    begin = 0
    for r, (n, length) in enumerate(zip(s["counts"], s["lens_host"])):
        j = torch.arange(length, device="cuda")
        page, inside = s["table"][r].long()[j // s["page"]], j % s["page"]
        for h in range(heads):
            k = torch.cat((s["prefix_k"][:, h // group], s["k_cache"][page, inside, h // group])).double()
            v = torch.cat((s["prefix_v"][:, h // group], s["v_cache"][page, inside, h // group])).double()
            score = torch.einsum("nd,md->nm", s["q"][begin:begin + n, h].double(), k) / dim ** 0.5
            key = torch.arange(k.shape[0], device="cuda") - s["prefix"] - (length - n)
            score = score.masked_fill(key > torch.arange(n, device="cuda")[:, None], -torch.inf)
            out[begin:begin + n, h] = torch.exp(score - torch.logsumexp(score, 1, keepdim=True)) @ v
        begin += n
    return out
