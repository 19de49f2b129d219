"""Refusals of the operators of a paged cache behind a shared prefix (no GPU: every check comes
before a device is touched)."""
from __future__ import annotations

import ctypes
import struct

import pytest


def _heads(ptr=16, heads=2, sb=2048, sn=128, sh=64):
    return struct.pack("Pi4xqqq", ptr, heads, sb, sn, sh)


def _plan(**kw):
    from msst_b200 import lib

    a = dict(new=16, lens=16, R=4, table=16, blocks=8, stride=8, free=16, pages=64, count=16, page=16, start=0, tokens=4,
             out_lens=16, out_count=16, starts=16, slots=16, positions=16)
    a.update(kw)
    return lib().msst_cache_plan(*a.values(), None)


@pytest.mark.parametrize("bad, word", [
    (dict(page=8), "page_size"), (dict(page=512), "page_size"), (dict(page=48), "page_size"), (dict(pages=0), "pages"),
    (dict(pages=1 << 27), "pages"), (dict(R=-1), "requests"), (dict(R=8193), "requests"), (dict(blocks=-1), "blocks"),
    (dict(blocks=1 << 27, stride=1 << 27), "blocks"), (dict(stride=7), "overlap"), (dict(table=None), "block_table"),
    (dict(tokens=-1), "tokens"), (dict(tokens=0x7fffffff), "tokens"), (dict(start=-1), "positions"),
    (dict(start=0x7fffffff), "positions"), (dict(new=None), "null"), (dict(lens=None), "null"), (dict(free=None), "null"),
    (dict(count=None), "null"), (dict(out_lens=None), "null"), (dict(out_count=None), "null"), (dict(starts=None), "null"),
    (dict(slots=None), "null"), (dict(positions=None), "null"),
])
def test_cache_plan_refuses(bad, word):
    from msst_b200 import MSST_ERR_INVALID, lib

    assert _plan(**bad) == MSST_ERR_INVALID
    assert word in lib().msst_last_error().decode()


def _append(**kw):
    from msst_b200 import lib

    a = dict(q=_heads(), k=_heads(), v=_heads(), tokens=4, d=64, positions=16, slots=16, freq=16, rot=64, amplitude=1.0,
             pairing=0, k_cache=_heads(), v_cache=_heads(), pages=4, page=16, dtype=0, out=_heads())
    a.update(kw)
    return lib().msst_rope_append(*a.values(), None)


@pytest.mark.parametrize("bad, word", [
    (dict(q=None), "q needs"), (dict(k=None), "k needs"), (dict(out=None), "q_out"), (dict(k_cache=None), "k_cache"),
    (dict(d=0), "head_dim"), (dict(d=60), "head_dim"), (dict(d=264), "head_dim"), (dict(rot=4), "rot_dim"),
    (dict(rot=72), "rot_dim"), (dict(rot=-8), "rot_dim"), (dict(pairing=2), "pairing"), (dict(dtype=2), "dtype"),
    (dict(amplitude=float("nan")), "amplitude"), (dict(page=17), "page_size"), (dict(pages=-1), "pages"),
    (dict(q=_heads(ptr=24)), "aligned"), (dict(k=_heads(sn=132)), "multiples of 8"), (dict(v=_heads(heads=1)), "same number"),
    (dict(v_cache=_heads(heads=1)), "same number"), (dict(out=_heads(heads=3)), "q's heads"), (dict(tokens=-1), "tokens"),
    (dict(k_cache=_heads(sb=0)), "strides above 0"), (dict(out=_heads(sn=0)), "strides above 0"),
    (dict(q=_heads(sn=-8)), "negative"), (dict(slots=None), "null"), (dict(positions=None), "null"), (dict(freq=None), "null"),
    (dict(tokens=1 << 29), "too many"),
])
def test_rope_append_refuses(bad, word):
    from msst_b200 import MSST_ERR_INVALID, lib

    assert _append(**bad) == MSST_ERR_INVALID
    assert word in lib().msst_last_error().decode()


def _attention(**kw):
    from msst_b200 import lib

    a = dict(q=_heads(), tokens=4, starts=16, requests=2, pk=_heads(), pv=_heads(), prefix=8, kc=_heads(), vc=_heads(),
             pages=4, page=16, table=16, blocks=2, stride=2, lens=16, d=64, scale=0.0, dtype=0, out=_heads(), rest=0, ws=None,
             wsb=0)
    a.update(kw)
    return lib().msst_prefix_attention(*a.values(), None)


@pytest.mark.parametrize("bad, word", [
    (dict(q=None), "q needs"), (dict(out=None), "out"), (dict(kc=None), "k_cache"), (dict(vc=None), "v_cache"),
    (dict(pk=None), "prefix_k"), (dict(pv=None), "prefix_v"), (dict(tokens=-1), "shape"), (dict(prefix=-1), "shape"),
    (dict(prefix=0x7fffffff), "too many"), (dict(starts=None), "one token"), (dict(requests=-1), "requests"),
    (dict(requests=9000), "requests"), (dict(d=136), "head_dim"), (dict(d=12), "head_dim"), (dict(scale=float("inf")), "scale"),
    (dict(dtype=2), "dtype"), (dict(page=12), "page_size"), (dict(pages=0), "pages"), (dict(blocks=-1), "blocks"),
    (dict(stride=1), "overlap"), (dict(table=None), "block_table"), (dict(lens=None), "lens"),
    (dict(q=_heads(heads=3), out=_heads(heads=3)), "multiple of it"), (dict(out=_heads(heads=4)), "q's heads"), (dict(vc=_heads(heads=1)), "same number"),
    (dict(pk=_heads(heads=1)), "caches' heads"), (dict(kc=_heads(sn=0)), "must not be 0"), (dict(q=_heads(sn=0)), "must not be 0"),
    (dict(pv=_heads(sn=0)), "must not be 0"), (dict(kc=_heads(ptr=8)), "aligned"), (dict(pk=_heads(sh=60)), "multiples of 8"),
    (dict(tokens=(1 << 30) + 1), "too many"),
])
def test_prefix_attention_refuses(bad, word):
    from msst_b200 import MSST_ERR_INVALID, lib

    assert _attention(**bad) == MSST_ERR_INVALID
    assert word in lib().msst_last_error().decode()


@pytest.mark.parametrize("q_heads, kv_heads, head_dim", [(2, 4, 64), (3, 2, 64), (4, 4, 136), (4, 4, 12), (0, 1, 64)])
def test_workspace_refuses_heads(q_heads, kv_heads, head_dim):
    from msst_b200 import MSST_ERR_INVALID, lib

    n = ctypes.c_longlong(-1)
    assert lib().msst_prefix_attention_workspace(8, 2, 64, q_heads, kv_heads, head_dim, ctypes.byref(n)) == MSST_ERR_INVALID
    assert n.value == -1


def test_calls_by_words():
    """msst_call hands each argument on to its place: the refusals of the calls themselves, one argument wrong at a time."""
    from msst_b200 import MSST_ERR_INVALID, MSST_OK, lib

    L, big = lib(), 1 << 40

    def call(op, form, words):
        return L.msst_call(op, struct.pack(form, *words))

    heads = [16, 2, 2048, 128, 64]
    plan = [16, 16, 4, 16, 8, 8, 16, 64, 16, 16, 0, 4, 16, 16, 16, 16, 16, 0]
    append = heads * 3 + [0, 64, 16, 16, 16, 64, 1.0, 0] + heads * 2 + [4, 16, 0] + heads + [0]
    attend = heads + [0, 16, 2] + heads * 2 + [8] + heads * 2 + [4, 16, 16, 2, 2, 16, 64, 0.0, 0] + heads + [0, 0, 0, 0]
    for op, form, good, bads in (
        (0, "18q", plan, ((0, 0, "null"), (1, 0, "null"), (2, 9000, "requests"), (3, 0, "block_table"), (4, big, "blocks"),
                          (5, 7, "overlap"), (6, 0, "null"), (7, 0, "pages"), (8, 0, "null"), (9, 48, "page_size"),
                          (10, -1, "positions"), (11, big, "tokens"), (11, -big, "tokens"), (12, 0, "null"), (13, 0, "null"),
                          (14, 0, "null"), (15, 0, "null"), (16, 0, "null"))),
        (1, "21qd20q", append, ((0, 24, "q must be"), (1, 0, "q needs"), (3, 132, "q needs strides"), (6, 0, "k needs"),
                                (9, 60, "k needs strides"), (10, 8, "v must be"), (15, -1, "tokens"), (16, 60, "head_dim"),
                                (20, 72, "rot_dim"), (21, float("nan"), "amplitude"), (22, 2, "pairing"), (24, 1, "same number"),
                                (25, 0, "k_cache is written"), (30, -8, "v_cache has a negative"), (33, 0, "pages"),
                                (34, 17, "page_size"), (35, 3, "dtype"), (37, 3, "q's heads"))),
        (2, "36qd10q", attend, ((1, 3, "q's heads"), (5, -1, "shape"), (7, -1, "requests"), (8, 8, "prefix_k must be"),
                               (9, 0, "prefix_k needs"), (14, 1, "caches' heads"), (18, -1, "shape"), (20, 0, "k_cache needs"),
                               (25, 1, "same number"), (29, 0, "pages"), (30, 12, "page_size"), (31, 0, "block_table"),
                               (32, -1, "blocks"), (33, 1, "overlap"), (35, 12, "head_dim"), (36, float("inf"), "scale"),
                               (37, 2, "dtype"), (39, 4, "q's heads"))),
    ):
        if op:
            assert call(op, form, good) == MSST_OK  # (no row: nothing is launched)
        for at, value, word in bads:
            wrong = list(good)
            if op:
                wrong[{1: 15, 2: 5}[op]] = 4  # rows, for which strides and pointers have to be right
            wrong[at] = value
            assert call(op, form, wrong) == MSST_ERR_INVALID, (op, at)
            assert word in L.msst_last_error().decode(), (op, at, L.msst_last_error())
    assert L.msst_call(3, struct.pack("q", 0)) == MSST_ERR_INVALID and L.msst_call(0, None) == MSST_ERR_INVALID


def test_empty_calls_need_no_device():
    from msst_b200 import MSST_OK

    assert _append(tokens=0) == MSST_OK and _attention(tokens=0) == MSST_OK and _attention(requests=0) == MSST_OK


def test_python_argument_checks():
    import torch
    from msst_b200 import ops

    def i32(*shape):
        return torch.zeros(*shape, dtype=torch.int32)

    plan = dict(new_tokens=i32(3), lens=i32(3), block_table=i32(3, 4), free_pages=i32(20), free_count=i32(1), page_size=16,
                tokens=3)
    t, h = torch.zeros(4, 2, 64, dtype=torch.float16), torch.zeros(5, 16, 2, 64, dtype=torch.float16)
    append = dict(q=t, k=t, v=t, positions=i32(4), slots=i32(4), inv_freq=torch.zeros(32, dtype=torch.float64), k_cache=h,
                  v_cache=h)
    attend = dict(q=t, prefix_k=t, prefix_v=t, k_cache=h, v_cache=h, block_table=i32(4, 2), lens=i32(4))
    for op, good, bads in (
        (ops.cache_plan, plan, (dict(new_tokens=i32(3, 1)), dict(lens=i32(2)), dict(lens=i32(3).long()),
                                dict(block_table=i32(2, 4)), dict(block_table=i32(4, 3).t()[:3]), dict(free_count=i32(2)),
                                dict(free_pages=i32(40)[::2]), dict(out_lens=i32(6)[::2]), dict(tokens=-1))),
        (ops.rope_append, append, (dict(q=t[0]), dict(k=t[:3]), dict(v=t[:, :1]), dict(k=t.bfloat16()), dict(q=t.float()),
                                   dict(positions=i32(3)), dict(positions=None), dict(slots=i32(4).long()),
                                   dict(inv_freq=torch.zeros(32)), dict(k_cache=h[..., :32]), dict(v_cache=h[:4]),
                                   dict(k_cache=h.transpose(2, 3)), dict(out_q=t[:, :1]))),
        (ops.prefix_attention, attend, (dict(q=t[0]), dict(prefix_k=None), dict(prefix_v=t[:3]), dict(prefix_k=t.bfloat16()),
                                        dict(k_cache=h[..., :32]), dict(v_cache=h.bfloat16()), dict(block_table=i32(3, 2)),
                                        dict(lens=i32(4).long()), dict(lens=i32(8)[::2]), dict(q_starts=i32(4)),
                                        dict(out=t[:3]), dict(q=t[:, :1].expand(4, 3, 64)))),
    ):
        for bad in bads:
            with pytest.raises(ValueError):
                op(**{**good, **bad})


def _source(name):
    import os

    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    with open(os.path.join(root, "cuda-msst-infer_b200", "csrc", name)) as f:
        return f.read()


@pytest.mark.parametrize("begin, end", [
    ("// ------------------------------------------------------------ softmax + epilogue", "  __syncthreads();\n  if (warp == 1) {"),
    ("// ------------------------------------------------------------ rows that nobody sees", "} else if (lane == 0) {"),
    ("// ------------------------------------------------------------ the team's tiles", "if (!ok && lane == 0) {"),
    ("  const int q_box =", "__global__"),
])
def test_whole_warp_roles_wait_together(begin, end):
    """Where a wait gives up, lanes of a warp must not part (full-mask instructions follow): a wait cannot be made
    to run out from outside, so the source is read."""
    text = _source("prefix_attn.cu")
    assert text.count(begin) == 1
    role = text[text.index(begin):]
    role = role[:role.index(end)]
    assert "mbar_wait_warp" in role and "mbar_wait<" not in role and "ring->wait(" not in role


def test_roles_end_after_their_own_copies():
    text = _source("prefix_attn.cu")
    assert text.count("mbar_drain_ring(") == 4  # K and V of the tile role, tiles and query rows of the token role
    assert text.count("umma_commit(mma_end)") == text.count("mbar_drain(mma_end, 0)") == 1


def test_rope_frequencies():
    import math

    import torch
    from msst_b200 import rope_frequencies

    plain, one = rope_frequencies(64, 10000.0)
    assert plain.dtype == torch.float64 and plain.shape == (32,) and one == 1.0
    assert torch.allclose(plain, 10000.0 ** (-torch.arange(32, dtype=torch.float64) / 32), rtol=1e-14)
    assert torch.equal(rope_frequencies(64, scaling="linear", factor=4.0)[0], plain / 4)
    wide, _ = rope_frequencies(64, scaling="base", factor=4.0)
    assert abs(float(wide[0] - plain[0])) < 1e-15 and abs(float(wide[-1] / plain[-1]) - 0.25) < 1e-12
    parts, amplitude = rope_frequencies(64, scaling="parts", factor=8.0, original=4096)
    turns = plain * 4096 / (2 * math.pi)
    assert torch.equal(parts[turns > 32], plain[turns > 32]) and amplitude == 1 + 0.1 * math.log(8.0)
    assert torch.allclose(parts[turns < 1], plain[turns < 1] / 8, rtol=1e-14)
    between = (turns >= 1) & (turns <= 32)
    assert bool((parts[between] <= plain[between]).all()) and bool((parts[between] >= plain[between] / 8).all())
    for bad in (dict(rot_dim=3), dict(rot_dim=0), dict(base=0.0), dict(scaling="ntk"), dict(factor=-1.0),
                dict(scaling="parts", slow=4.0, fast=2.0)):
        with pytest.raises(ValueError):
            rope_frequencies(**{"rot_dim": 64, **bad})


def test_tokens_of_a_request_within_a_tile_of_32_bits_are_refused():
    """Rounded up to a tile of keys they would pass 2^31 - 1 and count as none."""
    from msst_b200 import MSST_ERR_INVALID, lib

    most = dict(blocks=(1 << 27) - 1, stride=1 << 27)  # of 16 tokens
    for call in (_plan, _attention):
        assert call(**most) == MSST_ERR_INVALID and "blocks" in lib().msst_last_error().decode()
