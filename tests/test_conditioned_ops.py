"""Refusals of the conditioned-block operators (no GPU: every check comes before a device is touched)."""
from __future__ import annotations

import ctypes
import struct

import pytest


def _heads(ptr=16, heads=2, sb=1024, sn=128, sh=64):
    return struct.pack("Pi4xqqq", ptr, heads, sb, sn, sh)


def _qk(**kw):
    from msst_b200 import lib

    a = dict(q=_heads(), k=None, batch=1, seq=4, d=64, eps=1e-6, cos=16, sin=16, num_pos=8, rot=64, pos=None, pairing=0,
             dtype=0, qo=_heads(), ko=None)
    a.update(kw)
    return lib().msst_qk_norm_rope(a["q"], a["k"], a["batch"], a["seq"], a["d"], None, None, a["eps"], a["cos"],
                                   a["sin"], a["num_pos"], a["rot"], a["pos"], a["pairing"], a["dtype"], a["qo"],
                                   a["ko"], None)


@pytest.mark.parametrize("bad, word", [
    (dict(q=None), "q needs"), (dict(qo=None), "q_out"), (dict(d=0), "head_dim"), (dict(d=7), "head_dim"),
    (dict(d=258), "head_dim"), (dict(rot=66), "rot_dim"), (dict(rot=3), "rot_dim"), (dict(cos=None), "tables"),
    (dict(num_pos=3), "longer than the tables"), (dict(pairing=2), "pairing"), (dict(dtype=2), "dtype"),
    (dict(eps=-1.0), "eps"), (dict(eps=float("nan")), "eps"), (dict(q=_heads(heads=0)), "head"), (dict(k=_heads()), "k_out"),
    (dict(qo=_heads(heads=3)), "heads"), (dict(q=_heads(sn=-64)), "negative"), (dict(batch=-1), "shape"),
    (dict(q=_heads(ptr=0)), "null"), (dict(batch=1 << 20, seq=1 << 12, num_pos=1 << 12), "too many"),
])
def test_qk_norm_rope_refuses(bad, word):
    from msst_b200 import MSST_ERR_INVALID, lib

    assert _qk(**bad) == MSST_ERR_INVALID
    assert word in lib().msst_last_error().decode()


def _cross(**kw):
    from msst_b200 import lib

    a = dict(q=_heads(), k=_heads(), v=_heads(), batch=1, nq=4, nk=4, d=64, scale=0.0, dtype=0, out=_heads(),
             ws=None, wsb=0)
    a.update(kw)
    return lib().msst_cross_attention(a["q"], a["k"], a["v"], a["batch"], a["nq"], a["nk"], a["d"], a["scale"], None,
                                      None, a["dtype"], a["out"], a["ws"], a["wsb"], None)


@pytest.mark.parametrize("bad, word", [
    (dict(q=None), "q needs"), (dict(out=None), "out"), (dict(d=4), "head_dim"), (dict(d=136), "head_dim"),
    (dict(d=60), "head_dim"), (dict(scale=float("inf")), "scale"), (dict(dtype=7), "dtype"),
    (dict(nq=-1), "shape"), (dict(q=_heads(ptr=24)), "aligned"), (dict(k=_heads(sn=132)), "multiples of 8"),
    (dict(v=_heads(heads=1)), "same number of heads"), (dict(k=_heads(heads=4), v=_heads(heads=4)), "multiple of it"),
    (dict(out=_heads(heads=4)), "q's heads"), (dict(batch=1 << 20, nq=1 << 12), "too many"),
])
def test_cross_attention_refuses(bad, word):
    from msst_b200 import MSST_ERR_INVALID, lib

    assert _cross(**bad) == MSST_ERR_INVALID
    assert word in lib().msst_last_error().decode()


def _adapter(**kw):
    from msst_b200 import lib

    a = dict(x=16, rows=4, K=64, ldx=64, w=16, N=64, la=16, lb=16, count=2, rank=16, ids=16, dtype=0, out=16, ldo=64,
             ws=16, wsb=1 << 20)
    a.update(kw)
    return lib().msst_adapter_gemm(a["x"], a["rows"], a["K"], a["ldx"], a["w"], a["N"], None, a["la"], a["lb"], None,
                                   a["count"], a["rank"], a["ids"], a["dtype"], a["out"], a["ldo"], a["ws"], a["wsb"],
                                   None)


@pytest.mark.parametrize("bad, word", [
    (dict(x=None), "null"), (dict(ids=None), "null"), (dict(la=None), "null"), (dict(K=60), "multiples of 8"),
    (dict(N=0), "multiples of 8"), (dict(rank=4), "rank"), (dict(rank=264), "rank"), (dict(ldx=56), "ldx"),
    (dict(ldo=68), "ldo"), (dict(rows=-1), "rows"), (dict(rows=1 << 31), "rows"), (dict(count=-1), "adapters"),
    (dict(x=8), "aligned"), (dict(lb=8), "aligned"), (dict(dtype=2), "dtype"),
])
def test_adapter_gemm_refuses(bad, word):
    from msst_b200 import MSST_ERR_INVALID, lib

    assert _adapter(**bad) == MSST_ERR_INVALID
    assert word in lib().msst_last_error().decode()


def test_empty_calls_need_no_device():
    from msst_b200 import MSST_OK

    assert _qk(batch=0) == MSST_OK and _cross(nq=0) == MSST_OK and _adapter(rows=0) == MSST_OK


def test_workspaces():
    from msst_b200 import MSST_ERR_INVALID, lib

    n = ctypes.c_longlong(-1)
    L = lib()
    assert L.msst_cross_attention_workspace(1, 1, 1 << 20, 8, 0, 64, ctypes.byref(n)) == MSST_ERR_INVALID
    assert L.msst_adapter_gemm_workspace(-1, 64, 64, 1, 16, ctypes.byref(n)) == MSST_ERR_INVALID


def test_python_argument_checks():
    import torch
    from msst_b200 import ops

    h = torch.zeros(1, 4, 2, 64, dtype=torch.float16)
    f = torch.zeros(4, 32)
    ids = torch.zeros(4, dtype=torch.int32)
    x, w = torch.zeros(4, 64, dtype=torch.float16), torch.zeros(32, 64, dtype=torch.float16)
    la, lb = torch.zeros(2, 8, 64, dtype=torch.float16), torch.zeros(2, 32, 8, dtype=torch.float16)
    for call in (
        lambda: ops.qk_norm_rope(h.float()),
        lambda: ops.qk_norm_rope(h[0]),
        lambda: ops.qk_norm_rope(h, h[:, :2]),
        lambda: ops.qk_norm_rope(h, q_gamma=torch.zeros(32)),
        lambda: ops.qk_norm_rope(h, cos=f),
        lambda: ops.qk_norm_rope(h, cos=f, sin=f, positions=torch.zeros(1, 4)),
        lambda: ops.qk_norm_rope(h, out_q=h[:, :2]),
        lambda: ops.cross_attention(h, h, h[:, :3]),
        lambda: ops.cross_attention(h, h.bfloat16(), h),
        lambda: ops.cross_attention(h, h, h, key_lens=torch.zeros(1, dtype=torch.int64)),
        lambda: ops.cross_attention(h, h, h, key_mask=torch.zeros(1, 5, dtype=torch.bool)),
        lambda: ops.cross_attention(h, h, h, out=h[:, :2]),
        lambda: ops.adapter_gemm(x, w[:, :32], la, lb, ids),
        lambda: ops.adapter_gemm(x, w, la, lb[:1], ids),
        lambda: ops.adapter_gemm(x, w.bfloat16(), la, lb, ids),
        lambda: ops.adapter_gemm(x, w, la, lb, ids[:3]),
        lambda: ops.adapter_gemm(x, w, la, lb, ids.long()),
        lambda: ops.adapter_gemm(x, w, la, lb, ids, scales=torch.zeros(3)),
        lambda: ops.adapter_gemm(x, w, la, lb, ids, out=x),
    ):
        with pytest.raises(ValueError):
            call()
