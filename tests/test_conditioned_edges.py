"""Host side of the conditioned-block operators at the edges of their ranges (no GPU)."""
from __future__ import annotations

import ctypes
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "cuda-msst-infer_b200", "csrc")


def _run_on_host(tmp_path, program):
    """Compiles `program` against the kernels' headers and runs its host code."""
    nvcc = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not os.path.exists(nvcc):
        pytest.skip("nvcc not available")
    src, exe = tmp_path / "check.cu", tmp_path / "check"
    src.write_text(program)
    subprocess.run([nvcc, "-std=c++17", "-O1", "-gencode", "arch=compute_100a,code=sm_100a", "-I", CSRC, "-I",
                    os.path.join(ROOT, "include"), str(src), "-o", str(exe)], check=True, capture_output=True, timeout=300)
    out = subprocess.run([str(exe)], check=False, capture_output=True, text=True, timeout=300)
    assert out.returncode == 0, out.stdout + out.stderr


@pytest.mark.parametrize("q_heads, kv_heads, head_dim", [(2, 4, 64), (3, 2, 64), (1, 1 << 30, 8), (4, 4, 136), (4, 4, 12)])
def test_cross_attention_workspace_refuses_heads(q_heads, kv_heads, head_dim):
    """The sizes divide by q_heads / kv_heads: heads that the attention refuses are refused here too."""
    from msst_b200 import MSST_ERR_INVALID, lib

    n = ctypes.c_longlong(-1)
    assert lib().msst_cross_attention_workspace(1, 1, 64, q_heads, kv_heads, head_dim, ctypes.byref(n)) == MSST_ERR_INVALID
    assert n.value == -1


@pytest.mark.parametrize("Hq, Hk", [(2, 4), (3, 2), (2, 0), (0, 2)])
def test_cross_attention_refuses_heads_in_python(Hq, Hk):
    """Before anything is asked of the library."""
    import torch
    from msst_b200 import ops

    q = torch.zeros(1, 4, Hq, 64, dtype=torch.float16)
    k = torch.zeros(1, 5, Hk, 64, dtype=torch.float16)
    with pytest.raises(ValueError, match="heads"):
        ops.cross_attention(q, k, k)


def test_qk_norm_items_past_32_bits_of_threads(tmp_path):
    """The item of every thread against the same division in 64 bits, up to 2^31 items (the most head
    vectors that a call may have), where the threads' own numbers reach 2^36."""
    _run_on_host(tmp_path, r"""
#include <cstdio>
#include "operators.cuh"
int main() {
  for (unsigned lpv = 1; lpv <= 32; lpv *= 2) {
    const unsigned long long last = ((1ull << 31) * lpv + 127) / 128;  // blocks of the largest call
    for (unsigned long long b = 0; b < last; b = b < 1000 || b + 5 > last ? b + 1 : (b * 3 / 2 < last - 4 ? b * 3 / 2 : last - 4))
      for (unsigned t = 0; t < 128; ++t)
        if (msst::qk_norm_item((unsigned)b, t, lpv) != (b * 128 + t) / lpv) {
          std::printf("lpv %u block %llu thread %u\n", lpv, b, t);
          return 1;
        }
  }
}
""")


def test_device_errors_do_not_hide_one_another(tmp_path):
    """Every pair of codes, recorded in one translation unit or in two: a wait that gave up is reported
    as itself and before data errors, each data error as itself, and none is lost."""
    _run_on_host(tmp_path, r"""
#include <cstdio>
#include "device_errors.h"
using namespace msst;
static void record(DeviceErrors& e, unsigned code) {  // as the kernels' record_error
  if (code >= kFirstDataError) e.data |= 1u << (code - kFirstDataError);
  else if (!e.wait) e.wait = code;
}
int main() {
  static_assert(kErrPosition == 14 && kErrAdapter == 15 && kErrTimeoutFfnFlag == 13, "documented codes");
  for (unsigned a = 0; a <= 15; ++a)
    for (unsigned b = 0; b <= 15; ++b)
      for (int second = 0; second < 2; ++second) {
        DeviceErrors e[3] = {};
        if (a) record(e[0], a);
        if (b) record(e[second], b);
        unsigned want[3], n = 0;
        const bool wa = a && a < 14, wb = b && b < 14;
        if (wa || wb) want[n++] = wa ? a : b;
        for (unsigned k = 14; k <= 15; ++k)
          if (a == k || b == k) want[n++] = k;
        for (unsigned i = 0; i <= n; ++i) {
          const unsigned got = take_error(e, 3);
          if (got != (i < n ? want[i] : 0)) {
            std::printf("%u %u %d: %u\n", a, b, second, got);
            return 1;
          }
        }
      }
}
""")


def _source(name):
    with open(os.path.join(CSRC, name)) as f:
        return f.read()


@pytest.mark.parametrize("name, begin, end", [
    ("cross_attn.cu", "softmax + epilogue", "// Joins the partial results"),
    ("cross_attn.cu", "rows that are not kept", "softmax + epilogue"),
    ("cross_token.cu", "const int set = warp >> 2", "cudaError_t launch_k"),
    ("adapter_gemm.cu", "// ------------------------------------------------------------ epilogue", "if (split > 1) {"),
])
def test_whole_warp_roles_wait_together(name, begin, end):
    """Where a wait gives up, lanes must not part: one that left its loop never reaches the others'
    full-mask instructions, and a kernel that should return with its code hangs.  Such a wait cannot be
    made to run out from outside, so the sources are read: these roles wait by the warp."""
    text = _source(name)
    assert text.count(begin) == 1
    role = text[text.index(begin):]
    role = role[:role.index(end)]
    assert "mbar_wait_warp" in role and "mbar_wait<" not in role and "mbar_wait(" not in role


def test_roles_end_after_their_own_copies():
    """Every producer waits for its ring, every MMA issuer for its last commit, and the token kernel's
    warps leave their common barrier by one reading of the flag."""
    for name, rings in (("cross_attn.cu", 2), ("cross_token.cu", 1), ("adapter_gemm.cu", 1)):
        text = _source(name)
        assert text.count("mbar_drain_ring(") == rings
        if "umma_commit" in text:
            assert text.count("umma_commit(mma_end)") == text.count("mbar_drain(mma_end, 0)") == 1
    token = _source("cross_token.cu")
    assert token.count("= *abort_flag") == 1 and "ok = s_stop == 0" in token


def test_drain_of_a_ring():
    """mbar_drain_ring's parities against a ring walked use by use (a barrier's phase parity flips with
    each completed use; a wait for parity p returns where the current phase has the other one)."""
    for n in (1, 2, 3, 5, 9):
        uses, slot, phase = [0] * n, 0, 0
        for _ in range(4 * n + 3):
            for i in range(n):
                p = phase if i < slot else phase ^ 1
                # the last use counts as in flight: its phase is current and incomplete
                current = (uses[i] - 1) % 2 if uses[i] else 0
                assert (current == p) == (uses[i] > 0), (n, i, uses)
            uses[slot] += 1
            slot += 1
            if slot == n:
                slot, phase = 0, phase ^ 1


@pytest.mark.parametrize("out", [dict(sb=0), dict(sn=0), dict(sh=0)])
@pytest.mark.parametrize("op", ["q_out", "k_out", "cross"])
def test_outputs_that_share_places_are_refused(op, out):
    """An expanded output (stride 0 along an extent above 1) would be written by several threads, and
    normed several times where it is the input too."""
    from msst_b200 import MSST_ERR_INVALID, lib
    from test_conditioned_ops import _cross, _heads, _qk

    shape = dict(batch=2)
    if op == "cross":
        rc = _cross(out=_heads(**out), **shape)
    elif op == "q_out":
        rc = _qk(qo=_heads(**out), **shape)
    else:
        rc = _qk(k=_heads(), ko=_heads(**out), **shape)
    assert rc == MSST_ERR_INVALID and "strides above 0" in lib().msst_last_error().decode()
    # strides that nothing walks may be 0
    assert _qk(q=_heads(heads=1, sb=0, sn=0, sh=0), qo=_heads(heads=1, sb=0, sn=0, sh=0), batch=1, seq=1) != MSST_ERR_INVALID \
        or "strides above 0" not in lib().msst_last_error().decode()


def test_lengths_within_a_tile_of_32_bits_are_refused():
    """Rounded up to a tile they would pass 2^31 - 1 and come out negative: no tile, a result that is not
    written or not finished."""
    from msst_b200 import MSST_ERR_INVALID, lib
    from test_conditioned_ops import _adapter, _cross, _heads

    n, most = ctypes.c_longlong(-1), (1 << 31) - 1
    one = dict(q=_heads(heads=1), k=_heads(heads=1), v=_heads(heads=1), out=_heads(heads=1))
    for call, word in ((lambda: _cross(nq=most, **one), "too many"), (lambda: _cross(nk=most, **one), "too many"),
                       (lambda: _adapter(rows=most), "rows"), (lambda: _adapter(N=most - 7, ldo=most - 7), "N is too large"),
                       (lambda: _adapter(K=most - 7, ldx=most - 7), "N is too large")):
        assert call() == MSST_ERR_INVALID and word in lib().msst_last_error().decode()
    for nq, nk in ((most, 8), (8, most)):
        assert lib().msst_cross_attention_workspace(1, nq, nk, 1, 1, 8, ctypes.byref(n)) == MSST_ERR_INVALID
    for rows, K, N in ((most, 8, 8), (8, most - 7, 8), (8, 8, most - 7)):
        assert lib().msst_adapter_gemm_workspace(rows, K, N, 1, 8, ctypes.byref(n)) == MSST_ERR_INVALID


def test_workspace_is_asked_for_on_the_operands_device(monkeypatch):
    """With another GPU current, and once for each device and size."""
    import contextlib

    import msst_b200 as M
    import torch

    current, asked = [0], []

    @contextlib.contextmanager
    def device(d):
        before, current[0] = current[0], d
        yield
        current[0] = before

    class Lib:
        @staticmethod
        def msst_cross_attention_workspace(*args):
            asked.append(current[0])
            args[-1]._obj.value = 100 + 48 * current[0]
            return M.MSST_OK

    monkeypatch.setattr(M, "lib", lambda: Lib)
    monkeypatch.setattr(M, "_space", {})
    monkeypatch.setattr(torch.cuda, "device", device)
    sizes = (1, 2, 3, 4, 4, 64)
    assert [M._workspace("cross_attention", d, *sizes) for d in (1, 0, 1, 0)] == [148, 100, 148, 100]
    assert asked == [1, 0] and current == [0]
