"""Host side of the conditioned-block operators at the edges of their ranges (no GPU)."""
from __future__ import annotations

import ctypes

import pytest


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
