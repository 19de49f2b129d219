"""What the header promises of the paged-cache operators where no GPU is needed to see it."""
from __future__ import annotations

import struct

import pytest

from test_cache_ops import _attention, _heads


@pytest.mark.parametrize("words", [False, True])
def test_rows_without_a_request_are_not_skipped(words):
    """With zero_rest they are written, so that a call with operands that are no GPU's fails; without, and
    without a row, nothing is done."""
    from msst_b200 import MSST_OK, lib

    def call(tokens, rest):
        if not words:
            return _attention(requests=0, tokens=tokens, rest=rest)
        heads = [16, 2, 2048, 128, 64]
        return lib().msst_call(2, struct.pack("36qd10q", *heads, tokens, 16, 0, *heads, *heads, 8, *heads, *heads, 4, 16, 16,
                                              2, 2, 16, 64, 0.0, 0, *heads, rest, 0, 0, 0))

    assert _heads() == struct.pack("Pi4xqqq", 16, 2, 2048, 128, 64)
    assert call(4, 0) == MSST_OK and call(0, 1) == MSST_OK
    assert call(4, 1) != MSST_OK
