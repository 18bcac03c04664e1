"""Calls whose grid would reach HIP's 2^32 threads are refused before any launch. No GPU: the sizes alone
count, and no operand is touched."""
from __future__ import annotations

import pytest

from winnow_amd import _lib

P = 1 << 20      # an address that is never read, aligned for anything


def test_logits():
    def call(N, V):
        _lib.call("wn_adjust_logits", P, 0, V, P, V, N, V, None, 0, 0, None, None, None, None, None, 1.0, 0.0, 0.0, None, 0, None, 0, 0, None, 0, None)
    for N, V in ((2 ** 23, 70), (2 ** 30, 1), (2 ** 22, 100000)):
        with pytest.raises(_lib.WinnowHipError, match="grid too large"):
            call(N, V)


@pytest.mark.parametrize("B,Hq,Hkv,Q,D", [(2 ** 21, 8, 8, 1, 64), (64, 32, 8, 2 ** 18, 64), (2 ** 13, 8, 8, 5000, 32)])
def test_windowed_attention(B, Hq, Hkv, Q, D):
    with pytest.raises(_lib.WinnowHipError, match="grid too large"):
        _lib.call("wn_window_attention", P, 0, 0, 0, 0, P, P, P, P, P, 0, 0, P, 0, 0, P, 0, 0, P, 0, 0, P, 0, P, P, 0, P, 2 ** 62, B, Hq, Hkv, Q, D, 16, 4, 4, 1, 4,
                  8, 0, 0.1, 1, 1, 64, None, None, None)


@pytest.mark.parametrize("D,n", [(16, 2 ** 28), (256, 2 ** 27)])
def test_appends(D, n):
    """Of head_dims that the many-vector kernel, whose grid is the device's, does not take."""
    side = (P, P, 4)
    rows = (P, 0, 0, D)
    store = (P, 0, 0) * 4
    with pytest.raises(_lib.WinnowHipError, match="grid would be too large"):
        _lib.call("wn_append_kv", *rows, *rows, 0, *side, *side, P, 0, P, *store, 1, 1, n, D, 16, 4, 4, None, None, None)
    with pytest.raises(_lib.WinnowHipError, match="grid would be too large"):
        _lib.call("wn_append_rotated_kv", None, 0, 0, 0, 0, 0, None, P, 0, D, P, 0, D, 0, D, *rows, *rows, 0, *side, *side, P, 0, P, *store, 1, 1, n, D, 16, 4, 4,
                  None, None, None)
