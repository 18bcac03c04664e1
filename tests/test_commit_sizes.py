"""A commit over pages without rows is refused: it would write no lengths. No GPU."""
from __future__ import annotations

import pytest
import torch

from test_speculative_refusals import _commit, as_hip  # noqa: F401 - a fixture
from winnow_amd import _lib
from winnow_amd import packed_attention as pa


@pytest.mark.parametrize("axis", [0, 1, 2, 3])
def test_pages_without_rows(as_hip, axis):  # noqa: F811
    shape = [3, 6, 2, 16]
    shape[axis] = 0
    pages, norms = torch.zeros(*shape, 32, dtype=torch.uint8), torch.zeros(*shape, dtype=torch.float16)
    with pytest.raises(pa.UnsupportedLayout, match="no rows"):
        _commit(k_pages=pages, v_pages=pages, k_norms=norms, v_norms=norms)


@pytest.mark.parametrize("B", [0, 1])
@pytest.mark.parametrize("layers", [0, -1])
def test_the_entry_point_needs_a_layer(B, layers):
    i = 1 << 20   # an aligned address that is never read
    with pytest.raises(_lib.WinnowHipError, match=f"layers={layers}"):
        _lib.call("wn_commit_kv", i, 0, 64, 64, 4, i, 0, 64, 64, 4, i, 0, 0, 0, i, 0, 0, 0, i, 0, i, i, 0, i, 2 * i, layers, B, 1, 16, 1, 4,
                  1, 1, None)
