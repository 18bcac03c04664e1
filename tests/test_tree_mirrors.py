"""Host mirrors of a tree attention call that are not the operand's shape. No GPU."""
from __future__ import annotations

import pytest
import torch

from test_speculative_refusals import _tree, as_hip  # noqa: F401 - a fixture
from winnow_amd import packed_attention as pa


@pytest.mark.parametrize("shape", [(5,), (10,), (1, 5), (2, 4), (3, 5), (2, 5, 1), ()])
@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
def test_parents_host_of_another_shape(as_hip, shape, dtype):  # noqa: F811
    with pytest.raises(pa.UnsupportedLayout, match="parents_host is"):
        _tree(parents_host=torch.full(shape, -1, dtype=dtype))
