"""Norms that are not finite in the tree attention: on drafted tokens and behind a sequence's end."""
from __future__ import annotations

import pytest
import torch

from cases import to_device
from test_gpu_tree import DEV, _case, _pa, _wide_table

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("single", [False, True])
@pytest.mark.parametrize("D,bwk,bwv,columns", [(128, 4, 4, 0), (128, 4, 6, 2048), (128, 4, 4, 4096), (16, 4, 4, 0), (64, 8, 3, 0), (256, 4, 4, 0)])
def test_a_norm_that_is_not_finite_reaches_every_row_that_sees_it(D, bwk, bwv, columns, single):
    """Each head of each sequence: node 6 is seen by 6, 7 and 10, whose rows have no finite element
    (weight times an infinite value); the others' are those of finite norms."""
    lens = (21, 90, 200, 40)
    q, kv, parents = _case(4300 + D, lens, 8, 4, D, 12, bwk, bwv)
    parents[:] = torch.tensor([-1, 0, 0, 1, 2, 2, -1, 6, 4, 3, 7, 5], dtype=torch.int32)
    pa = _pa()

    def run():
        d = to_device(kv, DEV)
        return pa.packed_tree_attention(q.to(DEV), _wide_table(d, columns) if columns else d, 0.08, parents.to(DEV), allow_tf32=single)
    clean = run()
    for b, L in enumerate(lens):
        for side in ("k", "v"):
            norms = getattr(kv, f"{side}_norms")
            norms[int(kv.page_table[b, (L - 1) // 16]), :, (L - 1) % 16 + 1:] = float("nan")
            node = L - 12 + 6
            norms[int(kv.page_table[b, node // 16]), :, node % 16] = float("inf")
    got = run()
    rest = [i for i in range(12) if i not in (6, 7, 10)]
    assert torch.equal(got[:, :, rest], clean[:, :, rest])
    assert not torch.isfinite(got[:, :, [6, 7, 10]]).any()
