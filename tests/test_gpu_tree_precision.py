"""What ``allow_tf32`` chooses in the tree attention: without it a bf16 call has fp32 accuracy too,
so its result is the fp32 one rounded once. The tolerances of test_gpu_tree.py."""
from __future__ import annotations

import pytest
import torch

import tree_reference as ref
from test_gpu_tree import DEV, _case, _check, _pa, _wide_table
from cases import to_device

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("columns", [0, 2048])
@pytest.mark.parametrize("Hq,Hkv,D,T,bwk,bwv", [(32, 8, 128, 8, 4, 4), (28, 4, 128, 26, 4, 6), (16, 4, 128, 8, 6, 6), (14, 2, 64, 5, 8, 8),
                                                (8, 2, 256, 6, 4, 4), (8, 2, 16, 30, 4, 4)])
def test_bf16_is_the_fp32_result_rounded_once(Hq, Hkv, D, T, bwk, bwv, columns):
    """Also behind a table with room for long contexts. A result r within tol of the definition's
    w rounds into [bf16(w - tol), bf16(w + tol)]: rounding is monotone."""
    pa, scale = _pa(), D ** -0.5
    q, kv, parents = _case(3100 + D + T, (T, 130, 515, 2000), Hq, Hkv, D, T, bwk, bwv, dtype=torch.bfloat16)
    d = to_device(kv, DEV)
    if columns:
        d = _wide_table(d, columns)
    args = q.to(DEV), d, scale, parents.to(DEV)
    got, wide = pa.packed_tree_attention(*args), pa.packed_tree_attention(*args, out_dtype=torch.float32)
    assert got.dtype == torch.bfloat16 and torch.equal(got, wide.to(torch.bfloat16))
    _check(wide, q, kv, parents, scale, torch.float32)
    want = ref.tree_attention(q, kv, parents, scale)
    K, V, E = ref.bounds(q, kv, scale)
    tol = (2 * E * K + V) * 2.0 ** -19
    assert (got.cpu() >= (want - tol).to(torch.bfloat16)).all() and (got.cpu() <= (want + tol).to(torch.bfloat16)).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_single_terms_are_asked_for(dtype):
    """``allow_tf32`` takes the same products for every type of query."""
    pa = _pa()
    q, kv, parents = _case(3200, (9, 130, 515), 28, 4, 128, 9, 4, 4, dtype=torch.bfloat16)
    d = to_device(kv, DEV)
    got = pa.packed_tree_attention(q.to(dtype).to(DEV), d, 0.09, parents.to(DEV), allow_tf32=True, out_dtype=torch.float32)
    _check(got, q, kv, parents, 0.09, torch.float32, single=True)
    one = pa.packed_tree_attention(q.to(DEV), d, 0.09, parents.to(DEV), allow_tf32=True)
    assert torch.equal(one, got.to(torch.bfloat16))
