"""The tree attention's scan of long contexts (head_dim 128, 4 and 6 bits, ``allow_tf32``) and which
layouts it is chosen for: K rows that can be read by 16 bytes (8 at 6 bits) and norms by fours. Any
other layout is right too, in the other scan. The tolerances of test_gpu_tree.py."""
from __future__ import annotations

import pytest
import torch

from cases import to_device
from test_gpu_tree import DEV, _case, _check, _pa, _wide_table

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bwk,bwv", [(4, 4), (4, 6), (6, 4), (6, 6)])
@pytest.mark.parametrize("Hq,Hkv,T", [(16, 4, 1), (16, 4, 8), (28, 4, 9), (4, 4, 64)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_long_contexts(bwk, bwv, Hq, Hkv, T, dtype):
    lens = (0, max(1, T // 2), T + 63, 700, 3001)
    q, kv, parents = _case(4100 + T + bwk * bwv, lens, Hq, Hkv, 128, T, bwk, bwv, dtype=dtype)
    d = _wide_table(to_device(kv, DEV), 2048)
    assert _pa().wide_rows(d)
    for splits in (None, 1, 13):
        got = _pa().packed_tree_attention(q.to(DEV), d, 0.09, parents.to(DEV), num_splits=splits, allow_tf32=True)
        _check(got, q, kv, parents, 0.09, dtype, single=True)
        assert torch.equal(got, _pa().packed_tree_attention(q.to(DEV), d, 0.09, parents.to(DEV), num_splits=splits, allow_tf32=True))


def _shifted(t, off, row_gap, head_gap):
    """A copy of t (P, Hkv, S, ...) whose base lies ``off`` elements behind an aligned one, with gaps of
    so many elements behind each head's block and each page."""
    P, Hkv = t.shape[:2]
    block = t[0, 0].numel()
    head = block + head_gap
    page = Hkv * head + row_gap
    flat = torch.zeros(P * page + off, dtype=t.dtype, device=t.device)
    inner = (t.shape[3], 1) if t.dim() == 4 else (1,)
    out = flat.as_strided(t.shape, (page, head, *inner), off)
    out.copy_(t)
    return out


@pytest.mark.parametrize("bwk,bwv", [(4, 4), (6, 4), (4, 6), (6, 6)])
@pytest.mark.parametrize("where", ["k base 4", "k base 8", "k head 4", "k page 12", "kn base 1", "vn base 2", "kn head 1", "vn head 3", "kn page 1",
                                   "vn page 2", "all"])
def test_long_contexts_in_other_layouts(bwk, bwv, where):
    q, kv, parents = _case(4200 + bwk * bwv, (0, 5, 200, 1003), 8, 4, 128, 9, bwk, bwv, dtype=torch.bfloat16)
    pa, d = _pa(), _wide_table(to_device(kv, DEV), 4096)
    want = pa.packed_tree_attention(q.to(DEV), d, 0.09, parents.to(DEV), allow_tf32=True)
    _check(want, q, kv, parents, 0.09, torch.bfloat16, single=True)
    if where == "all":
        d.k_pages, d.v_pages = _shifted(d.k_pages, 4, 12, 4), _shifted(d.v_pages, 4, 4, 8)
        d.k_norms, d.v_norms = _shifted(d.k_norms, 1, 1, 1), _shifted(d.v_norms, 3, 2, 1)
    else:
        side, kind, n = where.split()
        name = {"k": "k_pages", "kn": "k_norms", "vn": "v_norms"}[side]
        gap = {"base": (int(n), 0, 0), "page": (0, int(n), 0), "head": (0, 0, int(n))}[kind]
        setattr(d, name, _shifted(getattr(d, name), *gap))
    # eight-byte K rows are enough at 6 bits
    assert pa.wide_rows(d) == (where == "k base 8" and bwk == 6)
    got = pa.packed_tree_attention(q.to(DEV), d, 0.09, parents.to(DEV), allow_tf32=True)
    _check(got, q, kv, parents, 0.09, torch.bfloat16, single=True)


@pytest.mark.parametrize("bwk,bwv", [(4, 4), (6, 4)])
def test_long_contexts_captured_at_lengths_that_grow(bwk, bwv):
    pa, B, T = _pa(), 5, 9
    q, kv, parents = _case(4400 + bwk, (3000,) * B, 8, 2, 128, T, bwk, bwv, dtype=torch.bfloat16)
    d, dq, dp = _wide_table(to_device(kv, DEV), 16384), q.to(DEV), parents.to(DEV)
    d.seq_lens_host = torch.tensor((3000, 20, 20, 20, 20), dtype=torch.int32)
    d.seq_lens.copy_(d.seq_lens_host)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = pa.packed_tree_attention(dq, d, 0.08, dp, allow_tf32=True, check_ranges=False)
    for lens in ((3000, 20, 20, 20, 20), (2977, 0, 1, 2945, 65), (0,) * B, (3000,) * B, (10, 700, 0, 0, 129)):
        kv.seq_lens.copy_(torch.tensor(lens, dtype=kv.seq_lens.dtype))
        d.seq_lens_host = torch.tensor(lens, dtype=torch.int32)
        d.seq_lens.copy_(d.seq_lens_host)
        graph.replay()
        torch.cuda.synchronize()
        _check(out, q, kv, parents, 0.08, torch.bfloat16, single=True)
        _check(pa.packed_tree_attention(dq, d, 0.08, dp, allow_tf32=True), q, kv, parents, 0.08, torch.bfloat16, single=True)


def test_long_contexts_of_many_sequences_some_of_them_empty():
    lens = [0, 0, 5] + [(37 * i) % 90 if i % 3 else 0 for i in range(135)] + [400, 0]
    q, kv, parents = _case(4500, lens, 4, 2, 128, 3, 4, 4, dtype=torch.bfloat16)
    d = _wide_table(to_device(kv, DEV), 1024)
    for splits in (None, 5):
        got = _pa().packed_tree_attention(q.to(DEV), d, 0.08, parents.to(DEV), num_splits=splits, allow_tf32=True)
        _check(got, q, kv, parents, 0.08, torch.bfloat16, single=True)
