"""A work-group of the tree attention that takes several units one after another: captured calls
whose lengths have grown, and fewer ``parts`` than there are. The tolerances of test_gpu_tree.py."""
from __future__ import annotations

import ctypes

import pytest
import torch

from test_gpu_tree import DEV, _case, _check, _pa
from cases import to_device

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("single", [False, True])
@pytest.mark.parametrize("D,bwk,bwv,Hq,Hkv,T", [
    (16, 4, 4, 8, 2, 9), (16, 4, 4, 8, 2, 16), (16, 3, 5, 12, 1, 17), (16, 8, 8, 4, 4, 30), (32, 4, 4, 8, 2, 9), (32, 5, 8, 12, 1, 17),
    (64, 4, 4, 8, 2, 9), (64, 8, 8, 12, 1, 17), (128, 4, 4, 8, 2, 9), (128, 4, 6, 12, 1, 17), (256, 4, 4, 8, 2, 9), (256, 6, 3, 12, 1, 17)])
def test_a_captured_call_whose_lengths_grow(D, bwk, bwv, Hq, Hkv, T, single):
    """Up to 32, 64 and more rows a kv head at every head_dim, captured with one long sequence (many
    splits to each) and four short ones (few in all): later lengths have five times as many units, and
    end 1 to 31 tokens into a chunk, so that a wave's half of it has no key for any row."""
    pa, B, scale = _pa(), 5, D ** -0.5
    q, kv, parents = _case(3300 + D + T, (3000,) * B, Hq, Hkv, D, T, bwk, bwv)
    d, dq, dp = to_device(kv, DEV), q.to(DEV), parents.to(DEV)
    d.seq_lens_host = torch.tensor((3000, 20, 20, 20, 20), dtype=torch.int32)
    d.seq_lens.copy_(d.seq_lens_host)
    splits, _, parts = pa.tree_plan_for(dq, d, not single)
    assert 5 * splits > 4 * parts
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = pa.packed_tree_attention(dq, d, scale, dp, allow_tf32=single, check_ranges=False)
    for lens in ((20,) * B, (2977, 0, 1, 2945, 65), (0,) * B, (3000,) * B, (65, 705, 0, 0, 129)):
        kv.seq_lens.copy_(torch.tensor(lens, dtype=kv.seq_lens.dtype))
        d.seq_lens_host = torch.tensor(lens, dtype=torch.int32)
        d.seq_lens.copy_(d.seq_lens_host)
        graph.replay()
        torch.cuda.synchronize()
        _check(out, q, kv, parents, scale, torch.float32, single)
        _check(pa.packed_tree_attention(dq, d, scale, dp, allow_tf32=single), q, kv, parents, scale, torch.float32, single)


@pytest.mark.parametrize("D", [16, 64, 128, 256])
@pytest.mark.parametrize("exact", [0, 1])
def test_one_part_for_the_whole_batch(D, exact, monkeypatch):
    """``parts`` = 1 and a short span through the C ABI: eight work-groups a row block take every unit."""
    from winnow_amd import _lib
    pa, call = _pa(), _lib.call
    q, kv, parents = _case(3400 + D, (700, 33, 0, 97, 1), 8, 2, D, 11, 4, 4)
    d, dq, dp = to_device(kv, DEV), q.to(DEV), parents.to(DEV)

    def one_part(name, *args):
        if name == "wn_tree_plan":
            assert call(name, *args) is None
            for p, v in zip(args[-3:], (11, 64, 1)):
                ctypes.cast(p, ctypes.POINTER(ctypes.c_int))[0] = v
            return None
        return call(name, *args)
    monkeypatch.setattr(_lib, "call", one_part)
    d.seq_lens_host = d.page_table_host = None
    got = pa.packed_tree_attention(dq, d, 0.1, dp, allow_tf32=not exact)
    _check(got, q, kv, parents, 0.1, torch.float32, single=not exact)
