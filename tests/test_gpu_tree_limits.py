"""The tree attention at the longest sequences and the largest spans it takes, where a sum of two
positions no longer fits 32 bits."""
from __future__ import annotations

import ctypes

import pytest
import torch

import tree_reference as ref
from cases import to_device
from test_gpu_tree import DEV, _case, _check, _pa

pytestmark = pytest.mark.gpu


def _uniform(D, S, width, T, seed):
    """A sequence that fills a table of ``width`` pages of S positions with two pages, the first in its
    first half. K norms are 0, so every visible position has the same weight; values are -1, 0 or 1 times
    2^-8 with norm 1. (q, handle on the device, parents, result in float64)

    Every sum of a split is then a whole number times a power of two, below 2^24 of them (a split has at
    most 2^23 positions), and exact in 32 bits; what is left are the merge's sums over at most 256
    splits, the division and the rotation, (8 + 1 + D / 16 + 5) roundings in a row at most: 2^-19 of |v|."""
    pa = _pa()
    g = torch.Generator().manual_seed(seed)
    quant = pa.Quantizer(torch.linalg.qr(torch.randn(D, D, generator=g))[0].contiguous(),
                         torch.tensor([0., 1., -1.] + [0.] * 13) / 256, 4)
    codes = torch.randint(0, 3, (2, 1, S, D), generator=g)
    pages = (codes[..., ::2] | codes[..., 1::2] << 4).to(torch.uint8)
    norms = torch.ones(2, 1, S, dtype=torch.float16)
    table = torch.zeros(1, width, dtype=torch.int32)
    table[:, width // 2:] = 1
    L = S * width
    lens = torch.tensor([L], dtype=torch.int32)
    parents = ref.random_parents(1, T, seed + 1)
    c = quant.centroids.double()[codes[:, 0]]                                        # (2, S, D)
    before = c[0].sum(0) * (width // 2) + c[1].sum(0) * (width - width // 2) - c[1, S - T:].sum(0)
    anc = ref.ancestors(parents[0], T).double()
    want = (before + anc @ c[1, S - T:]) / (L - T + anc.sum(-1, keepdim=True)) @ quant.Pi.double()
    q = torch.randn(1, 2, T, D, generator=g)
    dq = pa.Quantizer(quant.Pi.to(DEV), quant.centroids.to(DEV), 4)
    kv = pa.PackedKV(pages.to(DEV), torch.zeros_like(norms).to(DEV), pages.to(DEV), norms.to(DEV), table.to(DEV), lens.to(DEV),
                     dq, dq, D, seq_lens_host=lens, page_table_host=table)
    return q.to(DEV), kv, parents, want, float(c.norm(dim=-1).max())


@pytest.mark.parametrize("D,single", [(16, False), (16, True), (128, False), (128, True), (256, False)])
def test_the_longest_sequence(D, single):
    """2^31 - 512 positions in 256-token pages: the last of the planned splits would end at 2^31."""
    pa = _pa()
    q, kv, parents, want, V = _uniform(D, 256, (2 ** 31 - 257) // 256, 3, 40 + D)
    assert int(kv.seq_lens_host[0]) == 2 ** 31 - 512
    splits, span, _ = pa.tree_plan_for(q, kv, not single)
    assert splits * span >= 2 ** 31
    got = pa.packed_tree_attention(q, kv, 0.1, parents.to(DEV), allow_tf32=single)
    assert ((got[0].double().cpu() - want).abs() <= V * 2.0 ** -19).all()


@pytest.mark.parametrize("plan", [(1, 2 ** 31 - 64, 5), (3, 2 ** 31 - 64, 1), (2, 2 ** 30, 5), (4096, 64, 5)])
@pytest.mark.parametrize("D,single", [(64, False), (128, True)])
def test_any_span_and_number_of_splits(D, single, plan, monkeypatch):
    """Through the C ABI: spans that added to a length pass 2^31, fewer parts than there are."""
    from winnow_amd import _lib
    pa, call = _pa(), _lib.call
    q, kv, parents = _case(3500 + D, (300, 33, 0, 97, 1), 8, 2, D, 11, 4, 4)

    def planned(name, *args):
        if name == "wn_tree_plan":
            for p, v in zip(args[-3:], plan):
                ctypes.cast(p, ctypes.POINTER(ctypes.c_int))[0] = v
            return None
        return call(name, *args)
    monkeypatch.setattr(_lib, "call", planned)
    d = to_device(kv, DEV)
    d.seq_lens_host = d.page_table_host = None
    got = pa.packed_tree_attention(q.to(DEV), d, 0.1, parents.to(DEV), allow_tf32=single)
    _check(got, q, kv, parents, 0.1, torch.float32, single)
