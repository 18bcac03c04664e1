"""``PagedPackedCache.commit`` writes only pages that its sequences still hold. No GPU: the commit's
launch is recorded in place of being made."""
from __future__ import annotations

import pytest
import torch

from winnow_amd import packed_backend as pb
from winnow_amd.page_pool import PagePool, StalePage
from winnow_amd.quantizer import TurboQuantMSE

TREE = [-1, 0, 0, 2]


@pytest.fixture
def calls(monkeypatch):
    seen = []
    monkeypatch.setattr(pb, "commit_kv", lambda *a, **k: seen.append(a))
    return seen


def _forward(owners, lengths, num_pages=8, dense=None):
    tq = TurboQuantMSE(4, 64, "cpu", 1)
    pool = PagePool(num_layers=2, num_pages=num_pages, num_kv_heads=1, page_size=16, nb_k=32, nb_v=32, dense_dtype=dense)
    for o, n in zip(owners, lengths):
        pool.ensure(o, n + len(TREE))
    cache = pb.PagedPackedCache(pool, owners, lengths, k_quant=tq, v_quant=tq, head_dim=64, tree=TREE)
    cache.lengths = cache.begin(len(TREE), "cpu").seq_host.tolist()         # as after the last layer
    return pool, cache


@pytest.mark.parametrize("dense", [None, torch.bfloat16])
def test_a_released_lease_is_not_written(calls, dense):
    pool, cache = _forward(["a"], [30], 4, dense)
    pool.release("a")
    with pytest.raises(StalePage):
        cache.commit([[0, 2]])
    pool.ensure("b", 40)                                                   # the same pages, another's
    with pytest.raises(StalePage):
        cache.commit([[0, 2]])
    pool.release("b")
    pool.ensure("a", 40)                                                   # its own name, another lease
    with pytest.raises(StalePage):
        cache.commit([[0]])
    assert calls == [] and cache.lengths == [34]                           # the cache is as it was


def test_one_released_sequence_of_a_batch(calls):
    pool, cache = _forward(["a", "b", "c"], [30, 5, 12])
    pool.release("b")
    with pytest.raises(StalePage):
        cache.commit([[0], [0], [0, 2]])
    assert calls == []
    assert cache.commit([[0], [], [0, 2, 3]]) == [31, 5, 15]               # nothing of b is moved
    assert len(calls) == 1


def test_a_lease_that_grew_is_the_same_lease(calls):
    pool, cache = _forward(["a", "b"], [30, 1])
    pool.ensure("a", 70)
    assert cache.commit([[0, 2], [0]]) == [32, 2]
    assert len(calls) == 1
