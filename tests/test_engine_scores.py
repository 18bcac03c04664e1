"""A score that cannot be had ends the request that asked for it, not the others of its batch. No
GPU: a model of canned logits on the host, whose scores the operator refuses."""
from __future__ import annotations

from types import SimpleNamespace

import pytest
import torch

from winnow_amd.engine import Engine, EngineConfig, Request
from winnow_amd.page_pool import PagePool


class _Model(torch.nn.Module):
    def __init__(self):
        super().__init__()
        self.w = torch.nn.Parameter(torch.zeros(1))

    def forward(self, input_ids, past_key_values, **kwargs):
        B, n = input_ids.shape
        past_key_values.lengths = [L + n for L in past_key_values.lengths]     # as after the last layer
        return SimpleNamespace(logits=torch.nn.functional.one_hot(input_ids[:, -1:] + 1, 32).float())


def _run(tops, fail_from=0, monkeypatch=None):
    from winnow_amd import engine as mod
    pool = PagePool(num_layers=1, num_pages=16, num_kv_heads=1, page_size=16, nb_k=64, nb_v=64)
    e = Engine(_Model(), pool, None, None, 128, config=EngineConfig())
    steps = []

    def scores(logits, tokens, top):
        steps.append(len(logits))
        if len(steps) > fail_from:
            raise RuntimeError("no scores")
        n = len(logits)
        return SimpleNamespace(logprob=torch.zeros(n), entropy=torch.zeros(n), top_ids=torch.zeros(n, max(top, 1), dtype=torch.int64),
                               top_logprobs=torch.zeros(n, max(top, 1)))
    monkeypatch.setattr(mod, "token_logprobs", scores)
    reqs = [e.submit(Request(f"r{i}", [3 * i + 1, 3 * i + 2], 5, top_logprobs=t)) for i, t in enumerate(tops)]
    e.run_until_idle(50)
    assert pool.stats()["owned"] == 0
    return reqs


@pytest.mark.parametrize("tops", [[None, 0, None], [2, None, None], [None, None, 3], [0, 1, 2]])
@pytest.mark.parametrize("fail_from", [3, 4, 5])
def test_a_failed_score_is_its_requests_alone(tops, fail_from, monkeypatch):
    """Failing in the prefill step's score or in a later batch's."""
    asked = sum(t is not None for t in tops)
    reqs = _run(tops, fail_from * asked // 3, monkeypatch)
    for i, r in enumerate(reqs):
        if r.top_logprobs is None:
            assert r.status == "length" and r.generated == [3 * i + 3 + k for k in range(5)]
        else:
            assert r.status == "error" and "no scores" in r.detail and len(r.logprobs) == len(r.generated) < 5


def test_the_operators_own_refusal(monkeypatch):
    """Host logits: the operator refuses them."""
    pool = PagePool(num_layers=1, num_pages=16, num_kv_heads=1, page_size=16, nb_k=64, nb_v=64)
    e = Engine(_Model(), pool, None, None, 128, config=EngineConfig())
    a, b = e.submit(Request("a", [1, 2], 3)), e.submit(Request("b", [5, 6], 3, top_logprobs=1))
    e.run_until_idle(50)
    assert a.status == "length" and a.generated == [3, 4, 5]
    assert b.status == "error" and b.generated == [] and "HIP device" in b.detail
