"""Engines and caches that share a model: what one of them fuses is not fused for another."""
from __future__ import annotations

import pytest

from test_gpu_conversation import _engine, _generate, _prompts, model  # noqa: F401 - a fixture

pytestmark = pytest.mark.gpu


def _serve(e, prompts):
    from winnow_amd.engine import Request
    reqs = [e.submit(Request(f"r{i}", p, 8)) for i, p in enumerate(prompts)]
    e.run_until_idle()
    assert all(r.status == "length" for r in reqs)
    return [r.generated for r in reqs]


def test_engines_of_one_model(model, monkeypatch):  # noqa: F811
    from winnow_amd import packed_backend as pb
    calls, inner = [], pb.PagedPackedCache.update_rotated
    monkeypatch.setattr(pb.PagedPackedCache, "update_rotated", lambda self, *a: (calls.append(1), inner(self, *a))[1])
    prompts = _prompts(3)
    alone = _serve(_engine(model, prefill_chunk=40), prompts)
    _, logits, _ = _generate(model, prompts, 3)
    assert not calls                                        # nothing fused yet
    fused, plain, either = _engine(model, fuse_rotary=True, prefill_chunk=40), _engine(model, fuse_rotary=False, prefill_chunk=40), _engine(
        model, prefill_chunk=40)
    first = _serve(fused, prompts)
    assert len(calls) > 0
    n = len(calls)
    assert _serve(plain, prompts) == alone and _serve(either, prompts) == alone and len(calls) == n
    _, again, _ = _generate(model, prompts, 3)
    assert (again == logits).all() and len(calls) == n
    assert _serve(fused, prompts) == first and len(calls) == 2 * n
    assert pb.fuse_rotary(model) == 2                       # the caller's own choice, for who has none
    assert _serve(either, prompts) == first and len(calls) == 3 * n
    assert _serve(plain, prompts) == alone and len(calls) == 3 * n
    assert pb.fuse_rotary(model, False) == 2
    assert _serve(either, prompts) == alone and len(calls) == 3 * n
