"""The operators of a speculative step give values alone: where a derivative or a place in a trace is
asked of them they refuse, in place of leaving it out silently. No GPU: host tensors pass for HIP
ones, and a call into the library is recorded."""
from __future__ import annotations

import pytest
import torch
import torch.autograd.forward_ad as fwd
from torch.fx.experimental.proxy_tensor import make_fx
from torch.utils._python_dispatch import TorchDispatchMode

from test_speculative_refusals import _commit, _kv
from winnow_amd import _lib
from winnow_amd import packed_attention as pa
from winnow_amd.logprobs import token_logprobs


@pytest.fixture
def calls(monkeypatch):
    seen = []
    monkeypatch.setattr(_lib, "is_hip", lambda t: True)
    monkeypatch.setattr(_lib, "on", lambda device: _lib._here)
    monkeypatch.setattr(_lib, "stream_of", lambda device: 0)
    monkeypatch.setattr(_lib, "call", lambda name, *args: seen.append(name))
    return seen


PARENTS = torch.full((2, 5), -1, dtype=torch.int32)


def _tree(q):
    return pa.packed_tree_attention(q, _kv(), 0.1, PARENTS, num_splits=1)


def _rows(x):
    return token_logprobs(x).entropy


def _pages(k):
    return _commit(k_pages=k, v_pages=torch.zeros_like(k), k_norms=None, v_norms=None)


CASES = [(_tree, (2, 4, 5, 64), "wn_tree_attention"), (_rows, (3, 10), "wn_token_logprobs"), (_pages, (3, 6, 2, 16, 32), "wn_commit_kv")]


@pytest.mark.parametrize("f,shape,name", CASES)
def test_a_tangent(calls, f, shape, name):
    with fwd.dual_level():
        x = fwd.make_dual(torch.randn(shape), torch.randn(shape))
        with pytest.raises(pa.UnsupportedLayout, match="forward-mode"):
            f(x)
        assert calls == []
        f(fwd.unpack_dual(x).primal.detach())
    assert calls[-1] == name


@pytest.mark.parametrize("f,shape,name", CASES)
def test_a_gradient(calls, f, shape, name):
    x = torch.randn(shape, requires_grad=True)
    with pytest.raises(pa.UnsupportedLayout, match="no gradient"):
        f(x)
    assert calls == []
    with torch.no_grad():
        f(x)
    f(x.detach())
    assert [c for c in calls if c == name] == [name, name]


@pytest.mark.parametrize("f,shape,name", CASES)
def test_a_trace(calls, f, shape, name):
    x = torch.randn(shape)
    for trace in (lambda: torch.jit.trace(f, (x,), check_trace=False), lambda: make_fx(f)(x), lambda: make_fx(f, pre_dispatch=True)(x)):
        with pytest.raises(pa.UnsupportedLayout, match="traced"):
            trace()
    assert calls == []


class _Watch(TorchDispatchMode):
    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        return func(*args, **(kwargs or {}))


@pytest.mark.parametrize("f,shape,name", CASES)
def test_what_only_watches_or_casts_stays_served(calls, f, shape, name):
    x = torch.randn(shape)
    with _Watch():
        f(x)
    with torch.inference_mode():
        f(x)
    with torch.autocast("cpu", dtype=torch.bfloat16):
        f(x)
    f(torch.nn.Parameter(x, requires_grad=False))
    assert [c for c in calls if c == name] == [name] * 4
