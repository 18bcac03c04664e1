"""What a request asks of its next token, in the engine. No GPU: a model of canned logits on the
host, and the operator's place taken by its definition in float64."""
from __future__ import annotations

import math
from types import SimpleNamespace

import pytest
import torch

from winnow_amd.engine import Engine, EngineConfig, Refused, Request
from winnow_amd.logits import pack_allowed
from winnow_amd.page_pool import PagePool

V = 70


class _Model(torch.nn.Module):
    """Logits that fall from the token after the last one on, around the vocabulary."""

    def __init__(self):
        super().__init__()
        self.w = torch.nn.Parameter(torch.zeros(1))

    def forward(self, input_ids, past_key_values, **kwargs):
        B, n = input_ids.shape
        past_key_values.lengths = [L + n for L in past_key_values.lengths]     # as after the last layer
        d = (torch.arange(V)[None] - input_ids[:, -1:] - 1) % V
        return SimpleNamespace(logits=(3.0 - d.float())[:, None])


def defined(x, hist, made, r, p, f, bias, ok):
    y = x.double().clone()
    for t in set(hist):
        y[t] = y[t] / r if y[t] > 0 else y[t] * r
    for t in set(hist[made:]):
        y[t] -= f * hist[made:].count(t) + p
    for t, b in bias.items():
        if 0 <= t < len(y):
            y[t] += b
    return torch.where(ok, y, -math.inf)


def adjust(logits, *, history=None, lengths=None, prompt_lengths=None, repetition=1.0, presence=0.0, frequency=0.0, bias_ids=None, bias=None,
           allowed=None):
    """``adjust_logits`` on the host."""
    out = []
    for i, x in enumerate(logits):
        hist = [] if history is None else history[i, :int(lengths[i])].tolist()
        each = [float(t[i]) if isinstance(t, torch.Tensor) else t for t in (repetition, presence, frequency)]
        ids = {} if bias is None else dict(zip(bias_ids[i].tolist(), bias[i].tolist()))
        v = torch.arange(V)
        ok = torch.ones(V, dtype=torch.bool) if allowed is None else ((allowed[i].long()[v // 32] >> (v % 32)) & 1) > 0
        out.append(defined(x, hist, 0 if history is None else int(prompt_lengths[i]), *each, ids, ok))
    return torch.stack(out)


def _engine(monkeypatch, op=adjust, **cfg):
    from winnow_amd import engine as mod
    if op is not None:
        monkeypatch.setattr(mod, "adjust_logits", op)
    pool = PagePool(num_layers=1, num_pages=64, num_kv_heads=1, page_size=16, nb_k=64, nb_v=64)
    return Engine(_Model(), pool, None, None, 128, config=EngineConfig(**cfg))


def _expected(r, n):
    """The tokens that the definition gives, one by one."""
    made = []
    while len(made) < n:
        hist = r.prompt_ids + made
        x = 3.0 - ((torch.arange(V) - hist[-1] - 1) % V).float()
        probe = SimpleNamespace(prompt_ids=r.prompt_ids, generated=made)
        ok = torch.ones(V, dtype=torch.bool) if r.allowed_tokens is None else r.allowed_tokens(probe)
        made.append(int(defined(x, hist, len(r.prompt_ids), r.repetition_penalty, r.presence_penalty, r.frequency_penalty, r.logit_bias, ok).argmax()))
    return made


def _requests(n):
    some = torch.zeros(V, dtype=torch.bool)
    some[::3] = True
    return [Request("plain", [4, 5], n), Request("rep", [9, 10, 11, 12, 10], n, repetition_penalty=1.7),
            Request("freq", [1, 2, 3], n, presence_penalty=0.5, frequency_penalty=2.5), Request("bias", [30], n, logit_bias={33: 2.5, 34: 1.0, V + 9: 50.0}),
            Request("mask", [6] * 20, n, allowed_tokens=lambda r: some),
            Request("all", [68, 69, 0, 1], n, repetition_penalty=1.3, presence_penalty=1.5, frequency_penalty=0.25, logit_bias={2: -5.0, 7: 4.0},
                    allowed_tokens=lambda r: ~some if len(r.generated) % 2 else some)]


@pytest.mark.parametrize("batch", [1, 3, 8])
@pytest.mark.parametrize("chunk", [2, 64])
def test_tokens_follow_the_definition(monkeypatch, batch, chunk):
    """Alone and in batches, whole and partial ones, slots that change hands, prompts in chunks."""
    e = _engine(monkeypatch, max_batch=batch, prefill_chunk=chunk)
    reqs = [e.submit(r) for r in _requests(9)]
    e.run_until_idle(400)
    for r in reqs:
        assert r.status == "length" and r.generated == _expected(r, 9), r.request_id
    assert e.pool.stats()["owned"] == 0


def test_the_forms_of_a_mask(monkeypatch):
    e = _engine(monkeypatch)
    some = torch.zeros(V, dtype=torch.bool)
    some[[8, 20, 69]] = True
    forms = [lambda r: [8, 20, 69, 69, -4, V + 3], lambda r: some, lambda r: pack_allowed(some), lambda r: {8, 20, 69}, lambda r: some.tolist() and [69, 20, 8]]
    reqs = [e.submit(Request(f"r{i}", [10], 5, allowed_tokens=f)) for i, f in enumerate(forms)]
    free = e.submit(Request("free", [10], 5, allowed_tokens=lambda r: None))
    e.run_until_idle(200)
    assert [r.generated for r in reqs] == [[20, 69, 8, 20, 69]] * 5
    assert free.generated == [11, 12, 13, 14, 15]


@pytest.mark.parametrize("ask,says", [
    (dict(allowed_tokens=lambda r: [] if len(r.generated) == 2 else [5, 6]), "no token is allowed"),
    (dict(allowed_tokens=lambda r: 1 / 0 if len(r.generated) == 2 else None), "ZeroDivisionError"),
    (dict(allowed_tokens=lambda r: torch.zeros(V + 1, dtype=torch.bool) if len(r.generated) == 2 else None), "allowed_tokens gave")])
def test_a_mask_that_fails_ends_its_request_alone(monkeypatch, ask, says):
    e = _engine(monkeypatch)
    a, b, c = e.submit(Request("a", [4], 6)), e.submit(Request("b", [4], 6, **ask)), e.submit(Request("c", [4], 6, presence_penalty=1.0))
    e.run_until_idle(100)
    assert a.status == c.status == "length" and len(c.generated) == 6 and a.generated == [5, 6, 7, 8, 9, 10]
    assert b.status == "error" and says in b.detail and len(b.generated) == 2
    assert e.pool.stats()["owned"] == 0


def test_the_operators_own_refusal(monkeypatch):
    """Host logits: the operator refuses them, and those that asked end."""
    e = _engine(monkeypatch, op=None)
    a, b = e.submit(Request("a", [1, 2], 3)), e.submit(Request("b", [5, 6], 3, repetition_penalty=1.1))
    e.run_until_idle(50)
    assert a.status == "length" and a.generated == [3, 4, 5]
    assert b.status == "error" and b.generated == [] and "HIP device" in b.detail


def test_a_request_that_is_sent_again(monkeypatch):
    """The same object with another prompt, in the slot that it had."""
    e = _engine(monkeypatch, max_batch=1)
    r = Request("r", [1, 2, 3, 4, 5, 6, 7], 4, presence_penalty=9.0, frequency_penalty=3.0, repetition_penalty=2.0)
    e.submit(r)
    e.run_until_idle(50)
    again = Request("r", [40, 41], 4, presence_penalty=9.0, frequency_penalty=3.0, repetition_penalty=2.0)
    e.submit(again)
    e.run_until_idle(50)
    assert again.generated == _expected(again, 4)


def test_refusals():
    pool = PagePool(num_layers=1, num_pages=64, num_kv_heads=1, page_size=16, nb_k=64, nb_v=64)
    e = Engine(_Model(), pool, None, None, 128)
    for kw, why in ((dict(repetition_penalty=0.0), "bad_penalty"), (dict(repetition_penalty=math.inf), "bad_penalty"), (dict(presence_penalty=math.nan), "bad_penalty"),
                    (dict(frequency_penalty=-math.inf), "bad_penalty"), (dict(logit_bias={3: math.nan}), "bad_logit_bias"),
                    (dict(logit_bias={t: 1.0 for t in range(1025)}), "bad_logit_bias")):
        with pytest.raises(Refused) as err:
            e.submit(Request("r", [1], 3, **kw))
        assert err.value.reason == why


def test_sinks_without_a_window():
    pool = PagePool(num_layers=1, num_pages=4, num_kv_heads=1, page_size=16, nb_k=64, nb_v=64)
    with pytest.raises(ValueError, match="window"):
        Engine(_Model(), pool, None, None, 128, config=EngineConfig(sinks=4))
    assert Request("r", [1], 2, logit_bias=None).logit_bias == {}


@pytest.mark.parametrize("window,sinks", [(0, 0), (-3, 0), (2.5, 0), (8, -1)])
def test_a_window_that_is_none(window, sinks):
    pool = PagePool(num_layers=1, num_pages=4, num_kv_heads=1, page_size=16, nb_k=64, nb_v=64)
    with pytest.raises(ValueError, match="at least"):
        Engine(_Model(), pool, None, None, 128, config=EngineConfig(window=window, sinks=sinks))
