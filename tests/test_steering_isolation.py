"""What one request asks for does not end the others of its batch. No GPU."""
from __future__ import annotations

import pytest

from winnow_amd.engine import Refused, Request
from test_engine_steering import V, _engine, _expected


@pytest.mark.parametrize("bias", [{2 ** 70: 50.0}, {-2 ** 63 - 1: 50.0, 33: 2.5}, {2 ** 31: 1.0, 2 ** 63 - 1: 9.0}])
def test_biases_of_tokens_that_no_type_holds(monkeypatch, bias):
    """Ids outside the vocabulary are ignored, however far outside."""
    e = _engine(monkeypatch)
    a = e.submit(Request("a", [30], 5, logit_bias=bias))
    b = e.submit(Request("b", [1, 2, 3], 5, presence_penalty=0.5, frequency_penalty=2.5))
    e.run_until_idle(50)
    for r in (a, b):
        assert r.status == "length" and r.generated == _expected(r, 5), (r.request_id, r.detail)


@pytest.mark.parametrize("bias", [{"fifty": 1.0}, {None: 1.0}, {3: "much"}, {3: None}, {float("inf"): 1.0}])
def test_biases_that_are_none(monkeypatch, bias):
    e = _engine(monkeypatch)
    with pytest.raises(Refused) as err:
        e.submit(Request("r", [1], 3, logit_bias=bias))
    assert err.value.reason == "bad_logit_bias"


@pytest.mark.parametrize("prompt", [(9, 10, 11, 12, 10), range(4, 9)])
def test_prompts_that_are_other_sequences(monkeypatch, prompt):
    e = _engine(monkeypatch)
    a = e.submit(Request("a", prompt, 5, repetition_penalty=1.7))
    b = e.submit(Request("b", [1, 2, 3], 5, presence_penalty=0.5))
    e.run_until_idle(50)
    a.prompt_ids = list(prompt)
    for r in (a, b):
        assert r.status == "length" and r.generated == _expected(r, 5), (r.request_id, r.detail)


def test_biases_by_text_keys(monkeypatch):
    """As a request in JSON has them."""
    e = _engine(monkeypatch)
    r = e.submit(Request("r", [30], 3, logit_bias={"33": 2.5, str(V + 9): 50.0}))
    e.run_until_idle(20)
    r.logit_bias = {33: 2.5}
    assert r.generated == _expected(r, 3)


@pytest.mark.parametrize("ask", [dict(repetition_penalty=2.0), dict(frequency_penalty=3.0, presence_penalty=1.0)])
def test_a_request_object_that_is_used_again(monkeypatch, ask):
    """In the slot that it had, with a shorter prompt: its tokens of the first time, which the second run would
    make next, are not held against it."""
    e = _engine(monkeypatch, max_batch=1)
    r = Request("r", [42, 60, 43, 44, 44, 44, 60], 4, **ask)
    e.submit(r)
    e.run_until_idle(50)
    assert r.status == "length" and r.generated == _expected(r, 4)
    vars(r).update(vars(Request("r", [40, 41], 4, **ask)))
    e.submit(r)
    e.run_until_idle(50)
    assert r.status == "length" and r.generated == _expected(r, 4) == [42, 43, 44, 45]
