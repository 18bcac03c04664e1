"""Penalties that are numbers are refused by what fp32, the type that they are applied in, makes of
them. No GPU."""
from __future__ import annotations

import math

import pytest
import torch

from winnow_amd import _lib
from winnow_amd import packed_attention as pa
from winnow_amd.logits import adjust_logits
from test_conversation_refusals import as_hip  # noqa: F401 - a fixture
from test_engine_steering import _engine

FP32_MAX = float(torch.finfo(torch.float32).max)
OUT = [dict(repetition=1e39), dict(repetition=1e-46), dict(repetition=-1e-46), dict(presence=1e39), dict(presence=-1e39), dict(frequency=3.5e38),
       dict(frequency=-1e300), dict(repetition=10 ** 400), dict(presence=-10 ** 400)]
IDS = ["-".join(f"{k}{float(v) if abs(v) < 1e301 else 'huge'}" for k, v in kw.items()) for kw in OUT]
IN = [dict(repetition=FP32_MAX), dict(repetition=2.0 ** -149), dict(presence=-FP32_MAX), dict(presence=1e-46), dict(frequency=FP32_MAX)]


@pytest.mark.parametrize("kw", OUT, ids=IDS)
def test_the_operator(as_hip, kw):  # noqa: F811
    with pytest.raises(pa.UnsupportedLayout, match="finite"):
        adjust_logits(torch.zeros(3, 70), history=torch.zeros(3, 4, dtype=torch.int32), **kw)


@pytest.mark.parametrize("kw", IN, ids=str)
def test_the_operator_takes_what_fp32_holds(as_hip, monkeypatch, kw):  # noqa: F811
    seen = []
    monkeypatch.setattr(_lib, "call", lambda name, *a: seen.append(a))
    adjust_logits(torch.zeros(3, 70), history=torch.zeros(3, 4, dtype=torch.int32), **kw)
    name, value = next(iter(kw.items()))
    got = seen[0][15 + ("repetition", "presence", "frequency").index(name)]
    assert got == float(torch.tensor(value, dtype=torch.float32)) and math.isfinite(got)


@pytest.mark.parametrize("kw", OUT, ids=IDS)
def test_the_engine(monkeypatch, kw):
    from winnow_amd.engine import Refused, Request
    e = _engine(monkeypatch)
    with pytest.raises(Refused) as err:
        e.submit(Request("r", [1], 3, **{f"{k}_penalty": v for k, v in kw.items()}))
    assert err.value.reason == "bad_penalty"


@pytest.mark.parametrize("kw", IN, ids=str)
def test_the_engine_takes_what_fp32_holds(monkeypatch, kw):
    from winnow_amd.engine import Request
    e = _engine(monkeypatch)
    r = e.submit(Request("r", [1], 2, **{f"{k}_penalty": v for k, v in kw.items()}))
    e.run_until_idle(20)
    assert r.status == "length" and len(r.generated) == 2
