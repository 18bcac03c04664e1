"""What the operators of a step of a long conversation refuse. No GPU: the C ABI checks its
arguments before any launch, the Python layer is asked with host tensors that it is told to take
for HIP ones."""
from __future__ import annotations

import math
import types

import pytest
import torch

from winnow_amd import _lib
from winnow_amd import packed_attention as pa
from winnow_amd.logits import adjust_logits


@pytest.fixture
def as_hip(monkeypatch):
    """Host tensors pass for HIP ones; a call into the library fails the test."""
    monkeypatch.setattr(_lib, "is_hip", lambda t: True)
    monkeypatch.setattr(_lib, "on", lambda device: _lib._here)
    monkeypatch.setattr(_lib, "stream_of", lambda device: 0)

    def call(name, *args):
        raise AssertionError(f"{name} was called")
    monkeypatch.setattr(_lib, "call", call)


def test_logits_need_a_gpu():
    with pytest.raises(pa.UnsupportedLayout, match="HIP device"):
        adjust_logits(torch.zeros(2, 5))


X = torch.zeros(3, 70)


@pytest.mark.parametrize("x,kw,match", [
    (torch.zeros(3, 70, dtype=torch.float64), {}, "fp32, fp16 or bf16"),
    (torch.zeros(70), {}, r"\(N, V\)"),
    (torch.zeros(3, 0), {}, "non-empty"),
    (torch.zeros(70, 3).t(), {}, "contiguous"),
    (torch.zeros(3, 70, requires_grad=True), {}, "no gradient"),
    (X, dict(lengths=torch.zeros(3, dtype=torch.int32)), "of a history"),
    (X, dict(history=torch.zeros(2, 4, dtype=torch.int32)), "history must be"),
    (X, dict(history=torch.zeros(3, dtype=torch.int32)), "history must be"),
    (X, dict(history=torch.zeros(3, 4)), "history must be"),
    (X, dict(history=torch.zeros(3, 4, dtype=torch.int32), lengths=torch.zeros(4, dtype=torch.int32)), "lengths must be"),
    (X, dict(history=torch.zeros(3, 4, dtype=torch.int32), prompt_lengths=torch.zeros(3)), "prompt_lengths must be"),
    (X, dict(repetition=0.0), "above 0"), (X, dict(repetition=-1.0), "above 0"), (X, dict(repetition=math.nan), "finite"),
    (X, dict(presence=math.inf), "finite"), (X, dict(frequency=torch.zeros(2)), r"number or \(3,\)"),
    (X, dict(presence=torch.zeros(3, dtype=torch.float64)), r"number or \(3,\)"),
    (X, dict(repetition=torch.ones(3, requires_grad=True)), "no gradient"),
    (X, dict(bias=torch.zeros(3, 2)), "together"), (X, dict(bias_ids=torch.zeros(3, 2, dtype=torch.int32)), "together"),
    (X, dict(bias=torch.zeros(3, 2), bias_ids=torch.zeros(3, 3, dtype=torch.int32)), "bias_ids must be"),
    (X, dict(bias=torch.zeros(3, 2).half(), bias_ids=torch.zeros(3, 2, dtype=torch.int32)), "bias must be"),
    (X, dict(bias=torch.zeros(3, 1025), bias_ids=torch.zeros(3, 1025, dtype=torch.int32)), "J <= 1024"),
    (X, dict(allowed=torch.zeros(3, 2, dtype=torch.int32)), "allowed must be"), (X, dict(allowed=torch.zeros(3, 3)), "allowed must be"),
    (X, dict(allowed=torch.zeros(3, 6, dtype=torch.int32)[:, ::2]), "allowed must be"),
    (X, dict(out=torch.zeros(3, 71)), "out must be"), (X, dict(out=torch.zeros(3, 70).half()), "out must be"),
    (X, dict(out=torch.zeros(1, 70).expand(3, -1)), "out must be")])
def test_logits_operands(as_hip, x, kw, match):
    with pytest.raises(pa.UnsupportedLayout, match=match):
        adjust_logits(x, **kw)


def test_logits_out_that_shares(as_hip):
    big = torch.zeros(4, 80)
    with pytest.raises(pa.UnsupportedLayout, match="no other view"):
        adjust_logits(big[:3, :70], out=big[1:, :70])
    with pytest.raises(pa.UnsupportedLayout, match="no other view"):
        adjust_logits(big[:1, :70].expand(3, -1), out=big[:3, :70])
    bias = torch.zeros(3, 70)
    with pytest.raises(pa.UnsupportedLayout, match="another operand"):
        adjust_logits(X, bias=bias, bias_ids=torch.zeros(3, 70, dtype=torch.int32), out=bias)
    with pytest.raises(AssertionError, match="wn_adjust_logits"):
        adjust_logits(big[:3, :70], out=big[:3, :70])


def test_logits_under_a_trace(as_hip):
    with pytest.raises(pa.UnsupportedLayout, match="traced"):
        torch.jit.trace(lambda x: adjust_logits(x), X)


def test_logits_c_abi():
    """Nothing is launched for arguments outside the contract."""
    x = torch.zeros(4, 70)

    def call(**kw):
        a = dict(logits=x.data_ptr(), dtype=0, stride=70, out=x.data_ptr(), out_stride=70, N=4, V=70, history=None, hs=0, H=0, lengths=None,
                 prompts=None, r=None, p=None, f=None, ra=1.0, pa=0.0, fa=0.0, ids=None, ids_s=0, bias=None, bias_s=0, J=0, allowed=None, als=0)
        a.update(kw)
        _lib.call("wn_adjust_logits", *a.values(), None)
    for kw, match in ((dict(V=0), "bad sizes"), (dict(N=-1), "bad sizes"), (dict(H=1 << 30), "bad sizes"), (dict(H=3), "null"), (dict(J=2), "null"),
                      (dict(J=1025), "biases"), (dict(dtype=3), "dtype"), (dict(logits=None), "null"), (dict(out_stride=69), "overlap"),
                      (dict(stride=-1), "negative"), (dict(logits=x.data_ptr() + 2), "aligned"), (dict(V=2 ** 31 - 1), "V="),
                      (dict(N=2 ** 40, out_stride=70), "grid")):
        with pytest.raises(_lib.WinnowHipError, match=match):
            call(**kw)
    call(N=0, logits=None)


# ------------------------------------------------------------------------ rotated append

def _append(**kw):
    """``append_rotated_kv`` on host tensors: the GPU's place is checked first."""
    from winnow_amd.packed_backend import append_rotated_kv
    tq = types.SimpleNamespace(Pi=torch.eye(64), boundaries=torch.zeros(15), centroids=torch.zeros(16), bit_width=4)
    g = dict(q=torch.zeros(2, 4, 3, 64), k=torch.zeros(2, 2, 3, 64), v=torch.zeros(2, 2, 3, 64), cos=torch.zeros(2, 3, 64), sin=torch.zeros(2, 3, 64),
             k_tq=tq, v_tq=tq, k_pages=torch.zeros(6, 2, 16, 32, dtype=torch.uint8), v_pages=torch.zeros(6, 2, 16, 32, dtype=torch.uint8),
             k_norms=torch.zeros(6, 2, 16, dtype=torch.float16), v_norms=torch.zeros(6, 2, 16, dtype=torch.float16),
             page_table=torch.tensor([[0, 1, -1], [2, 3, 4]], dtype=torch.int32), start_pos=torch.tensor([10, 30], dtype=torch.int32))
    g.update(kw)
    names = ("q", "k", "v", "cos", "sin", "k_tq", "v_tq", "k_pages", "v_pages", "k_norms", "v_norms", "page_table", "start_pos")
    args = [g.pop(n) for n in names]
    return append_rotated_kv(*args, **g)


def test_append_needs_a_gpu():
    with pytest.raises(pa.UnsupportedLayout, match="HIP device"):
        _append()


@pytest.mark.parametrize("name", ["q", "k", "v", "cos", "sin"])
def test_append_has_no_gradient(name):
    shape = (2, 3, 64) if name in ("cos", "sin") else (2, 4 if name == "q" else 2, 3, 64)
    with pytest.raises(pa.UnsupportedLayout, match="no gradient"):
        _append(**{name: torch.zeros(shape, requires_grad=True)})


def test_append_c_abi():
    """Nothing is launched for arguments outside the contract."""
    x = torch.zeros(4096)
    p = x.data_ptr()

    def call(**kw):
        a = dict(q=p, qb=0, qh=0, qn=0, qd=0, Hq=4, qo=p, cos=p, cb=0, cn=0, sin=p, sb=0, sn=0, rd=0, R=64, k=p, kb=0, kh=0, kn=0, v=p, vb=0, vh=0,
                 vn=0, xd=0, pik=p, bk=p, bwk=4, piv=p, bv=p, bwv=4, table=p, ts=0, start=p, kp=p, kpp=0, kph=0, vp=p, vpp=0, vph=0, knp=p, knpp=0,
                 knph=0, vnp=p, vnpp=0, vnph=0, B=1, Hkv=2, n=1, D=64, S=16, P=1, mp=1)
        a.update(kw)
        _lib.call("wn_append_rotated_kv", *a.values(), None, None, None)
    for kw, match in ((dict(R=0), "rotated channels"), (dict(R=63), "rotated channels"), (dict(R=66), "rotated channels"), (dict(rd=3), "dtype"),
                      (dict(qd=-1), "dtype"), (dict(Hq=0), "query heads"), (dict(cos=None), "null"), (dict(qo=None), "null"), (dict(cos=p + 2), "aligned"),
                      (dict(qo=p + 8), "aligned"), (dict(B=2 ** 16, n=2 ** 16), "too many"), (dict(D=96), "head_dim"), (dict(k=None), "null"),
                      (dict(v=None, pik=p + 4), "16-byte"), (dict(S=24), "power of two")):
        with pytest.raises(_lib.WinnowHipError, match=match):
            call(**kw)
    call(n=0, k=None, cos=None)
