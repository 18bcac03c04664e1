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


# --------------------------------------------------------------------- windowed attention

def _kv(D=64, P=6, Hkv=2, S=16, bw=4, B=2, lens=(20, 33)):
    quant = pa.Quantizer(torch.eye(D), torch.linspace(-1, 1, 2 ** bw), bw)
    pages, norms = torch.zeros(P, Hkv, S, D * bw // 8, dtype=torch.uint8), torch.ones(P, Hkv, S, dtype=torch.float16)
    table = torch.tensor([[0, 1, -1], [2, 3, 4]], dtype=torch.int32)[:B]
    return pa.PackedKV(pages, norms, pages.clone(), norms.clone(), table, torch.tensor(lens, dtype=torch.int32), quant, quant, D)


def _window(q=None, kv=None, window=8, sinks=2, **kw):
    return pa.packed_window_attention(torch.zeros(2, 4, 5, 64) if q is None else q, kv or _kv(), 0.1, window=window, sinks=sinks, **kw)


def test_window_needs_a_gpu():
    with pytest.raises(pa.UnsupportedLayout, match="HIP device"):
        _window()


@pytest.mark.parametrize("kw,match", [
    (dict(window=0), "at least 1"), (dict(window=-5), "at least 1"), (dict(sinks=-1), "at least"), (dict(window=2.5), "whole"), (dict(window=True), "whole"),
    (dict(q=torch.zeros(2, 4, 0, 64)), "queries a sequence"), (dict(q=torch.zeros(2, 3, 5, 64)), "multiple"),
    (dict(q=torch.zeros(1, 1, 1, 64).expand(2, 4, 2 ** 20, 64)), "queries a sequence"),
    (dict(q=torch.zeros(2, 4, 64, 5).transpose(2, 3)), "contiguous head_dim"), (dict(q=torch.zeros(2, 4, 5, 64, dtype=torch.float64)), "fp32/fp16/bf16"),
    (dict(q=torch.zeros(2, 4, 5, 64, requires_grad=True)), "no gradient"), (dict(out_dtype=torch.float64), "output dtype"),
    (dict(q=torch.zeros(2, 4, 5, 8), kv=_kv(D=8)), "head_dim 8"), (dict(kv=_kv(S=24, lens=(3, 4))), "power of two"),
    (dict(kv=_kv(lens=(20, 49))), "out of range"), (dict(kv=_kv(lens=(-1, 4))), "out of range")])
def test_window_operands(as_hip, kw, match):
    with pytest.raises(pa.UnsupportedLayout, match=match):
        _window(**kw)


def _in_range(lens, table, P, S, Q, window, sinks):
    """Page by page, from the definition."""
    for L, row in zip(lens.tolist(), table.tolist()):
        if not 0 <= L <= len(row) * S:
            return False
        for j in range(L):
            if any(j <= p and (p - j < window or j < sinks) for p in range(L - Q, L)) and not 0 <= row[j // S] < P:
                return False
    return True


@pytest.mark.parametrize("native", [True, False])
def test_window_ranges_are_those_in_view(monkeypatch, native):
    """Random lengths, tables with ids out of range here and there, windows and sinks: a call is refused
    exactly where a page in view is."""
    lib = _lib.lib()
    if not native:
        monkeypatch.setattr(_lib, "_lib", None)
    g = torch.Generator().manual_seed(3)
    seen = set()
    for _ in range(400):
        r = lambda lo, hi: int(torch.randint(lo, hi, (1,), generator=g))  # noqa: E731
        S, width, P, Q = 2 ** r(0, 4), r(1, 7), 5, r(1, 6)
        lens = torch.randint(-1 if r(0, 9) == 0 else 0, width * S + (2 if r(0, 9) == 0 else 1), (2,), generator=g).int()
        table = torch.randint(0, P, (2, width), generator=g).int()
        if r(0, 3):
            table[r(0, 2), r(0, width)] = (-1, P, 2 ** 31 - 1)[r(0, 3)]
        window, sinks = r(1, 20), r(0, 9)
        ok = _in_range(lens, table, P, S, Q, window, sinks)
        seen.add(ok)
        if native:
            assert bool(lib.wn_window_in_range(lens.data_ptr(), table.data_ptr(), width, 2, width, P, S, Q, window, sinks)) == ok
        if ok:
            pa.check_window_ranges(lens, table, P, S, Q, window, sinks)
        else:
            with pytest.raises(pa.UnsupportedLayout):
                pa.check_window_ranges(lens, table, P, S, Q, window, sinks)
    assert seen == {True, False}


def test_window_c_abi():
    """Nothing is launched for arguments outside the contract."""
    x = torch.zeros(4096)
    p = x.data_ptr()

    def call(**kw):
        a = dict(q=p, qd=0, qb=0, qh=0, qq=0, pik=p, piv=p, cbk=p, cbv=p, kp=p, kpp=0, kph=0, vp=p, vpp=0, vph=0, knp=p, knpp=0, knph=0, vnp=p, vnpp=0,
                 vnph=0, table=p, ts=0, lens=p, out=p, od=0, ws=None, wb=0, B=1, Hq=4, Hkv=2, Q=1, D=64, S=16, bwk=4, bwv=4, P=1, mp=4, window=8,
                 sinks=0, scale=0.1, exact=1, ns=1, span=64)
        a.update(kw)
        _lib.call("wn_window_attention", *a.values(), None, None, None)
    for kw, match in ((dict(window=0), "at least 1"), (dict(sinks=-1), "sinks"), (dict(Hq=3), "need"), (dict(Q=0), "need"), (dict(Q=2 ** 20), "need"),
                      (dict(D=96), "need"), (dict(bwk=7), "widths"), (dict(S=8), "page size"), (dict(ns=0), "num_splits"), (dict(ns=4097), "num_splits"),
                      (dict(span=32), "span"), (dict(mp=0), "max_pages"), (dict(mp=2 ** 30), "max_pages"), (dict(kp=p + 2), "4-byte"), (dict(kph=6), "4-byte"),
                      (dict(vnpp=-1), "negative"), (dict(q=None), "null"), (dict(out=p + 1), "aligned"), (dict(), "workspace"), (dict(od=5), "dtype")):
        with pytest.raises(_lib.WinnowHipError, match=match):
            call(**kw)
    call(B=0, q=None)
    size = _lib.lib().wn_window_workspace_bytes       # B, Hq, Hkv, Q, D, S, max_pages, window, sinks, num_splits, span
    for bad in ((1, 3, 2, 1, 64, 16, 4, 8, 0, 1, 64), (1, 4, 2, 1, 64, 16, 4, 8, 0, 0, 64), (1, 4, 2, 1, 64, 16, 4, 0, 0, 1, 64),
                (1, 4, 2, 2, 128, 16, 4, 8, 0, 8, 0), (1, 4, 2, 1, 64, 16, 4, 8, 0, 8, 0), (1, 4, 2, 1, 128, 24, 4, 8, 0, 8, 0)):
        assert size(*bad) == -1
    assert size(1, 4, 2, 1, 128, 16, 4, 8, 0, 8, 0) > 0 and size(1, 4, 2, 1, 64, 16, 4, 8, 0, 1, 64) > 0


@pytest.mark.parametrize("call", [lambda x: adjust_logits(x.reshape(-1, 64)), lambda x: _append(q=x), lambda x: _window(q=x[:, :, :1].expand(2, 4, 5, 64))],
                         ids=["logits", "append", "window"])
def test_tangents_and_traces(as_hip, call):
    """A forward-mode derivative and a place in a trace are refused, on tensors that pass else."""
    import torch.autograd.forward_ad as fwd
    from torch.fx.experimental.proxy_tensor import make_fx
    x = torch.randn(2, 4, 3, 64)
    with fwd.dual_level():
        with pytest.raises(pa.UnsupportedLayout, match="forward-mode"):
            call(fwd.make_dual(x, torch.ones_like(x)))
    with pytest.raises(pa.UnsupportedLayout, match="traced"):
        make_fx(lambda t: call(t))(x)
