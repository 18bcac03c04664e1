"""GPU parity of ``adjust_logits`` (``wn_adjust_logits``) against float64 on the host.

Tolerance. A logit goes through at most 3 + J fp32 roundings (division or product, two
subtractions, one addition per bias of its token), each off by at most 2^-24 of a value below
M = |x| max(r, 1 / r) + frequency c + presence + sum |bias| (1 + a few 2^-24, taken as 1.01), and
is rounded once to its type, by half a step of it: eps / 2 of the value, or half the least
subnormal. A logit that nothing applies to keeps its bits.
"""
from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda"
TYPES = [torch.float32, torch.float16, torch.bfloat16]


def _adjust(*a, **k):
    from winnow_amd.logits import adjust_logits
    return adjust_logits(*a, **k)


def _row(x, hist, made, r, p, f, ids, bias, allowed):
    """One row in float64: (values, tolerance before the type's own, touched)."""
    V = len(x)
    total, count = torch.zeros(V), torch.zeros(V, dtype=torch.float64)
    for k, t in enumerate(hist):
        if 0 <= t < V:
            total[t] = 1
            count[t] += k >= made
    y, size, ops = x.clone(), x.abs(), torch.full((V,), 3.0, dtype=torch.float64)
    seen = total > 0
    y[seen] = torch.where(x[seen] > 0, x[seen] / r, x[seen] * r)
    size = torch.where(seen, size * max(r, 1 / r), size)
    y = torch.where(count > 0, y - f * count - p, y)
    size = size + torch.where(count > 0, abs(f) * count + abs(p), 0)
    touched = seen.clone()
    for t, b in zip(ids, bias):
        if 0 <= t < V:
            y[t] += b
            size[t] += abs(b)
            ops[t] += 1
            touched[t] = True
    y = torch.where(allowed, y, -math.inf)
    return y, ops * 1.01 * size * 2.0 ** -24, touched | ~allowed


def _check(x, got, history=None, lengths=None, prompt_lengths=None, repetition=1.0, presence=0.0, frequency=0.0,
           bias_ids=None, bias=None, allowed=None):
    N, V = x.shape
    assert got.shape == x.shape and got.dtype == x.dtype
    info = torch.finfo(x.dtype)
    least = info.smallest_normal * info.eps
    per_row = [t.double().cpu().tolist() if isinstance(t, torch.Tensor) else [float(torch.tensor(t, dtype=torch.float32))] * N
               for t in (repetition, presence, frequency)]
    x64, got64 = x.cpu(), got.cpu()
    for i in range(N):
        n = history.shape[1] if history is not None and lengths is None else 0 if history is None else min(max(int(lengths[i]), 0), history.shape[1])
        hist = history[i].tolist()[:n] if n else []
        made = int(prompt_lengths[i]) if prompt_lengths is not None else 0
        ids, b = ([], []) if bias is None else (bias_ids[i].tolist(), bias[i].double().tolist())
        ok = torch.ones(V, dtype=torch.bool)
        if allowed is not None:
            v = torch.arange(V)
            ok = ((allowed[i].cpu().long()[v // 32] >> (v % 32)) & 1) > 0
        want, tol, touched = _row(x64[i].double(), hist, made, *(t[i] for t in per_row), ids, b, ok)
        one = torch.int32 if x.dtype == torch.float32 else torch.int16
        assert torch.equal(got64[i].view(one)[~touched], x64[i].view(one)[~touched])
        w, g = want[touched], got64[i].double()[touched]
        tol = tol[touched] + w.abs() * (info.eps / 2) + least / 2
        over = w.abs() + tol >= info.max            # may be infinite in the type
        fine = ((g - w).abs() <= tol) | (g == w) | (g.isnan() & w.isnan()) | (over & ((g == w.sign() * math.inf) | (g.abs() == info.max)))
        assert fine.all(), (i, w[~fine], g[~fine])


def _case(N, V, H, J, mask, dtype, seed, penalties="rows"):
    g = torch.Generator(device=DEV).manual_seed(seed)
    kw = {}
    x = (3 * torch.randn(N, V, generator=g, device=DEV)).to(dtype)
    if H:
        pool = torch.randint(-1, V + 1, (max(1, min(V, H // 2 + 1)),), generator=g, device=DEV)   # repeats, and ids of no token
        kw["history"] = pool[torch.randint(len(pool), (N, H), generator=g, device=DEV)].int()
        kw["lengths"] = torch.randint(0, H + 2, (N,), generator=g, device=DEV).int()
        kw["prompt_lengths"] = torch.randint(-1, H + 2, (N,), generator=g, device=DEV).int()
        if penalties == "rows":
            kw["repetition"] = 0.5 + torch.rand(N, generator=g, device=DEV)
            kw["presence"], kw["frequency"] = torch.randn(N, generator=g, device=DEV), torch.randn(N, generator=g, device=DEV)
        else:
            kw.update(repetition=1.3, presence=0.25, frequency=-0.125)
    if J:
        kw["bias_ids"] = torch.randint(-1, min(V + 1, 2 * J), (N, J), generator=g, device=DEV).int()   # the same token twice and more
        kw["bias"] = 4 * torch.randn(N, J, generator=g, device=DEV)
    if mask:
        kw["allowed"] = torch.randint(-2 ** 31, 2 ** 31, (N, -(-V // 32)), generator=g, device=DEV).int()
    return x, kw


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("N,V,H,J,mask", [
    (1, 1, 1, 1, True), (3, 7, 5, 3, True), (2, 31, 40, 2, True), (2, 33, 0, 0, True), (4, 1003, 300, 0, False), (3, 8192, 2100, 70, True),
    (2, 8193, 17, 64, True), (5, 50257, 5000, 1, False), (1, 128256, 900, 1024, True), (70, 2049, 33, 5, True), (2, 300, 0, 4, False),
    (300, 65, 1, 0, True)])
def test_matches_float64(dtype, N, V, H, J, mask):
    """One row to many, vocabularies of one token to large, at and around the segments' size and the
    words' 32; empty and partial histories, ids of no token, tokens listed twice."""
    x, kw = _case(N, V, H, J, mask, dtype, V + 10 * N)
    _check(x, _adjust(x, **kw), **kw)


@pytest.mark.parametrize("dtype", TYPES)
def test_each_part_alone(dtype):
    x, kw = _case(3, 5000, 700, 9, True, dtype, 5, "all")
    for names in (("history", "repetition"), ("history", "presence"), ("history", "frequency", "lengths"), ("history",), ("bias", "bias_ids"),
                  ("allowed",), ("history", "lengths", "prompt_lengths", "presence", "frequency"), ()):
        part = {n: kw[n] for n in names}
        got = _adjust(x, **part)
        assert got.data_ptr() != x.data_ptr()
        _check(x, got, **part)


@pytest.mark.parametrize("dtype", TYPES)
def test_strides_and_wide_integers(dtype):
    """Rows with gaps that start at any element, shared rows, int64 operands with ids past 32 bits,
    operands with gaps; out with a stride of its own; in place."""
    x, kw = _case(6, 1111, 50, 6, True, dtype, 6)
    big, _ = _case(6, 1400, 0, 0, False, dtype, 7)
    for lo in (0, 1, 3):
        y = big[:, lo:lo + 1111]
        _check(y, _adjust(y, **kw), **kw)
        out = torch.full((6, 1500), 7.0, dtype=dtype, device=DEV)
        got = _adjust(y, out=out[:, 5 + lo:5 + lo + 1111], **kw)
        assert got.data_ptr() == out[:, 5 + lo:].data_ptr()
        _check(y, got, **kw)
        assert (out[:, :5 + lo] == 7).all() and (out[:, 5 + lo + 1111:] == 7).all()
    shared = x[:1].expand(6, -1)
    _check(shared, _adjust(shared, **kw), **kw)
    wide = dict(kw, history=kw["history"].long(), lengths=kw["lengths"].long(), prompt_lengths=kw["prompt_lengths"].long(),
                bias_ids=kw["bias_ids"].long())
    wide["history"][:, 0] = 2 ** 32 + 5
    wide["bias_ids"][:, 0] = -2 ** 32 + 1
    narrow = dict(kw, history=wide["history"].clamp(-1, 2000).int(), bias_ids=wide["bias_ids"].clamp(-1, 2000).int())
    assert torch.equal(_adjust(x, **wide), _adjust(x, **narrow))
    gaps = dict(kw, history=torch.stack([kw["history"]] * 2, 2)[..., 0], lengths=torch.stack([kw["lengths"]] * 2, 1)[:, 0],
                allowed=torch.cat([kw["allowed"]] * 2, 1)[:, :kw["allowed"].shape[1]])
    want = _adjust(x, **kw)
    assert torch.equal(_adjust(x, **gaps), want)
    y = x.clone()
    assert _adjust(y, out=y, **kw) is y and torch.equal(y, want)


@pytest.mark.parametrize("dtype", TYPES)
def test_values_that_are_not_finite(dtype):
    """NaN, infinities, the type's extremes, +-0, with and without what applies to them: in their own
    places only; a row that allows nothing is -inf, whatever it held."""
    info = torch.finfo(dtype)
    special = torch.tensor([math.nan, math.inf, -math.inf, info.max, info.min, 0.0, -0.0, info.smallest_normal], dtype=torch.float64).to(dtype).to(DEV)
    x = special.repeat(4, 40)
    V = x.shape[1]
    hist = torch.arange(0, V, 3, device=DEV).int().expand(4, -1)
    allowed = torch.full((4, V // 32), -1, dtype=torch.int32, device=DEV)
    allowed[1] = 0
    allowed[2, 1] = 0x0f0f0f0f
    kw = dict(history=hist, repetition=1.5, presence=0.5, frequency=0.25, allowed=allowed, bias_ids=torch.tensor([[1, 2, 9, -1]] * 4, device=DEV).int(),
              bias=torch.tensor([[-math.inf, math.inf, 2.0, math.nan]] * 4, device=DEV))
    got = _adjust(x, **kw)
    _check(x, got, **kw)
    assert (got[1] == -math.inf).all()


def test_counts_in_any_order():
    """A token that fills the history, and the same tokens in another order: the same bits."""
    x, _ = _case(2, 9000, 0, 0, False, torch.float32, 8)
    hist = torch.randint(0, 50, (2, 20000), device=DEV, generator=torch.Generator(device=DEV).manual_seed(1)).int()
    hist[1] = 8999
    kw = dict(repetition=1.1, presence=0.3, frequency=0.001)
    a = _adjust(x, history=hist, **kw)
    _check(x, a, history=hist, **kw)
    order = torch.randperm(20000, device=DEV)
    for _ in range(3):
        assert torch.equal(_adjust(x, history=hist[:, order].contiguous(), **kw), a)


def test_rows_past_two_to_the_31():
    V, N = 1 << 20, 2100
    x = torch.zeros(N, V, dtype=torch.bfloat16, device=DEV)
    x[N - 1] = _case(1, V, 0, 0, False, torch.bfloat16, 3)[0][0]
    last = x[N - 1:].clone()
    hist = torch.randint(0, V, (N, 8), device=DEV).int()
    allowed = torch.full((N, V // 32), -1, dtype=torch.int32, device=DEV)
    allowed[:, ::7] = 0x55555555
    _adjust(x, history=hist, presence=1.0, allowed=allowed, out=x)
    kw = dict(history=hist[N - 1:], presence=1.0, allowed=allowed[N - 1:])
    _check(last, x[N - 1:], **kw)


def test_graph_replays_and_own_stream():
    x, kw = _case(9, 70001, 500, 12, True, torch.bfloat16, 4)
    want = _adjust(x, **kw)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = _adjust(x, **kw)
    side.synchronize()
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = _adjust(x, **kw)
    for k in range(4):
        y, new = _case(9, 70001, 500, 12, True, torch.bfloat16, 40 + k)
        x.copy_(y)
        for name, t in kw.items():
            t.copy_(new[name])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, _adjust(x, **kw))
    assert torch.equal(got, _adjust(y, **new))


def test_pack_allowed():
    from winnow_amd.logits import mask_words, pack_allowed
    g = torch.Generator().manual_seed(2)
    for V in (1, 31, 32, 33, 1000):
        ok = torch.rand(3, V, generator=g) < 0.5
        words = pack_allowed(ok)
        assert words.shape == (3, mask_words(V)) and words.dtype == torch.int32
        v = torch.arange(V)
        assert torch.equal(((words.long()[:, v // 32] >> (v % 32)) & 1) > 0, ok)
        x = torch.zeros(3, V, device=DEV)
        assert torch.equal(_adjust(x, allowed=words.to(DEV)) == 0, ok.to(DEV))
