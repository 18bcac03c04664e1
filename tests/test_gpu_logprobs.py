"""GPU parity of ``token_logprobs`` (``wn_token_logprobs``) against float64 torch.

Tolerance. A lane adds at most V / 256 + 64 terms in a row (one work-group a row; fewer with
segments), a tree joins the rest: the sums are off by at most (V / 256 + 80) 2^-24 of themselves,
e^d by |d| 2^-23 (its argument's rounding, |d| weighted by a share that falls as e^d: at most
2^-22 in the sum). With n = V / 256 + 100: the log of the sum is off by n 2^-24, a log
probability by that and 2^-23 of itself and of the logits' magnitude (x - m); the entropy by
n 2^-24 (1 + H).
"""
from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda"


def _lp(*a, **k):
    from winnow_amd.logprobs import token_logprobs
    return token_logprobs(*a, **k)


def _check(x, tokens, top, got=None):
    """x on the device, any shape and strides."""
    got = got or _lp(x, tokens, top=top)
    V, rows = x.shape[-1], x.shape[:-1]
    x64 = x.double().cpu()
    want = torch.log_softmax(x64, -1)
    n = V / 256 + 100
    if tokens is not None:
        w = want.gather(-1, tokens.cpu().long()[..., None])[..., 0]
        tol = n * 2.0 ** -24 + 2.0 ** -22 * w.abs().nan_to_num(posinf=0)
        assert got.logprob.shape == rows and got.logprob.dtype == torch.float32
        same = (got.logprob.double().cpu() - w).abs() <= tol
        assert (same | (got.logprob.cpu() == w)).all(), (got.logprob, w)
    p = want.exp()
    H = -(torch.where(p > 0, p * want, 0.0)).sum(-1)
    assert got.entropy.shape == rows
    assert ((got.entropy.double().cpu() - H).abs() <= n * 2.0 ** -24 * (1 + H)).all(), (got.entropy, H)
    if top == 0:
        assert got.top_ids is None and got.top_logprobs is None
        return
    ids = torch.sort(x64, dim=-1, descending=True, stable=True).indices[..., :top]
    assert got.top_ids.dtype == torch.int64 and torch.equal(got.top_ids.cpu(), ids)
    w = want.gather(-1, ids)
    tol = n * 2.0 ** -24 + 2.0 ** -22 * w.abs().nan_to_num(posinf=0)
    assert (((got.top_logprobs.double().cpu() - w).abs() <= tol) | (got.top_logprobs.cpu() == w)).all()


def _logits(shape, dtype, seed, spread=3.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return (spread * torch.randn(*shape, generator=g, device=DEV)).to(dtype)


def _tokens(shape, V, seed):
    return torch.randint(V, shape, generator=torch.Generator(device=DEV).manual_seed(seed), device=DEV)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("N,V,top", [(1, 1, 1), (1, 1, 0), (3, 2, 2), (1, 64, 64), (7, 100, 5), (5, 2047, 20), (1, 32003, 1),
                                     (2, 128256, 64), (33, 50257, 10), (600, 4097, 3), (1200, 1000, 20), (1030, 8, 8)])
def test_matches_float64(dtype, N, V, top):
    """One row to many (segments joined by a second launch, and a work-group a row), vocabularies
    of one token, below a wave, odd and large; the ties of 16-bit logits."""
    _check(_logits((N, V), dtype, V + N), _tokens((N,), V, N), top)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_shapes_and_strides(dtype):
    """(V,), (B, T, V), rows with gaps that start at any element, tokens left out or int32."""
    x = _logits((5, 4, 1003), dtype, 1)
    _check(x, _tokens((5, 4), 1003, 2), 7)
    _check(x[2, 1], _tokens((), 1003, 3), 3)
    _check(x[1:4, :, 5:906], _tokens((3, 4), 901, 4).int(), 5)
    _check(x.transpose(0, 1), _tokens((4, 5), 1003, 5), 2)
    _check(x[:, -1], None, 4)
    _check(x[:, :1].expand(5, 3, 1003), _tokens((5, 3), 1003, 6), 1)
    _check(x[:0, 0], _tokens((0,), 1003, 7), 0)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("V", [37, 5000, 70001])
def test_masked_and_equal_logits(dtype, V):
    """Rows of equal logits, of -inf but for a few, of the type's lowest value (all, or all but a
    few), one certain token, +-0 beside each other; alternatives beyond the allowed tokens."""
    low = torch.finfo(dtype).min
    x = _logits((9, V), dtype, V)
    x[0] = 1.5
    x[1] = -math.inf
    x[1, [V - 1, 3]] = torch.tensor([0.5, 0.5], dtype=dtype, device=DEV)
    x[2] = low
    x[3, 4:] = low
    x[4] = -math.inf
    x[4, V // 2] = -7
    x[5, V - 2] = 60
    x[6] = 0.0
    x[6, ::2] = -0.0
    x[7] = -math.inf
    x[7, 5:9] = low
    tokens = torch.tensor([0, V - 1, V - 1, 2, V // 2, V - 2, 1, 6, 0], device=DEV)
    _check(x, tokens, 20)
    out = torch.tensor([V - 1, 0, 0, V - 1, 0, 0, 0, 0, 1], device=DEV)
    _check(x, out, 0)


@pytest.mark.parametrize("V", [300, 40000])
def test_rows_without_an_answer(V):
    """NaN and +inf rows, rows of -inf alone, tokens that are none: NaN, in their rows only, and
    ids inside the vocabulary."""
    x = _logits((6, V), torch.float32, 9)
    clean = _lp(x.clone(), _tokens((6,), V, 10), top=5)
    tokens = _tokens((6,), V, 10)
    x[1, V // 3] = math.nan
    x[2, 7] = math.inf
    x[3] = -math.inf
    tokens[4] = -1
    tokens[5] = V
    got = _lp(x, tokens, top=5)
    assert got.logprob[1:].isnan().all() and got.entropy[1:4].isnan().all() and got.top_logprobs[[1, 3]].isnan().all()
    assert ((got.top_ids >= 0) & (got.top_ids < V)).all()
    for name in ("logprob", "entropy", "top_logprobs", "top_ids"):
        assert torch.equal(getattr(got, name)[0], getattr(clean, name)[0])
    assert torch.equal(got.entropy[4:], clean.entropy[4:]) and torch.equal(got.top_ids[4:], clean.top_ids[4:])


def test_rows_past_two_to_the_31():
    """Row offsets above 2^31 elements."""
    V, N = 1 << 20, 2100
    x = torch.zeros(N, V, dtype=torch.bfloat16, device=DEV)
    x[N - 1] = _logits((V,), torch.bfloat16, 3)
    t = torch.full((N,), V - 5, device=DEV)
    got = _lp(x, t, top=3)
    one = _lp(x[N - 1:].clone(), t[:1], top=3)
    assert torch.equal(got.top_ids[N - 1], one.top_ids[0])
    assert (got.logprob[N - 1] - one.logprob[0]).abs() <= (V / 256 + 100) * 2.0 ** -23
    assert torch.equal(got.top_ids[0].cpu(), torch.arange(3))


def test_graph_replays_and_own_stream():
    x, t = _logits((9, 70001), torch.bfloat16, 4), _tokens((9,), 70001, 5)
    want = _lp(x, t, top=6)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = _lp(x, t, top=6)
    side.synchronize()
    assert torch.equal(got.logprob, want.logprob) and torch.equal(got.top_ids, want.top_ids)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = _lp(x, t, top=6)
    for k in range(4):
        x.copy_(_logits((9, 70001), torch.bfloat16, 40 + k))
        graph.replay()
        torch.cuda.synchronize()
        want = _lp(x, t, top=6)
        for name in ("logprob", "entropy", "top_logprobs", "top_ids"):
            assert torch.equal(getattr(got, name), getattr(want, name))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("N,V,top", [(1, 128256, 64), (3, 9001, 20), (1100, 4100, 7), (2, 70001, 1)])
@pytest.mark.parametrize("order", ["rising", "falling", "sawtooth", "one_wave"])
def test_alternatives_of_logits_in_an_order(dtype, N, V, top, order):
    """Every logit of a rising row is the best so far; a falling row's are all in the first pieces;
    a sawtooth repeats its values (equal logits, the lowest index first); a row whose best lie in
    one piece, which one wave of the four reads."""
    i = torch.arange(V, dtype=torch.float64)
    x = {"rising": i / V * 20, "falling": -i / V * 20, "sawtooth": (i % 97) / 8,
         "one_wave": torch.where((i >= V // 2) & (i < V // 2 + 100), 5 + (i % 13), -(i % 31) / 4)}[order]
    x = x.to(dtype).expand(N, V).contiguous()
    _check(x.to(DEV), (torch.arange(N) % V).to(DEV), top)
