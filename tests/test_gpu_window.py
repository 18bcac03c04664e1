"""GPU parity of the windowed attention (``packed_window_attention``, ``wn_window_attention``)
against a plain float64 computation over the oracle's packed pages.

Tolerances, per element of the result, from the inputs that are in view, as for the tree
attention, whose arithmetic it shares. K = scale |q| |k|, V = |v| (vectors), E = the largest |v|
element. A score's error d (in nats) changes a row's weights by at most a factor e^(+-2d), so the
result by at most 2 d E to first order.

* fp32 accuracy: each factor is two fp16 terms, off by at most 2^-22, and the product of the two
  low terms is left out (2^-22): 3 2^-22 K; a score's fp32 sums round nine times, 9 2^-24 K; the
  rotation the same again. d = 2^-19 K, and the value product adds the same relative error of
  sum p |v| <= V: tol = (2 E K + V) 2^-19 plus half a step of the result.
* single terms: compared with queries and codebooks rounded the same way, so only a weight's
  rounding is left, 2^-11 V; a rotated query within fp32 rounding of a midpoint may round the
  other way: four such flips, 24 2^-10 K E / D; plus the fp32 bound and half a step of the result.
"""
from __future__ import annotations

import pytest
import torch

import window_reference as ref
from cases import build, to_device

pytestmark = pytest.mark.gpu

DEV = "cuda"
HALF_STEP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def _pa():
    from winnow_amd import packed_attention as pa
    return pa


def _case(seed, lens, Hq, Hkv, D, Q, bwk, bwv, S=16, q_scale=1.0, dtype=torch.float32, num_pages=None):
    _, kv = build(seed, len(lens), Hq, Hkv, D, lens, S, bwk, bw_v=bwv, num_pages=num_pages)
    g = torch.Generator().manual_seed(seed + 1)
    return (torch.randn(len(lens), Hq, Q, D, generator=g) * q_scale).to(dtype), kv


def _check(got, q, kv, scale, window, sinks, dtype, single=False):
    want, K, V, E = ref.window_attention(q, kv, scale, window, sinks, single)
    tol = (2 * E * K + V) * 2.0 ** -19
    if single:
        tol += 2.0 ** -11 * V + 24 * 2.0 ** -10 * K * E / q.shape[-1]
    tol = tol + HALF_STEP[dtype] * want.abs() + (2.0 ** -25 if dtype == torch.float16 else 0)
    assert got.dtype == dtype and got.shape == q.shape
    err = (got.double().cpu() - want).abs()
    assert torch.isfinite(got).all() and (err <= tol).all(), f"max err {err.max():.3e}, tol {float(tol.min()):.3e}"
    for b in range(q.shape[0]):
        hidden = q.shape[2] - int(kv.seq_lens[b])      # queries before position 0
        if hidden > 0:
            assert (got[b, :, :hidden] == 0).all()


def _run(q, kv, scale, window, sinks, **kw):
    return _pa().packed_window_attention(q.to(DEV), kv if kv.k_pages.is_cuda else to_device(kv, DEV), scale, window=window, sinks=sinks, **kw)


@pytest.mark.parametrize("D,bwk,bwv,Hq,Hkv,Q", [
    (128, 4, 4, 32, 8, 1), (128, 4, 4, 28, 4, 26), (128, 4, 6, 16, 2, 70), (128, 6, 4, 8, 8, 1), (128, 8, 8, 28, 4, 1), (128, 3, 3, 10, 1, 1),
    (128, 2, 3, 12, 4, 7), (128, 5, 8, 16, 1, 33), (128, 6, 6, 5, 1, 1), (128, 4, 8, 8, 2, 1), (128, 5, 5, 32, 2, 1), (128, 2, 2, 17, 1, 1),
    (64, 4, 4, 14, 2, 1), (64, 3, 5, 8, 8, 64), (64, 8, 2, 40, 8, 13), (256, 4, 4, 8, 2, 1), (256, 8, 8, 8, 8, 40), (256, 5, 3, 28, 4, 17),
    (32, 4, 4, 8, 2, 1), (32, 3, 8, 6, 6, 50), (16, 4, 4, 8, 2, 30), (16, 6, 2, 17, 1, 1)])
def test_window_matches_float64(D, bwk, bwv, Hq, Hkv, Q):
    """Every head_dim, every width on both sides, n_rep from 1 to 17, one query to many; lengths of
    nothing, shorter than the queries, of them alone, across chunks and pages; windows of one
    position, odd ones, wider than the sequence; no sinks, few, more than a chunk of them."""
    lens = (0, max(1, Q // 2), Q, Q + 1, Q + 63, 700)
    q, kv = _case(500 + D + 7 * Q + bwk, lens, Hq, Hkv, D, Q, bwk, bwv)
    dkv, scale = to_device(kv, DEV), D ** -0.5
    for window, sinks, splits in ((1, 0, None), (1, 3, 2), (17, 0, 1), (100, 4, None), (129, 70, 5), (333, 1, 13), (2 ** 31, 0, None), (64, 2 ** 40, None)):
        _check(_run(q, dkv, scale, window, sinks, num_splits=splits), q, kv, scale, window, sinks, torch.float32)
    _check(_run(q, dkv, scale, 150, 5, allow_tf32=True), q, kv, scale, 150, 5, torch.float32, single=True)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("Hq,Hkv,D,Q", [(32, 8, 128, 1), (28, 4, 128, 40), (8, 2, 64, 20), (8, 2, 256, 1)])
def test_window_half_types(dtype, Hq, Hkv, D, Q):
    q, kv = _case(900 + Q, (Q, 130, 515), Hq, Hkv, D, Q, 4, 4, dtype=dtype)
    scale = D ** -0.5
    _check(_run(q, kv, scale, 90, 4), q, kv, scale, 90, 4, dtype)
    _check(_run(q, kv, scale, 90, 4, out_dtype=torch.float32), q, kv, scale, 90, 4, torch.float32)


@pytest.mark.parametrize("S", [32, 64, 128, 256])
@pytest.mark.parametrize("Q", [1, 9])
def test_window_page_sizes(S, Q):
    """Pages larger than a chunk: a window that starts in the second half of one, sinks that end there."""
    q, kv = _case(40 + S, (9, 300, 257, 1000), 8, 2, 128, Q, 4, 6, S=S)
    for window, sinks in ((1, 0), (60, 4), (130, 200), (200, 65)):
        _check(_run(q, kv, 0.1, window, sinks), q, kv, 0.1, window, sinks, torch.float32)


@pytest.mark.parametrize("Q", [1, 12])
@pytest.mark.parametrize("q_scale,scale", [(50.0, 128 ** -0.5), (1e-3, 128 ** -0.5), (1.0, 0.0), (1.0, -0.1)])
def test_window_score_ranges(q_scale, scale, Q):
    q, kv = _case(77, (40, 300), 8, 2, 128, Q, 4, 4, q_scale=q_scale)
    _check(_run(q, kv, scale, 100, 4), q, kv, scale, 100, 4, torch.float32)


@pytest.mark.parametrize("Q", [1, 12])
@pytest.mark.parametrize("factor", [2.0 ** -18, 2.0 ** -8, 2.0 ** 8])
def test_window_norm_ranges(factor, Q):
    """Values whose norms are tiny or large keep their precision, whatever the norms outside the view."""
    q, kv = _case(78, (900,), 8, 2, 128, Q, 4, 4)
    kv.v_norms.copy_((kv.v_norms.float() * factor).half())
    table = kv.page_table[0].long()
    kv.v_norms[table[2:40]] = 60000.0
    kv.k_norms[table[2:40]] = 60000.0
    _check(_run(q, kv, 0.05, 200, 4), q, kv, 0.05, 200, 4, torch.float32)


@pytest.mark.parametrize("Q,S", [(1, 16), (1, 64), (1, 256), (12, 16), (12, 128), (100, 16)])
@pytest.mark.parametrize("D,bw", [(128, 4), (64, 8)])
def test_what_is_out_of_view_does_not_count(Q, S, D, bw):
    """Released pages (-1, ids of others, ids outside the pool), and NaN, infinities and the largest
    norms in every position out of view, in the pages that are partly in view too: the same bits."""
    lens = (Q + 900, 700 + Q, Q, 333 + Q)
    for window, sinks in ((50, 5), (129, 0), (1, 70), (300, 17)):
        q, kv = _case(5 + Q + window, lens, 8, 2, D, Q, bw, bw, S=S, num_pages=8 + sum(-(-L // S) for L in lens))
        clean = _run(q, kv, 0.1, window, sinks)
        _check(clean, q, kv, 0.1, window, sinks, torch.float32)
        kv.page_table = kv.page_table.clone()
        bad = torch.tensor([float("nan"), float("inf"), -float("inf"), 65504.0, -65504.0], dtype=torch.float16)
        width = kv.page_table.shape[1]
        for b, L in enumerate(lens):
            view = ref.sees(L, Q, window, sinks).any(0)
            for j in range(-(-L // S)):
                on = view[j * S:(j + 1) * S]
                page = int(kv.page_table[b, j])
                hide = torch.ones(S, dtype=torch.bool)
                hide[:len(on)] = ~on
                for norms in (kv.k_norms, kv.v_norms):
                    norms[page, :, hide] = bad[torch.arange(int(hide.sum())) % 5]
                if not on.any():
                    kv.page_table[b, j] = (-1, 0, kv.k_pages.shape[0] + 5, 2 ** 31 - 1)[j % 4]
            kv.page_table[b, -(-L // S):] = -7
        assert width == kv.page_table.shape[1]
        again = _run(q, kv, 0.1, window, sinks)
        assert torch.equal(again, clean), (window, sinks)


@pytest.mark.parametrize("Q", [1, 8])
def test_a_value_that_is_not_finite_reaches_the_rows_that_see_it(Q):
    q, kv = _case(6, (400,), 8, 2, 128, Q, 4, 4)
    clean = _run(q, kv, 0.1, 64, 2).cpu()
    at = 400 - 64 - 3                     # in view of the first queries alone, of none for Q = 1
    kv.v_norms[kv.page_table[0, at // 16], :, at % 16] = float("inf")
    got = _run(q, kv, 0.1, 64, 2).cpu()
    for i in range(Q):
        if 400 - Q + i - at < 64:
            assert not torch.isfinite(got[0, :, i]).any()
        else:
            assert torch.equal(got[0, :, i], clean[0, :, i])


@pytest.mark.parametrize("Hq,Hkv,bwk,bwv", [(32, 8, 4, 4), (28, 4, 8, 8), (8, 8, 3, 3), (24, 2, 6, 4), (5, 1, 4, 8)])
def test_row_scan_plans(Hq, Hkv, bwk, bwv):
    """The row scan of one query over any number of waves: fewer than kv heads, one, many more than there
    are chunks; ragged lengths, some empty or shorter than the sinks; and the tile scan beside it."""
    lens = (0, 3, 64, 65, 700, 1, 1300)
    q, kv = _case(60 + Hq + bwk, lens, Hq, Hkv, 128, 1, bwk, bwv)
    dkv = to_device(kv, DEV)
    for window, sinks in ((100, 4), (1, 0), (257, 33)):
        for plan in ((1, 0), (3, 0), (Hkv, 0), (17 * Hkv, 0), (2048, 0), (2, 64), (1, 128)):
            _check(_run(q, dkv, 0.09, window, sinks, plan=plan), q, kv, 0.09, window, sinks, torch.float32)
    if bwk in (4, 6) and bwv in (4, 6):
        _check(_run(q, dkv, 0.09, 100, 4, allow_tf32=True, plan=(40, 0)), q, kv, 0.09, 100, 4, torch.float32, single=True)


def test_a_plan_that_the_layout_does_not_take():
    """The row scan asks for the decode's alignments: refused where they are not met, or for other shapes."""
    import dataclasses
    from winnow_amd import _lib
    pa = _pa()
    q, kv = _case(3, (70, 300), 8, 2, 128, 1, 4, 4)
    dkv = to_device(kv, DEV)
    flat = torch.zeros(dkv.k_pages.numel() + 4, dtype=torch.uint8, device=DEV)
    odd = dataclasses.replace(dkv, k_pages=flat[4:].view(dkv.k_pages.shape).copy_(dkv.k_pages))
    assert pa.window_plan_for(q.to(DEV), dkv, 50, 4, True)[1] == 0 and pa.window_plan_for(q.to(DEV), odd, 50, 4, True)[1] > 0
    with pytest.raises(_lib.WinnowHipError, match="row scan"):
        _run(q, odd, 0.1, 50, 4, plan=(64, 0))
    _check(_run(q, odd, 0.1, 50, 4), q, kv, 0.1, 50, 4, torch.float32)
    q, kv = _case(4, (70, 300), 8, 2, 128, 2, 4, 4)
    with pytest.raises(pa.UnsupportedLayout, match="sizes"):
        _run(q, kv, 0.1, 50, 4, plan=(64, 0))
    q, kv = _case(5, (70, 300), 8, 2, 64, 1, 4, 4)
    with pytest.raises(pa.UnsupportedLayout, match="sizes"):
        _run(q, kv, 0.1, 50, 4, plan=(64, 0))


def test_a_wide_window_is_the_causal_mask():
    pa = _pa()
    q, kv = _case(11, (5, 64, 200), 32, 8, 128, 1, 4, 4)
    _check(pa.packed_decode_attention(q.to(DEV), to_device(kv, DEV), 0.09), q, kv, 0.09, 1000, 0, torch.float32)
    _check(_run(q, kv, 0.09, 200, 0), q, kv, 0.09, 1000, 0, torch.float32)
    q, kv = _case(12, (9, 64, 200), 32, 8, 128, 9, 4, 4)
    chain = torch.arange(-1, 8, dtype=torch.int32)[None].expand(3, -1).to(DEV)
    tree = pa.packed_tree_attention(q.to(DEV), to_device(kv, DEV), 0.09, chain)
    _check(tree, q, kv, 0.09, 10 ** 6, 0, torch.float32)
    _check(_run(q, kv, 0.09, 10 ** 6, 0), q, kv, 0.09, 10 ** 6, 0, torch.float32)


@pytest.mark.parametrize("Q", [1, 7])
@pytest.mark.parametrize("bwk,bwv", [(4, 4), (3, 6), (5, 5)])
def test_strided_operands(Q, bwk, bwv):
    """q as (B, Q, Hq, D) memory with a gap; pages and norms as one layer of a pool, 4-byte aligned
    only; a page table that is a window of a wider one; a handle without host mirrors."""
    import dataclasses
    q, kv = _case(21, (70, 300), 8, 2, 128, Q, bwk, bwv)
    want = _run(q, kv, 0.1, 77, 3)
    dkv = to_device(kv, DEV)
    qm = torch.zeros(2, Q, 8, 131, device=DEV)
    qm[..., 1:129] = q.to(DEV).transpose(1, 2)

    def pool(pages):
        P, Hkv, S, NB = pages.shape
        flat = torch.zeros(P * (Hkv * S * NB + 12) + 4, dtype=torch.uint8, device=DEV)
        view = flat[4:].as_strided((P, Hkv, S, NB), (Hkv * S * NB + 12, S * NB, NB, 1))
        return view.copy_(pages)

    def wide(norms):
        P, Hkv, S = norms.shape
        return torch.zeros(P * (Hkv * S + 3) + 1, dtype=norms.dtype, device=DEV)[1:].as_strided((P, Hkv, S), (Hkv * S + 3, S, 1)).copy_(norms)
    table = torch.full((2, kv.page_table.shape[1] + 5), -1, dtype=torch.int32, device=DEV)
    table[:, 2:-3] = dkv.page_table
    other = dataclasses.replace(dkv, k_pages=pool(dkv.k_pages), v_pages=pool(dkv.v_pages), k_norms=wide(dkv.k_norms), v_norms=wide(dkv.v_norms),
                                page_table=table[:, 2:-3], seq_lens_host=None, page_table_host=None)
    got = _pa().packed_window_attention(qm[..., 1:129].transpose(1, 2), other, 0.1, window=77, sinks=3)
    _check(got, q, kv, 0.1, 77, 3, torch.float32)
    _check(want, q, kv, 0.1, 77, 3, torch.float32)


@pytest.mark.parametrize("Q", [1, 5])
def test_plans_workspaces_and_streams(Q):
    """A plan made for other lengths, a caller's workspace (too small: refused), another stream."""
    pa = _pa()
    q, kv = _case(31, (900, 30, 400), 8, 2, 128, Q, 4, 4)
    dkv, dq = to_device(kv, DEV), q.to(DEV)
    want = pa.packed_window_attention(dq, dkv, 0.1, window=300, sinks=4)
    _check(want, q, kv, 0.1, 300, 4, torch.float32)
    need = pa.window_workspace_bytes(3, 8, 2, Q, 128, 16, dkv.page_table.shape[1], 300, 4, 7, 64)
    ws = torch.full((need,), 255, dtype=torch.uint8, device=DEV)
    got = pa.packed_window_attention(dq, dkv, 0.1, window=300, sinks=4, num_splits=7, workspace=ws)
    _check(got, q, kv, 0.1, 300, 4, torch.float32)
    with pytest.raises(pa.UnsupportedLayout, match="workspace"):
        pa.packed_window_attention(dq, dkv, 0.1, window=300, sinks=4, num_splits=7, workspace=ws[:-1])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = pa.packed_window_attention(dq, dkv, 0.1, window=300, sinks=4)
    side.synchronize()
    assert torch.equal(got, want)


@pytest.mark.parametrize("Q", [1, 6])
@pytest.mark.parametrize("D", [128, 64])
def test_graph_replays_with_lengths_that_change(Q, D):
    """Captured once, replayed as the sequences grow, shrink and empty, between eager calls."""
    pa = _pa()
    q, kv = _case(41, (1000, 500, 64), 8, 2, D, Q, 4, 4)
    dkv, dq = to_device(kv, DEV), q.to(DEV)
    call = lambda: pa.packed_window_attention(dq, dkv, 0.1, window=170, sinks=4, check_ranges=False)  # noqa: E731
    dkv.seq_lens_host = None
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for lens in ((1000, 500, 64), (10, 499, 1), (0, 0, 64), (999, 3, 0), (640, 320, 50)):
        kv.seq_lens.copy_(torch.tensor(lens))
        dkv.seq_lens.copy_(torch.tensor(lens))
        graph.replay()
        torch.cuda.synchronize()
        _check(out, q, kv, 0.1, 170, 4, torch.float32)
        _check(call(), q, kv, 0.1, 170, 4, torch.float32)


def test_a_long_prompt_chunk():
    """Many row blocks, each with a window of its own."""
    q, kv = _case(51, (1500,), 4, 2, 128, 700, 4, 4)
    for window, sinks in ((64, 4), (500, 0), (900, 33)):
        _check(_run(q, kv, 0.09, window, sinks), q, kv, 0.09, window, sinks, torch.float32)
        _check(_run(q, kv, 0.09, window, sinks, allow_tf32=True), q, kv, 0.09, window, sinks, torch.float32, single=True)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("D,Hq,Hkv,Q,splits", [(128, 32, 8, 70, None), (64, 6, 2, 500, 3), (32, 10, 2, 171, None), (16, 8, 8, 99, 17),
                                               (256, 8, 4, 133, 2)])
def test_window_many_rows(D, Hq, Hkv, Q, splits, dtype):
    """Rows whose merge has more tiles of sixteen than the device's work-groups that stay, or fewer;
    sequences of nothing and of fewer positions than queries between long ones."""
    lens = (Q + 40, 0, 300 + Q, Q // 3, Q, 90 + Q, 1, 2 * Q, Q + 7, Q + 129, Q, 64 + Q) * (3 if D == 128 else 1)
    q, kv = _case(60 + D, lens, Hq, Hkv, D, Q, 4, 4, dtype=dtype)
    for window, sinks in ((100, 4), (33, 0)):
        _check(_run(q, kv, D ** -0.5, window, sinks, num_splits=splits), q, kv, D ** -0.5, window, sinks, dtype)


@pytest.mark.parametrize("single", [False, True])
@pytest.mark.parametrize("D,bwk,bwv", [(128, 4, 4), (128, 8, 3), (64, 4, 4), (64, 5, 6), (32, 4, 4), (32, 2, 8), (16, 4, 4), (16, 3, 3)])
@pytest.mark.parametrize("Q", [61, 64])
def test_window_blocks_of_256_rows(D, bwk, bwv, Q, single):
    """Enough (sequence, kv head) pairs of 244 and 256 rows for the widest row blocks, every kind of kernel:
    lengths of nothing, of part of the queries, across chunks; windows that begin and end inside one."""
    lens = (Q + 300, 0, Q // 2, Q + 7, 2 * Q, 777)
    q, kv = _case(70 + D + Q, lens, 24, 6, D, Q, bwk, bwv)
    dkv, scale = to_device(kv, DEV), D ** -0.5
    for window, sinks, splits in ((100, 5, None), (1, 0, 2), (2 ** 31, 0, 1), (64, 66, 7)):
        got = _run(q, dkv, scale, window, sinks, num_splits=splits, allow_tf32=single)
        _check(got, q, kv, scale, window, sinks, torch.float32, single=single)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("D,Hq,Hkv,Q", [(128, 16, 4, 150), (256, 8, 2, 131)])
def test_window_many_rows_strided(D, Hq, Hkv, Q, dtype):
    """As (B, Q, Hq, D) memory, aligned, and with rows of an odd length; the same bits."""
    lens = (Q + 40, Q // 2, 300 + Q, Q, 90 + Q, Q + 7, 2 * Q, 1, 0, Q + 129, Q, Q) * 3
    q, kv = _case(33 + D, lens, Hq, Hkv, D, Q, 4, 6, dtype=dtype)
    dkv = to_device(kv, DEV)
    want = _run(q, dkv, 0.1, 70, 3)
    _check(want, q, kv, 0.1, 70, 3, dtype)
    heads = q.to(DEV).transpose(1, 2).contiguous().transpose(1, 2)
    odd = torch.zeros(len(lens), Q, Hq, D + 3, dtype=dtype, device=DEV)[..., 1:D + 1].transpose(1, 2)
    odd.copy_(q)
    for view in (heads, odd):
        got = _pa().packed_window_attention(view, dkv, 0.1, window=70, sinks=3)
        assert torch.equal(got.view(torch.uint8), want.view(torch.uint8))
