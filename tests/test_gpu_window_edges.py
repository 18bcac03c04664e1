"""``packed_window_attention`` at the edges of what it is given: queries and norms that are not finite.

Tolerances as in test_gpu_window.py, whose checks these are.
"""
from __future__ import annotations

import pytest
import torch

from cases import to_device
from test_gpu_window import DEV, _case, _check, _run

pytestmark = pytest.mark.gpu

# D, Hq, Hkv, Q, splits: rows merged sixteen at a time from few splits and from many, by fours, and the row scan
ROWS = [(128, 8, 2, 12, None), (128, 8, 2, 12, 13), (128, 8, 2, 200, None), (64, 14, 2, 5, 1), (64, 8, 8, 33, 12), (256, 4, 2, 9, 2),
        (32, 8, 2, 7, None), (16, 8, 4, 3, 2), (128, 32, 8, 1, None), (64, 8, 2, 1, None)]


@pytest.mark.parametrize("single", [False, True])
@pytest.mark.parametrize("D,Hq,Hkv,Q,splits", ROWS)
def test_a_query_that_is_not_finite_has_no_finite_answer(D, Hq, Hkv, Q, splits, single):
    """Every score of its row is NaN, in every split; no other row shows it."""
    q, kv = _case(900 + D + Q, (Q + 300, Q + 5, Q + 77), Hq, Hkv, D, Q, 4, 4)
    dkv = to_device(kv, DEV)
    bad = q.clone()
    for b, h, i in ((0, 1, Q // 2), (1, Hq - 1, Q - 1), (2, 0, 0)):
        bad[b, h, i, (b + 5) % D] = float("nan")
    for window, sinks in ((100, 4), (1, 0), (2 ** 31, 0)):
        got = _run(bad, dkv, 0.1, window, sinks, num_splits=splits, allow_tf32=single)
        hit = bad.isnan().any(-1)
        assert not torch.isfinite(got.cpu()[hit]).any()
        clean = _run(q, dkv, 0.1, window, sinks, num_splits=splits, allow_tf32=single)
        got[hit.to(DEV)] = clean[hit.to(DEV)]
        _check(got, q, kv, 0.1, window, sinks, torch.float32, single=single)


@pytest.mark.parametrize("D,Hq,Hkv,Q,splits", ROWS)
def test_the_only_key_in_view_is_not_finite(D, Hq, Hkv, Q, splits):
    """A window of one position: the row whose own key's norm is NaN has nothing else to answer with."""
    q, kv = _case(950 + D + Q, (Q + 130, Q + 5), Hq, Hkv, D, Q, 4, 4)
    clean = _run(q, kv, 0.1, 1, 0, num_splits=splits)
    _check(clean, q, kv, 0.1, 1, 0, torch.float32)
    at = Q + 130 - 1 - Q // 2
    kv.k_norms[kv.page_table[0, at // 16], :, at % 16] = float("nan")
    got = _run(q, kv, 0.1, 1, 0, num_splits=splits)
    row = Q - 1 - Q // 2
    assert not torch.isfinite(got[0, :, row]).any()
    got[0, :, row] = clean[0, :, row]
    assert torch.equal(got, clean)


def test_one_query_of_many_sequences():
    """Enough (sequence, kv head) pairs for the merge of four heads at once."""
    lens = tuple(20 + 3 * b for b in range(72))
    q, kv = _case(71, lens, 16, 8, 128, 1, 4, 4)
    bad = q.clone()
    bad[3, 5], bad[70, 15] = float("nan"), float("nan")
    got, clean = _run(bad, kv, 0.1, 30, 2).cpu(), _run(q, kv, 0.1, 30, 2).cpu()
    _check(clean, q, kv, 0.1, 30, 2, torch.float32)
    hit = bad.isnan().any(-1)
    assert got[hit].isnan().all()
    got[hit] = clean[hit]
    _check(got, q, kv, 0.1, 30, 2, torch.float32)


@pytest.mark.parametrize("L,Q,window", [(9000, 129, 64), (9000, 130, 1), (9000, 257, 16), (9000, 400, 700), (300, 200, 64), (9000, 128, 64)])
def test_a_plan_has_splits_for_its_longest_row_block(L, Q, window):
    """Full row blocks span more positions than a partial last one. Planned for one sequence on an idle
    device, every chunk of the longest block has a split of its own."""
    from winnow_amd import packed_attention as pa
    q, kv = _case(7, (L,), 2, 2, 128, Q, 4, 4)
    splits, span = pa.window_plan_for(q.to(DEV), to_device(kv, DEV), window, 4, True)
    rows, longest = 32 if Q <= 32 else 64 if Q <= 64 else 128, 0
    for r0 in range(0, Q, rows):
        p = range(L - Q + r0, L - Q + min(r0 + rows, Q))
        lo, hi = max(p[0] - window + 1, 0), p[-1] + 1
        longest = max(longest, len({j // 64 for j in range(lo, hi)} | {0}))
    assert span == 64 and splits >= longest


@pytest.mark.parametrize("Q", [1, 9])
@pytest.mark.parametrize("S", [1024, 4096])
@pytest.mark.parametrize("D,bw", [(128, 4), (64, 8)])
def test_pages_of_many_chunks(D, bw, S, Q):
    """Views that begin and end inside a page much longer than the window."""
    q, kv = _case(40 + S + Q, (9, S + 1, 2 * S + 700, 3 * S), 4, 2, D, Q, bw, bw, S=S)
    for window, sinks in ((1, 0), (64, 4), (200, 1100), (5000, 65)):
        _check(_run(q, kv, 0.1, window, sinks), q, kv, 0.1, window, sinks, torch.float32)


@pytest.mark.parametrize("value", [float("inf"), -float("inf")])
@pytest.mark.parametrize("D,Hq,Hkv,Q,splits", ROWS)
@pytest.mark.parametrize("single", [False, True])
def test_an_infinite_query_beside_large_ones(D, Hq, Hkv, Q, splits, single, value):
    """A head of infinities does not move its neighbours."""
    q, kv = _case(300 + D + Q, (Q + 300, Q + 5), Hq, Hkv, D, Q, 4, 4, q_scale=30.0)
    dkv = to_device(kv, DEV)
    bad = q.clone()
    bad[0, 1, Q // 2, 3:] = value
    bad[1, Hq - 1, Q - 1, :] = value
    got = _run(bad, dkv, 0.1, 100, 4, num_splits=splits, allow_tf32=single)
    clean = _run(q, dkv, 0.1, 100, 4, num_splits=splits, allow_tf32=single)
    hit = (bad != q).any(-1).to(DEV)
    assert not torch.isfinite(got[hit]).any()
    got[hit] = clean[hit]
    _check(got, q, kv, 0.1, 100, 4, torch.float32, single=single)


@pytest.mark.parametrize("side", ["k_norms", "v_norms"])
@pytest.mark.parametrize("D,Hq,Hkv,Q,splits", ROWS)
def test_a_norm_in_view_that_is_nan(D, Hq, Hkv, Q, splits, side):
    """Among many other keys: the rows that see it are NaN, the others' bits are those without it."""
    L = Q + 300
    q, kv = _case(350 + D + Q, (L, Q + 5), Hq, Hkv, D, Q, 4, 4)
    clean = _run(q, kv, 0.1, 64, 2, num_splits=splits)
    at = L - 32 - (Q + 1) // 2
    getattr(kv, side)[kv.page_table[0, at // 16], :, at % 16] = float("nan")
    got = _run(q, kv, 0.1, 64, 2, num_splits=splits)
    for i in range(Q):
        p = L - Q + i
        if at <= p < at + 64:
            assert got[0, :, i].isnan().all()
        else:
            assert torch.equal(got[0, :, i], clean[0, :, i])
    assert torch.equal(got[1], clean[1])
