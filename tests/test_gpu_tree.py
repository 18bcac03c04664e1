"""GPU parity of the tree attention (``packed_tree_attention``, ``wn_tree_attention``) against a
plain float64 computation over the oracle's packed pages.

Tolerances, per element of the result, from the inputs. K = scale |q| |k|, V = |v| (vectors), E =
the largest |v| element. A score's error d (in nats) changes a row's weights by at most a factor
e^(+-2d), so the result by at most 2 d E to first order.

* fp32 accuracy: each factor is two fp16 terms, off by at most 2^-22 (half a step of the second
  term, 2^-11 of 2^-11), and the product of the two low terms is left out (2^-22): 3 2^-22 K; the
  fp32 sums of a score round nine times on the way (five levels of a 32-term product, four
  K-steps), 9 2^-24 K; the rotation the same again. d = 2^-19 K, and the value product adds the
  same relative error of sum p |v| <= V: tol = (2 E K + V) 2^-19 plus half a step of the result.
* single terms: compared with queries and codebooks rounded the same way, so only a weight's
  rounding is left, 2^-11 of it (|error| <= 2^-11 V); a rotated query within fp32 rounding of a
  midpoint may round the other way: four such flips of one of D terms, each 2^-10 of a term of at
  most 3 / sqrt(D) of K over sqrt(D) of its length: tol = 2^-11 V + 24 2^-10 K E / D, plus the
  fp32 bound, plus half a step of the result.
"""
from __future__ import annotations

import pytest
import torch

import tree_reference as ref
from cases import build, to_device

pytestmark = pytest.mark.gpu

DEV = "cuda"
HALF_STEP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def _pa():
    from winnow_amd import packed_attention as pa
    return pa


def _case(seed, lens, Hq, Hkv, D, T, bwk, bwv, S=16, q_scale=1.0, dtype=torch.float32, num_pages=None):
    _, kv = build(seed, len(lens), Hq, Hkv, D, lens, S, bwk, bw_v=bwv, num_pages=num_pages)
    g = torch.Generator().manual_seed(seed + 1)
    q = (torch.randn(len(lens), Hq, T, D, generator=g) * q_scale).to(dtype)
    return q, kv, ref.random_parents(len(lens), T, seed + 2)


def _tol(q, kv, scale, want, dtype, single):
    K, V, E = ref.bounds(q, kv, scale)
    tol = (2 * E * K + V) * 2.0 ** -19
    if single:
        tol += 2.0 ** -11 * V + 24 * 2.0 ** -10 * K * E / q.shape[-1]
    return tol + HALF_STEP[dtype] * want.abs() + (2.0 ** -25 if dtype == torch.float16 else 0)


def _check(got, q, kv, parents, scale, dtype, single=False):
    want = ref.tree_attention(q, kv, parents, scale, single)
    err = (got.double().cpu() - want).abs()
    assert got.dtype == dtype and got.shape == q.shape
    tol = _tol(q, kv, scale, want, dtype, single)
    assert torch.isfinite(got).all() and (err <= tol).all(), f"max err {err.max():.3e}, tol {float(tol.min()):.3e}"
    for b in range(q.shape[0]):
        if int(kv.seq_lens[b]) == 0:
            assert (got[b] == 0).all()


@pytest.mark.parametrize("D,bwk,bwv,Hq,Hkv,T", [
    (128, 4, 4, 32, 8, 8), (128, 4, 4, 28, 4, 26), (128, 4, 6, 16, 2, 64), (128, 6, 4, 8, 8, 1), (128, 8, 8, 28, 4, 5),
    (128, 2, 3, 12, 4, 7), (128, 5, 8, 16, 1, 33), (64, 4, 4, 14, 2, 5), (64, 3, 5, 8, 8, 64), (64, 8, 2, 40, 8, 13),
    (64, 6, 6, 64, 4, 11), (256, 4, 4, 8, 2, 9), (256, 8, 8, 8, 8, 64), (256, 5, 3, 28, 4, 17), (32, 4, 4, 8, 2, 16),
    (32, 3, 8, 6, 6, 2), (16, 4, 4, 8, 2, 30), (16, 3, 5, 8, 8, 3), (16, 6, 2, 17, 1, 6)])
def test_tree_matches_float64(D, bwk, bwv, Hq, Hkv, T):
    """Every head_dim, every width on both sides, n_rep from 1 to 17, one node to 64; lengths of
    nothing, shorter than the tree (its first nodes do not exist), of the tree alone, one more,
    across chunks and pages; the library's splits, one, and more than chunks."""
    lens = (0, max(1, T // 2), T, T + 1, T + 63, 700)
    q, kv, parents = _case(500 + D + 7 * T + bwk, lens, Hq, Hkv, D, T, bwk, bwv)
    scale = D ** -0.5
    dkv = to_device(kv, DEV)
    for splits in (None, 1, 13):
        got = _pa().packed_tree_attention(q.to(DEV), dkv, scale, parents.to(DEV), num_splits=splits)
        _check(got, q, kv, parents, scale, torch.float32)
    one = _pa().packed_tree_attention(q.to(DEV), dkv, scale, parents.to(DEV), allow_tf32=True)
    _check(one, q, kv, parents, scale, torch.float32, single=True)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("Hq,Hkv,D,T", [(32, 8, 128, 8), (28, 4, 128, 40), (8, 2, 64, 20), (8, 2, 256, 6)])
def test_tree_half_types(dtype, Hq, Hkv, D, T):
    """bf16 takes single-term products, fp16 fp32-accurate ones; each result rounded once."""
    q, kv, parents = _case(900 + T, (T, 130, 515), Hq, Hkv, D, T, 4, 4, dtype=dtype)
    scale = D ** -0.5
    got = _pa().packed_tree_attention(q.to(DEV), to_device(kv, DEV), scale, parents.to(DEV))
    _check(got, q, kv, parents, scale, dtype, single=dtype == torch.bfloat16)
    wide = _pa().packed_tree_attention(q.to(DEV), to_device(kv, DEV), scale, parents.to(DEV), out_dtype=torch.float32)
    _check(wide, q, kv, parents, scale, torch.float32)


@pytest.mark.parametrize("S", [32, 64, 256])
def test_tree_page_sizes(S):
    q, kv, parents = _case(40 + S, (9, 300, 257), 8, 2, 128, 9, 4, 6, S=S)
    got = _pa().packed_tree_attention(q.to(DEV), to_device(kv, DEV), 0.1, parents.to(DEV))
    _check(got, q, kv, parents, 0.1, torch.float32)


@pytest.mark.parametrize("q_scale,scale", [(50.0, 128 ** -0.5), (1e-3, 128 ** -0.5), (1.0, 0.0), (1.0, -0.1)])
def test_tree_score_ranges(q_scale, scale):
    """Scores in the hundreds, tiny queries, no scale and a negative one."""
    q, kv, parents = _case(77, (40, 300), 8, 2, 128, 12, 4, 4, q_scale=q_scale)
    got = _pa().packed_tree_attention(q.to(DEV), to_device(kv, DEV), scale, parents.to(DEV))
    want = ref.tree_attention(q, kv, parents, scale)
    K, V, E = ref.bounds(q, kv, abs(scale))
    tol = (2 * E * K + V) * 2.0 ** -19 + 2.0 ** -24 * want.abs()
    assert ((got.double().cpu() - want).abs() <= tol).all()


@pytest.mark.parametrize("factor", [2.0 ** -18, 2.0 ** -8, 2.0 ** 8])
def test_tree_norm_ranges(factor):
    """Values whose norms are tiny (down to fp16's smallest) or large keep their precision, also
    behind a chunk of zero vectors and one of other magnitude."""
    q, kv, parents = _case(78, (300,), 8, 2, 128, 12, 4, 4)
    kv.v_norms.copy_((kv.v_norms.float() * factor).half())
    S, table = 16, kv.page_table[0]
    kv.v_norms[table[:4].long()] = 0
    kv.v_norms[table[4:8].long()] *= 0.01
    got = _pa().packed_tree_attention(q.to(DEV), to_device(kv, DEV), 0.05, parents.to(DEV))
    _check(got, q, kv, parents, 0.05, torch.float32)


def test_a_chain_is_the_causal_mask():
    """parents[i] = i - 1 is the prefill's offset causal mask."""
    pa = _pa()
    q, kv, _ = _case(11, (5, 64, 200), 32, 8, 128, 16, 4, 4)
    chain = torch.arange(-1, 15, dtype=torch.int32)[None].expand(3, -1)
    got = pa.packed_tree_attention(q.to(DEV), to_device(kv, DEV), 0.09, chain.to(DEV), allow_tf32=True)
    pre = pa.packed_prefill_attention(q.to(DEV), to_device(kv, DEV), 0.09)
    assert (got - pre).abs().max() < 4e-3     # both round each factor to 11 bits, the weights apart
    _check(pa.packed_tree_attention(q.to(DEV), to_device(kv, DEV), 0.09, chain.to(DEV)), q, kv, chain, 0.09, torch.float32)


def test_one_tree_for_all_and_strided_operands():
    """A parents row shared by stride 0; q as (B, T, Hq, D) memory with a gap; pages and norms as
    one layer of a pool with odd page gaps; a page table that is a window of a wider one."""
    q, kv, parents = _case(12, (17, 100, 333), 8, 2, 128, 10, 4, 6)
    parents = parents[:1].expand(3, -1)
    d = to_device(kv, DEV)
    wide = torch.zeros(3, 10, 9, 132, device=DEV)
    wide[:, :, :8, :128] = q.to(DEV).transpose(1, 2)
    qs = wide[:, :, :8, :128].transpose(1, 2)
    P = d.k_pages.shape[0]
    for name in ("k_pages", "v_pages", "k_norms", "v_norms"):
        t = getattr(d, name)
        pool = torch.zeros(P, 3, 2, *t.shape[1:], dtype=t.dtype, device=DEV)
        pool[:, 1, 1] = t
        setattr(d, name, pool[:, 1, 1])
    table = torch.full((3, d.page_table.shape[1] + 5), -7, dtype=torch.int32, device=DEV)
    table[:, 2:-3] = d.page_table
    d.page_table = table[:, 2:-3]
    got = _pa().packed_tree_attention(qs, d, 0.08, parents[:1].to(DEV).expand(3, -1))
    _check(got, q, kv, parents, 0.08, torch.float32)


def test_what_a_row_does_not_see_does_not_reach_it():
    """Norms that are infinite or NaN behind the sequence's end and on drafted tokens: only rows
    that see such a token are touched by it."""
    q, kv, parents = _case(13, (21, 90), 8, 2, 128, 12, 4, 4)
    parents[:] = torch.tensor([-1, 0, 0, 1, 2, 2, -1, 6, 4, 3, 7, 5], dtype=torch.int32)
    clean = _pa().packed_tree_attention(q.to(DEV), to_device(kv, DEV), 0.08, parents.to(DEV))
    for b, L in enumerate((21, 90)):
        for side in ("k", "v"):
            norms = getattr(kv, f"{side}_norms")
            last = int(kv.page_table[b, (L - 1) // 16])
            norms[last, :, L % 16:] = float("nan")                  # neither length fills its last page
            node = L - 12 + 6                                       # node 6: seen by 6, 7 and 10
            norms[int(kv.page_table[b, node // 16]), :, node % 16] = float("inf")
    got = _pa().packed_tree_attention(q.to(DEV), to_device(kv, DEV), 0.08, parents.to(DEV))
    rest = [i for i in range(12) if i not in (6, 7, 10)]
    assert torch.equal(got[:, :, rest], clean[:, :, rest])
    assert not torch.isfinite(got[:, :, [6, 7, 10]]).any(-1).all()


def test_parents_out_of_order_hang_on_the_history_without_the_check():
    """With ``check_ranges`` off a parent that is no earlier node counts as -1 (no read goes astray)."""
    q, kv, _ = _case(14, (40,), 8, 2, 64, 6, 4, 4)
    bad = torch.tensor([[5, 0, 9, -3, 4, 2 ** 31 - 1]], dtype=torch.int32)
    good = torch.tensor([[-1, 0, -1, -1, -1, -1]], dtype=torch.int32)
    d = to_device(kv, DEV)
    a = _pa().packed_tree_attention(q.to(DEV), d, 0.1, bad.to(DEV), check_ranges=False)
    assert torch.equal(a, _pa().packed_tree_attention(q.to(DEV), d, 0.1, good.to(DEV)))


def test_the_result_is_the_same_every_time_and_for_each_sequence_alone():
    q, kv, parents = _case(15, (70, 400, 33), 28, 4, 128, 20, 4, 4, dtype=torch.bfloat16)
    pa, d = _pa(), to_device(kv, DEV)
    a = pa.packed_tree_attention(q.to(DEV), d, 0.08, parents.to(DEV), num_splits=3)
    assert torch.equal(a, pa.packed_tree_attention(q.to(DEV), d, 0.08, parents.to(DEV), num_splits=3))
    for b in range(3):
        one = pa.PackedKV(d.k_pages, d.k_norms, d.v_pages, d.v_norms, d.page_table[b:b + 1], d.seq_lens[b:b + 1].clone(),
                          d.k_quant, d.v_quant, 128)
        got = pa.packed_tree_attention(q[b:b + 1].to(DEV), one, 0.08, parents[b:b + 1].to(DEV), num_splits=3)
        assert torch.equal(got, a[b:b + 1])


def test_own_stream_and_graph_replays():
    """On a stream of its own, and captured: every replay equals the eager result on the operands
    as they are then, with eager work between the replays."""
    pa = _pa()
    q, kv, parents = _case(16, (50, 300), 8, 2, 128, 9, 4, 4)
    d, dq, dp = to_device(kv, DEV), q.to(DEV), parents.to(DEV)
    want = pa.packed_tree_attention(dq, d, 0.08, dp)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = pa.packed_tree_attention(dq, d, 0.08, dp)
    side.synchronize()
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = pa.packed_tree_attention(dq, d, 0.08, dp, check_ranges=False)
    for k in range(4):
        dq.copy_(q.to(DEV) * (1 + k))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, pa.packed_tree_attention(dq, d, 0.08, dp))


def test_a_workspace_of_the_callers():
    pa = _pa()
    q, kv, parents = _case(17, (50, 300), 8, 2, 128, 9, 4, 4)
    d = to_device(kv, DEV)
    need = pa.tree_workspace_bytes(2, 8, 2, 9, 128, 4)
    ws = torch.full((need + 512,), 255, dtype=torch.uint8, device=DEV)
    got = pa.packed_tree_attention(q.to(DEV), d, 0.08, parents.to(DEV), num_splits=4, workspace=ws[:need])
    _check(got, q, kv, parents, 0.08, torch.float32)
    assert (ws[need:] == 255).all()
    with pytest.raises(pa.UnsupportedLayout, match="workspace"):
        pa.packed_tree_attention(q.to(DEV), d, 0.08, parents.to(DEV), num_splits=4, workspace=ws[:need - 256])


def test_pages_past_four_gigabytes():
    """Page ids whose byte offset passes 2^32 on both sides."""
    q, kv, parents = _case(18, (100,), 8, 8, 128, 9, 4, 4)
    d = to_device(kv, DEV)
    P, n = (1 << 32) // (8 * 16 * 64) + 4096, d.k_pages.shape[0]
    ids = torch.arange(P - n, P)
    for name in ("k_pages", "v_pages", "k_norms", "v_norms"):
        t = getattr(d, name)
        big = torch.empty(P, *t.shape[1:], dtype=t.dtype, device=DEV)
        big[P - n:] = t
        setattr(d, name, big)
    table = kv.page_table.clone()
    table[table >= 0] = ids[table[table >= 0].long()].int()
    d.page_table, d.page_table_host = table.to(DEV), table
    got = _pa().packed_tree_attention(q.to(DEV), d, 0.08, parents.to(DEV))
    _check(got, q, kv, parents, 0.08, torch.float32)


def _wide_table(d, columns):
    """The same sequences behind a page table with room for ``columns`` pages each: what the kernel
    variants are chosen by."""
    table = torch.zeros(d.page_table.shape[0], columns, dtype=torch.int32, device=DEV)
    table[:, :d.page_table.shape[1]] = d.page_table
    d.page_table = table
    return d


@pytest.mark.parametrize("bwk,bwv", [(4, 4), (4, 6), (6, 4), (6, 6)])
@pytest.mark.parametrize("Hq,Hkv,T", [(16, 4, 1), (16, 4, 8), (28, 4, 9), (4, 4, 64)])
def test_tree_of_long_contexts(bwk, bwv, Hq, Hkv, T):
    """What a table with room for 5 x 4 x 32,768 positions takes (4 and 6 bits, single terms), at
    lengths of nothing, inside the tree, across chunks and long; partial blocks of 32 rows."""
    lens = (0, max(1, T // 2), T + 63, 700, 3001)
    q, kv, parents = _case(1700 + T + bwk * bwv, lens, Hq, Hkv, 128, T, bwk, bwv, dtype=torch.bfloat16)
    d = _wide_table(to_device(kv, DEV), 2048)
    for splits in (None, 1, 13):
        got = _pa().packed_tree_attention(q.to(DEV), d, 0.09, parents.to(DEV), num_splits=splits)
        _check(got, q, kv, parents, 0.09, torch.bfloat16, single=True)
    again = _pa().packed_tree_attention(q.to(DEV), d, 0.09, parents.to(DEV), num_splits=13)
    assert torch.equal(got, again)


def test_long_contexts_what_a_row_does_not_see_does_not_reach_it():
    q, kv, parents = _case(18, (21, 90, 200, 40), 8, 4, 128, 12, 4, 6, dtype=torch.bfloat16)
    parents[:] = torch.tensor([-1, 0, 0, 1, 2, 2, -1, 6, 4, 3, 7, 5], dtype=torch.int32)
    clean = _pa().packed_tree_attention(q.to(DEV), _wide_table(to_device(kv, DEV), 2048), 0.08, parents.to(DEV))
    for b, L in enumerate((21, 90, 200, 40)):
        for side in ("k", "v"):
            norms = getattr(kv, f"{side}_norms")
            norms[int(kv.page_table[b, (L - 1) // 16]), :, (L - 1) % 16 + 1:] = float("nan")
            node = L - 12 + 6                                       # node 6: seen by 6, 7 and 10
            norms[int(kv.page_table[b, node // 16]), :, node % 16] = float("inf")
    got = _pa().packed_tree_attention(q.to(DEV), _wide_table(to_device(kv, DEV), 2048), 0.08, parents.to(DEV))
    rest = [i for i in range(12) if i not in (6, 7, 10)]
    assert torch.equal(got[:, :, rest], clean[:, :, rest])
    assert not torch.isfinite(got[:, :, [6, 7, 10]].float()).any(-1).all()


@pytest.mark.parametrize("columns", [0, 2048])
def test_a_captured_call_at_lengths_that_grow_and_end(columns):
    """Captured at short lengths (few splits planned), replayed at longer, shorter and empty ones."""
    pa = _pa()
    B, T = 5, 9
    q, kv, parents = _case(19, (3000,) * B, 8, 2, 128, T, 4, 4, dtype=torch.bfloat16)
    d, dq, dp = to_device(kv, DEV), q.to(DEV), parents.to(DEV)
    if columns:
        d = _wide_table(d, 16 * columns)
    d.seq_lens.fill_(20)
    d.seq_lens_host = torch.full((B,), 20, dtype=torch.int32)
    assert pa.tree_plan_for(dq, d, False)[2] <= B
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = pa.packed_tree_attention(dq, d, 0.08, dp, check_ranges=False)
    for lens in ((20,) * B, (3000, 0, 1, 2999, 64), (0,) * B, (3000,) * B, (10, 700, 0, 0, 129)):
        kv.seq_lens.copy_(torch.tensor(lens, dtype=kv.seq_lens.dtype))
        d.seq_lens_host = torch.tensor(lens, dtype=torch.int32)
        d.seq_lens.copy_(d.seq_lens_host)
        graph.replay()
        torch.cuda.synchronize()
        _check(out, q, kv, parents, 0.08, torch.bfloat16, single=True)
        _check(pa.packed_tree_attention(dq, d, 0.08, dp), q, kv, parents, 0.08, torch.bfloat16, single=True)


@pytest.mark.parametrize("columns", [0, 1024])
def test_many_sequences_some_of_them_empty(columns):
    """More sequences than a wave has lanes, empty ones between and at both ends."""
    lens = [0, 0, 5] + [(37 * i) % 90 if i % 3 else 0 for i in range(135)] + [400, 0]
    q, kv, parents = _case(20, lens, 4, 2, 128, 3, 4, 4, dtype=torch.bfloat16)
    d = to_device(kv, DEV)
    if columns:
        d = _wide_table(d, columns)
    for splits in (None, 5):
        got = _pa().packed_tree_attention(q.to(DEV), d, 0.08, parents.to(DEV), num_splits=splits)
        _check(got, q, kv, parents, 0.08, torch.bfloat16, single=True)


@pytest.mark.parametrize("bwk,bwv", [(4, 4), (8, 3)])
@pytest.mark.parametrize("D", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("Hq,Hkv,T", [(6, 2, 33), (12, 1, 64)])
def test_more_rows_than_a_block(D, bwk, bwv, Hq, Hkv, T):
    """99 and 768 rows a kv head: whole row blocks, and ones whose last waves have none."""
    q, kv, parents = _case(1900 + D + T + bwk, (T + 5, 0, 333), Hq, Hkv, D, T, bwk, bwv)
    d, scale = to_device(kv, DEV), D ** -0.5
    got = _pa().packed_tree_attention(q.to(DEV), d, scale, parents.to(DEV))
    _check(got, q, kv, parents, scale, torch.float32)
    one = _pa().packed_tree_attention(q.to(DEV), d, scale, parents.to(DEV), allow_tf32=True)
    _check(one, q, kv, parents, scale, torch.float32, single=True)


def test_a_workspace_that_is_no_buffer_is_refused():
    pa = _pa()
    q, kv, parents = _case(21, (50,), 8, 2, 128, 5, 4, 4)
    d = to_device(kv, DEV)
    need = pa.tree_workspace_bytes(1, 8, 2, 5, 128, 2)
    one = torch.zeros(1, dtype=torch.uint8, device=DEV)
    for ws in (one.expand(need), torch.zeros(2 * need, dtype=torch.uint8, device=DEV)[::2]):
        with pytest.raises(pa.UnsupportedLayout, match="workspace"):
            pa.packed_tree_attention(q.to(DEV), d, 0.1, parents.to(DEV), num_splits=2, workspace=ws)


def test_host_mirrors_are_checked_and_need_not_be_int32():
    """The mirrors in other types and strides, and out of range: as without them."""
    pa = _pa()
    q, kv, parents = _case(22, (50, 300), 8, 2, 128, 5, 4, 4)
    d, dq, dp = to_device(kv, DEV), q.to(DEV), parents.to(DEV)
    want = pa.packed_tree_attention(dq, d, 0.1, dp)
    lens, table = kv.seq_lens.to(torch.int32), kv.page_table.to(torch.int32)
    wide = torch.stack([table, table], -1).transpose(1, 2)[:, 0]
    for h_lens, h_table, h_parents in ((lens, table, parents), (lens.long(), table.long(), parents.long()),
                                       (lens, wide, parents.t().contiguous().t())):
        d.seq_lens_host, d.page_table_host = h_lens, h_table
        assert torch.equal(pa.packed_tree_attention(dq, d, 0.1, dp, parents_host=h_parents), want)
    far, low = lens.clone(), table.clone()
    far[1] = table.shape[1] * 16 + 1
    low[0, 0] = -1
    late = parents.clone()
    late[1, 2] = 2
    for h_lens, h_table, h_parents in ((far, table, parents), (lens, low, parents), (lens, table, late), (lens, table, parents[:1])):
        d.seq_lens_host, d.page_table_host = h_lens, h_table
        with pytest.raises(pa.UnsupportedLayout):
            pa.packed_tree_attention(dq, d, 0.1, dp, parents_host=h_parents)
