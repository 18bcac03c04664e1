"""GPU parity of ``commit_kv`` (``wn_commit_kv``): rows move, bit for bit, nothing else changes."""
from __future__ import annotations

import pytest
import torch

import tree_reference as ref

pytestmark = pytest.mark.gpu

DEV = "cuda"


def _commit(*a, **k):
    from winnow_amd.packed_backend import commit_kv
    return commit_kv(*a, **k)


def _table(B, need, S, g, spare=3):
    order = torch.randperm(B * need + spare, generator=g)
    return order[:B * need].view(B, need).int(), B * need + spare


def _fill(shape, dtype, g):
    t = torch.randint(0, 256, (*shape[:-1], shape[-1] * (1 if dtype == torch.uint8 else dtype.itemsize)), generator=g, dtype=torch.uint8)
    return t.view(dtype)


def _bits(t):
    return t.contiguous().view(torch.uint8)


def _check(kp, vp, kn, vn, table, start, path, counts, nodes, **kw):
    dev = [None if t is None else t.to(DEV) for t in (kp, vp, kn, vn)]
    lengths = _commit(*dev, table.to(DEV), start.to(DEV), path.to(DEV), counts.to(DEV), nodes=nodes, **kw)
    assert torch.equal(lengths.cpu(), start + counts.clamp(0, path.shape[1]))
    axis = kp.dim() - 4
    for got, was in zip(dev, (kp, vp, kn, vn)):
        if was is not None:
            assert torch.equal(_bits(got.cpu()), _bits(ref.commit(was, table, start, path, counts, nodes, axis)))


def _branches(B, A, nodes, g):
    return torch.stack([torch.randperm(nodes, generator=g)[:A].sort().values for _ in range(B)]).int()


@pytest.mark.parametrize("D,bwk,bwv,S", [(128, 4, 4, 16), (128, 6, 3, 32), (64, 8, 5, 16), (256, 8, 2, 16), (16, 3, 5, 16),
                                         (16, 2, 6, 64), (32, 3, 3, 16)])
@pytest.mark.parametrize("layers", [None, 3])
def test_packed_pages(D, bwk, bwv, S, layers):
    """Row lengths from 4 to 256 bytes, one layer or a pool of three; branches of every length,
    none accepted and all, over page borders."""
    g = torch.Generator().manual_seed(D + bwk)
    B, nodes, A, Hkv = 5, 23, 9, 3
    start = torch.tensor([0, 1, S - 1, 2 * S - 5, 40], dtype=torch.int32)
    table, P = _table(B, -(-(int(start.max()) + nodes) // S), S, g)
    lead = (P, Hkv, S) if layers is None else (layers, P, Hkv, S)
    kp, vp = (_fill((*lead, D * bw // 8), torch.uint8, g) for bw in (bwk, bwv))
    kn, vn = _fill((*lead,), torch.float16, g), _fill((*lead,), torch.float16, g)
    counts = torch.tensor([0, 1, 4, 9, 7], dtype=torch.int32)
    _check(kp, vp, kn, vn, table, start, _branches(B, A, nodes, g), counts, nodes, page_table_host=table, start_pos_host=start)


@pytest.mark.parametrize("dtype,D", [(torch.bfloat16, 128), (torch.float16, 64), (torch.float32, 256)])
def test_unquantized_pages(dtype, D):
    g = torch.Generator().manual_seed(D)
    start = torch.tensor([3, 30], dtype=torch.int32)
    table, P = _table(2, 6, 16, g)
    kp, vp = _fill((2, P, 2, 16, D), dtype, g), _fill((2, P, 2, 16, D), dtype, g)
    _check(kp, vp, None, None, table, start, _branches(2, 64, 64, g), torch.tensor([64, 31], dtype=torch.int32), 64)


def test_the_widest_tree_over_itself_in_any_order():
    """64 nodes onto one another, in a path that is no branch: every row is read first."""
    g = torch.Generator().manual_seed(3)
    table, P = _table(3, 8, 16, g)
    start = torch.tensor([0, 17, 63], dtype=torch.int32)
    path = torch.stack([torch.randperm(64, generator=g) for _ in range(3)]).int()
    path[2] = path[2, :1]                                           # the same node everywhere
    kp, vp = _fill((P, 2, 16, 128), torch.uint8, g), _fill((P, 2, 16, 256), torch.uint8, g)
    kn, vn = _fill((P, 2, 16), torch.float16, g), _fill((P, 2, 16), torch.float16, g)
    _check(kp, vp, kn, vn, table, start, path, torch.tensor([64, 50, 64], dtype=torch.int32), 64)


def test_what_names_nothing_moves_nothing():
    """Nodes, positions and pages out of range, counts below and above the path (checks off)."""
    g = torch.Generator().manual_seed(4)
    table, P = _table(4, 3, 16, g)
    table[1, 1], table[2, 2] = -1, P
    start = torch.tensor([40, 10, 30, -3], dtype=torch.int32)       # 40 + 12 passes the table's 48
    path = torch.tensor([[2, 5, 9, 11], [0, 3, 7, 11], [-1, 12, 8, 2 ** 31 - 1], [1, 4, 6, 7]], dtype=torch.int32)
    counts = torch.tensor([4, 9, 4, 3], dtype=torch.int32)
    kp, vp = _fill((P, 2, 16, 64), torch.uint8, g), _fill((P, 2, 16, 48), torch.uint8, g)
    kn, vn = _fill((P, 2, 16), torch.float16, g), _fill((P, 2, 16), torch.float16, g)
    _check(kp, vp, kn, vn, table, start, path, counts, 12, check_ranges=False)
    _check(kp, vp, kn, vn, table, start, path, -counts, 12, check_ranges=False)


@pytest.mark.parametrize("shift", [1, 2, 4, 8])
def test_pages_at_any_alignment_and_stride(shift):
    """Pages that start anywhere, of a pool whose page axis comes first, with gaps."""
    g = torch.Generator().manual_seed(5)
    table, P = _table(2, 4, 16, g)
    start = torch.tensor([5, 20], dtype=torch.int32)
    path, counts = _branches(2, 7, 20, g), torch.tensor([7, 5], dtype=torch.int32)
    pools = [torch.randint(0, 256, (P * 3 * 2 * 16 * 64 + 16,), generator=g, dtype=torch.uint8) for _ in range(2)]
    norms = [_fill((P, 3, 2, 16), torch.float16, g).transpose(0, 1)[:2] for _ in range(2)]
    host = [p[shift:shift + P * 3 * 2 * 16 * 64].view(P, 3, 2, 16, 64).transpose(0, 1)[:2] for p in pools]
    dev = [p.to(DEV)[shift:shift + P * 3 * 2 * 16 * 64].view(P, 3, 2, 16, 64).transpose(0, 1)[:2] for p in pools]
    dn = [n.transpose(0, 1).contiguous().to(DEV).transpose(0, 1) for n in norms]
    _commit(*dev, *dn, table.to(DEV), start.to(DEV), path.to(DEV), counts.to(DEV), nodes=20)
    for got, was in zip(dev + dn, host + norms):
        assert torch.equal(_bits(got.cpu()), _bits(ref.commit(was, table, start, path, counts, 20, 1)))


def test_graph_replays():
    """Captured once, replayed on other branches; eager work between the replays."""
    g = torch.Generator().manual_seed(6)
    table, P = _table(3, 5, 16, g)
    start = torch.tensor([0, 20, 33], dtype=torch.int32)
    kp, vp = _fill((2, P, 2, 16, 64), torch.uint8, g), _fill((2, P, 2, 16, 64), torch.uint8, g)
    kn, vn = _fill((2, P, 2, 16), torch.float16, g), _fill((2, P, 2, 16), torch.float16, g)
    dev = [t.to(DEV) for t in (kp, vp, kn, vn)]
    path, counts = torch.zeros(3, 6, dtype=torch.int32, device=DEV), torch.zeros(3, dtype=torch.int32, device=DEV)
    dt, ds = table.to(DEV), start.to(DEV)
    _commit(*dev, dt, ds, path, counts, nodes=30)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        lengths = _commit(*dev, dt, ds, path, counts, nodes=30, check_ranges=False)
    for k in range(3):
        p, c = _branches(3, 6, 30, g), torch.tensor([6, k, 3], dtype=torch.int32)
        path.copy_(p)
        counts.copy_(c)
        for t, was in zip(dev, (kp, vp, kn, vn)):
            t.copy_(was)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(lengths.cpu(), start + c)
        for t, was in zip(dev, (kp, vp, kn, vn)):
            assert torch.equal(_bits(t.cpu()), _bits(ref.commit(was, table, start, p, c, 30, 1)))
