"""``append_rotated_kv`` (``wn_append_rotated_kv``).

The pages must hold, bit for bit, what ``append_kv`` (tested against the oracle) writes for K
rotated in float64 and rounded once to fp32, and V; every other byte stays as it was. That fp32 K
is itself held to a float64 rotation by complex products. The returned q against the float64
rotation: one rounding to fp32 and one to its type, (1 + 2^-23) (2^-24 + eps / 2) of the value
(eps / 2 half a step of the type; for fp32 one rounding: 2^-24) and half the least subnormal.
"""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda"
TYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}


def _rotated64(x, cos, sin):
    """x (B, H, n, D) rotated by complex products in float64."""
    R = cos.shape[-1]
    a, c, s = x.double(), cos.double()[:, None], sin.double()[:, None]
    lo, hi = a[..., :R // 2], a[..., R // 2:R]
    return torch.cat([lo * c[..., :R // 2] - hi * s[..., :R // 2], hi * c[..., R // 2:] + lo * s[..., R // 2:], a[..., R:]], -1)


def _quantizers(bwk, bwv, D):
    from winnow_amd.quantizer import get_quantizer
    return get_quantizer(bwk, D, DEV, 42), get_quantizer(bwv, D, DEV, 7)


def _pool(lens, n, Hkv, S, D, bwk, bwv, seed, spare=2):
    g = torch.Generator().manual_seed(seed)
    need = [-(-(L + n) // S) for L in lens]
    P = sum(need) + spare
    order = torch.randperm(P, generator=g).tolist()
    table = torch.full((len(lens), max(need + [1])), -1, dtype=torch.int32)
    at = 0
    for b, m in enumerate(need):
        table[b, :m] = torch.tensor(order[at:at + m], dtype=torch.int32)
        at += m
    page = lambda bw: torch.randint(0, 256, (P, Hkv, S, D * bw // 8), dtype=torch.uint8, generator=g).to(DEV)  # noqa: E731
    norm = lambda: torch.randn(P, Hkv, S, generator=g).half().to(DEV)  # noqa: E731
    return table.to(DEV), torch.tensor(lens, dtype=torch.int32, device=DEV), [page(bwk), page(bwv), norm(), norm()]


def _inputs(B, Hq, Hkv, n, D, R, dtype, rot, seed, shared=False):
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = [torch.randn(B, n, h, D, generator=g, device=DEV).to(dtype).transpose(1, 2) for h in (Hq, Hkv, Hkv)]
    pos = torch.randint(0, 100000, (1 if shared else B, n, 1), generator=g, device=DEV).double()
    ang = pos * 10000.0 ** (-torch.arange(0, R, 2, device=DEV).double() / R)
    ang = torch.cat([ang, ang], -1)
    return x, ang.cos().to(rot), ang.sin().to(rot)


def _check_q(got, q, cos, sin):
    assert got.shape == q.shape and got.dtype == q.dtype and got.is_contiguous()
    want, info = _rotated64(q, cos, sin), torch.finfo(q.dtype)
    rel = 2.0 ** -24 + (0 if q.dtype == torch.float32 else info.eps / 2 * (1 + 2.0 ** -23))
    assert ((got.double() - want).abs() <= rel * want.abs() + info.smallest_normal * info.eps / 2).all()


def _run(case, seed=0, shared=False, has_q=True, has_v=True, k=None, v=None):
    from winnow_amd.packed_backend import append_kv, append_rotated_kv
    B, Hq, Hkv, n, D, R, bwk, bwv, S, dtype, rot = case
    (q, k0, v0), cos, sin = _inputs(B, Hq, Hkv, n, D, R, TYPES[dtype], TYPES[rot], seed, shared)
    k, v = k0 if k is None else k, v0 if v is None else v
    lens = [(7 * b + 3) % 41 for b in range(B)]
    table, start, pages = _pool(lens, n, Hkv, S, D, bwk, bwv, seed)
    kq, vq = _quantizers(bwk, bwv, D)
    want = [t.clone() for t in pages]
    k32 = _rotated64(k, cos, sin).float()
    vs = (lambda p: (vq, p[0], p[1], p[2], p[3])) if has_v else (lambda p: (None, p[0], None, p[2], None))
    append_kv(k32, v.float() if has_v else None, kq, *vs(want), table, start)
    got = append_rotated_kv(q if has_q else None, k, v if has_v else None, cos, sin, kq, *vs(pages), table, start)
    for name, a, b in zip(("K pages", "V pages", "K norms", "V norms"), pages, want):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8)), name
    if has_q:
        _check_q(got, q, cos, sin)
    else:
        assert got is None
    return q, k, v, cos, sin, table, start


@pytest.mark.parametrize("case", [
    # B, Hq, Hkv, n, D, R, widths, S, type of q / K / V, type of the tables
    (1, 32, 8, 1, 128, 128, 4, 4, 16, "bf16", "bf16"), (3, 28, 4, 1, 128, 128, 8, 8, 16, "bf16", "fp32"), (2, 14, 2, 5, 64, 64, 4, 6, 16, "fp16", "fp16"),
    (2, 14, 2, 37, 64, 32, 3, 5, 32, "fp16", "fp32"), (1, 4, 2, 3, 128, 2, 2, 3, 16, "fp32", "fp32"), (2, 3, 1, 19, 256, 256, 6, 4, 16, "bf16", "bf16"),
    (2, 5, 5, 7, 16, 16, 8, 2, 16, "fp32", "bf16"), (1, 2, 1, 33, 32, 18, 5, 5, 16, "fp16", "fp16"), (4, 8, 8, 2, 128, 96, 4, 4, 64, "fp32", "fp32"),
    (70, 4, 2, 1, 128, 64, 4, 4, 16, "bf16", "bf16"), (2, 7, 1, 1, 64, 6, 6, 6, 16, "bf16", "fp16")], ids=str)
def test_the_pages_are_those_of_the_rotated_k(case):
    """One token to many, every head_dim, whole and partial rotations, an odd number of pairs, types
    of the tables that are not the tensors'."""
    _run(case, seed=sum(x for x in case if isinstance(x, int)))


@pytest.mark.parametrize("dtype,rot", [("bf16", "bf16"), ("fp16", "fp32"), ("fp32", "fp16"), ("fp32", "fp32"), ("bf16", "fp32"), ("fp16", "fp16")])
@pytest.mark.parametrize("D,R,bwk,bwv", [(128, 128, 4, 4), (64, 64, 8, 4), (128, 32, 6, 3), (64, 16, 4, 4), (128, 24, 4, 8)])
def test_many_vectors(D, R, bwk, bwv, dtype, rot):
    """Enough vectors for the tile kernel (from 12,288 or 16,384), and rotations that it does not take."""
    _run((2, 12, 4, 2100, D, R, bwk, bwv, 16, dtype, rot), seed=D + R)


@pytest.mark.parametrize("n", [1, 3000])
def test_tables_without_a_batch_and_sides_left_out(n):
    for kw in (dict(shared=True), dict(has_q=False), dict(has_v=False), dict(has_q=False, has_v=False, shared=True)):
        _run((3, 8, 4, n, 128, 128, 4, 4, 16, "bf16", "bf16"), seed=n, **kw)


def _misaligned(t):
    """The same values, two bytes (or four) off a 16-byte address."""
    flat = torch.empty(t.numel() + 1, dtype=t.dtype, device=t.device)
    return flat[1:].view(t.shape).copy_(t)


@pytest.mark.parametrize("n", [2, 2100])
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_strides_and_alignment(n, dtype):
    """Heads before tokens in memory, expanded heads, odd row strides and bases."""
    from winnow_amd.packed_backend import append_kv, append_rotated_kv
    (q, k, v), cos, sin = _inputs(2, 8, 4, n, 128, 64, TYPES[dtype], TYPES[dtype], 5)
    table, start, pages = _pool([3, 30], n, 4, 16, 128, 4, 6, 5)
    kq, vq = _quantizers(4, 6, 128)
    wide = torch.empty(2, n, 67, dtype=cos.dtype, device=DEV)
    wide[..., 1:65] = cos
    views = {
        "contiguous": (q.contiguous(), k.contiguous(), v.contiguous(), cos, sin),
        "off": (_misaligned(q), _misaligned(k), _misaligned(v), _misaligned(cos), _misaligned(sin)),
        "tables": (q, k, v, wide[..., 1:65], sin.transpose(0, 1).contiguous().transpose(0, 1)),
        "expanded": (q[:, :1].expand(-1, 8, -1, -1), k[:, :1].expand(-1, 4, -1, -1), v[:1].expand(2, -1, -1, -1), cos[:, :1].expand(-1, n, -1), sin[:, :1].expand(-1, n, -1))}
    for name, (q1, k1, v1, c1, s1) in views.items():
        got, want = [t.clone() for t in pages], [t.clone() for t in pages]
        append_kv(_rotated64(k1, c1, s1).float(), v1.float(), kq, vq, *want, table, start)
        out = append_rotated_kv(q1, k1, v1, c1, s1, kq, vq, *got, table, start)
        assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(got, want)), name
        _check_q(out, q1, c1, s1)


def test_a_zero_vector_and_values_that_are_not_finite():
    """Zero and tiny vectors keep the norm's floor; a vector with a NaN or an infinity changes no other's."""
    case = (1, 4, 2, 6, 128, 128, 4, 4, 16, "fp32", "fp32")
    (_, k, v), cos, sin = _inputs(1, 4, 2, 6, 128, 128, torch.float32, torch.float32, 9)
    k = k.contiguous()
    k[0, 0, 0] = 0
    k[0, 0, 1] *= 1e-30
    k[0, 1, 2, 5] = float("nan")
    k[0, 1, 3, 100] = float("inf")
    k[0, 0, 4] *= 1e30
    _run(case, seed=9, k=k, v=v)


def test_pages_outside_are_refused_and_neighbours_kept():
    from winnow_amd import packed_attention as pa
    from winnow_amd.packed_backend import append_rotated_kv
    (q, k, v), cos, sin = _inputs(2, 4, 2, 3, 64, 64, torch.bfloat16, torch.bfloat16, 1)
    table, start, pages = _pool([3, 30], 3, 2, 16, 64, 4, 4, 1)
    kq, vq = _quantizers(4, 4, 64)
    keep = [t.clone() for t in pages]
    bad = table.clone()
    bad[1, 1] = pages[0].shape[0]
    bad[1, 2:] = pages[0].shape[0]
    with pytest.raises(pa.UnsupportedLayout, match="outside"):
        append_rotated_kv(q, k, v, cos, sin, kq, vq, *pages, bad, start)
    with pytest.raises(pa.UnsupportedLayout, match="outside its"):
        append_rotated_kv(q, k, v, cos, sin, kq, vq, *pages, table, start + 1000)
    assert all(torch.equal(a, b) for a, b in zip(pages, keep))


def test_graph_replays_and_own_stream():
    from winnow_amd.packed_backend import append_rotated_kv
    for n in (1, 2100):
        (q, k, v), cos, sin = _inputs(2, 8, 4, n, 128, 128, torch.bfloat16, torch.bfloat16, 2)
        table, start, pages = _pool([5, 20], n, 4, 16, 128, 4, 4, 2)
        kq, vq = _quantizers(4, 4, 128)
        call = lambda p: append_rotated_kv(q, k, v, cos, sin, kq, vq, *p, table, start, check_ranges=False)  # noqa: E731
        side, other = torch.cuda.Stream(), [t.clone() for t in pages]
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            a = call(other)
        side.synchronize()
        b = call(pages)
        assert torch.equal(a, b) and all(torch.equal(x, y) for x, y in zip(pages, other))
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = call(pages)
        for i in range(4):
            (q1, k1, v1), c1, s1 = _inputs(2, 8, 4, n, 128, 128, torch.bfloat16, torch.bfloat16, 50 + i)
            for dst, src in zip((q, k, v, cos, sin), (q1, k1, v1, c1, s1)):
                dst.copy_(src)
            graph.replay()
            torch.cuda.synchronize()
            eager = [t.clone() for t in pages]
            for t in eager:
                t.view(torch.uint8).zero_()
            for t in pages:
                t.view(torch.uint8).zero_()
            graph.replay()
            want = call(eager)
            assert torch.equal(out, want) and all(torch.equal(x, y) for x, y in zip(pages, eager))


@pytest.mark.parametrize("dtype,rot", [("bf16", "bf16"), ("fp16", "fp32"), ("fp32", "fp16"), ("fp32", "fp32")])
@pytest.mark.parametrize("B,n,R,bwk,bwv", [(1, 1, 256, 4, 4), (3, 1, 64, 8, 8), (2, 17, 6, 3, 5), (2, 700, 256, 4, 6), (5, 33, 128, 2, 8)])
def test_head_dim_256(B, n, R, bwk, bwv, dtype, rot):
    """The matrix cores against ``append_kv``'s vector ALU: one vector, parts of a work-group's sixteen, many;
    rotations that 16-byte loads read and ones that they do not."""
    case = (B, 8, 2, n, 256, R, bwk, bwv, 16, dtype, rot)
    q, k, v, *_ = _run(case, seed=B + n + R)
    _run(case, seed=B + n, k=_misaligned(k), v=v)
    _run(case, seed=B + n + 1, has_v=False, has_q=False)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_head_dim_256_extremes(dtype):
    """Zero vectors, one channel, tiny and huge norms, values that are not finite."""
    (_, k, v), _, _ = _inputs(2, 2, 2, 40, 256, 256, TYPES[dtype], TYPES[dtype], 3)
    k, v = k.clone(), v.clone()
    for x in (k, v):
        x[:, :, 0] = 0
        x[:, :, 1] = 0
        x[:, :, 1, 77] = 3.0
        x[:, :, 2] *= 1e-20
        x[:, :, 3] *= 1e15
        x[0, 0, 4, 9] = float("inf")
        x[0, 1, 5, 200] = float("nan")
    _run((2, 2, 2, 40, 256, 256, 4, 4, 16, dtype, dtype), seed=3, k=k, v=v, has_q=False)


@pytest.mark.parametrize("rotated", [False, True])
def test_start_positions_with_gaps_are_refused(rotated):
    """They are read as a contiguous row."""
    from winnow_amd.packed_attention import UnsupportedLayout
    from winnow_amd.packed_backend import append_kv, append_rotated_kv
    (q, k, v), cos, sin = _inputs(3, 4, 2, 2, 64, 64, torch.float32, torch.float32, 1)
    table, start, (kp, vp, kn, vn) = _pool([1, 20, 33], 2, 2, 16, 64, 4, 4, 1)
    before = kp.clone()
    gaps = torch.stack([start, start + 7], 1)[:, 0]
    kq, vq = _quantizers(4, 4, 64)
    with pytest.raises(UnsupportedLayout, match="contiguous"):
        if rotated:
            append_rotated_kv(q, k, v, cos, sin, kq, vq, kp, vp, kn, vn, table, gaps)
        else:
            append_kv(k, v, kq, vq, kp, vp, kn, vn, table, gaps)
    assert torch.equal(kp, before)
