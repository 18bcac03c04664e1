"""What the operators of a speculative step refuse, and their host-side helpers. No GPU: the C ABI
checks its arguments before any launch, the Python layer is asked with host tensors that it is told
to take for HIP ones."""
from __future__ import annotations

import pytest
import torch

import tree_reference as ref
from winnow_amd import _lib
from winnow_amd import packed_attention as pa
from winnow_amd import packed_backend as pb
from winnow_amd.logprobs import token_logprobs


@pytest.fixture
def as_hip(monkeypatch):
    """Host tensors pass for HIP ones; a call into the library fails the test."""
    monkeypatch.setattr(_lib, "is_hip", lambda t: True)

    def call(name, *args):
        raise AssertionError(f"{name} was called")
    monkeypatch.setattr(_lib, "call", call)


def _kv(D=64, P=6, Hkv=2, S=16, bw=4, B=2, lens=(20, 33)):
    quant = pa.Quantizer(torch.eye(D), torch.linspace(-1, 1, 2 ** bw), bw)
    pages, norms = torch.zeros(P, Hkv, S, D * bw // 8, dtype=torch.uint8), torch.ones(P, Hkv, S, dtype=torch.float16)
    table = torch.tensor([[0, 1, -1], [2, 3, 4]], dtype=torch.int32)[:B]
    return pa.PackedKV(pages, norms, pages.clone(), norms.clone(), table, torch.tensor(lens, dtype=torch.int32), quant, quant, D)


def _tree(q=None, kv=None, parents=None, **kw):
    kv = kv or _kv()
    q = torch.zeros(2, 4, 5, 64) if q is None else q
    parents = torch.full((2, 5), -1, dtype=torch.int32) if parents is None else parents
    return pa.packed_tree_attention(q, kv, 0.1, parents, **kw)


def test_tree_needs_a_gpu():
    with pytest.raises(pa.UnsupportedLayout, match="HIP device"):
        _tree()


@pytest.mark.parametrize("parents,match", [
    (torch.tensor([[-1, 0, 1, 2, 3], [-1, 0, 2, 0, 0]], dtype=torch.int32), "node 2 has parent 2"),
    (torch.tensor([[-1, 0, 1, 4, 3], [-1, 0, 1, 0, 0]], dtype=torch.int32), "node 3 has parent 4"),
    (torch.tensor([[-2, 0, 1, 2, 3], [-1, 0, 1, 0, 0]], dtype=torch.int32), "parent -2"),
    (torch.zeros(2, 4, dtype=torch.int32), "parents must be"),
    (torch.full((2, 5), -1), "parents must be"),
    (torch.full((5, 2), -1, dtype=torch.int32).t(), "contiguous rows")])
def test_tree_parents(as_hip, parents, match):
    with pytest.raises(pa.UnsupportedLayout, match=match):
        _tree(parents=parents)


def test_tree_shapes(as_hip):
    with pytest.raises(pa.UnsupportedLayout, match="1 to 64"):
        _tree(q=torch.zeros(2, 4, 65, 64), parents=torch.full((2, 65), -1, dtype=torch.int32))
    with pytest.raises(pa.UnsupportedLayout, match="1 to 64"):
        _tree(q=torch.zeros(2, 4, 0, 64), parents=torch.zeros(2, 0, dtype=torch.int32))
    with pytest.raises(pa.UnsupportedLayout, match="multiple"):
        _tree(q=torch.zeros(2, 3, 5, 64))
    with pytest.raises(pa.UnsupportedLayout, match="contiguous head_dim"):
        _tree(q=torch.zeros(2, 4, 64, 5).transpose(2, 3))
    with pytest.raises(pa.UnsupportedLayout, match="fp32/fp16/bf16"):
        _tree(q=torch.zeros(2, 4, 5, 64, dtype=torch.float64))
    with pytest.raises(pa.UnsupportedLayout, match="no gradient"):
        _tree(q=torch.zeros(2, 4, 5, 64, requires_grad=True))
    with pytest.raises(pa.UnsupportedLayout, match="output dtype"):
        _tree(out_dtype=torch.float64)
    with pytest.raises(pa.UnsupportedLayout, match="head_dim 8"):
        _tree(q=torch.zeros(2, 4, 5, 8), kv=_kv(D=8))
    with pytest.raises(pa.UnsupportedLayout, match="parents_host"):
        _tree(parents_host=torch.full((1, 5), -1, dtype=torch.int32))


def test_tree_pages(as_hip):
    kv = _kv()
    kv.k_pages = torch.zeros(6, 2, 16, 64, dtype=torch.uint8)[..., :32]
    with pytest.raises(pa.UnsupportedLayout, match="contiguous"):
        _tree(kv=kv)
    kv = _kv()
    kv.v_pages = torch.zeros(6 * 2 * 16 * 32 + 4, dtype=torch.uint8)[2:-2].view(6, 2, 16, 32)
    with pytest.raises(pa.UnsupportedLayout, match="4-byte"):
        _tree(kv=kv)
    kv = _kv()
    kv.page_table[1, 2] = 6
    with pytest.raises(pa.UnsupportedLayout, match="outside"):
        _tree(kv=kv)
    kv = _kv(lens=(20, 49))
    with pytest.raises(pa.UnsupportedLayout, match="out of range"):
        _tree(kv=kv)
    with pytest.raises(pa.UnsupportedLayout, match="powers? of two"):
        _tree(kv=_kv(S=24, lens=(3, 4)))


def _commit(**kw):
    g = dict(k_pages=torch.zeros(3, 6, 2, 16, 32, dtype=torch.uint8), v_pages=torch.zeros(3, 6, 2, 16, 48, dtype=torch.uint8),
             k_norms=torch.zeros(3, 6, 2, 16, dtype=torch.float16), v_norms=torch.zeros(3, 6, 2, 16, dtype=torch.float16),
             page_table=torch.tensor([[0, 1, -1], [2, 3, 4]], dtype=torch.int32), start_pos=torch.tensor([10, 30], dtype=torch.int32),
             path=torch.zeros(2, 4, dtype=torch.int32), counts=torch.zeros(2, dtype=torch.int32), nodes=8)
    g.update(kw)
    names = ("k_pages", "v_pages", "k_norms", "v_norms", "page_table", "start_pos", "path", "counts")
    args = [g.pop(n) for n in names]
    return pb.commit_kv(*args, **g)


def test_commit_needs_a_gpu():
    with pytest.raises(pa.UnsupportedLayout, match="HIP device"):
        _commit()


@pytest.mark.parametrize("kw,match", [
    (dict(nodes=65), "1 <= A"), (dict(nodes=3), "1 <= A"), (dict(path=torch.zeros(2, 0, dtype=torch.int32)), "1 <= A"),
    (dict(path=torch.zeros(2, 4)), "path"), (dict(path=torch.zeros(3, 4, dtype=torch.int32)), "path"),
    (dict(path=torch.zeros(4, 2, dtype=torch.int32).t()), "path"),
    (dict(counts=torch.zeros(2)), "counts"), (dict(counts=torch.zeros(3, dtype=torch.int32)), "counts"),
    (dict(start_pos=torch.zeros(2)), "start_pos"), (dict(start_pos=torch.zeros(4, dtype=torch.int32)[::2]), "start_pos"),
    (dict(page_table=torch.zeros(2, 3)), "page_table"), (dict(page_table=torch.zeros(3, 2, dtype=torch.int32).t()), "page_table"),
    (dict(k_norms=None), "uint8 with norms"), (dict(v_pages=torch.zeros(3, 6, 2, 16, 48)), "without"),
    (dict(v_pages=torch.zeros(3, 6, 2, 16, 48), v_norms=None), "V pages are|K pages are"),
    (dict(v_pages=torch.zeros(2, 6, 2, 16, 48, dtype=torch.uint8)), "V pages must be"),
    (dict(k_norms=torch.zeros(3, 6, 2, 16)), "norms must be fp16"),
    (dict(k_pages=torch.zeros(3, 6, 2, 16, 64, dtype=torch.uint8)[..., :32]), "contiguous"),
    (dict(k_pages=torch.zeros(1, 6, 2, 16, 32, dtype=torch.uint8).expand(3, -1, -1, -1, -1)), "expanded"),
    (dict(start_pos=torch.tensor([10, 45], dtype=torch.int32)), "outside its 3-page"),
    (dict(start_pos=torch.tensor([30, 10], dtype=torch.int32)), "outside \\[0, 6\\)"),
    (dict(start_pos=torch.tensor([-1, 10], dtype=torch.int32)), "outside its 3-page")])
def test_commit_refusals(as_hip, kw, match):
    with pytest.raises(pa.UnsupportedLayout, match=match):
        _commit(**kw)


def test_logprobs_refusals(monkeypatch):
    x = torch.zeros(3, 10)
    with pytest.raises(pa.UnsupportedLayout, match="HIP device"):
        token_logprobs(x)
    monkeypatch.setattr(_lib, "is_hip", lambda t: True)
    for bad, kw, match in [(x.double(), {}, "fp32, fp16 or bf16"), (torch.zeros(1, 1, 1, 1), {}, "fp32, fp16 or bf16"),
                           (torch.zeros(()), {}, "fp32, fp16 or bf16"), (x.t(), {}, "contiguous"), (x[:, :0], {}, "non-empty"),
                           (x, dict(top=11), "top 11"), (x, dict(top=-1), "top -1"), (torch.zeros(1, 100), dict(top=65), "top 65"),
                           (x, dict(tokens=torch.zeros(4, dtype=torch.int64)), "tokens"), (x, dict(tokens=torch.zeros(3)), "tokens"),
                           (torch.zeros(3, 10, requires_grad=True), {}, "no gradient")]:
        with pytest.raises(pa.UnsupportedLayout, match=match):
            token_logprobs(bad, **kw)


def test_c_abi_refusals():
    i = 1 << 20   # an aligned address that is never read
    tree = lambda **k: _lib.call("wn_tree_attention", *{**dict(  # noqa: E731
        q=i, dt=0, qb=0, qh=0, qt=0, pk=i, pv=i, ck=i, cv=i, kp=i, ksp=0, ksh=0, vp=i, vsp=0, vsh=0, kn=i, knp=0, knh=0, vn=i, vnp=0,
        vnh=0, table=i, tsb=0, lens=i, par=i, psb=0, out=i, odt=0, ws=i, wsb=1 << 40, B=1, Hq=4, Hkv=2, T=5, D=64, S=16, bwk=4, bwv=4,
        P=4, maxp=4, scale=1.0, exact=1, ns=1, span=64, parts=1, stream=None, e0=None, e1=None), **k}.values())
    for k, match in [(dict(T=65), "T<=64"), (dict(T=0), "T<="), (dict(D=96), "power of two"), (dict(Hq=5), "Hq"), (dict(bwk=7), "widths"),
                     (dict(S=8), "page size"), (dict(S=24), "page size"), (dict(dt=3), "dtype"), (dict(ns=0), "num_splits"), (dict(ns=4097), "num_splits"), (dict(span=0), "span"), (dict(span=96), "span"), (dict(parts=0), "parts"),
                     (dict(P=0), "num_pages"), (dict(maxp=1 << 28), "max_pages"), (dict(q=None), "null"), (dict(par=None), "null"),
                     (dict(kp=i + 2), "4-byte"), (dict(vsh=6), "4-byte"), (dict(knp=-1), "negative"), (dict(pk=i + 4), "16-byte"),
                     (dict(wsb=100), "workspace"), (dict(ws=i + 16), "workspace"), (dict(ws=None), "workspace")]:
        with pytest.raises(_lib.WinnowHipError, match=match):
            tree(**k)
    tree(B=0)                                                        # nothing to do, nothing launched
    assert _lib.lib().wn_tree_workspace_bytes(1, 4, 2, 65, 64, 1) == -1
    assert pa.tree_workspace_bytes(2, 32, 8, 16, 128, 4) > 2 * 32 * 16 * 4 * 128 * 4
    commit = lambda **k: _lib.call("wn_commit_kv", *{**dict(  # noqa: E731
        k=i, kl=0, kp=64, kh=64, kr=4, v=i, vl=0, vp=64, vh=64, vr=4, kn=i, knl=0, knp=0, knh=0, vn=i, vnl=0, vnp=0, vnh=0, t=i, tsb=0,
        start=i, path=i, psb=0, counts=i, lengths=2 * i, layers=1, B=1, Hkv=1, S=16, A=1, nodes=4, P=1, maxp=1, stream=None), **k}.values())
    for k, match in [(dict(nodes=65), "nodes"), (dict(A=5), "A <= nodes"), (dict(A=0), "1 <= A"), (dict(S=24), "page size"), (dict(kr=0), "sizes"),
                     (dict(k=None), "null"), (dict(kn=None), "null"), (dict(lengths=i), "start_pos itself"), (dict(layers=70000), "grid")]:
        with pytest.raises(_lib.WinnowHipError, match=match):
            commit(**k)
    commit(B=0)
    lp = lambda **k: _lib.call("wn_token_logprobs", *{**dict(  # noqa: E731
        x=i, dt=0, so=0, si=0, inner=1, tok=i, lp=i, h=i, tl=i, ti=i, N=1, V=10, top=1, ws=None, wsb=0, stream=None), **k}.values())
    for k, match in [(dict(top=11), "top"), (dict(top=65, V=100), "top"), (dict(V=0), "sizes"), (dict(inner=0), "sizes"), (dict(dt=9), "dtype"),
                     (dict(x=None), "null"), (dict(lp=None), "null"), (dict(tl=None), "null"), (dict(x=i + 2), "aligned"),
                     (dict(V=100000), "workspace")]:
        with pytest.raises(_lib.WinnowHipError, match=match):
            lp(**k)
    lp(N=0)


def test_tree_helpers():
    parents = ref.random_parents(3, 20, 5)
    lens = torch.tensor([7, 20, 50])
    mask, live = pb._tree_mask(parents, lens, 50, "cpu")
    for b, L in enumerate(lens.tolist()):
        anc = ref.ancestors(parents[b], 20)
        for i in range(20):
            want = [j < L - 20 or (L - 20 <= j < L and bool(anc[i, j - (L - 20)])) for j in range(50)]
            assert mask[b, 0, i].tolist() == want
        assert live[b, 0, :, 0].tolist() == mask[b, 0].any(-1).tolist()
    assert pb.tree_positions([-1, 0, 0, 1, -1], [10, 3]).tolist() == [[10, 11, 11, 12, 10], [3, 4, 4, 5, 3]]
    for bad in ([], [0], [-1, 1], [[-1, 0]] * 3, [-1] * 65):
        with pytest.raises(pa.UnsupportedLayout):
            pb.tree_positions(bad, [4, 5])


def test_cache_refuses_what_is_no_branch():
    from winnow_amd.page_pool import PagePool
    from winnow_amd.quantizer import TurboQuantMSE
    tq = TurboQuantMSE(4, 64, "cpu", 1)
    pool = PagePool(num_layers=1, num_pages=8, num_kv_heads=1, page_size=16, nb_k=32, nb_v=32)
    pool.ensure("a", 40)
    cache = pb.PagedPackedCache(pool, ["a"], [10], k_quant=tq, v_quant=tq, head_dim=64, tree=[-1, 0, 0, 2])
    with pytest.raises(RuntimeError, match="follows a forward"):
        cache.commit([[0]])
    with pytest.raises(ValueError, match="4 tokens, the forward 3"):
        cache.begin(3, "cpu")
    meta = cache.begin(4, "cpu")
    cache.lengths = meta.seq_host.tolist()                           # as after the last layer
    for paths, match in [([], "0 paths"), ([[1]], "not a branch"), ([[0, 3]], "not a branch"), ([[0, 2, 3, 1]], "not a branch"),
                         ([[4]], "not a branch"), ([[-1]], "not a branch")]:
        with pytest.raises(ValueError, match=match):
            cache.commit(paths)


def test_engine_refuses_too_many_alternatives():
    from winnow_amd.engine import Engine, Refused, Request
    from winnow_amd.page_pool import PagePool
    pool = PagePool(num_layers=1, num_pages=8, num_kv_heads=1, page_size=16, nb_k=32, nb_v=32)
    e = Engine(torch.nn.Linear(1, 1), pool, None, None, 64)
    for n in (-1, 65):
        with pytest.raises(Refused, match="bad_top_logprobs"):
            e.submit(Request("r", [1], 2, top_logprobs=n))
    assert e.submit(Request("r", [1], 2, top_logprobs=0)).logprobs == []


def test_the_native_range_checks_agree_with_the_plain_ones(monkeypatch):
    """Positions of lengths and of appended tokens, and parents: random small metadata, some of it
    out of range, strided tables, other types; the message names what the plain check finds."""
    import random

    from winnow_amd import packed_attention as pa
    from winnow_amd import packed_backend as pb
    _lib.lib()
    r = random.Random(5)

    def said(check, *args):
        try:
            return check(*args)
        except pa.UnsupportedLayout as e:
            return str(e)

    refused = 0
    for k in range(600):
        B, W, S, P = r.randint(0, 5), r.choice([1, 2, 7]), r.choice([1, 16, 12]), r.choice([1, 5])
        odd = [-1, P, 2 ** 31 - 1, -2 ** 31]
        ids = [[r.choice(odd) if r.random() < 0.03 else r.randrange(P) for _ in range(W + 2)] for _ in range(B)]
        table = torch.tensor(ids, dtype=torch.int32).reshape(B, W + 2)[:, 1:1 + W]
        start = torch.tensor([r.choice([0, W * S, W * S + 1, -1, 2 ** 31 - 1]) if r.random() < 0.2 else r.randint(0, W * S)
                              for _ in range(B)], dtype=torch.int32)
        n = r.choice([0, 1, 2, S, 2 ** 31 - 1])
        parents = torch.tensor([[r.choice([-2, i, i + 1, 2 ** 31 - 1]) if r.random() < 0.03 else r.randint(-1, i - 1)
                                 for i in range(W)] for _ in range(B)], dtype=torch.int32).reshape(B, W)
        if k % 3 == 0:
            table, start = table.long(), start.long()  # not the mirrors' type: the plain checks look
        calls = [(pa.check_page_ranges, start, table, P, S), (pb._positions_in_range, start, table, n, P, S),
                 (pa.check_parents, parents)]
        got = [said(*c) for c in calls]
        with monkeypatch.context() as m:
            m.setattr(_lib, "positions_in_range", lambda *a: False)
            m.setattr(_lib, "parents_in_order", lambda *a: False)
            assert got == [said(*c) for c in calls], (start, table, n, P, S, parents)
        refused += sum(x is not None for x in got)
    assert 300 < refused < 1500
