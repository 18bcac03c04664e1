"""The operators of a step of a long conversation together, as a program uses them: a tiny seeded
Qwen2 over the packed cache with a window and sinks, the rotation in the append, and penalties,
biases and masks on what it answers.

Every operator is checked where the model calls it, on the model's own q, K and V and the pool's own
bytes, against its definition in float64 and with the bounds of its own tests (a whole run against
another one has no such bound: a rounding in one layer moves a code over a bucket border in the
next).
"""
from __future__ import annotations

import math

import pytest
import torch

DEV = "cuda"
pytestmark = pytest.mark.gpu


@pytest.fixture()
def model():
    from tiny_qwen import tiny_qwen
    return tiny_qwen(DEV)


@torch.no_grad()
def _generate(model, prompts, n, *, chunk=10 ** 6, dense=False, **cache_kw):
    """Greedy tokens and the logits of every step; prompts in chunks."""
    from winnow_amd import packed_backend as pb
    cfg = model.config
    cfg._attn_implementation = pb.ATTN_NAME
    pool = pb.make_pool(cfg, bit_width=None if dense else 8, num_pages=96, page_size=16, device=DEV, dense_dtype=torch.float32 if dense else None)
    kq, vq = pb.quantizers_for(cfg, 8, DEV)
    kw = dict(k_quant=kq, v_quant=vq, head_dim=pb.head_dim_of(cfg), **cache_kw)
    owners, last = [f"r{i}" for i in range(len(prompts))], []
    for o, p in zip(owners, prompts):
        pool.ensure(o, len(p) + n)
        for lo in range(0, len(p), chunk):
            part = p[lo:lo + chunk]
            out = model(input_ids=torch.tensor([part], device=DEV), position_ids=torch.arange(lo, lo + len(part), device=DEV)[None],
                        past_key_values=pb.PagedPackedCache(pool, [o], [lo], **kw), use_cache=True, logits_to_keep=1)
        last.append(out.logits[0, -1].float())
    toks, steps, lengths = [[int(x.argmax())] for x in last], [torch.stack(last)], [len(p) for p in prompts]
    for _ in range(n - 1):
        cache = pb.PagedPackedCache(pool, owners, lengths, **kw)
        out = model(input_ids=torch.tensor([[t[-1]] for t in toks], device=DEV), position_ids=torch.tensor(lengths, device=DEV)[:, None],
                    past_key_values=cache, use_cache=True, logits_to_keep=1)
        lengths = cache.lengths
        steps.append(out.logits[:, -1].float())
        for t, x in zip(toks, steps[-1]):
            t.append(int(x.argmax()))
    return toks, torch.stack(steps, 1), pool


def _prompts(n, lo=30, hi=120):
    from tiny_qwen import prompts
    return prompts(n, seed=4, lo=lo, hi=hi)


def _checked_window(counts):
    """The windowed route, each call held to float64 over the same bytes."""
    import window_reference as ref
    from cases import to_host
    from winnow_amd import packed_backend as pb

    def route(query, kv, scale):
        out = pb._hip_window(query, kv, scale)
        want, K, V, E = ref.window_attention(query.cpu(), to_host(kv), scale, kv.window, kv.sinks)
        tol = (2 * E * K + V) * 2.0 ** -19 + 2.0 ** -24 * want.abs()
        assert ((out.double().cpu() - want).abs() <= tol).all()
        counts.append(query.shape[2])
        return out
    return route


@pytest.mark.parametrize("window,sinks,chunk", [(24, 4, 10 ** 6), (24, 0, 16), (7, 20, 33), (1000, 0, 40)])
def test_a_windowed_cache(model, monkeypatch, window, sinks, chunk):
    from winnow_amd import packed_backend as pb
    prompts = _prompts(3)
    pb.BACKEND_COUNTS.clear()
    counts = []
    monkeypatch.setitem(pb._ROUTES, "window_hip_packed", _checked_window(counts))
    toks, logits, _ = _generate(model, prompts, 8, chunk=chunk, window=window, sinks=sinks)
    assert set(pb.BACKEND_COUNTS) == {"window_hip_packed"} and pb.BACKEND_COUNTS["window_hip_packed"] == len(counts)
    assert counts.count(1) >= 2 * 7 and max(counts) > 1                   # decode steps and prompt chunks of both layers
    assert all(len(t) == 8 for t in toks) and torch.isfinite(logits).all()
    if window < 1000:
        _, whole, _ = _generate(model, prompts, 8, chunk=chunk)
        assert (logits[:, 0] - whole[:, 0]).abs().max() > 1e-2 * whole.abs().max()       # the window shows


def test_a_windowed_dense_cache(model, monkeypatch):
    """Unquantized pages under the same window: SDPA with its mask, against the definition in float64
    with the bound of an fp32 product of this size (128 + 60 terms, 2^-24 each of |q| |k| and |v|)."""
    from winnow_amd import packed_backend as pb
    calls = []

    def route(query, kv, scale):
        out = pb._dense_sdpa(query, kv, scale)
        lens, n = kv.seq_lens_host.long(), query.shape[1] // kv.num_kv_heads
        for b, L in enumerate(lens.tolist()):
            t = torch.arange(L)
            page = kv.page_table_host[b].long()[t // kv.page_size].to(DEV)
            k, v = (p[page, :, (t % kv.page_size).to(DEV)].transpose(0, 1).double().repeat_interleave(n, 0) for p in (kv.k_pages, kv.v_pages))
            pos, j = torch.arange(L - query.shape[2], L, device=DEV)[:, None], torch.arange(L, device=DEV)[None]
            s = torch.matmul(query[b].double(), k.transpose(1, 2).contiguous()) * scale
            hidden = (j > pos) | ((pos - j >= kv.window) & (j >= kv.sinks))
            want = torch.softmax(s.masked_fill(hidden, -math.inf), -1) @ v
            K = float(scale * query[b].double().norm(dim=-1).max() * k.norm(dim=-1).max())
            V, E = float(v.norm(dim=-1).max()), float(v.abs().max())
            assert ((out[b].double() - want).abs() <= 200 * 2.0 ** -24 * (2 * E * K + V)).all()
        calls.append(query.shape[2])
        return out
    monkeypatch.setitem(pb._ROUTES, "window_dense_sdpa", route)
    pb.BACKEND_COUNTS.clear()
    _generate(model, _prompts(2, 20, 40), 6, dense=True, window=12, sinks=2)
    assert set(pb.BACKEND_COUNTS) == {"window_dense_sdpa"} and min(calls) == 1 < max(calls)


def test_the_rotation_in_the_append(model, monkeypatch):
    """fuse_rotary: every append of the model holds, bit for bit, what ``append_kv`` writes for K rotated
    in float64, and q is its own rotation; calls that the fused path does not serve go the module's way."""
    from test_gpu_append_rotated import _check_q, _rotated64
    from winnow_amd import packed_backend as pb
    calls, inner = [], pb.PagedPackedCache.update_rotated

    def checked(self, q, k, v, cos, sin, layer):
        out, handle = inner(self, q, k, v, cos, sin, layer)
        _check_q(out, q, cos, sin)
        pages = (handle.k_pages, handle.v_pages, handle.k_norms, handle.v_norms)
        want = [t.clone() for t in pages]
        pb.append_kv(_rotated64(k, cos, sin).float(), v.float(), self.kq, self.vq, *want, self.meta.table, self.meta.start)
        assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(pages, want))
        calls.append(q.shape[2])
        return out, handle
    monkeypatch.setattr(pb.PagedPackedCache, "update_rotated", checked)
    assert pb.fuse_rotary(model) == 2 and pb.fuse_rotary(model) == 2
    prompts = _prompts(3)
    toks, logits, _ = _generate(model, prompts, 8, chunk=40)
    assert calls.count(1) >= 2 * 7 and max(calls) == 40 and torch.isfinite(logits).all()
    n = len(calls)
    _generate(model, prompts[:1], 2, dense=True)                               # an unquantized cache: own forward
    pool = pb.make_pool(model.config, bit_width=8, num_pages=8, page_size=16, device=DEV)
    pool.ensure("g", 20)
    kq, vq = pb.quantizers_for(model.config, 8, DEV)
    with torch.enable_grad():                                                   # a gradient: own forward
        cache = pb.PagedPackedCache(pool, ["g"], [0], k_quant=kq, v_quant=vq, head_dim=128)
        model(input_ids=torch.tensor([prompts[0][:4]], device=DEV), position_ids=torch.arange(4, device=DEV)[None], past_key_values=cache)
    assert len(calls) == n and cache.lengths == [4]


def test_a_copy_of_a_fused_model_has_its_own_weights(model):
    import copy
    from winnow_amd import packed_backend as pb
    pb.fuse_rotary(model)
    other = copy.deepcopy(model)
    with torch.no_grad():
        for m in other.modules():
            if isinstance(m, torch.nn.Linear) and m.weight.shape[0] == 512 and m.bias is not None:
                m.weight.mul_(0.5)
    _, a, _ = _generate(model, _prompts(1), 2)
    _, b, _ = _generate(other, _prompts(1), 2)
    _, again, _ = _generate(model, _prompts(1), 2)
    assert torch.equal(a, again) and not torch.equal(a, b)


def test_fuse_rotary_refuses_other_models(model):
    from winnow_amd import packed_backend as pb
    model.config.architectures = ["OtherForCausalLM"]
    with pytest.raises(pb.UnsupportedModel):
        pb.fuse_rotary(model)


def _engine(model, **cfg):
    from winnow_amd import packed_backend as pb
    from winnow_amd.engine import Engine, EngineConfig
    model.config._attn_implementation = pb.ATTN_NAME
    pool = pb.make_pool(model.config, bit_width=8, num_pages=96, page_size=16, device=DEV)
    kq, vq = pb.quantizers_for(model.config, 8, DEV)
    return Engine(model, pool, kq, vq, pb.head_dim_of(model.config), config=EngineConfig(**cfg))


def test_the_engine_over_all_of_it(model):
    """Windowed attention, the rotation in the append, penalties, biases and masks, with scores: every
    token is the greedy choice of the definition, in float64, over the logits that the model gave."""
    from winnow_amd.engine import Request
    e = _engine(model, window=24, sinks=4, fuse_rotary=True, prefill_chunk=20, max_batch=3)
    seen = {}
    e.on_logits = lambda reqs, x: [seen.setdefault(r.request_id, []).append(row.double().cpu()) for r, row in zip(reqs, x)]
    even = torch.zeros(128, dtype=torch.bool)
    even[::2] = True
    p = _prompts(5)
    reqs = [Request("plain", p[0], 10), Request("penalties", p[1], 10, repetition_penalty=1.4, presence_penalty=0.7, frequency_penalty=0.3),
            Request("bias", p[2], 10, logit_bias={5: 100.0, 6: -100.0}, top_logprobs=2),
            Request("mask", p[3], 10, allowed_tokens=lambda r: even if len(r.generated) % 2 else ~even),
            Request("all", p[4], 10, repetition_penalty=1.2, frequency_penalty=0.5, logit_bias={7: 3.0}, allowed_tokens=lambda r: ~even, top_logprobs=0)]
    for r in reqs:
        e.submit(r)
    e.run_until_idle()
    for r in reqs:
        assert r.status == "length" and len(r.generated) == 10
        steps = seen[r.request_id][-10:]
        for i, (x, t) in enumerate(zip(steps, r.generated)):
            hist = r.prompt_ids + r.generated[:i]
            y = x.clone()
            for k in set(hist):
                y[k] = y[k] / r.repetition_penalty if y[k] > 0 else y[k] * r.repetition_penalty
            for k in set(r.generated[:i]):
                y[k] -= r.frequency_penalty * r.generated[:i].count(k) + r.presence_penalty
            for k, b in r.logit_bias.items():
                y[k] += b
            if r.request_id in ("mask", "all"):
                ok = even if r.request_id == "mask" and i % 2 else ~even
                y[~ok] = -math.inf
            assert y[t] >= y.max() - 1e-4 * x.abs().max()      # fp32 arithmetic: equal but for its rounding
            if r.request_id in ("mask", "all"):
                assert ok[t]
    assert reqs[2].generated == [5] * 10
    # scores are the model's, before what was asked
    for s, x in zip(reqs[2].logprobs, seen["bias"][-10:]):
        assert abs(s.logprob - float(torch.log_softmax(x, -1)[5])) < 1e-4 * max(1, float(x.abs().max()))
    assert e.pool.stats()["owned"] == 0


def test_batched_requests_are_those_of_one(model):
    from winnow_amd.engine import Request
    cfg = dict(window=40, sinks=3, fuse_rotary=True, prefill_chunk=32)
    ask = [dict(repetition_penalty=1.3), dict(), dict(frequency_penalty=1.0, logit_bias={3: 1.0}), dict(presence_penalty=2.0)]
    p = _prompts(4)
    together = [Request(f"r{i}", x, 12, **a) for i, (x, a) in enumerate(zip(p, ask))]
    e = _engine(model, **cfg)
    for r in together:
        e.submit(r)
    e.run_until_idle()
    for r, x, a in zip(together, p, ask):
        one = Request("solo", x, 12, **a)
        e = _engine(model, **cfg)
        e.submit(one)
        e.run_until_idle()
        assert one.generated == r.generated


def test_caches_that_are_refused(model):
    from winnow_amd import packed_attention as pa
    from winnow_amd import packed_backend as pb
    pool = pb.make_pool(model.config, bit_width=8, num_pages=8, page_size=16, device=DEV)
    kq, vq = pb.quantizers_for(model.config, 8, DEV)
    kw = dict(k_quant=kq, v_quant=vq, head_dim=128)
    for bad, err in ((dict(sinks=3), ValueError), (dict(window=0), pa.UnsupportedLayout), (dict(window=4, sinks=-1), pa.UnsupportedLayout),
                     (dict(window=4, tree=[-1, 0]), ValueError)):
        with pytest.raises(err):
            pb.PagedPackedCache(pool, ["a"], [0], **kw, **bad)
    for backend in ("reconstruct_sdpa", "hip_dense", "nonsense"):
        with pytest.raises(ValueError, match="no window"):
            _generate(model, _prompts(1), 2, window=8, decode_backend=backend)
    with pytest.raises(ValueError, match="no window"):
        _generate(model, _prompts(1), 2, window=8, dense=True, decode_backend="hip_dense")
