"""The operators of a speculative step together, as a program uses them: drafted trees through a
tiny seeded Qwen2 and the paged cache, scored, the accepted branch kept. Decoding is greedy, so the
tokens must be those of one-token decoding, and so must the logits, to the bar of the model tests
(1e-3 of the logit scale at 8 bits, whose K and V may differ by a code at a bucket border; 2e-2 over
bf16 pages, read by SDPA in fp32 on one side and by the dense decode on the other)."""
from __future__ import annotations

import pytest
import torch

DEV = "cuda"
pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def model():
    from tiny_qwen import tiny_qwen
    return tiny_qwen(DEV)


def _setup(model, prompts, room, dense):
    from winnow_amd import packed_backend as pb
    cfg = model.config
    model.config._attn_implementation = pb.ATTN_NAME
    pool = pb.make_pool(cfg, bit_width=None if dense else 8, num_pages=96, page_size=16, device=DEV,
                        dense_dtype=torch.bfloat16 if dense else None)
    kq, vq = pb.quantizers_for(cfg, 8, DEV)
    kw = dict(k_quant=kq, v_quant=vq, head_dim=pb.head_dim_of(cfg))
    owners, first = [f"r{i}" for i in range(len(prompts))], []
    for o, p in zip(owners, prompts):
        pool.ensure(o, len(p) + room)
        cache = pb.PagedPackedCache(pool, [o], [0], **kw)
        out = model(input_ids=torch.tensor([p], device=DEV), position_ids=torch.arange(len(p), device=DEV)[None],
                    past_key_values=cache, use_cache=True, logits_to_keep=1)
        first.append(int(out.logits[0, -1].argmax()))
    return pool, kw, owners, first


@torch.no_grad()
def _one_by_one(model, prompts, n, dense):
    """Greedy tokens (B, n) and the logits that followed each of them."""
    from winnow_amd import packed_backend as pb
    pool, kw, owners, first = _setup(model, prompts, n, dense)
    toks, lengths, logits = [[t] for t in first], [len(p) for p in prompts], []
    for _ in range(n - 1):
        cache = pb.PagedPackedCache(pool, owners, lengths, **kw)
        out = model(input_ids=torch.tensor([[t[-1]] for t in toks], device=DEV),
                    position_ids=torch.tensor(lengths, device=DEV)[:, None], past_key_values=cache, use_cache=True)
        lengths = cache.lengths
        logits.append(out.logits[:, -1].float())
        for t, x in zip(toks, logits[-1]):
            t.append(int(x.argmax()))
    return toks, torch.stack(logits, 1)


def _draft(known, done, T, g):
    """A tree of T tokens for one sequence: node 0 is the last token decided, a branch of right
    guesses (known[done:]) among wrong ones that hang anywhere. (tokens, parents)"""
    right = int(torch.randint(0, 5, (1,), generator=g))
    tokens, parents, tip = [known[done - 1]], [-1], 0
    for i in range(1, T):
        if right > 0 and done + len(tokens) - 1 < len(known) and float(torch.rand((), generator=g)) < 0.5:
            depth, n = 0, tip
            while n > 0:
                n, depth = parents[n], depth + 1
            if done + depth < len(known):
                parents.append(tip)
                tokens.append(known[done + depth])
                tip, right = i, right - 1
                continue
        parents.append(int(torch.randint(0, i, (1,), generator=g)))
        tokens.append(int(torch.randint(0, 128, (1,), generator=g)))
    return tokens, parents


@pytest.mark.parametrize("dense", [False, True])
@torch.no_grad()
def test_drafted_trees_give_the_tokens_of_one_by_one_decoding(model, dense):
    from tiny_qwen import prompts as make
    from winnow_amd import packed_backend as pb
    from winnow_amd.logprobs import token_logprobs
    prompts, n, T = make(3, 4), 24, 11
    want, steps = _one_by_one(model, prompts, n, dense)
    pool, kw, owners, first = _setup(model, prompts, n + T, dense)
    toks, lengths, forwards = [[t] for t in first], [len(p) for p in prompts], 0
    g = torch.Generator().manual_seed(8)
    pb.BACKEND_COUNTS.clear()
    while min(len(t) for t in toks) < n:
        drafts = [_draft(w, min(len(t), n), T, g) for w, t in zip(want, toks)]
        ids, tree = torch.tensor([d[0] for d in drafts], device=DEV), [d[1] for d in drafts]
        cache = pb.PagedPackedCache(pool, owners, lengths, tree=tree, **kw)
        out = model(input_ids=ids, position_ids=pb.tree_positions(tree, lengths).to(DEV), past_key_values=cache, use_cache=True)
        forwards += 1
        scores = token_logprobs(out.logits, ids, top=1)
        best, paths = scores.top_ids[..., 0].tolist(), []
        for b, (tokens, parents) in enumerate(drafts):
            path = [0]
            while len(toks[b]) < n:
                at = path[-1]
                scale = float(steps[b].abs().max())
                err = float((out.logits[b, at].float() - steps[b, len(toks[b]) - 1]).abs().max())
                assert err <= (2e-2 if dense else 1e-3) * scale, (b, at, err)
                toks[b].append(best[b][at])
                nxt = [i for i in range(T) if parents[i] == at and tokens[i] == best[b][at]]
                if not nxt:
                    break
                path.append(nxt[0])
            paths.append(path if len(toks[b]) < n else [])           # one that is done stays where it is
        before = lengths
        lengths = cache.commit(paths)
        assert lengths == [L + len(p) for L, p in zip(before, paths)]
        if forwards > n:
            break
    assert toks == want
    assert forwards < n - 3                                          # some steps kept more than one token
    route = "tree_dense_sdpa" if dense else "tree_hip_packed"
    assert set(pb.BACKEND_COUNTS) == {route} and pb.BACKEND_COUNTS[route] == 2 * forwards


def test_the_engine_scores_its_tokens(model):
    """``Request.top_logprobs``: a score per generated token, beside requests that ask for none or
    another number; the tokens stay those of an unscored run."""
    from tiny_qwen import prompts as make
    from winnow_amd import packed_backend as pb
    from winnow_amd.engine import Engine, EngineConfig, Request
    prompts = make(3, 6)

    def run(tops):
        model.config._attn_implementation = pb.ATTN_NAME
        pool = pb.make_pool(model.config, bit_width=8, num_pages=64, page_size=16, device=DEV)
        kq, vq = pb.quantizers_for(model.config, 8, DEV)
        e = Engine(model, pool, kq, vq, pb.head_dim_of(model.config), config=EngineConfig(prefill_chunk=16))
        seen, events = {}, []
        # the logits of a request's last prompt token and of every step after it
        e.on_logits = lambda rs, lg: [seen.setdefault(r.request_id, []).append(lg[i].double().cpu()) for i, r in enumerate(rs)]
        reqs = [Request(f"r{i}", p, 6, top_logprobs=t, on_event=lambda r, ev: events.append((r.request_id, ev)))
                for i, (p, t) in enumerate(zip(prompts, tops))]
        for r in reqs:
            e.submit(r)
        e.run_until_idle()
        return reqs, seen, events
    plain, _, events = run([None] * 3)
    assert not any("score" in ev for _, ev in events) and all(r.logprobs == [] for r in plain)
    reqs, seen, events = run([None, 0, 5])
    assert [r.generated for r in reqs] == [r.generated for r in plain] and all(r.status == "length" for r in reqs)
    assert reqs[0].logprobs == []
    for r in reqs[1:]:
        assert len(r.logprobs) == 6
        assert [ev["score"] for rid, ev in events if rid == r.request_id and ev["kind"] == "token"] == r.logprobs
        for s, token, x in zip(r.logprobs, r.generated, seen[r.request_id][-6:]):
            lp = torch.log_softmax(x, -1)
            assert abs(s.logprob - float(lp[token])) < 1e-5 * (1 + abs(float(lp[token])))
            assert abs(s.entropy + float((lp.exp() * lp).sum())) < 1e-4
            order = torch.sort(x, descending=True, stable=True).indices[:r.top_logprobs].tolist()
            assert [i for i, _ in s.alternatives] == order
            assert all(abs(v - float(lp[i])) < 1e-5 * (1 + abs(float(lp[i]))) for i, v in s.alternatives)
