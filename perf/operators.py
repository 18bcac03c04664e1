"""The operators of a speculative decoding step, with the sizes they are called at.

A draft proposes a small tree of tokens per sequence; the model runs once over all of
them and the longest branch that it agrees with is kept. Three operators carry that step
over the packed cache:

``tree``      ``packed_tree_attention``: each drafted token attends to its sequence's
              packed history and to its own ancestors among the drafted tokens, whose
              K and V the cache already holds in its last positions.
``commit``    ``commit_kv``: the cache rows of the accepted branch move to the positions
              right behind the history, in every layer, and the lengths follow.
``logprobs``  ``token_logprobs``: the log probability of the drafted token, the entropy
              and the most likely alternatives of every row of the model's logits.

Codes are those of vectors N(0, 1/D) under a Lloyd-Max codebook, as the cache's random
rotation leaves them, norms are log-normal, page tables shuffled. Where ``own`` is false
``run`` computes an operator from its formula with elementary torch operations in 32 bits.
"""
import functools
import math
import random

import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
ESIZE = {"bf16": 2, "fp16": 2, "fp32": 4}
MAX_NODES = 64          # drafted tokens per sequence
WIDTHS = ((4, 4), (4, 4), (4, 4), (6, 6), (4, 6), (6, 4), (8, 8), (3, 3), (5, 5), (2, 2), (8, 4))
HEADS = ((32, 8), (28, 4), (64, 8), (8, 8), (8, 2), (14, 2), (40, 8), (16, 1))


# ------------------------------------------------------------------------------ cases

def _tree(name, B, Hq, Hkv, D, T, Lmin, Lmax, bwk, bwv, S, dtype):
    return dict(name=name, op="tree", B=B, Hq=Hq, Hkv=Hkv, D=D, T=T, Lmin=Lmin, Lmax=Lmax, bwk=bwk, bwv=bwv, S=S, dtype=dtype)


def listed():
    return [
        # one user mid-conversation, a draft of eight tokens: latency counts
        _tree("tree_one_user", 1, 32, 8, 128, 8, 300, 300, 4, 4, 16, "bf16"),
        # a serving batch of ragged conversations, a bushy tree, seven query heads per kv head
        _tree("tree_batch", 8, 28, 4, 128, 26, 500, 6000, 4, 4, 16, "bf16"),
        # the decode benchmark's batch at 32k context, sixteen drafted tokens
        _tree("tree_32k", 16, 32, 8, 128, 16, 32768, 32768, 4, 4, 16, "bf16"),
        # few long contexts, the widest tree, K and V of different widths, half precision
        _tree("tree_wide_k4v6", 4, 64, 8, 128, 64, 15000, 20000, 4, 6, 16, "fp16"),
        # a small model with 64-wide heads at 8 bits, in single precision
        _tree("tree_hd64_fp32", 3, 14, 2, 64, 5, 100, 1000, 8, 8, 32, "fp32"),
        # one user's accepted branch, 28 layers at 8 bits
        dict(name="commit_one_user", op="commit", layers=28, B=1, Hkv=4, D=128, T=8, A=5, Lmin=300, Lmax=300, bwk=8, bwv=8, S=16),
        # a full batch over 32 layers, wide trees, long accepted branches
        dict(name="commit_batch", op="commit", layers=32, B=16, Hkv=8, D=128, T=64, A=12, Lmin=500, Lmax=4000, bwk=4, bwv=4, S=16),
        # an unquantized (bf16) cache's pages
        dict(name="commit_dense", op="commit", layers=32, B=24, Hkv=8, D=128, T=26, A=7, Lmin=100, Lmax=1000, bwk=0, bwv=0, S=32),
        # the next token of one request, five alternatives shown to the user
        dict(name="logprobs_one_row", op="logprobs", N=1, V=128256, top=5, dtype="fp32"),
        # every node of a batch of drafts, a vocabulary that is no multiple of anything
        dict(name="logprobs_odd_fp16", op="logprobs", N=208, V=50257, top=1, dtype="fp16"),
        # every node of a full batch of wide trees, the most alternatives
        dict(name="logprobs_many_rows", op="logprobs", N=1024, V=128256, top=20, dtype="bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["tree", "tree", "tree", "commit", "logprobs", "logprobs"])
    if op == "logprobs":
        case = dict(op=op, N=_log(rng, 1, 1024), V=_log(rng, 100, 128256), top=rng.choice([0, 1, 2, 5, 20, rng.randint(1, 32)]),
                    dtype=rng.choice(["bf16", "fp16", "fp32"]))
        while case["N"] * case["V"] * ESIZE[case["dtype"]] > 1024 * 128256 * 2:
            case["N"] //= 2
        return case
    if op == "commit":
        bwk, bwv = rng.choice(WIDTHS + ((0, 0),))
        T = rng.randint(1, MAX_NODES)
        lo = _log(rng, 1, 2000)
        case = dict(op=op, layers=_log(rng, 1, 40), B=_log(rng, 1, 24), Hkv=rng.choice([1, 2, 4, 8]), D=rng.choice([64, 128, 128, 256]), T=T,
                    A=rng.randint(1, min(T, 12)), Lmin=lo, Lmax=rng.randint(lo, 2 * lo), bwk=bwk, bwv=bwv, S=rng.choice([16, 16, 32, 64]))
        while case["layers"] > 1 and case["layers"] * _vectors(case) * (_row_bytes(case, "bwk") + _row_bytes(case, "bwv")) > 1_500_000_000:
            case["layers"] //= 2
        return case
    Hq, Hkv = rng.choice(HEADS)
    bwk, bwv = rng.choice(WIDTHS)
    lo = _log(rng, 1, 20000)
    case = dict(op=op, B=_log(rng, 1, 24), Hq=Hq, Hkv=Hkv, D=rng.choice([64, 128, 128, 128, 256]), T=_log(rng, 1, MAX_NODES), Lmin=lo,
                Lmax=rng.randint(lo, min(32768, 3 * lo)), bwk=bwk, bwv=bwv, S=rng.choice([16, 16, 32, 64]), dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]))
    while case["B"] > 1 and (_vectors(case) > 4_000_000 or _scores(case) > 200_000_000):
        case["B"] //= 2
    while _vectors(case) > 4_000_000 or _scores(case) > 200_000_000:
        case["Lmin"], case["Lmax"] = case["Lmin"] // 2, case["Lmax"] // 2
    return case


def _lens(case):
    """History lengths, before the drafted tokens: fixed by the case, spread over its range."""
    r = random.Random(case["Lmin"] * 31 + case["Lmax"])
    return [r.randint(case["Lmin"], case["Lmax"]) for _ in range(case["B"])]


def _counts(case):
    """Accepted tokens per sequence, 1 .. A."""
    return [1 + (5 * b + 3) % case["A"] for b in range(case["B"])]


def _vectors(case):
    return (sum(_lens(case)) + case["B"] * case["T"]) * case["Hkv"]


def _scores(case):
    return (sum(_lens(case)) + case["B"] * case["T"]) * case["Hq"] * case["T"]


def work(case):
    if case["op"] == "logprobs":
        n, top = case["N"], case["top"]
        return {"bytes": n * case["V"] * ESIZE[case["dtype"]] + n * (8 + 4 + 4 + 12 * top), "flops": 4.0 * n * case["V"]}
    D, Hkv = case["D"], case["Hkv"]
    row = _row_bytes(case, "bwk") + _row_bytes(case, "bwv")
    if case["op"] == "commit":
        moved = sum(_counts(case))
        return {"bytes": 2 * case["layers"] * Hkv * moved * row + 4 * moved + 12 * case["B"], "flops": 0}
    B, Hq, T = case["B"], case["Hq"], case["T"]
    pages = sum(-(-(L + T) // case["S"]) for L in _lens(case))
    io = 2 * B * Hq * T * D * ESIZE[case["dtype"]] + 8 * D * D + 4 * pages + 4 * B * (T + 1)
    return {"bytes": _vectors(case) * row + io, "flops": 4.0 * D * _scores(case) + 4.0 * B * Hq * T * D * D}


def _row_bytes(case, side):
    """Bytes of one token's row of one head, norm included."""
    return case["D"] * case[side] // 8 + 2 if case[side] else 2 * case["D"]


# ----------------------------------------------------------------------------- inputs

@functools.lru_cache(maxsize=None)
def _codebook(bits, dim):
    """Lloyd-Max levels of N(0, 1/dim), float64 on the host."""
    c = math.sqrt(2) * torch.special.erfinv((2 * torch.arange(2 ** bits, dtype=torch.float64) + 1) / 2 ** bits - 1)
    inf = torch.tensor([math.inf], dtype=torch.float64)
    for _ in range(200):
        e = torch.cat([-inf, (c[1:] + c[:-1]) / 2, inf])
        cdf, pdf = (1 + torch.erf(e / math.sqrt(2))) / 2, torch.exp(-e * e / 2) / math.sqrt(2 * math.pi)
        c = (pdf[:-1] - pdf[1:]) / (cdf[1:] - cdf[:-1])
    return c / math.sqrt(dim)


def _rotation(D, g):
    return torch.linalg.qr(torch.randn(D, D, generator=g, device=DEV))[0].contiguous()


def _pages(lead, D, bits, g):
    """Random packed rows (*lead, D bits / 8) uint8, codes LSB-first along D, and norms."""
    mids = _codebook(bits, D)
    mids = ((mids[1:] + mids[:-1]) / 2).to(DEV, torch.float32)
    out = torch.empty(*lead, D * bits // 8, dtype=torch.uint8, device=DEV)
    flat = out.view(-1, D // 8, bits)
    at = torch.arange(8, device=DEV)
    for i in range(0, len(flat), 1 << 20):
        part = flat[i:i + (1 << 20)]
        y = torch.randn(*part.shape[:-1], 8, generator=g, device=DEV) / math.sqrt(D)
        word = (torch.bucketize(y, mids) << (bits * at)).sum(-1, keepdim=True)
        part.copy_((word >> (8 * at[:bits])) & 255)
    norms = torch.exp(0.3 * torch.randn(lead, generator=g, device=DEV)) * math.sqrt(D)
    return out, norms.half()


def _parents(B, T, r):
    """A tree of T drafted tokens per sequence: a node's parent comes before it, -1 is the history's end."""
    chain = r.choice([0.2, 0.5, 0.8])
    return [[-1 if i == 0 or r.random() < 0.08 else (i - 1 if r.random() < chain else r.randrange(i)) for i in range(T)] for _ in range(B)]


def _table(lens, S, r):
    """A shuffled page table, -1 past a sequence's pages, and the pool's page count."""
    need = [-(-L // S) for L in lens]
    order = list(range(sum(need) + 3))
    r.shuffle(order)
    table = torch.full((len(lens), max(need)), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = torch.tensor(order[at:at + n], dtype=torch.int32)
        at += n
    return table, len(order)


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    r = random.Random(seed)
    st = dict(case=case)
    if case["op"] == "logprobs":
        # most of a model's mass lies on few tokens
        x = torch.randn(case["N"], case["V"], generator=g, device=DEV) * 2
        peak = torch.randint(case["V"], (case["N"], 6), generator=g, device=DEV)
        x.scatter_add_(1, peak, 12 * torch.rand(case["N"], 6, generator=g, device=DEV))
        st["logits"] = x.to(DTYPES[case["dtype"]])
        st["tokens"] = torch.where(torch.rand(case["N"], generator=g, device=DEV) < 0.7, peak[:, 0],
                                   torch.randint(case["V"], (case["N"],), generator=g, device=DEV))
        return st
    B, T, S, D, Hkv = case["B"], case["T"], case["S"], case["D"], case["Hkv"]
    hist = _lens(case)
    table, P = _table([L + T for L in hist], S, r)
    st["table_host"], st["table"] = table, table.to(DEV)
    st["start_host"] = torch.tensor(hist, dtype=torch.int32)
    st["seq_host"] = st["start_host"] + T
    st["start"], st["seq"] = st["start_host"].to(DEV), st["seq_host"].to(DEV)
    lead = (P, Hkv, S) if case["op"] == "tree" else (case["layers"], P, Hkv, S)
    for side in "kv":
        bits = case["bw" + side]
        if bits:
            st[side], st[side + "n"] = _pages(lead, D, bits, g)
        else:
            st[side], st[side + "n"] = torch.randn(*lead, D, generator=g, device=DEV).bfloat16(), None
    if case["op"] == "commit":
        counts = _counts(case)
        path = [sorted(r.sample(range(T), n)) + [0] * (case["A"] - n) for n in counts]
        st["path"] = torch.tensor(path, dtype=torch.int32, device=DEV)
        st["counts"] = torch.tensor(counts, dtype=torch.int32, device=DEV)
        return st
    for side in "kv":
        st["pi_" + side] = _rotation(D, g)
        st["cb_" + side] = _codebook(case["bw" + side], D).to(DEV, torch.float32)
    parents = torch.tensor(_parents(B, T, r), dtype=torch.int32)
    st["parents_host"], st["parents"] = parents, parents.to(DEV)
    st["q"] = (1.5 * torch.randn(B, case["Hq"], T, D, generator=g, device=DEV)).to(DTYPES[case["dtype"]])
    st["scale"] = 1.0 / math.sqrt(D)
    return st


# ------------------------------------------------------------------------- plain forms

def _unpack(rows, D, bits):
    """(..., D bits / 8) bytes -> (..., D) codes."""
    at = torch.arange(8, device=rows.device)
    word = (rows.view(*rows.shape[:-1], D // 8, bits).to(torch.int64) << (8 * at[:bits])).sum(-1, keepdim=True)
    return ((word >> (bits * at)) & (2 ** bits - 1)).flatten(-2)


def _history(st, side, L):
    """(B, Hkv, L, D) vectors of one side, the first L positions of every table row."""
    case, S = st["case"], st["case"]["S"]
    t = torch.arange(L, device=DEV)
    page, slot = st["table"].long()[:, t // S].clamp(min=0), (t % S)[None, :]
    codes = _unpack(st[side][page, :, slot], case["D"], case["bw" + side])          # (B, L, Hkv, D)
    x = (st["cb_" + side][codes] @ st["pi_" + side]) * st[side + "n"][page, :, slot].float()[..., None]
    return x.transpose(1, 2).contiguous()


def _ancestors(parents):
    """(B, T, T) whether node i descends from node j or is it: paths of up to T steps to a parent or nowhere."""
    T = parents.shape[1]
    eye = torch.eye(T, device=DEV)[None]
    up = (parents.long()[:, :, None] == torch.arange(T, device=DEV)).float()
    return torch.linalg.matrix_power(eye + up, T) > 0


def _visible(st, L):
    """(B, T, L) whether drafted token i sees the key at position j."""
    T = st["parents"].shape[1]
    j = torch.arange(L, device=DEV)[None, :] - st["start"].long()[:, None]            # (B, L): node of a position
    anc = _ancestors(st["parents"]).gather(2, j.clamp(0, T - 1)[:, None, :].expand(-1, T, -1))
    return (j < 0)[:, None, :] | (anc & (j < T)[:, None, :])


def _tree_plain(st):
    case, q = st["case"], st["q"]
    B, Hq, T, D = q.shape
    L, n = int(st["seq_host"].max()), Hq // case["Hkv"]
    k, v = _history(st, "k", L), _history(st, "v", L)
    rows = q.float().view(B, case["Hkv"], n * T, D)
    s = (rows @ k.transpose(2, 3).contiguous()) * st["scale"]
    s = s.view(B, case["Hkv"], n, T, L).masked_fill(~_visible(st, L)[:, None, None], -math.inf)
    p = torch.exp(s - s.amax(-1, keepdim=True))
    o = (p / p.sum(-1, keepdim=True)).view(B, case["Hkv"], n * T, L) @ v
    return o.view(B, Hq, T, D).to(q.dtype)


def _commit_plain(st):
    case, S = st["case"], st["case"]["S"]
    counts, A = st["counts"].long(), case["A"]
    i = torch.arange(A, device=DEV)[None, :]
    live = i < counts[:, None]
    # entries past a sequence's count repeat its first one (of no accepted token: position 0 onto itself)
    first = torch.where(counts > 0, st["path"][:, 0].long(), 0)[:, None]
    src = st["start"].long()[:, None] + torch.where(live, st["path"].long(), first)
    dst = st["start"].long()[:, None] + torch.where(live, i, 0)
    table = st["table"].long()
    sp, ss, dp, ds = table.gather(1, src // S), src % S, table.gather(1, dst // S), dst % S
    st["k"][:, dp, :, ds] = st["k"][:, sp, :, ss]
    st["v"][:, dp, :, ds] = st["v"][:, sp, :, ss]
    if st["kn"] is not None:
        st["kn"][:, dp, :, ds] = st["kn"][:, sp, :, ss]
        st["vn"][:, dp, :, ds] = st["vn"][:, sp, :, ss]
    return st["start"] + st["counts"]


def _order(x):
    """Whole numbers in the order of (value, then the lowest index first) along the last axis of a float32 tensor."""
    b = (x + 0.0).view(torch.int32).long()
    b = torch.where(b < 0, -(b & 0x7FFFFFFF), b)
    return (b << 32) - torch.arange(x.shape[-1], device=x.device)


def _logprobs_plain(st):
    x, top = st["logits"].float(), st["case"]["top"]
    d = x - x.amax(-1, keepdim=True)
    e = torch.exp(d)
    total = e.sum(-1, keepdim=True)
    lp = d - torch.log(total)
    got = lp.gather(1, st["tokens"][:, None])[:, 0]
    entropy = torch.log(total)[:, 0] - (e * d).sum(-1) / total[:, 0]
    if not top:
        return {"logprob": got, "entropy": entropy}
    ids = torch.topk(_order(x), top, dim=-1).indices
    return {"logprob": got, "entropy": entropy, "top_logprobs": lp.gather(1, ids), "top_ids": ids}


# -------------------------------------------------------------------------------- run

def run(st):
    op = st["case"]["op"]
    if own:
        return _OWN[op](st)
    if op == "tree":
        return _tree_plain(st)
    if op == "commit":
        return {"lengths": _commit_plain(st), "k": st["k"], "v": st["v"], "kn": st["kn"], "vn": st["vn"]}
    return _logprobs_plain(st)


def _tree_own(st):
    from winnow_amd import packed_attention as pa
    case = st["case"]
    kv = pa.PackedKV(st["k"], st["kn"], st["v"], st["vn"], st["table"], st["seq"], pa.Quantizer(st["pi_k"], st["cb_k"], case["bwk"]),
                     pa.Quantizer(st["pi_v"], st["cb_v"], case["bwv"]), case["D"], seq_lens_host=st["seq_host"], page_table_host=st["table_host"])
    return pa.packed_tree_attention(st["q"], kv, st["scale"], st["parents"], parents_host=st["parents_host"])


def _commit_own(st):
    from winnow_amd.packed_backend import commit_kv
    lengths = commit_kv(st["k"], st["v"], st["kn"], st["vn"], st["table"], st["start"], st["path"], st["counts"], nodes=st["case"]["T"],
                        page_table_host=st["table_host"], start_pos_host=st["start_host"])
    return {"lengths": lengths, "k": st["k"], "v": st["v"], "kn": st["kn"], "vn": st["vn"]}


def _logprobs_own(st):
    from winnow_amd.logprobs import token_logprobs
    r = token_logprobs(st["logits"], st["tokens"], top=st["case"]["top"])
    if not st["case"]["top"]:
        return {"logprob": r.logprob, "entropy": r.entropy}
    return {"logprob": r.logprob, "entropy": r.entropy, "top_logprobs": r.top_logprobs, "top_ids": r.top_ids}


_OWN = {"tree": _tree_own, "commit": _commit_own, "logprobs": _logprobs_own}


# -------------------------------------------------------------------- in 64 bits, apart

def exact(case, seed):
    """The operators by their definitions, in 64 bits, a sequence (or a block of rows) at a time."""
    st = prepare(case, seed)
    return {"tree": _tree_exact, "commit": _commit_exact, "logprobs": _logprobs_exact}[case["op"]](case, st)


def _vectors_exact(case, st, side, b, n):
    bits, D, S = case["bw" + side], case["D"], case["S"]
    ids = st["table_host"][b, :-(-n // S)].long().to(DEV)
    rows = st[side][ids].transpose(1, 2).reshape(-1, case["Hkv"], D * bits // 8)[:n]                 # (n, Hkv, NB)
    bit = (rows[..., None].int() >> torch.arange(8, device=DEV, dtype=torch.int32)) & 1
    code = (bit.flatten(-2).view(n, case["Hkv"], D, bits) << torch.arange(bits, device=DEV, dtype=torch.int32)).sum(-1)
    y = st["cb_" + side].double()[code]
    norm = st[side + "n"][ids].transpose(1, 2).reshape(-1, case["Hkv"])[:n].double()
    return torch.matmul(y, st["pi_" + side].double()) * norm[..., None]


def _tree_exact(case, st):
    B, Hq, T, D = st["q"].shape
    n = Hq // case["Hkv"]
    out = torch.zeros(B, Hq, T, D, dtype=torch.float64, device=DEV)
    for b in range(B):
        past = int(st["start_host"][b])
        k, v = (_vectors_exact(case, st, side, b, past + T) for side in "kv")
        sees = torch.zeros(T, past + T, dtype=torch.bool)
        sees[:, :past] = True
        for i in range(T):
            node = i
            while node >= 0:
                sees[i, past + node] = True
                node = int(st["parents_host"][b, node])
        sees = sees.to(DEV)
        for h in range(Hq):
            s = (st["q"][b, h].double() @ k[:, h // n].t()) / math.sqrt(D)
            out[b, h] = torch.softmax(s.masked_fill(~sees, -math.inf), -1) @ v[:, h // n]
    return out


def _commit_exact(case, st):
    S, start = case["S"], st["start_host"].tolist()
    table, path, counts = st["table_host"].tolist(), st["path"].tolist(), st["counts"].tolist()
    new = {name: st[name].clone() if st[name] is not None else None for name in ("k", "v", "kn", "vn")}
    for b in range(case["B"]):
        for i in range(counts[b]):
            s, d = start[b] + path[b][i], start[b] + i
            for name, pages in new.items():
                if pages is not None:
                    pages[:, table[b][d // S], :, d % S] = st[name][:, table[b][s // S], :, s % S]
    # what moves keeps its type: the only floating outputs are norms and unquantized rows
    return {"lengths": torch.tensor([a + n for a, n in zip(start, counts)], dtype=torch.int32), **new}


def _logprobs_exact(case, st):
    lp, entropy, values, ids = [], [], [], []
    for i in range(0, case["N"], 64):
        x = st["logits"][i:i + 64].double()
        rows = torch.log_softmax(x, -1)
        lp.append(rows.gather(1, st["tokens"][i:i + 64, None])[:, 0])
        entropy.append(-(torch.exp(rows) * rows).sum(-1))
        if case["top"]:
            ids.append(torch.sort(x, dim=-1, descending=True, stable=True).indices[:, :case["top"]])
            values.append(rows.gather(1, ids[-1]))
    out = {"logprob": torch.cat(lp), "entropy": torch.cat(entropy)}
    return {**out, "top_logprobs": torch.cat(values), "top_ids": torch.cat(ids)} if case["top"] else out
