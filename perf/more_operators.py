"""The operators of a step of a long conversation over the packed cache, with the sizes they are called at.

A step appends the new tokens' K and V, attends to what of the conversation is kept in
view, and picks the next token from logits that penalties and a grammar have been applied
to. Three operators carry it:

``append``  ``append_rotated_kv``: the position rotation of q and k (the model's cos and sin
            tables), K and V quantized, bit-packed and written to the pages, q' returned.
``window``  ``packed_window_attention``: the query at position p sees the last ``W``
            positions up to its own and the conversation's first ``sinks``.
``logits``  ``adjust_logits``: penalties for tokens of the history, biases of single tokens,
            and a bit mask of the tokens that a grammar allows.

Codes are those of vectors N(0, 1/D) under a Lloyd-Max codebook, as the cache's random
rotation leaves them, norms are log-normal, page tables shuffled. Where ``own`` is false
``run`` computes an operator from its formula with elementary torch operations, in 32 bits;
in 64 what decides a code (the packed bytes are whole numbers: every code is the bucket of
a correctly rounded value).
"""
import functools
import math
import random
import types

import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
ESIZE = {"bf16": 2, "fp16": 2, "fp32": 4}
WIDTHS = ((4, 4), (4, 4), (4, 4), (6, 6), (4, 6), (6, 4), (8, 8), (3, 3), (5, 5), (2, 2), (8, 4))
HEADS = ((32, 8), (28, 4), (64, 8), (8, 8), (8, 2), (14, 2), (40, 8), (16, 1))


# ------------------------------------------------------------------------------ cases

def _window(name, B, Hq, Hkv, D, Q, W, sinks, Lmin, Lmax, bwk, bwv, S, dtype):
    return dict(name=name, op="window", B=B, Hq=Hq, Hkv=Hkv, D=D, Q=Q, W=W, sinks=sinks, Lmin=Lmin, Lmax=Lmax, bwk=bwk, bwv=bwv, S=S, dtype=dtype)


def _append(name, B, Hq, Hkv, D, n, R, Lmin, Lmax, bwk, bwv, S, dtype):
    return dict(name=name, op="append", B=B, Hq=Hq, Hkv=Hkv, D=D, n=n, R=R, Lmin=Lmin, Lmax=Lmax, bwk=bwk, bwv=bwv, S=S, dtype=dtype)


def listed():
    return [
        # one user's next token, a window of 1,024 and four sinks: latency counts
        _window("window_one_user", 1, 32, 8, 128, 1, 1024, 4, 5000, 5000, 4, 4, 16, "bf16"),
        # a full serving batch of long conversations, a wide window
        _window("window_batch", 32, 32, 8, 128, 1, 8192, 4, 9000, 16000, 4, 4, 16, "bf16"),
        # a small model with 64-wide heads at 8 bits, in single precision, some histories shorter than the window
        _window("window_hd64_fp32", 3, 14, 2, 64, 1, 512, 1, 100, 1000, 8, 8, 32, "fp32"),
        # a prompt chunk as the engine cuts them, deep in a long prompt
        _window("window_prompt_chunk", 1, 32, 8, 128, 512, 4096, 4, 9000, 9000, 4, 4, 16, "bf16"),
        # ragged batch of short continuations, an odd window without sinks, K and V of different widths
        _window("window_ragged_k4v6", 5, 28, 4, 128, 37, 300, 0, 40, 2000, 4, 6, 16, "fp16"),
        # one user's next token
        _append("append_one_user", 1, 32, 8, 128, 1, 128, 300, 300, 4, 4, 16, "bf16"),
        # a decode step of a large batch at 8 bits
        _append("append_batch", 64, 28, 4, 128, 1, 128, 100, 1000, 8, 8, 16, "bf16"),
        # a whole prompt
        _append("append_prompt", 1, 32, 8, 128, 8191, 128, 0, 0, 4, 4, 16, "bf16"),
        # short continuations of a small model, half of each head rotated, widths that share bytes
        _append("append_ragged_hd64", 6, 14, 2, 64, 37, 32, 20, 500, 3, 5, 32, "fp16"),
        # the next token of one request under a grammar, with penalties over its history
        dict(name="logits_one_row", op="logits", N=1, V=128256, H=900, J=20, mask=True, dtype="fp32"),
        # a batch without a grammar, a vocabulary that is no multiple of anything
        dict(name="logits_odd_fp16", op="logits", N=208, V=50257, H=333, J=5, mask=False, dtype="fp16"),
        # many rows under grammars, long histories
        dict(name="logits_many_rows", op="logits", N=1024, V=128256, H=4096, J=32, mask=True, dtype="bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["window", "window", "window", "append", "append", "logits", "logits"])
    if op == "logits":
        case = dict(op=op, N=_log(rng, 1, 1024), V=_log(rng, 100, 128256), H=_log(rng, 1, 4096), J=rng.choice([0, 1, 7, rng.randint(1, 64)]),
                    mask=rng.random() < 0.6, dtype=rng.choice(["bf16", "fp16", "fp32"]))
        while case["N"] * case["V"] * ESIZE[case["dtype"]] > 1024 * 128256 * 2:
            case["N"] //= 2
        return case
    Hq, Hkv = rng.choice(HEADS)
    bwk, bwv = rng.choice(WIDTHS)
    base = dict(op=op, Hq=Hq, Hkv=Hkv, D=rng.choice([64, 128, 128, 128, 256]), bwk=bwk, bwv=bwv, S=rng.choice([16, 16, 32, 64]),
                dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]))
    if op == "append":
        lo = _log(rng, 1, 1000)
        case = dict(base, B=_log(rng, 1, 64), n=rng.choice([1, 1, _log(rng, 2, 4096)]), Lmin=lo, Lmax=rng.randint(lo, 2 * lo),
                    R=base["D"] // rng.choice([1, 1, 1, 2, 4]))
        while case["B"] > 1 and case["B"] * case["n"] * (Hq + 2 * Hkv) * case["D"] > 8191 * 48 * 128:
            case["B"] //= 2
        while case["B"] * case["n"] * (Hq + 2 * Hkv) * case["D"] > 8191 * 48 * 128:
            case["n"] //= 2
        return case
    lo = _log(rng, 1, 20000)
    case = dict(base, B=_log(rng, 1, 32), Q=rng.choice([1, 1, 1, _log(rng, 2, 512)]), W=_log(rng, 16, 8192), sinks=rng.choice([0, 0, 1, 4, 4, 16, rng.randint(1, 200)]),
                Lmin=lo, Lmax=rng.randint(lo, 2 * lo))
    case["Lmin"], case["Lmax"] = max(case["Lmin"], case["Q"]), max(case["Lmax"], case["Q"])
    while case["B"] > 1 and (sum(_lens(case)) * Hkv > 3_200_000 or _pairs(case) * Hq * case["D"] > 512 * 4100 * 32 * 128):
        case["B"] //= 2
    while _pairs(case) * Hq * case["D"] > 512 * 4100 * 32 * 128:
        case["Q"] //= 2
    return case


def _lens(case):
    """Lengths (of an append: before it), fixed by the case, spread over its range."""
    r = random.Random(case["Lmin"] * 31 + case["Lmax"])
    return [r.randint(case["Lmin"], case["Lmax"]) for _ in range(case["B"])]


def _pairs(case):
    """Visible (query, key) pairs of one head over the batch."""
    Q, W, sinks = case["Q"], case["W"], case["sinks"]
    return sum(min(p + 1, W) + min(sinks, max(0, p + 1 - W)) for L in _lens(case) for p in range(L - Q, L))


def _keys(case):
    """Keys of one head that some query sees, over the batch."""
    return sum(min(L, case["W"] + case["Q"] - 1) + min(case["sinks"], max(0, L - case["W"] - case["Q"] + 1)) for L in _lens(case))


def work(case):
    if case["op"] == "logits":
        n, es = case["N"], ESIZE[case["dtype"]]
        mask = 4 * n * -(-case["V"] // 32) if case["mask"] else 0
        return {"bytes": 2 * n * case["V"] * es + mask + n * (4 * case["H"] + 8 * case["J"] + 20), "flops": 4.0 * n * case["V"]}
    D, Hq, Hkv, B, es = case["D"], case["Hq"], case["Hkv"], case["B"], ESIZE[case["dtype"]]
    row = D * (case["bwk"] + case["bwv"]) // 8 + 4
    if case["op"] == "append":
        t = B * case["n"]
        return {"bytes": t * (2 * Hq * D * es + 2 * Hkv * D * es + 2 * case["R"] * es + Hkv * row) + 8 * D * D + 8 * B,
                "flops": t * (4.0 * Hkv * D * D + 3.0 * (Hq + Hkv) * case["R"])}
    rows = B * case["Q"] * Hq
    return {"bytes": _keys(case) * Hkv * row + 2 * rows * D * es + 8 * D * D, "flops": 4.0 * D * _pairs(case) * Hq + 4.0 * rows * D * D}


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


def _boundaries(bits, dim):
    c = _codebook(bits, dim)
    return ((c[1:] + c[:-1]) / 2).to(DEV, torch.float32)


def _pages(lead, D, bits, g):
    """Random packed rows (*lead, D bits / 8) uint8, codes LSB-first along D, and norms."""
    mids = _boundaries(bits, D)
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


def _prepare_logits(case, g):
    N, V, H, J = case["N"], case["V"], case["H"], case["J"]
    st = dict(case=case)
    st["logits"] = (torch.randn(N, V, generator=g, device=DEV) * 3).to(DTYPES[case["dtype"]])
    # histories repeat themselves: a third of the tokens come from a few of the row's own
    few = torch.randint(V, (N, 16), generator=g, device=DEV)
    some = few.gather(1, torch.randint(16, (N, H), generator=g, device=DEV))
    st["history"] = torch.where(torch.rand(N, H, generator=g, device=DEV) < 0.33, some, torch.randint(V, (N, H), generator=g, device=DEV)).int()
    st["lengths"] = torch.randint((H + 1) // 2, H + 1, (N,), generator=g, device=DEV).int()
    st["prompts"] = (st["lengths"] * torch.rand(N, generator=g, device=DEV)).int()
    st["repetition"] = 1 + 0.4 * torch.rand(N, generator=g, device=DEV)
    st["presence"] = 0.5 * torch.rand(N, generator=g, device=DEV)
    st["frequency"] = 0.5 * torch.rand(N, generator=g, device=DEV)
    if J:  # a row's ids differ from one another
        first, step = torch.randint(V, (N, 1), generator=g, device=DEV), max(1, V // (J + 1))
        st["bias_ids"] = ((first + step * torch.arange(J, device=DEV)) % V).int()
        st["bias"] = 5 * torch.randn(N, J, generator=g, device=DEV)
    if case["mask"]:  # words of a grammar's mask: all, none or some of 32 neighbours
        words = torch.randint(-2 ** 31, 2 ** 31, (N, -(-V // 32)), generator=g, device=DEV)
        kind = torch.rand(words.shape, generator=g, device=DEV)
        st["allowed"] = torch.where(kind < 0.4, 0, torch.where(kind < 0.8, -1, words)).int()
    return st


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    if case["op"] == "logits":
        return _prepare_logits(case, g)
    r = random.Random(seed)
    st = dict(case=case)
    B, S, D, Hkv, Hq = case["B"], case["S"], case["D"], case["Hkv"], case["Hq"]
    n = case["Q"] if case["op"] == "window" else case["n"]
    new = 0 if case["op"] == "window" else n
    lens = _lens(case)
    table, P = _table([L + new for L in lens], S, r)
    st["table_host"], st["table"] = table, table.to(DEV)
    st["lens_host"] = torch.tensor(lens, dtype=torch.int32)
    st["lens"] = st["lens_host"].to(DEV)
    for side in "kv":
        st[side], st[side + "n"] = _pages((P, Hkv, S), D, case["bw" + side], g)
        st["tq_" + side] = types.SimpleNamespace(Pi=_rotation(D, g), centroids=_codebook(case["bw" + side], D).to(DEV, torch.float32),
                                                 boundaries=_boundaries(case["bw" + side], D), bit_width=case["bw" + side])
    # a model's projections: (B, n, heads, D) in memory
    q = 1.5 * torch.randn(B, n, Hq, D, generator=g, device=DEV)
    st["q"] = q.to(DTYPES[case["dtype"]]).transpose(1, 2)
    if case["op"] == "window":
        st["scale"] = 1.0 / math.sqrt(D)
        return st
    for side in "kv":
        x = torch.randn(B, n, Hkv, D, generator=g, device=DEV) * torch.exp(0.3 * torch.randn(B, n, Hkv, 1, generator=g, device=DEV))
        st["new_" + side] = x.to(DTYPES[case["dtype"]]).transpose(1, 2)
    # the model's cos and sin of these positions, in its type: far positions have their angles in 64 bits
    freq = 10000.0 ** (-torch.arange(0, case["R"], 2, dtype=torch.float64, device=DEV) / case["R"])
    at = st["lens"].double()[:, None] + torch.arange(n, device=DEV)
    angle = at[..., None] * freq
    angle = torch.cat([angle, angle], -1)
    st["cos"], st["sin"] = angle.cos().to(DTYPES[case["dtype"]]), angle.sin().to(DTYPES[case["dtype"]])
    return st


# ------------------------------------------------------------------------- plain forms

def _unpack(rows, D, bits):
    """(..., D bits / 8) bytes -> (..., D) codes."""
    at = torch.arange(8, device=rows.device)
    word = (rows.view(*rows.shape[:-1], D // 8, bits).to(torch.int64) << (8 * at[:bits])).sum(-1, keepdim=True)
    return ((word >> (bits * at)) & (2 ** bits - 1)).flatten(-2)


def _vectors(st, side, at):
    """(B, Hkv, n, D) vectors of one side at positions ``at`` (B, n) of every sequence."""
    case, S, tq = st["case"], st["case"]["S"], st["tq_" + side]
    page, slot = st["table"].long().gather(1, at // S).clamp(min=0), at % S
    codes = _unpack(st[side][page, :, slot], case["D"], case["bw" + side])          # (B, n, Hkv, D)
    x = (tq.centroids[codes] @ tq.Pi) * st[side + "n"][page, :, slot].float()[..., None]
    return x.transpose(1, 2).contiguous()


def _window_plain(st):
    case, q = st["case"], st["q"]
    B, Hq, Q, D = q.shape
    Hkv, W, sinks, L = case["Hkv"], case["W"], case["sinks"], st["lens"].long()[:, None]
    longest = int(st["lens_host"].max())
    n = min(W + Q - 1, longest)                                   # positions that end with the last one ...
    last = L - n + torch.arange(n, device=DEV)
    first = torch.arange(min(sinks, longest - n), device=DEV).expand(B, -1)   # ... and the sinks before them
    at = torch.cat([torch.where(first < L - n, first, -1), last], 1)
    p = L - Q + torch.arange(Q, device=DEV)                       # (B, Q)
    sees = (at[:, None] >= 0) & (at[:, None] <= p[..., None]) & ((p[..., None] - at[:, None] < W) | (at[:, None] < sinks))
    k, v = _vectors(st, "k", at.clamp(min=0)), _vectors(st, "v", at.clamp(min=0))
    s = (q.float().reshape(B, Hkv, Hq // Hkv * Q, D) @ k.transpose(2, 3).contiguous()) * st["scale"]
    s = s.view(B, Hkv, Hq // Hkv, Q, -1).masked_fill(~sees[:, None, None], -math.inf)
    e = torch.exp(s - s.amax(-1, keepdim=True))
    o = (e / e.sum(-1, keepdim=True)).view(B, Hkv, Hq // Hkv * Q, -1) @ v
    return o.view(B, Hq, Q, D).to(q.dtype)


def _rotated(x, cos, sin):
    """x (B, H, n, D) with its first R channels rotated, fp32: each value rounded once."""
    R = cos.shape[-1]
    a, half = x[..., :R].double(), R // 2
    turned = torch.cat([-a[..., half:], a[..., :half]], -1)
    return torch.cat([(a * cos.double()[:, None] + turned * sin.double()[:, None]).float(), x[..., R:].float()], -1)


def _quantized(x, tq):
    """Packed rows and fp16 norms of fp32 vectors: codes are the buckets of correctly rounded values."""
    D, bits = x.shape[-1], tq.bit_width
    norm = x.double().square().sum(-1).sqrt().float().clamp(min=1e-10)
    unit = (x.double() / norm.double()[..., None]).float()
    y = (unit.double() @ tq.Pi.double().t()).float()
    code = torch.bucketize(y, tq.boundaries).view(*x.shape[:-1], D // 8, 8)
    at = torch.arange(8, device=DEV)
    word = (code << (bits * at)).sum(-1, keepdim=True)
    return ((word >> (8 * at[:bits])) & 255).to(torch.uint8).flatten(-2), norm.half()


def _append_plain(st):
    case, S, n = st["case"], st["case"]["S"], st["case"]["n"]
    at = st["lens"].long()[:, None] + torch.arange(n, device=DEV)
    page, slot = st["table"].long().gather(1, at // S), at % S
    q = _rotated(st["q"], st["cos"], st["sin"]).to(st["q"].dtype)
    k = _rotated(st["new_k"], st["cos"], st["sin"])
    for side, x in (("k", k), ("v", st["new_v"].float())):
        rows, norm = _quantized(x, st["tq_" + side])
        st[side][page, :, slot] = rows.transpose(1, 2)
        st[side + "n"][page, :, slot] = norm.transpose(1, 2)
    return q


def _logits_plain(st):
    x, hist = st["logits"].float(), st["history"].long()
    j = torch.arange(hist.shape[1], device=DEV)
    live = j < st["lengths"][:, None]
    made = live & (j >= st["prompts"][:, None])
    total = torch.zeros_like(x).scatter_add_(1, hist, live.float())
    count = torch.zeros_like(x).scatter_add_(1, hist, made.float())
    r = st["repetition"][:, None]
    x = torch.where(total > 0, torch.where(x > 0, x / r, x * r), x)
    x = x - st["frequency"][:, None] * count - st["presence"][:, None] * (count > 0)
    if st["case"]["J"]:
        x = x.scatter_add(1, st["bias_ids"].long(), st["bias"])
    if st["case"]["mask"]:
        bits = (st["allowed"][:, :, None] >> torch.arange(32, device=DEV)) & 1
        x = x.masked_fill(bits.flatten(1)[:, :x.shape[1]] == 0, -math.inf)
    return x.to(st["logits"].dtype)


# -------------------------------------------------------------------------------- run

def run(st):
    op = st["case"]["op"]
    if op == "append":
        q = _append_own(st) if own else _append_plain(st)
        return {"q": q, "k": st["k"], "v": st["v"], "kn": st["kn"], "vn": st["vn"]}
    if op == "window":
        return _window_own(st) if own else _window_plain(st)
    return _logits_own(st) if own else _logits_plain(st)


def _window_own(st):
    from winnow_amd import packed_attention as pa
    case = st["case"]
    kv = pa.PackedKV(st["k"], st["kn"], st["v"], st["vn"], st["table"], st["lens"], pa.Quantizer.from_tq(st["tq_k"]),
                     pa.Quantizer.from_tq(st["tq_v"]), case["D"], seq_lens_host=st["lens_host"], page_table_host=st["table_host"])
    return pa.packed_window_attention(st["q"], kv, st["scale"], window=case["W"], sinks=case["sinks"])


def _append_own(st):
    from winnow_amd.packed_backend import append_rotated_kv
    return append_rotated_kv(st["q"], st["new_k"], st["new_v"], st["cos"], st["sin"], st["tq_k"], st["tq_v"], st["k"], st["v"], st["kn"], st["vn"],
                             st["table"], st["lens"], page_table_host=st["table_host"], start_pos_host=st["lens_host"])


def _logits_own(st):
    from winnow_amd.logits import adjust_logits
    return adjust_logits(st["logits"], history=st["history"], lengths=st["lengths"], prompt_lengths=st["prompts"], repetition=st["repetition"],
                         presence=st["presence"], frequency=st["frequency"], bias_ids=st.get("bias_ids"), bias=st.get("bias"), allowed=st.get("allowed"))


# -------------------------------------------------------------------- in 64 bits, apart

def exact(case, seed):
    """The operators by their definitions, in 64 bits, a sequence (or a block of rows) at a time."""
    st = prepare(case, seed)
    return {"window": _window_exact, "append": _append_exact, "logits": _logits_exact}[case["op"]](case, st)


def _history_exact(case, st, side, b, positions):
    """(n, Hkv, D) float64 vectors of sequence b at ``positions``."""
    bits, D, S, tq = case["bw" + side], case["D"], case["S"], st["tq_" + side]
    page = st["table_host"][b].to(DEV).long()[positions // S]
    rows = st[side][page, :, positions % S]                                                       # (n, Hkv, NB)
    bit = (rows[..., None].int() >> torch.arange(8, device=DEV, dtype=torch.int32)) & 1
    code = (bit.flatten(-2).view(len(positions), case["Hkv"], D, bits) << torch.arange(bits, device=DEV, dtype=torch.int32)).sum(-1)
    return torch.matmul(tq.centroids.double()[code], tq.Pi.double()) * st[side + "n"][page, :, positions % S].double()[..., None]


def _window_exact(case, st):
    B, Hq, Q, D = st["q"].shape
    n, W, sinks = Hq // case["Hkv"], case["W"], case["sinks"]
    out = torch.zeros(B, Hq, Q, D, dtype=torch.float64, device=DEV)
    for b in range(B):
        L = int(st["lens_host"][b])
        lo = max(0, L - Q - W + 1)
        at = torch.tensor([j for j in range(min(sinks, lo))] + list(range(lo, L)), device=DEV)
        k, v = (_history_exact(case, st, side, b, at) for side in "kv")
        p = torch.arange(L - Q, L, device=DEV)[:, None]
        hidden = (at > p) | ((at <= p - W) & (at >= sinks))
        for h in range(Hq):
            s = (st["q"][b, h].double() @ k[:, h // n].t()) / math.sqrt(D)
            out[b, h] = torch.softmax(s.masked_fill(hidden, -math.inf), -1) @ v[:, h // n]
    return out


def _append_exact(case, st):
    S, R, n, bits = case["S"], case["R"], case["n"], {"k": case["bwk"], "v": case["bwv"]}
    turn = torch.complex(st["cos"].double(), st["sin"].double())[..., :R // 2][:, None]
    turned = {}
    for name in ("q", "new_k"):
        x = st[name].double()
        z = torch.complex(x[..., :R // 2].contiguous(), x[..., R // 2:R].contiguous()) * turn
        turned[name] = torch.cat([z.real, z.imag, x[..., R:]], -1)
    new = {name: st[name].clone() for name in ("k", "v", "kn", "vn")}
    norms = {"k": st["kn"].double(), "v": st["vn"].double()}
    for side, x in (("k", turned["new_k"].float().double()), ("v", st["new_v"].double())):
        # a stored vector's codes: the cache's format rounds norm, direction and rotated direction to fp32
        norm = torch.linalg.vector_norm(x, dim=-1, keepdim=True).float().double()
        y = torch.matmul((x / norm).float().double(), st["tq_" + side].Pi.double().t().contiguous()).float()
        code = torch.zeros(y.shape, dtype=torch.int32, device=DEV)
        for edge in st["tq_" + side].boundaries:
            code += y > edge
        bit = (code[..., None] >> torch.arange(bits[side], device=DEV, dtype=torch.int32)) & 1
        byte = (bit.flatten(-2).view(*y.shape[:-1], -1, 8) << torch.arange(8, device=DEV, dtype=torch.int32)).sum(-1).to(torch.uint8)
        for b in range(case["B"]):
            at = int(st["lens_host"][b]) + torch.arange(n)
            page, slot = st["table_host"][b].long()[at // S].to(DEV), (at % S).to(DEV)
            new[side][page, :, slot] = byte[b].transpose(0, 1)
            norms[side][page, :, slot] = norm[b, ..., 0].transpose(0, 1)
    return {"q": turned["q"], "k": new["k"], "v": new["v"], "kn": norms["k"], "vn": norms["v"]}


def _logits_exact(case, st):
    N, V = case["N"], case["V"]
    out = torch.empty(N, V, dtype=torch.float64, device=DEV)
    for i in range(0, N, 64):
        rows = slice(i, min(N, i + 64))
        x, hist = st["logits"][rows].double(), st["history"][rows].long()
        place = torch.arange(case["H"], device=DEV)
        count = [torch.zeros_like(x).index_put_((torch.arange(len(x), device=DEV)[:, None], hist),
                                                ((place >= lo) & (place < st["lengths"][rows, None])).double(), accumulate=True)
                 for lo in (torch.zeros(len(x), 1, device=DEV), st["prompts"][rows, None])]
        r, f, p = (st[name][rows, None].double() for name in ("repetition", "frequency", "presence"))
        x = torch.where(count[0] > 0, x * torch.where(x > 0, 1 / r, r), x) - f * count[1] - torch.where(count[1] > 0, p, 0)
        if case["J"]:
            x.scatter_add_(1, st["bias_ids"][rows].long(), st["bias"][rows].double())
        if case["mask"]:
            v = torch.arange(V, device=DEV)
            x[(st["allowed"][rows][:, v // 32] >> (v % 32).int()) & 1 == 0] = -math.inf
        out[rows] = x
    return out
