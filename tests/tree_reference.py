"""Plain float64 references of tree attention and of the branch commit (CPU, test infrastructure)."""
from __future__ import annotations

import math

import torch


def ancestors(parents, T):
    """(T, T) bool: node i is node j or descends from it."""
    sees = torch.zeros(T, T, dtype=torch.bool)
    for i in range(T):
        n = i
        while n >= 0:
            sees[i, n] = True
            n = int(parents[n])
    return sees


def random_parents(B, T, seed, root=0.1):
    """Trees whose nodes hang on any earlier node, some of them on the history itself."""
    g = torch.Generator().manual_seed(seed)
    p = torch.full((B, T), -1, dtype=torch.int32)
    for b in range(B):
        for i in range(1, T):
            if torch.rand((), generator=g) > root:
                p[b, i] = int(torch.randint(0, i, (1,), generator=g))
    return p


def codes_of(rows, bits, D):
    """(..., D bits / 8) uint8 -> (..., D) int64 codes, LSB-first."""
    bit = (rows[..., None].long() >> torch.arange(8)) & 1
    return (bit.flatten(-2).view(*rows.shape[:-1], D, bits) << torch.arange(bits)).sum(-1)


def side_of(kv, side, b, n):
    """Codebook vectors (Hkv, n, D) and norms (Hkv, n) of the first n positions of sequence b, float64."""
    pages, norms, quant = getattr(kv, f"{side}_pages"), getattr(kv, f"{side}_norms"), getattr(kv, f"{side}_quant")
    S, D = pages.shape[2], kv.head_dim
    t = torch.arange(n)
    ids = kv.page_table[b].long()[t // S]
    rows, nrm = pages[ids, :, t % S], norms[ids, :, t % S]
    c = quant.centroids.double()[codes_of(rows, quant.bit_width, D)]
    return c.transpose(0, 1), nrm.double().t()


def half_rows(x):
    """x with each row rounded to fp16 after the power of two that takes its largest value below 2^15."""
    top = x.abs().amax(-1, keepdim=True)
    e = 15 - torch.frexp(torch.where(top > 0, top, torch.ones_like(top))).exponent.double()
    return (x * 2.0 ** e).half().double() * 2.0 ** -e


def tree_attention(q, kv, parents, scale, single=False):
    """(B, Hq, T, D) float64. single: the rotated queries and the codebooks rounded to fp16 as the
    single-term products round them (the probabilities are not)."""
    B, Hq, T, D = q.shape
    Hkv = kv.k_pages.shape[1]
    n_rep = Hq // Hkv
    out = torch.zeros(B, Hq, T, D, dtype=torch.float64)
    for b in range(B):
        L = int(kv.seq_lens[b])
        if L == 0:
            continue
        (ck, nk), (cv, nv) = side_of(kv, "k", b, L), side_of(kv, "v", b, L)
        if single:
            ck, cv = (ck * 256).half().double() / 256, (cv * 256).half().double() / 256
        sees = torch.ones(T, L, dtype=torch.bool)
        anc = ancestors(parents[b], T)
        for j in range(T):
            if 0 <= L - T + j:
                sees[:, L - T + j] = anc[:, j]
        for h in range(Hq):
            qr = q[b, h].double() @ kv.k_quant.Pi.double().t()
            if single:
                qr = half_rows(qr)
            s = scale * (qr @ ck[h // n_rep].t()) * nk[h // n_rep]
            s = s.masked_fill(~sees, -math.inf)
            live = sees.any(-1)
            p = torch.softmax(s[live], -1) * nv[h // n_rep]
            out[b, h, live] = (p @ cv[h // n_rep]) @ kv.v_quant.Pi.double()
    return out


def bounds(q, kv, scale):
    """(largest scale |q| |k|, largest |v| of a vector, largest |v| of an element) over the batch."""
    k = v = e = 0.0
    for b in range(q.shape[0]):
        L = int(kv.seq_lens[b])
        if L:
            (ck, nk), (cv, nv) = side_of(kv, "k", b, L), side_of(kv, "v", b, L)
            k = max(k, float((ck.norm(dim=-1) * nk).max()))
            w = (cv @ kv.v_quant.Pi.double()) * nv[..., None]
            v, e = max(v, float(w.norm(dim=-1).max())), max(e, float(w.abs().max()))
    return scale * float(q.double().norm(dim=-1).max()) * k, v, e


def commit(pages, table, start, path, counts, nodes, page_axis):
    """A copy of ``pages`` after the moves (axes from ``page_axis``: page, head, slot): every
    source is read from the original. Moves that name no node, position or page are left out."""
    new = pages.clone()
    P, S = pages.shape[page_axis], pages.shape[page_axis + 2]
    lead = (slice(None),) * page_axis

    def at(b, pos):
        if not 0 <= pos < table.shape[1] * S:
            return None
        page = int(table[b, pos // S])
        return (*lead, page, slice(None), pos % S) if 0 <= page < P else None

    for b in range(table.shape[0]):
        for i in range(max(0, min(int(counts[b]), path.shape[1]))):
            node = int(path[b, i])
            if 0 <= node < nodes:
                src, dst = at(b, int(start[b]) + node), at(b, int(start[b]) + i)
                if src is not None and dst is not None:
                    new[dst] = pages[src]
    return new
