"""A plain float64 reference of the windowed attention (CPU, test infrastructure)."""
from __future__ import annotations

import math

import torch

from tree_reference import codes_of, half_rows


def sides(kv, b, L):
    """((Hkv, L, D) codebook vectors, (Hkv, L) norms) of K and of V, float64; a page id outside the pool as page 0's."""
    out = []
    for side in "kv":
        pages, norms, quant = getattr(kv, f"{side}_pages"), getattr(kv, f"{side}_norms"), getattr(kv, f"{side}_quant")
        P, S, t = pages.shape[0], pages.shape[2], torch.arange(L)
        ids = kv.page_table[b].long()[t // S]
        ids = torch.where((ids >= 0) & (ids < P), ids, 0)
        c = quant.centroids.double()[codes_of(pages[ids, :, t % S], quant.bit_width, kv.head_dim)]
        out.append((c.transpose(0, 1), norms[ids, :, t % S].double().t()))
    return out


def sees(L, Q, window, sinks):
    """(Q, L) bool, from the definition, element by element."""
    m = torch.zeros(Q, L, dtype=torch.bool)
    for i in range(Q):
        p = L - Q + i
        for j in range(L):
            m[i, j] = j <= p and (p - j < window or j < sinks)
    return m


def window_attention(q, kv, scale, window, sinks, single=False):
    """((B, Hq, Q, D) float64, largest scale |q| |k|, largest |v| of a vector, of an element), over what is in view."""
    B, Hq, Q, D = q.shape
    Hkv = kv.k_pages.shape[1]
    n_rep = Hq // Hkv
    out = torch.zeros(B, Hq, Q, D, dtype=torch.float64)
    K = V = E = 0.0
    for b in range(B):
        L = int(kv.seq_lens[b])
        if L == 0:
            continue
        m = sees(L, Q, window, sinks) if Q * L <= 300000 else None
        if m is None:
            p, j = torch.arange(L - Q, L)[:, None], torch.arange(L)[None]
            m = (j <= p) & ((p - j < window) | (j < sinks))
        (ck, nk), (cv, nv) = sides(kv, b, L)
        view = m.any(0)
        w = (cv @ kv.v_quant.Pi.double()) * nv[..., None]
        if view.any():
            K = max(K, float((ck.norm(dim=-1) * nk)[:, view].max()))
            V, E = max(V, float(w[:, view].norm(dim=-1).max())), max(E, float(w[:, view].abs().max()))
        if single:
            ck, cv = (ck * 256).half().double() / 256, (cv * 256).half().double() / 256
        live = m.any(-1)
        for h in range(Hq):
            qr = q[b, h].double() @ kv.k_quant.Pi.double().t()
            if single:
                qr = half_rows(qr)
            s = (scale * (qr @ ck[h // n_rep].t()) * nk[h // n_rep]).masked_fill(~m, -math.inf)
            p = torch.softmax(s[live], -1)
            pv = torch.where(m[live], p * nv[h // n_rep], 0.0)
            out[b, h, live] = (pv @ cv[h // n_rep]) @ kv.v_quant.Pi.double()
    return out, abs(scale) * float(q.double().norm(dim=-1).max()) * K, V, E
