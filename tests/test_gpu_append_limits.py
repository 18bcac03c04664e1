"""Appends of nearly as many vectors as a grid takes. The operands are one row, expanded; the pages of
2^28 positions are real."""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda"


@pytest.mark.parametrize("vec", [True, False])
def test_q_beside_a_grid_of_nearly_2_to_32_threads(vec):
    """2^28 - 16 vectors of K, 2^32 - 256 threads: q's items and a step of them pass 2^32 together."""
    from winnow_amd.packed_backend import append_rotated_kv
    from winnow_amd.quantizer import get_quantizer
    D, n, S = 16, 2 ** 28 - 16, 1 << 20
    tq = get_quantizer(4, D, DEV, 42)
    g = torch.Generator(device=DEV).manual_seed(5)
    odd = 0 if vec else 1       # rows that 16-byte loads do not take
    row = lambda: torch.randn(1, 1, 1, D + odd, generator=g, device=DEV).bfloat16()[..., odd:]  # noqa: E731
    q, k = row(), row()
    ang = torch.rand(1, 1, D, generator=g, device=DEV)
    cos, sin = ang.cos().bfloat16(), ang.sin().bfloat16()
    P = -(-n // S)

    def append(n, P):
        pages = torch.zeros(P, 1, S, D // 2, dtype=torch.uint8, device=DEV)
        norms = torch.zeros(P, 1, S, dtype=torch.float16, device=DEV)
        table, start = torch.arange(P, dtype=torch.int32, device=DEV)[None], torch.zeros(1, dtype=torch.int32, device=DEV)
        out = append_rotated_kv(q.expand(1, 1, n, D), k.expand(1, 1, n, D), None, cos.expand(1, n, D), sin.expand(1, n, D), tq, None, pages, None, norms,
                                None, table, start)
        return out, pages.view(-1, D // 2), norms.view(-1)
    few = append(5, 1)
    out, pages, norms = append(n, P)
    torch.cuda.synchronize()
    assert (out[0, 0] == few[0][0, 0, 0]).all()
    assert (pages[:n] == few[1][0]).all() and (norms[:n] == few[2][0]).all()
    assert not pages[n:].any() and not norms[n:].any()
