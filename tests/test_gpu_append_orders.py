"""One order of sums for every append: a vector whose norm depends on the order in which its squares are
added gets the same codes from ``append_kv``, from ``append_rotated_kv`` and from ``quantize``'s kernel.

The squares of ORDERED are 1, 2^-24 twice, 2^-48 and fifteen of 2^-54, in float64. Added one by one to
a sum of 1 the last fifteen are lost (half a step is 2^-53), and the root of (1 + 2^-24)^2 is a tie
that rounds to 1 in fp32; added to each other first they move it to 1 + 2^-23. x / n is then 1 or
1 - 2^-23, on the two sides of the boundary 1 - 2^-24. No answer is the wrong one; two are.
"""
from __future__ import annotations

import types

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda"


def _ordered(D):
    x = torch.zeros(D)
    x[0], x[1:3], x[3], x[16::16] = 1.0, 2.0 ** -12, 2.0 ** -24, 2.0 ** -27
    return x


@pytest.mark.parametrize("D", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("n", [1, 40, 9000])
@pytest.mark.parametrize("shift", [0, 1, 5])
def test_the_codes_do_not_depend_on_the_entry_point(D, n, shift):
    from winnow_amd.packed_backend import append_kv, append_rotated_kv
    bounds = torch.cat([torch.linspace(-0.9, 0.9, 14), torch.tensor([1 - 2.0 ** -24])]).to(DEV)
    tq = types.SimpleNamespace(Pi=torch.eye(D, device=DEV), boundaries=bounds, centroids=torch.zeros(16, device=DEV), bit_width=4)
    k = _ordered(D).roll(shift).expand(1, 2, n, D).contiguous().to(DEV)
    cos, sin = torch.ones(1, n, D, device=DEV), torch.zeros(1, n, D, device=DEV)
    P = -(-n // 16)
    table, start = torch.arange(P, dtype=torch.int32, device=DEV)[None], torch.zeros(1, dtype=torch.int32, device=DEV)

    def pages():
        return [torch.zeros(P, 2, 16, D // 2, dtype=torch.uint8, device=DEV) for _ in range(2)] + [
            torch.zeros(P, 2, 16, dtype=torch.float16, device=DEV) for _ in range(2)]
    plain, turned = pages(), pages()
    append_kv(k, k, tq, tq, *plain, table, start)
    append_rotated_kv(None, k, k, cos, sin, tq, tq, *turned, table, start)
    for a, b in zip(plain, turned):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    assert torch.equal(turned[0], turned[1])
