"""Cross attention on the GPU through its public entry points: calls at the edges of what their documentation allows."""
import os
import sys

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, os.path.join(ROOT, "tests"))

from rlipv2_amd.attention import cross_attention  # noqa: E402

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("Lq,Lk", [(1, 0), (0, 1), (70_000, 0), (0, 70_000)])
def test_an_empty_axis_with_more_groups_than_the_card_holds(dtype, Lq, Lk):
    """no tile to stream, and a grid that fills the 256 compute units more than once"""
    H, D = (300, 256) if Lq + Lk == 1 else (8, 32)
    q = torch.randn(1, Lq, H, D, device=DEV, dtype=dtype, requires_grad=True)
    k = torch.randn(1, Lk, H, D, device=DEV, dtype=dtype, requires_grad=True)
    v = torch.randn(1, Lk, H, D, device=DEV, dtype=dtype, requires_grad=True)
    out = cross_attention(q, k, v)
    for t in (out, *torch.autograd.grad(out.sum(), (q, k, v))):
        assert not bool(t.any())
