"""Cross attention on the GPU through its public entry points: calls at the edges of what their documentation allows."""
import os
import sys

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, os.path.join(ROOT, "tests"))
from attention_reference import make  # noqa: E402

from rlipv2_amd.attention import cross_attention  # noqa: E402

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def run(x, scale=None):
    q, k, v = (x[n].detach().requires_grad_(True) for n in ("q", "k", "v"))
    out = cross_attention(q, k, v, key_padding_mask=x["padding"], key_lengths=x["lengths"], scale=scale, keep=x["keep"],
                          keep_scale=x["keep_scale"])
    return (out.detach(), *torch.autograd.grad(out, (q, k, v), x["g"]))


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


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("case", [(2, 700, 900, 2, 1, 32, False), (2, 3000, 40, 2, 1, 128, False), (2, 20, 5000, 2, 1, 128, False),
                                  (2, 3000, 64, 2, 2, 256, False), (2, 64, 1000, 2, 2, 256, True)], ids=str)
def test_masked_keys_get_zero_gradients_whatever_grad_out_holds(case, dtype):
    """a NaN and an infinite row of grad_out: P = 0 times them is NaN; keys that do not count and queries without any key get zeros"""
    x = make(*case[:6], dtype, "hl", case[6], seed=4, device=DEV)
    x["g"][:, 0], x["g"][:, 1] = float("nan"), float("inf")
    _, gq, gk, gv = run(x)
    dead = x["dead"]
    assert bool(dead[0].any()) and not bool(dead[0].all()) and bool(dead[-1].all())
    for g in (gk, gv):
        assert not bool(g[dead].any()) and bool(torch.isnan(g[~dead]).any())
    assert not bool(gq[-1].any()) and bool(torch.isfinite(gq[0, 2:]).all())


def test_forward_mode_derivatives_are_refused():
    import torch.autograd.forward_ad as fwad
    x = [torch.randn(1, 3, 2, 8, device=DEV) for _ in range(3)]
    with fwad.dual_level():
        dual = fwad.make_dual(x[0], torch.ones_like(x[0]))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            cross_attention(dual, x[1], x[2])
