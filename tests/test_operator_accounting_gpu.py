"""The operators report their operands to the step's roofline accounting while a probe runs."""
import pytest
import torch

from rlipv2_amd import roofline
from rlipv2_amd.attention import cross_attention
from rlipv2_amd.optim import GradientClipper

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("train", [False, True])
def test_cross_attention_is_counted(train):
    B, Lq, Lk, H, Hk, D = 2, 30, 70, 4, 2, 32
    q, k, v = (torch.randn(B, L, h, D, device=DEV, requires_grad=train) for L, h in ((Lq, H), (Lk, Hk), (Lk, Hk)))
    pad = torch.zeros(B, Lk, dtype=torch.bool, device=DEV)

    def step():
        out = cross_attention(q, k, v, key_padding_mask=pad)
        if train:
            torch.autograd.grad(out, (q, k, v), torch.ones_like(out))
    got = roofline.probe(step)
    once = 4 * (2 * q.numel() + 2 * k.numel()) + pad.numel()
    # forward q, k, v, out; backward q, k, v, out's gradient read (and out, whose bytes delta takes) and three gradients written
    assert got["library_bytes"] == (once if not train else 2 * once + 4 * (2 * q.numel() + 2 * k.numel()))
    assert got["library_flops"] == (14 if train else 4) * B * H * Lq * Lk * D


def test_gradient_clipping_is_counted():
    grads = [torch.randn(n, device=DEV) for n in (1000, 7)]
    outs = [torch.empty(n, dtype=torch.bfloat16, device=DEV) for n in (1000, 7)]
    clipper = GradientClipper(grads, out=outs)
    assert roofline.probe(lambda: clipper.norm())["library_bytes"] == 4 * 1007
    assert roofline.probe(lambda: clipper.clip(0.1))["library_bytes"] == (4 + 4 + 2) * 1007
