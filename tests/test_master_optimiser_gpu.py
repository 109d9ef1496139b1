"""MasterWeightAdamW(fused_clip=True) with the real clipper: the gradients a step finds are the ones it uses, and it frees them."""
import pytest
import torch

from rlipv2_amd.train import MasterWeightAdamW

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _model(sizes):
    torch.manual_seed(1)
    return torch.nn.Sequential(*[torch.nn.Linear(a, b) for a, b in sizes]).to(DEV, torch.bfloat16)


def test_replaced_gradient_memory_is_what_the_next_step_uses():
    a, b = _model([(37, 50), (50, 3)]), _model([(37, 50), (50, 3)])
    oa, ob = MasterWeightAdamW(a, lr=1e-2), MasterWeightAdamW(b, lr=1e-2, fused_clip=True)
    gen = torch.Generator().manual_seed(2)
    for step in range(4):
        for p, q in zip(a.parameters(), b.parameters()):
            g = torch.randn(p.shape, generator=gen).bfloat16().to(DEV)
            if step in (0, 3):                              # (a fresh object, then other memory under the same object)
                p.grad, q.grad = g, g.clone()
            else:
                p.grad.data, q.grad.data = g, g.clone()
        oa.step(0.1)
        ob.step(0.1)
        # the norm's sum in float32 against float64, one rounding of the coefficient: 2^-24 times a few
        for x, y in zip(oa.gbuf, ob.gbuf):
            torch.testing.assert_close(y, x, rtol=2e-6, atol=0)


def test_dropped_gradients_give_their_memory_back():
    m = _model([(2048, 2048), (2048, 2048)])
    opt = MasterWeightAdamW(m, fused_clip=True)
    def grads():
        for p in m.parameters():
            p.grad = torch.ones_like(p)
    grads()
    opt.step()
    opt.zero_grad()
    torch.cuda.synchronize()
    without = torch.cuda.memory_allocated()
    grads()
    opt.step()
    for p in m.parameters():
        p.grad = None
    torch.cuda.synchronize()
    assert torch.cuda.memory_allocated() <= without + 4096
