"""MasterWeightAdamW(fused_clip=True): what a step clips are the gradients it finds, and nothing of them is kept for the next one.  (On the
CPU, with a plain stand-in for the clipper: as the real one, it works on the memory that the tensors have when it is made.)"""
import weakref

import pytest
import torch

from rlipv2_amd import train


class PlainClipper:
    def __init__(self, tensors, out):
        self.tensors, self.out = list(tensors), list(out)
        self.memory = [t.detach() for t in self.tensors]

    def clip(self, max_norm):
        norm = torch.sqrt(sum(m.double().square().sum() for m in self.memory))
        for m, o in zip(self.memory, self.out):
            o.copy_(m.float() * float((max_norm / (norm + 1e-6)).clamp(max=1.0)))


def _model(seed):
    torch.manual_seed(seed)
    return torch.nn.Sequential(torch.nn.Linear(7, 5), torch.nn.Linear(5, 3)).bfloat16()


def _fill(model, gen):
    return [torch.randn(p.shape, generator=gen).bfloat16() for p in model.parameters()]


@pytest.fixture
def pair(monkeypatch):
    monkeypatch.setattr(train, "GradientClipper", PlainClipper)
    a, b = _model(1), _model(1)
    return a, b, train.MasterWeightAdamW(a, lr=1e-2), train.MasterWeightAdamW(b, lr=1e-2, fused_clip=True)


def _same(oa, ob):
    for x, y in zip(oa.gbuf, ob.gbuf):
        torch.testing.assert_close(y, x, rtol=2e-6, atol=0)


def test_replaced_gradient_memory_is_what_the_next_step_uses(pair):
    """`p.grad.data = ...` leaves the gradient the same object with other memory"""
    a, b, oa, ob = pair
    gen = torch.Generator().manual_seed(2)
    for step in range(3):
        for p, q, g in zip(a.parameters(), b.parameters(), _fill(a, gen)):
            if step == 0:
                p.grad, q.grad = g.clone(), g.clone()
            else:
                p.grad.data, q.grad.data = g.clone(), g.clone()
        oa.step(0.1)
        ob.step(0.1)
        _same(oa, ob)


def test_dropped_gradients_are_freed(pair):
    a, b, _, ob = pair
    for zero in (ob.zero_grad, b.zero_grad):
        for q, g in zip(b.parameters(), _fill(b, torch.Generator().manual_seed(3))):
            q.grad = g
        memory = [weakref.ref(q.grad.untyped_storage()) for q in b.parameters()]
        objects = [weakref.ref(q.grad) for q in b.parameters()]
        del g, q
        ob.step(0.1)
        zero()
        assert all(o() is None for o in objects) and all(m() is None for m in memory)
