"""An error that an earlier HIP call left behind is not reported by the operators as theirs."""
import pytest
import torch

from rlipv2_amd import _lib
from rlipv2_amd.attention import cross_attention
from rlipv2_amd.optim import GradientClipper

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def leave_an_error():
    hip = _lib.lib()                            # (its symbols include those of the HIP runtime that it uses)
    assert hip.hipSetDevice(1000) != 0
    assert hip.hipPeekAtLastError() != 0


def test_pending_error():
    q, k = torch.randn(1, 3, 2, 32, device=DEV, requires_grad=True), torch.randn(1, 5, 2, 32, device=DEV)
    clipper = GradientClipper([torch.ones(4, device=DEV)])
    want = cross_attention(q, k, k)
    (gq,) = torch.autograd.grad(want, (q,), torch.ones_like(want), retain_graph=True)
    ones, two = torch.ones_like(want), torch.tensor(2.0, device=DEV)
    torch.cuda.synchronize()
    leave_an_error()
    out = cross_attention(q, k, k)
    leave_an_error()
    (again,) = torch.autograd.grad(want, (q,), ones)
    leave_an_error()
    norm = clipper.norm()
    leave_an_error()
    clipper.clip(1.0)
    assert torch.equal(out, want) and torch.equal(again, gq) and torch.equal(norm, two)
