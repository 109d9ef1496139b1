"""Cross attention: what its host side refuses before any kernel."""
import pytest
import torch
import torch.autograd.forward_ad as fwad

from rlipv2_amd import _lib


@pytest.mark.parametrize("which", [0, 1, 2])
@pytest.mark.parametrize("requires_grad", [False, True])
def test_forward_mode_derivatives_are_refused(which, requires_grad):
    """a dual tensor does not require grad: without the check its tangent is lost silently"""
    x = [torch.randn(1, 3, 2, 8) for _ in range(3)]
    with fwad.dual_level():
        x[which] = fwad.make_dual(x[which], torch.ones_like(x[which]))
        if requires_grad:
            x[(which + 1) % 3].requires_grad_(True)
        with pytest.raises(NotImplementedError, match="forward-mode"):
            _lib.operators().cross_attention(*x, None, None, None, 0.3, 1.0)
