"""Cross attention: what its host side refuses before any kernel."""
import os
import sys

import pytest
import torch
import torch.autograd.forward_ad as fwad

from rlipv2_amd import _lib
from rlipv2_amd.attention import CrossAttention, cross_attention

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
from attention_reference import BACK, HEAD, NO_WORK, WORK  # noqa: E402


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


@pytest.mark.parametrize("B,Lq,Lk,H,Hk,D", [(4, 22223, 22223, 8, 8, 256), (1, 65536, 65536, 32, 8, 128), (1, 300, 22223, 64, 64, 256),
                                            (1, 1, 1 << 24, 8, 8, 128), (1, 1 << 24, 64, 8, 8, 256), (16, 1 << 20, 1 << 20, 16, 16, 32)])
@pytest.mark.parametrize("dtype", [_lib.MSDA_F32, _lib.MSDA_BF16])
def test_workspaces_do_not_grow_with_the_product_of_the_lengths(dtype, B, Lq, Lk, H, Hk, D):
    """splits only fill the card: at most as many workgroups as fit on it, each with 128 rows of two float32 results of 256 elements; a
    float32 row of several stretches keeps its maximum and its sum"""
    L = _lib.lib()
    for backward in (0, 1):
        head = HEAD.pack(dtype, B, H, Hk, Lq, Lk, D, 1.0, 1.0, 0, 16, 16, 16, *(0,) * 9, 0, 0, 0, 0, 16, 0, 16)
        need = L.cross_attention_workspace_bytes(head + BACK.pack(16, 0, 0, 0, 16, 16, 16, 16) + NO_WORK, backward)
        assert need <= 256 * 9 * 128 * 2 * 256 * 4 + B * H * Lq * 8, need


def _entries(**change):
    """what the two C entries say to a call (addresses that nothing may touch: it must end in the checks)"""
    a = {**dict(dtype=_lib.MSDA_BF16, B=1, H=4, Hk=4, Lq=4, Lk=4, D=8, scale=1.0), **change}
    st = (a["Lq"] * 32, 32, 8)
    head = HEAD.pack(a["dtype"], a["B"], a["H"], a["Hk"], a["Lq"], a["Lk"], a["D"], a["scale"], 1.0, 0, 4096, 4096, 4096, *st, *st, *st, 0, 0, 0, 0,
                     4096, 0, 4096)
    args = head + BACK.pack(4096, *st, 4096, 4096, 4096, 4096) + WORK.pack(4096, 1 << 40)
    L = _lib.lib()
    return L.cross_attention_forward(args, None), L.cross_attention_backward(args, None), L.cross_attention_supported(args)


@pytest.mark.parametrize("change", [{"Lq": 1 << 30}, {"Lk": 1 << 30}, {"B": 1 << 23}, {"B": 1 << 14, "Lq": 1 << 15}], ids=str)
def test_launches_of_more_threads_than_32_bits_count_are_refused(change):
    assert _entries(**change) == (-2, -2, 0)


@pytest.mark.parametrize("dtype", [_lib.MSDA_BF16, _lib.MSDA_F32])
def test_a_scale_whose_reciprocal_overflows_is_refused(dtype):
    """the backward pass starts its logits from -L / (scale log2 e)"""
    for scale in (1e-31, 1e-38, 1e-45):
        assert _entries(dtype=dtype, scale=scale) == (-2, -2, 0)
    q, k = torch.zeros(1, 3, 2, 8), torch.zeros(1, 3, 2, 8)
    for scale in (1e-31, 1e-50, 1e39):
        with pytest.raises(ValueError, match="scale"):
            cross_attention(q, k, k, scale=scale)
    with pytest.raises(RuntimeError, match="Not implemented on the CPU"):
        cross_attention(q, k, k, scale=1e-30)


def test_module_refuses_a_dropout_that_keeps_nothing():
    """(kept probabilities are divided by 1 - dropout)"""
    for p in (1.0, -0.1, 1.5, float("nan")):
        with pytest.raises(ValueError, match="dropout"):
            CrossAttention(64, 4, dropout=p)
    assert CrossAttention(64, 4, dropout=0.999).dropout == 0.999
