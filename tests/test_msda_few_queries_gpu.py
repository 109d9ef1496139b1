"""The shape-agnostic sampling backward where queries are few: every query gets its own waves, two float64 ones share them."""
import os
import sys

import numpy as np
import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, os.path.join(ROOT, "tests"))

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _call(dtype, N, M, D, Lq, seed=0):
    gen = torch.Generator().manual_seed(seed)
    shapes = torch.tensor([[9, 14], [5, 7], [2, 4]])
    starts = torch.cat((shapes.new_zeros(1), (shapes[:, 0] * shapes[:, 1]).cumsum(0)[:-1]))
    S = int((shapes[:, 0] * shapes[:, 1]).sum())
    value, go = torch.randn(N, S, M, D, generator=gen), torch.randn(N, Lq, M * D, generator=gen)
    loc, aw = torch.rand(N, Lq, M, 3, 4, 2, generator=gen), torch.rand(N, Lq, M, 3, 4, generator=gen)
    return [t.to(DEV, dtype) for t in (value,)] + [shapes.to(DEV), starts.to(DEV)] + [t.to(DEV, dtype) for t in (loc, aw, go)]


@pytest.mark.parametrize("Lq", [1, 2])
def test_float64_gradients_of_two_queries_repeat_bit_for_bit(Lq):
    from rlipv2_amd import msda
    args = _call(torch.float64, 2, 2, 1500, Lq)
    first = msda.ms_deform_attn_backward(*args, 64)
    for _ in range(5):
        assert all(torch.equal(a, b) for a, b in zip(first, msda.ms_deform_attn_backward(*args, 64)))


@pytest.mark.parametrize("dtype", [torch.float32, torch.float64])
@pytest.mark.parametrize("N,M,D,Lq", [(2, 3, 40, 1), (2, 3, 40, 2), (3, 2, 71, 5), (1, 8, 64, 16), (2, 4, 48, 17)])
def test_few_queries_against_the_oracle(dtype, N, M, D, Lq):
    from oracle import msda_oracle
    from rlipv2_amd import msda
    args = _call(dtype, N, M, D, Lq, seed=Lq)
    got = msda.ms_deform_attn_backward(*args, 64)
    value, shapes, starts, loc, aw, go = (t.cpu().double().numpy() if t.is_floating_point() else t.cpu().numpy() for t in args)
    want = msda_oracle.backward(value, shapes, starts, loc, aw, go)
    # sums of at most N Lq M-independent 4 * 12 * Lq products per element of grad_value and D per location: 2^-24 (2^-53) times their number
    eps = 2.0 ** -24 if dtype == torch.float32 else 2.0 ** -53
    for g, w in zip(got, want):
        w = np.asarray(w).reshape(g.shape)
        assert np.abs(g.double().cpu().numpy() - w).max() <= eps * (48 * Lq + D + 64) * 4 * np.abs(w).max()
