"""What the gradient of the query may be off by where its delta = rowsum(dO O) is not taken from a rounded O.

q = 0: every logit is 0, an unnormalised probability is exactly 1 in the operands' type, P = 1 / Lk, O = mean V.  K = 1: the exact gradient is
scale sum_j P (dP_j - delta) = 0, so that the rounding of the result does not hide anything.  For calls of few probabilities the bound has
u^2 (u = 2^-8 for bf16) where dS, and what rounding took from O, are rounded a second time, and float32 steps w = 2^-24 elsewhere; a
delta from the rounded O, off by about u |dO O|, exceeds it."""
import torch

from attention_reference import make

CASES = [(1, 20, 40, 2, 1, 128), (1, 150, 64, 1, 1, 256), (1, 20, 100, 2, 1, 128), (1, 70, 90, 2, 2, 64), (1, 33, 70, 1, 1, 32)]


def inputs(case, device="cpu"):
    x = make(*case, torch.bfloat16, seed=sum(case), device=device)
    x["q"].zero_()
    x["k"].fill_(1.0)
    return x


def check_grad_query(got, x, scale):
    B, Lq, H, D = x["q"].shape
    Lk, G = x["k"].shape[1], H // x["k"].shape[2]
    u, w = 2.0 ** -8, 2.0 ** -24
    V, dO = x["v"].double().transpose(1, 2).repeat_interleave(G, 1), x["g"].double().transpose(1, 2)
    O, absO, dP = V.mean(2, keepdim=True), V.abs().mean(2, keepdim=True), dO @ V.transpose(-1, -2)
    p_rel = 2 * (8 + Lk) * w
    delta = (dO * O).sum(-1, keepdim=True)
    o_err = (u * u + 2 * w) * O.abs() + (p_rel + Lk * w) * absO
    d_err = (dO.abs() * o_err).sum(-1, keepdim=True) + D * w * (dO.abs() * O.abs()).sum(-1, keepdim=True)
    dp_err = D * w * (dO.abs() @ V.abs().transpose(-1, -2))
    ds_b = ((u * u + p_rel + (4 + Lk) * w) * (dP.abs() + delta.abs()) + d_err + dp_err) / Lk
    bound = (scale * ds_b.sum(-1, keepdim=True) * (1 + u)).transpose(1, 2)
    exact = (scale * (dP - delta).mean(-1, keepdim=True)).transpose(1, 2)               # 0 but for float64's steps
    err = (got.double().cpu() - exact.cpu()).abs()
    assert bool((err <= bound.cpu() * 1.0001 + 1e-12).all()), float((err / bound.cpu()).max())
