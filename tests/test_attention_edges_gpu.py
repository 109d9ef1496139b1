"""Cross attention on the GPU through its public entry points: calls at the edges of what their documentation allows."""
import os
import sys

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, os.path.join(ROOT, "tests"))
from attention_delta import CASES, check_grad_query, inputs  # noqa: E402
from attention_reference import check, make, reference  # noqa: E402

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


def at_odd_address(t):
    """the same values as a contiguous view one element into a buffer"""
    buf = torch.zeros(t.numel() + 1, dtype=t.dtype, device=t.device)
    view = buf[1:].view(t.shape)
    view.copy_(t)
    assert view.is_contiguous() and view.data_ptr() % 16
    return view


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("case", [(2, 5, 70, 2, 1, 32), (1, 1, 40, 2, 2, 128), (3, 20, 7, 1, 1, 8)], ids=str)
def test_contiguous_operands_at_an_odd_address_are_copied(dtype, case):
    x = make(*case, dtype, "h", seed=1, device=DEV)
    want = run(x)
    for names in (("q",), ("k",), ("v",), ("g",), ("q", "k", "v", "g")):
        got = run(dict(x, **{n: at_odd_address(x[n]) for n in names}))
        assert all(torch.equal(a, b) for a, b in zip(got, want)), names


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_gradient_that_is_a_slice_of_a_concatenation(dtype):
    """autograd hands over a contiguous view of the concatenation's gradient, behind an odd number of elements"""
    x = make(1, 6, 9, 2, 2, 16, dtype, seed=2, device=DEV)
    want = run(x)
    q, k, v = (x[n].detach().requires_grad_(True) for n in ("q", "k", "v"))
    other = torch.zeros(3, dtype=dtype, device=DEV, requires_grad=True)
    both = torch.cat((other, cross_attention(q, k, v).flatten()))
    got = torch.autograd.grad(both, (q, k, v), torch.cat((torch.ones(3, dtype=dtype, device=DEV), x["g"].flatten())))
    assert all(torch.equal(a, b) for a, b in zip(got, want[1:]))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_strides_of_dimensions_of_one_element_are_ignored(dtype):
    """one sequence cut out of rows with a pad, one token and one head out of odd buffers: such strides are arbitrary"""
    x = make(1, 1, 50, 1, 1, 64, dtype, "h", seed=3, device=DEV)
    want = run(x)
    odd = lambda t, i: t.as_strided(t.shape, tuple(s if j != i else 12803 for j, s in enumerate(t.stride())))
    far = lambda t: t.as_strided(t.shape, tuple(s if j != 1 else 1 << 40 for j, s in enumerate(t.stride())))
    for change in ({"q": odd(x["q"], 0)}, {"q": odd(x["q"], 1)}, {"q": odd(x["q"], 2)}, {"k": odd(x["k"], 0), "v": odd(x["v"], 2)},
                   {"g": odd(x["g"], 1)}, {"q": far(x["q"]), "g": far(x["g"])}):
        got = run(dict(x, **change))
        assert all(torch.equal(a, b) for a, b in zip(got, want)), change.keys()


@pytest.mark.parametrize("states", ["trained", "frozen", "asked for the query alone"])
@pytest.mark.parametrize("case", CASES, ids=str)
def test_delta_does_not_carry_the_rounding_of_the_result(case, states):
    x = inputs(case, DEV)
    q, k, v = (x[n].detach().requires_grad_(n == "q" or states != "frozen") for n in ("q", "k", "v"))
    out = cross_attention(q, k, v, scale=0.3)
    check_grad_query(torch.autograd.grad(out, (q, k, v) if states == "trained" else (q,), x["g"])[0], x, 0.3)


@pytest.mark.parametrize("case", [(1, 3, 5000, 260, 260, 128, "h"), (1, 5000, 3, 260, 260, 128, ""), (1, 2, 4200, 300, 300, 256, "hl"),
                                  (1, 4200, 2, 300, 300, 256, "f"), (2, 5, 9000, 600, 300, 32, "hl"), (1, 2, 9000, 150, 150, 128, "h"),
                                  (1, 4500, 33, 70, 70, 200, "h")], ids=str)
def test_float32_sums_of_several_stretches(case):
    """a card full of groups leaves one or two splits, whose float32 sums are added up in memory every 2048 rows"""
    x = make(*case[:6], torch.float32, case[6], seed=sum(case[:6]), device=DEV)
    names = ("out", "grad_query", "grad_key", "grad_value")
    got = dict(zip(names, run(x, 0.1)))
    check(got, reference(x["q"], x["k"], x["v"], x["g"], x["dead"], 0.1))
    again = dict(zip(names, run(x, 0.1)))
    assert all(torch.equal(got[n], again[n]) for n in names)


def test_float32_rows_whose_maximum_grows_from_stretch_to_stretch():
    """the logits rise along the keys, so that every stretch scales down what was held; masked stretches in front, between and behind"""
    B, Lq, Lk, H, D = 1, 2, 9000, 260, 128
    x = make(B, Lq, Lk, H, H, D, torch.float32, seed=9, device=DEV)
    x["q"].fill_(1.0)
    x["k"].mul_(0.01).add_(torch.linspace(-2.0, 2.0, Lk, device=DEV)[None, :, None, None])
    x["padding"] = torch.zeros(B, Lk, dtype=torch.bool, device=DEV)
    x["padding"][:, :2500] = x["padding"][:, 4000:6300] = x["padding"][:, 8200:] = True
    x["dead"] = x["padding"]
    got = dict(zip(("out", "grad_query", "grad_key", "grad_value"), run(x, 0.25)))
    check(got, reference(x["q"], x["k"], x["v"], x["g"], x["dead"], 0.25))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("case", [(2, 300, 1, 4, 2, 32), (3, 3000, 1, 2, 2, 128), (1, 40, 1, 1, 1, 256), (2, 700, 900, 2, 1, 64), (2, 3000, 40, 2, 1, 128),
                                  (2, 20, 5000, 2, 1, 128), (1, 5000, 1, 300, 300, 128)], ids=str)
def test_one_key_leaves_no_gradient_for_query_and_key(case, dtype):
    """dS = P (dP - delta) is 0 where P = 1, not what the two sums' orders leave of it; the last sequence, or all"""
    x = make(*case, dtype, "", seed=5, device=DEV)
    x["lengths"] = torch.full((case[0],), case[2], dtype=torch.int32, device=DEV)
    x["lengths"][-1] = 1
    x["dead"] = torch.arange(case[2], device=DEV)[None] >= x["lengths"][:, None]
    got = dict(zip(("out", "grad_query", "grad_key", "grad_value"), run(x, 0.3)))
    check(got, reference(x["q"], x["k"], x["v"], x["g"], x["dead"], 0.3))
    assert not bool(got["grad_query"][-1].any()) and not bool(got["grad_key"][-1].any()) and bool(got["grad_value"][-1, 0].any())
