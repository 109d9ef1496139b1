"""Cross attention kernels on the lane-level workgroup model: calls at the edges of what their C ABI allows."""
import os
import sys

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, os.path.join(ROOT, "tests"))
from attention_delta import CASES, check_grad_query, inputs  # noqa: E402
from attention_reference import make  # noqa: E402
from test_attention_emulated import CLANG, lib, run  # noqa: E402, F401

pytestmark = pytest.mark.skipif(not os.path.exists(CLANG), reason="needs the ROCm clang++ as host compiler")


@pytest.mark.parametrize("Lq,Lk", [(1, 0), (0, 1)])
def test_an_empty_axis_with_more_groups_than_the_card_holds(lib, Lq, Lk):  # noqa: F811
    """no tile to stream, and a grid that fills the 256 compute units (one workgroup each: float32 heads of 256) more than once"""
    x = make(1, Lq, Lk, 300, 300, 256, torch.float32)
    got = run(lib, x, 0.5)
    assert not any(bool(t.any()) for t in got.values())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("case", [(2, 70, 90, 2, 1, 32, False), (2, 70, 40, 2, 1, 128, False), (2, 20, 100, 2, 1, 128, False),
                                  (2, 20, 100, 2, 2, 256, True)], ids=str)
def test_masked_keys_get_zero_gradients_whatever_grad_out_holds(lib, case, dtype):  # noqa: F811
    """a NaN and an infinite row of grad_out: P = 0 times them is NaN.  Keys that do not count, and queries without any key (the last
    sequence), still get zeros; so do the keys that count in what the two rows do not reach"""
    x = make(*case[:6], dtype, "hl", case[6], seed=4)
    x["g"][:, 0], x["g"][:, 1] = float("nan"), float("inf")
    got = run(lib, x, 0.2)
    dead = x["dead"]
    assert bool(dead[0].any()) and not bool(dead[0].all()) and bool(dead[-1].all())
    for name in ("grad_key", "grad_value"):
        assert not bool(got[name][dead].any()), name
        assert bool(torch.isnan(got[name][~dead]).any()), name
    assert not bool(got["grad_query"][-1].any()) and bool(torch.isfinite(got["grad_query"][0, 2:]).all())


@pytest.mark.parametrize("states", [True, False])
@pytest.mark.parametrize("case", CASES, ids=str)
def test_delta_does_not_carry_the_rounding_of_the_result(lib, case, states):  # noqa: F811
    """also where only the query is trained"""
    x = inputs(case)
    check_grad_query(run(lib, x, 0.3, states)["grad_query"], x, 0.3)


ONE_KEY = [(2, 40, 1, 2, 1, 32, False), (2, 70, 1, 2, 1, 128, False), (1, 40, 1, 1, 1, 256, True)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("case", ONE_KEY, ids=str)
def test_one_key_leaves_no_gradient_for_query_and_key(lib, case, dtype):  # noqa: F811
    """dS = P (dP - delta) is 0 where P = 1, not what the two sums' orders leave of it"""
    x = make(*case[:6], dtype, "", case[6], seed=5)
    got = run(lib, x, 0.3)
    assert not bool(got["grad_query"].any()) and not bool(got["grad_key"].any()) and bool(got["grad_value"].any())


@pytest.mark.parametrize("case", [(2, 40, 90, 2, 1, 32), (2, 70, 40, 2, 1, 128), (2, 20, 100, 2, 1, 128)], ids=str)
def test_a_sequence_whose_length_is_one(lib, case):  # noqa: F811
    x = make(*case, torch.bfloat16, "", seed=6)
    x["lengths"] = torch.tensor([case[2], 1], dtype=torch.int32)
    got = run(lib, x, 0.3)
    for name in ("grad_query", "grad_key"):
        assert not bool(got[name][1].any()) and bool(got[name][0].any())
    assert bool(got["grad_value"][1, 0].any())
