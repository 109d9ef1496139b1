"""Cross attention kernels on the lane-level workgroup model: calls at the edges of what their C ABI allows."""
import os
import sys

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, os.path.join(ROOT, "tests"))
from attention_reference import make  # noqa: E402
from test_attention_emulated import CLANG, lib, run  # noqa: E402, F401

pytestmark = pytest.mark.skipif(not os.path.exists(CLANG), reason="needs the ROCm clang++ as host compiler")


@pytest.mark.parametrize("Lq,Lk", [(1, 0), (0, 1)])
def test_an_empty_axis_with_more_groups_than_the_card_holds(lib, Lq, Lk):  # noqa: F811
    """no tile to stream, and a grid that fills the 256 compute units (one workgroup each: float32 heads of 256) more than once"""
    x = make(1, Lq, Lk, 300, 300, 256, torch.float32)
    got = run(lib, x, 0.5)
    assert not any(bool(t.any()) for t in got.values())
