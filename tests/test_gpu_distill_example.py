"""The distillation example runs the operators together: its loss falls, and both forms of the gradient take the same steps."""

from __future__ import annotations

import math
import sys
from pathlib import Path

import pytest
import torch

pytestmark = pytest.mark.gpu

sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "examples"))


@pytest.mark.parametrize("one_pass", [False, True])
def test_a_binary_student_learns_from_its_teacher(one_pass):
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    import distill

    got = distill.main(steps=61, vocab=1003, d=128, layers=2, batch=4, seq=64, top=16, one_pass=one_pass, verbose=False)
    # tokens drawn from the teacher: the mean of some 200 log probabilities is near its entropy
    assert abs(got["teacher"][0] + got["teacher"][1]) < 0.6
    assert all(math.isfinite(v) for v in got["losses"])
    assert got["losses"][-1] < 0.7 * got["losses"][0]
    assert got["after"][0] > got["before"][0]
