"""Which types token numbers may have."""

from __future__ import annotations

import pytest
import torch


@pytest.mark.parametrize("dtype", [torch.uint8, torch.int8, torch.int16, torch.int32, torch.int64])
def test_integers_are_taken(dtype):
    from qste_amd.kernels import _row_tokens

    marks = torch.tensor([[3, 0], [100, 7]], dtype=dtype)
    if dtype != torch.uint8:
        marks[0, 1] = -1
    got = _row_tokens(marks.t(), (2, 2), "tokens")
    assert got.dtype == torch.int64 and got.is_contiguous() and torch.equal(got, marks.t().long())


@pytest.mark.parametrize("dtype", [torch.bool, torch.float32, torch.bfloat16])
def test_others_are_refused(dtype):
    from qste_amd.kernels import _row_tokens

    with pytest.raises(TypeError, match="integers"):
        _row_tokens(torch.zeros(2, 2).to(dtype), (2, 2), "tokens")
