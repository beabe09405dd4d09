"""8-bit blocks of a row of more than 2^31 columns whose last block is a short one.

Column 2^31 + 8 k of such a row passes 32 bits with a sign, in an index that is
a column's and not an element's of many rows.
"""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda"
COLUMNS = (1 << 31) + 40
LAST = (1 << 31) - 64  # a whole block before the last ones


@pytest.fixture(autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    from qste_amd import kernels

    assert kernels.native_available(), kernels.status()
    yield
    torch.cuda.empty_cache()


def _row(seed):
    """Zeros but for the first and the last values of the row."""

    g = torch.Generator(device=DEV).manual_seed(seed)
    x = torch.zeros(COLUMNS, dtype=torch.bfloat16, device=DEV)
    for part in (x[:96], x[LAST:]):
        part.copy_(torch.randn(part.shape, generator=g, device=DEV))
    return x


def test_blocks_of_a_long_row():
    from qste_amd import nn as qnn

    x = _row(1)
    b = qnn.quantize_blocks(x)
    back = qnn.dequantize_blocks(b)
    for part in (slice(0, 96), slice(LAST, COLUMNS)):
        want = qnn.quantize_blocks(x[part].clone())
        codes = slice(part.start // 32, -(-part.stop // 32))
        assert torch.equal(b.payload[part], want.payload) and torch.equal(b.codes[codes], want.codes)
        assert torch.equal(back[part], qnn.dequantize_blocks(want))
    assert not bool(b.payload[96:LAST].any()) and not bool(back[96:LAST].any())


def test_gate_of_a_long_row():
    from qste_amd import nn as qnn

    gate, up, grad = (_row(seed) for seed in (2, 3, 4))
    short = [[t[part].clone() for t in (gate, up, grad)] for part in (slice(0, 96), slice(LAST, COLUMNS))]
    gate.requires_grad_(), up.requires_grad_()
    h = qnn.swiglu(gate, up, checkpoint=True)
    h.backward(grad)
    for (g, u, w), part in zip(short, (slice(0, 96), slice(LAST, COLUMNS))):
        g.requires_grad_(), u.requires_grad_()
        want = qnn.swiglu(g, u, checkpoint=True)
        want.backward(w)
        for got, expected in ((h.detach()[part], want.detach()), (gate.grad[part], g.grad), (up.grad[part], u.grad)):
            assert torch.equal(got, expected)
    assert not bool(h.detach()[96:LAST].any())
