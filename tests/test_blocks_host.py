"""What the 8-bit blocks and the gated block refuse, without a GPU."""

from __future__ import annotations

import ctypes

import pytest
import torch

import qste_amd as qste
from qste_amd import kernels
from qste_amd.kernels import _lib

E_DTYPE, E_SHAPE, E_NULL, E_WORKSPACE, E_ALIGN = -1, -2, -3, -4, -6
F32, F16, BF16 = 0, 1, 2


def test_tensors_that_are_not_on_the_gpu():
    x = torch.zeros(4, 64)
    packed, scale = torch.zeros(8, 8, dtype=torch.uint8), torch.ones(8)
    blocks = kernels.Blocks8(torch.zeros(4, 64, dtype=torch.int8), torch.zeros(4, 2, dtype=torch.uint8), torch.float32)
    layer = qste.PackedLinear(packed, scale, 64, None)
    for call in (lambda: qste.nn.quantize_blocks(x), lambda: qste.nn.dequantize_blocks(blocks),
                 lambda: kernels.swiglu_forward_blocks(x, x), lambda: kernels.swiglu_backward_blocks(x, blocks, blocks),
                 lambda: kernels.gated_forward(x, packed, scale, None, packed, scale, None, 64),
                 lambda: qste.nn.gated(x, layer, layer)):
        with pytest.raises(RuntimeError, match="GPU only"):
            call()


def test_blocks_that_do_not_fit_together():
    payload, codes = torch.zeros(4, 64, dtype=torch.int8), torch.zeros(4, 2, dtype=torch.uint8)
    Blocks8 = qste.nn.Blocks8
    with pytest.raises(ValueError, match="codes of shape"):
        qste.nn.dequantize_blocks(Blocks8(payload, codes[:, :1], torch.float32))
    with pytest.raises(TypeError, match="int8 payload"):
        qste.nn.dequantize_blocks(Blocks8(payload.float(), codes, torch.float32))
    with pytest.raises(TypeError, match="unsupported dtype"):
        qste.nn.dequantize_blocks(Blocks8(payload, codes, torch.float64))
    with pytest.raises(ValueError, match="codes of shape"):
        qste.nn.dequantize_blocks(Blocks8(payload[0, 0], codes[0, 0], torch.float32))


def test_layers_that_are_no_pair():
    packed, scale = torch.zeros(8, 8, dtype=torch.uint8), torch.ones(8)
    layer = qste.PackedLinear(packed, scale, 64, None)
    other = qste.PackedLinear(packed, scale, 60, None)
    with pytest.raises(TypeError, match="two QSTELinear or two PackedLinear"):
        qste.nn.gated(torch.zeros(2, 64), layer, torch.nn.Linear(64, 8))
    with pytest.raises(TypeError, match="two QSTELinear or two PackedLinear"):
        qste.nn.gated(torch.zeros(2, 64), layer, qste.PackedEmbedding(packed, scale, 64))
    with pytest.raises(TypeError, match="two QSTELinear or two PackedLinear"):
        qste.nn.gated(torch.zeros(2, 64), layer, lambda x: x)
    with pytest.raises(ValueError, match="columns"):
        qste.nn.gated(torch.zeros(2, 64), layer, other)


def _gated(lib, *, dtype=BF16, m=4, rows=64, cols=64, at=4096, x=None, out=None, values=(None, None),
           blocks=(None,) * 4, scale=4096, ws=None, ws_bytes=0):
    p = ctypes.c_void_p
    return lib.qste_gated(p(at if x is None else x), dtype, p(at), p(scale), None, p(at), p(at), None,
                          p(at if out is None else out), *[None if v is None else p(v) for v in values],
                          *[None if b is None else p(b) for b in blocks], m, rows, cols, None if ws is None else p(ws),
                          ws_bytes, None)


def test_c_entries_refuse_before_any_launch():
    lib = _lib.load()
    assert _gated(lib, dtype=7) == E_DTYPE
    assert _gated(lib, m=-1) == E_SHAPE
    assert _gated(lib, m=0) == 0 and _gated(lib, rows=0) == 0
    assert _gated(lib, scale=0) == E_NULL
    assert _gated(lib, values=(4096, None)) == E_NULL
    assert _gated(lib, blocks=(4096, 4096, 4096, None)) == E_NULL
    assert _gated(lib, x=4098) == E_ALIGN
    assert _gated(lib, out=4104) == E_ALIGN
    assert _gated(lib, blocks=(4100, 4096, 4096, 4096)) == E_ALIGN
    # columns that the one kernel does not take need room for g and u
    assert lib.qste_gated_route(100, 63, 60, BF16, 0) == 0
    assert _gated(lib, m=100, rows=63, cols=60) == E_WORKSPACE
    need = lib.qste_gated_workspace_bytes(100, 63, 60, BF16, 0)
    assert need >= 2 * 100 * 63 * 2
    assert _gated(lib, m=100, rows=63, cols=60, ws=4096, ws_bytes=need - 1) == E_WORKSPACE
    assert _gated(lib, m=100, rows=63, cols=60, ws=4100, ws_bytes=need) == E_ALIGN
    p = ctypes.c_void_p
    ones = [p(4096)] * 9
    back = lambda dtype=BF16, kept=(None,) * 6, rows=4, cols=64, grads=4096, ws=None, n=0: lib.qste_gated_backward(  # noqa: E731
        p(4096), dtype, *kept, p(grads), *ones[:4], rows, cols, ws, n, None)
    values = (p(4096), p(4096), None, None, None, None)
    assert back(F32, values) == E_DTYPE and back(kept=values, cols=60) == E_SHAPE and back(kept=values, rows=0) == E_SHAPE
    assert back() == E_NULL and back(kept=(p(4096), None, None, None, None, None)) == E_NULL
    assert back(kept=tuple(ones[:6])) == E_NULL  # both
    assert back(kept=values, grads=4104) == E_ALIGN
    assert back(kept=values) == E_WORKSPACE
    assert lib.qste_linear_backward_operands(*ones[:2], F32, *ones[:8], 4, 8, 8, None, 0, None) == E_DTYPE
    assert lib.qste_linear_backward_operands(*ones[:2], F16, *ones[:8], 0, 8, 8, None, 0, None) == E_SHAPE
    assert lib.qste_linear_backward_operands(p(4096), None, F16, *ones[:8], 4, 8, 8, None, 0, None) == E_NULL
    assert lib.qste_linear_backward_operands(*ones[:2], F16, *ones[:8], 4, 8, 8, None, 0, None) == E_WORKSPACE
    bounds = (1e-6, 4.0)
    assert lib.qste_pair_scale(p(4096), 5, *bounds, p(4096), F32, *bounds, p(4096), p(4096), 4, 8, None) == E_DTYPE
    assert lib.qste_pair_scale(p(4096), F32, *bounds, p(4096), F32, *bounds, p(4096), p(4096), 9, 8, None) == E_SHAPE
    assert lib.qste_pair_scale(p(4096), F32, *bounds, None, F32, *bounds, p(4096), p(4096), 4, 8, None) == E_NULL
    assert lib.qste_pair_scale_backward(p(4096), p(4096), p(4096), F32, *bounds, None, F32, *bounds, 4, 8, None) == E_NULL
    assert lib.qste_quantize_blocks(None, 9, None, None, 1, 1, None) == E_DTYPE
    assert lib.qste_quantize_blocks(None, F32, None, None, -1, 1, None) == E_SHAPE
    assert lib.qste_quantize_blocks(None, F32, None, None, 1, 1, None) == E_NULL
    assert lib.qste_quantize_blocks(None, F32, None, None, 0, 8, None) == 0
    assert lib.qste_dequantize_blocks(None, None, None, F16, 2, 2, None) == E_NULL
    assert lib.qste_swiglu_forward_blocks(*[None] * 2, F16, *[None] * 8, 2, 2, None) == E_NULL
    assert lib.qste_swiglu_backward_blocks(None, F16, *[None] * 6, 2, 2, None) == E_NULL
    assert lib.qste_swiglu_backward_blocks_sums(None, F16, *[None] * 6, 1, None, None, None, 2, 2, None, 0, None) == E_SHAPE


def test_routes():
    """Which way sizes go: few rows, tiles, one by one."""

    route = _lib.load().qste_gated_route
    assert route(1, 14336, 4096, BF16, 0) == 1 and route(5, 2816, 1024, F32, 0) == 1
    assert route(1, 999, 4096, BF16, 0) == 1  # rows of any number
    assert route(500, 8192, 2048, BF16, 0) == 2 and route(8190, 14336, 4096, F16, 2) == 2
    assert route(1, 14336, 4096, BF16, 2) == 2  # with something kept
    assert route(500, 8191, 2048, BF16, 0) == 2 and route(500, 8192, 2041, BF16, 0) == 2  # ragged ones
    assert route(500, 8191, 2048, BF16, 1) == 0 and route(500, 8192, 2041, BF16, 2) == 2
    assert route(500, 8192, 2048, F32, 0) == 2 and route(22, 8192, 2048, F32, 0) == 2
    assert route(500, 8192, 2048, F32, 1) == 0 and route(1, 2816, 1000, F32, 0) == 1
    assert route(4, 64, 0, BF16, 0) == 0 and route(300, 64, 100, BF16, 0) == 0
    for m in (1, 16, 17, 64, 65, 300):
        for keep in (0, 1, 2):
            for dtype in (F32, F16, BF16):
                assert _lib.load().qste_gated_workspace_bytes(m, 1000, 2048, dtype, keep) < 1 << 30
