"""The gated block's entry point without a GPU: what it refuses, and which way it goes."""

from __future__ import annotations

import pytest
import torch
from torch.autograd import forward_ad

import qste_amd as qste


def _packed(rows=8, cols=64):
    return qste.PackedLinear(torch.zeros(rows, cols // 8, dtype=torch.uint8), torch.ones(rows), cols, None)


def test_tangents_of_packed_layers_are_refused():
    """A packed pair carries no gradient of either mode, and drops none silently: also where gradients are off and in a
    tensor that asks for one."""

    layer = _packed()
    for wants in (False, True):
        with forward_ad.dual_level():
            dual = forward_ad.make_dual(torch.zeros(2, 64, requires_grad=wants), torch.ones(2, 64))
            with pytest.raises(NotImplementedError, match="forward-mode"):
                qste.nn.gated(dual, layer, layer)
            with torch.no_grad(), pytest.raises(NotImplementedError, match="forward-mode"):
                qste.nn.gated(dual, layer, layer)
            # a tensor without a tangent goes on to the kernels
            with pytest.raises(RuntimeError, match="GPU only"):
                qste.nn.gated(torch.zeros(2, 64), layer, layer)
    with pytest.raises(RuntimeError, match="GPU only"):
        qste.nn.gated(torch.zeros(2, 64), layer, layer)


def test_tangents_of_values_to_quantize_are_refused():
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(torch.zeros(2, 64), torch.ones(2, 64))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            qste.nn.quantize_blocks(dual)
