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


class _Doubling(qste.PackedLinear):
    """A packed layer with a forward of its own."""

    calls = 0

    def forward(self, inputs):
        self.calls += 1
        return inputs[..., :self.out_features] * 2


class _Named(qste.PackedLinear):
    """A packed layer that adds a name and no forward."""

    name = "named"


def test_a_forward_of_its_own_is_called(monkeypatch):
    """A subclass's forward, and one set on a layer, run: the block's kernel does not stand for them."""

    gates = []
    monkeypatch.setattr(qste.nn, "swiglu", lambda g, u, *, checkpoint=False: gates.append((g, u, checkpoint)) or g * u)
    x = torch.ones(2, 64)
    packed, scale = torch.zeros(8, 8, dtype=torch.uint8), torch.ones(8)
    own, plain = _Doubling(packed, scale, 64, None), _Doubling(packed, scale, 64, None)
    assert torch.equal(qste.nn.gated(x, own, plain, checkpoint=True), torch.full((2, 8), 4.0))
    assert own.calls == plain.calls == 1 and gates.pop()[2]
    wrapped = _packed()
    wrapped.forward = lambda inputs: inputs[..., :8] * 3
    assert torch.equal(qste.nn.gated(x, own, wrapped), torch.full((2, 8), 6.0)) and not gates.pop()[2]
    assert not gates
    with pytest.raises(RuntimeError, match="GPU only"):  # a subclass without one takes the kernel
        qste.nn.gated(x, _Named(packed, scale, 64, None), _packed())


def test_mlp_of_packed_layers_goes_layer_by_layer():
    """What swiglu_mlp says of everything that its node does not take: an exported model's layers reach the kernels."""

    gate, up, down = _packed(64, 128), _packed(64, 128), _packed(128, 64)
    for checkpoint in (False, True):
        with pytest.raises(RuntimeError, match="GPU only"):
            qste.nn.swiglu_mlp(torch.zeros(2, 128), gate, up, down, checkpoint=checkpoint)


def test_mlp_of_functions(monkeypatch):
    """Anything that can be called is composed."""

    monkeypatch.setattr(qste.nn, "swiglu", lambda g, u, *, checkpoint=False: g * u)
    got = qste.nn.swiglu_mlp(torch.ones(2, 8), lambda x: x * 2, lambda x: x * 3, lambda x: x + 1)
    assert torch.equal(got, torch.full((2, 8), 7.0))


def test_encoding_of_an_inference_tensor(monkeypatch):
    """Layers in inference mode: their inputs have no version counter, so no encoding is remembered of them."""

    from qste_amd import functional

    monkeypatch.setattr(functional, "encode_activation", lambda flat: (flat, flat + 1))
    functional.forget_encodings()
    with torch.inference_mode():
        x = torch.zeros(2, 8)
        payload, aux = functional._encoding_of(x, x, 8)
        assert torch.equal(aux, payload + 1)
    assert functional._last_encoding is None
