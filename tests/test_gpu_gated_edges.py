"""The gated block and its checkpoints at the ends of what they take: second
derivatives and tangents, layers of a program's own, values at the ends of the
types' ranges."""

from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda"


@pytest.fixture(autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    from qste_amd import kernels

    assert kernels.native_available(), kernels.status()


def _randn(shape, dtype, seed, std=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randn(shape, generator=g, device=DEV) * std).to(dtype)


def _layer(rows, cols, seed, bias=False):
    """A training layer whose evidence goes to a list of its own."""

    import qste_amd as qste

    g = torch.Generator(device=DEV).manual_seed(seed)
    coordinate = torch.randint(-127, 128, (rows, cols), generator=g, device=DEV, dtype=torch.int8)
    log_scale = torch.randn(rows, generator=g, device=DEV) * 0.1 - 0.5 * math.log(cols)
    layer = qste.QSTELinear(qste.Surface.from_state(coordinate, log_scale),
                            torch.randn(rows, generator=g, device=DEV) * 0.1 if bias else None).to(DEV)
    layer.evidence = []
    layer.surface.route_evidence(lambda s, e: layer.evidence.append(e.clone()))
    return layer


def _mlp_gradient(ffn):
    import qste_amd as qste

    layers = _layer(ffn, 64, 1), _layer(ffn, 64, 2), _layer(64, ffn, 3)
    x = _randn((10, 64), torch.bfloat16, 4).requires_grad_()
    loss = qste.nn.swiglu_mlp(x, *layers, checkpoint=True).float().square().sum()
    grad, = torch.autograd.grad(loss, x, create_graph=True)
    assert all(len(layer.evidence) == 1 for layer in layers)
    return grad, loss


def test_no_second_derivative_of_the_mlp():
    """A gradient of a checkpointed MLP that reached it with a graph of its own is not differentiated again: it is
    refused, and not taken for a constant."""

    grad, loss = _mlp_gradient(192)
    assert grad.requires_grad
    with pytest.raises(RuntimeError, match="differentiate twice"):
        (grad.float().square().sum() + loss).backward()


def test_gradient_of_an_mlp_of_layers():
    """A hidden size that the one node does not take: the last layer's gradient, a layer's as ever, has no graph."""

    grad, _ = _mlp_gradient(200)
    assert not grad.requires_grad


def test_no_second_derivative_of_the_gated_block():
    import qste_amd as qste

    gate, up = _layer(96, 64, 1), _layer(96, 64, 2)
    for checkpoint in (False, True):
        x = _randn((10, 64), torch.bfloat16, 4).requires_grad_()
        loss = qste.nn.gated(x, gate, up, checkpoint=checkpoint).float().square().sum()
        grad, = torch.autograd.grad(loss, x, create_graph=True)
        with pytest.raises(RuntimeError, match="differentiate twice"):
            grad.float().square().sum().backward()


@pytest.mark.parametrize("checkpoint", [False, True])
@pytest.mark.parametrize("d,ffn,dtype", [(64, 192, torch.bfloat16), (72, 200, torch.float16)])
def test_mlp_trained_then_served(d, ffn, dtype, checkpoint):
    """A model written with swiglu_mlp, exported: its packed layers give what its training layers give."""

    import qste_amd as qste

    class MLP(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.gate, self.up, self.down = _layer(ffn, d, 1, True), _layer(ffn, d, 2), _layer(d, ffn, 3)

        def forward(self, x):
            return qste.nn.swiglu_mlp(x, self.gate, self.up, self.down, checkpoint=checkpoint)

    model = MLP()
    x = _randn((150, d), dtype, 4)
    with torch.no_grad():
        want = qste.nn.gated(x, model.gate, model.up) if checkpoint else qste.nn.swiglu(model.gate(x), model.up(x))
        want = model.down(want)
    served = qste.export_packed(model)
    assert isinstance(served.down, qste.PackedLinear)
    got = served(x)
    assert not got.requires_grad and torch.equal(got, want)
