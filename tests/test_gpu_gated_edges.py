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


@pytest.mark.parametrize("call", ["gated", "gated kept", "mlp kept"])
def test_the_input_as_it_is_now(call):
    """A forward whose backward never came, a write to the input that its version does not count, a forward with a
    backward: its gradients are those of a new tensor of the same values."""

    import qste_amd as qste

    layers = [_layer(192, 64, 1), _layer(192, 64, 2)]
    if call == "mlp kept":
        layers.append(_layer(64, 192, 6))
    x, other = (_randn((30, 64), torch.bfloat16, seed) for seed in (3, 4))

    def forward(t):
        return (qste.nn.gated(t, *layers, checkpoint=call == "gated kept") if len(layers) == 2
                else qste.nn.swiglu_mlp(t, *layers, checkpoint=True))

    w = _randn(forward(x).shape, torch.bfloat16, 5)
    x.data.copy_(other)
    results = []
    for t in (x, other):
        for layer in layers:
            layer.surface.reset_tracking()
            layer.surface.log_scale.grad = None
        forward(t).backward(w)
        results.append([layer.evidence.pop() for layer in layers] + [layer.surface.log_scale.grad for layer in layers])
    assert all(torch.equal(a, b) for a, b in zip(*results))


def test_captured_after_a_forward_alone():
    """A graph of a step, captured after a forward of the same input whose backward never came, encodes its input
    itself: every replay equals the eager step."""

    import qste_amd as qste

    gate, up = _layer(96, 64, 1), _layer(96, 64, 2)
    x, w = _randn((30, 64), torch.bfloat16, 3), _randn((30, 96), torch.bfloat16, 4)
    leaves = gate.surface.log_scale, up.surface.log_scale

    def step():
        grads = torch.autograd.grad(qste.nn.gated(x, gate, up, checkpoint=True), leaves, w)
        return (*grads, gate.evidence.pop(), up.evidence.pop())

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
        qste.nn.gated(x, gate, up, checkpoint=True)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    for layer in (gate, up):
        layer.surface.reset_tracking()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for seed in (5, 6, 7):
        x.copy_(_randn((30, 64), torch.bfloat16, seed))
        graph.replay()
        torch.cuda.synchronize()
        kept = [t.clone() for t in captured]
        assert all(torch.equal(a, b) for a, b in zip(kept, step()))
