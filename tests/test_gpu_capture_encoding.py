"""What layers share of their input stays within one graph capture.

Two layers that read one tensor encode it once.  A step captured after a
forward of the same tensor whose backward never came, and one captured after
another capture, each encode it for themselves, so that a replay follows what
the tensor holds then.
"""

from __future__ import annotations

import math

import pytest
import torch

DEV = "cuda"


def test_the_remembered_encoding_is_of_one_capture(monkeypatch):
    """On the CPU: the number of the capture is part of what an encoding is remembered by."""

    from qste_amd import functional, kernels

    made = []
    monkeypatch.setattr(functional, "encode_activation", lambda flat: made.append(1) or (flat, flat))
    now = [0]
    monkeypatch.setattr(kernels, "capture_id", lambda t: now[0])
    functional.forget_encodings()
    x = torch.zeros(2, 8)
    for capture, encodings in ((0, 1), (0, 1), (3, 2), (3, 2), (4, 3), (0, 4), (0, 4)):
        now[0] = capture
        functional._encoding_of(x, x, 8)
        assert len(made) == encodings
    functional.remember_encoding(x, x, x)
    functional._encoding_of(x, x, 8)
    assert len(made) == 4
    now[0] = 5
    functional._encoding_of(x, x, 8)
    assert len(made) == 5
    functional.forget_encodings()


@pytest.mark.gpu
def test_replays_follow_the_input():
    import qste_amd as qste
    from qste_amd import kernels

    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    gen = torch.Generator(device=DEV).manual_seed(1)
    layers = []
    for _ in range(2):
        coordinate = torch.randint(-127, 128, (96, 64), generator=gen, device=DEV, dtype=torch.int8)
        layer = qste.QSTELinear(qste.Surface.from_state(coordinate, torch.full((96,), -0.5 * math.log(64), device=DEV)))
        layer = layer.to(DEV)
        layer.evidence = []
        layer.surface.route_evidence(lambda s, e, to=layer.evidence: to.append(e.clone()))
        layers.append(layer)
    x, w = (torch.randn(30, n, generator=gen, device=DEV).bfloat16() for n in (64, 96))
    leaves = [layer.surface.log_scale for layer in layers]

    def forward():
        return layers[0](x) + layers[1](x)

    def step():
        grads = torch.autograd.grad(forward(), leaves, w)
        return (*grads, *(layer.evidence.pop() for layer in layers))

    def fresh():
        for layer in layers:
            layer.surface.reset_tracking()

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
        forward()  # its backward never comes
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert kernels.capture_id(x) == 0
    numbers, graphs = [], []
    for alone in (True, False):  # a graph of a forward alone, then one of the step
        fresh()
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            numbers.append(kernels.capture_id(x))
            if alone:
                forward()  # dropped: no autograd graph of these leaves lives while a backward is captured
            else:
                captured = step()
    assert numbers[0] and numbers[1] and numbers[0] != numbers[1]
    fresh()
    for seed in (5, 6, 7):
        x.copy_(torch.randn(30, 64, generator=torch.Generator(device=DEV).manual_seed(seed), device=DEV))
        graphs[-1].replay()
        torch.cuda.synchronize()
        kept = [t.clone() for t in captured]
        assert all(torch.equal(a, b) for a, b in zip(kept, step()))
