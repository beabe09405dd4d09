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


def test_evidence_of_the_largest_gradients():
    """fp16 gradients at the end of the type's range under scales that it rounds down: where dg and du are finite the
    evidence's operands are, and stay at the type's largest value where dg c passes it.

    dg and du are within 2^-24 (|g| + 10) of theirs, relative (the exponential's argument, two units each for it and
    the reciprocal, one for an addition or a product), times 4 for dg, a sum of terms of up to that size of it; c and
    its product add 2; the operand is then rounded, by half a step."""

    from qste_amd import kernels

    dtype = torch.float16
    e, most = torch.finfo(dtype).eps / 2, torch.finfo(dtype).max
    # scales just below the middle between two values of the type, and subnormal ones
    scales = [1 + e * (1 - 2.0 ** -8), 3 + 2 * e * (1 - 2.0 ** -8), 1.49 * 2.0 ** -24, 5.4 * 2.0 ** -24]
    xs = torch.tensor(scales, device=DEV).repeat_interleave(8)
    m = xs.numel()
    # dg is dh at g = 20, du nearly dh at g = 1.2783
    g = torch.full((m, 16), -3.0, device=DEV, dtype=dtype)
    g[:, :4], g[:, 4:8] = 20.0, 1.2783
    u = torch.ones(m, 16, device=DEV, dtype=dtype)
    dh = torch.linspace(0.3, 1.0, m * 16, device=DEV).double().view(m, 16)
    dh[:, :4] = dh[:, 4:8] = torch.linspace(0.99, 1.0, 4, device=DEV).double()
    dh[::2] *= -1
    dh = dh.mul(most).to(dtype)
    both, operand, _ = kernels._gated_grads(dh, g, u, torch.zeros(m, device=DEV), xs)
    a, d = g.double(), dh.double()
    s = torch.sigmoid(a)
    dy = torch.cat((d * u.double() * s * (1 + a * (1 - s)), d * a * s), 1)
    c = (xs.double() / xs.to(dtype).double())[:, None]
    held = torch.isfinite(both)
    past = held & ((dy * c).abs() > most)
    assert bool(past[:16, :16].any()) and bool(past[:16, 16:].any())  # the end is passed, by dg c and by du c
    assert bool(torch.isfinite(operand)[held].all())
    want = (dy * c).clamp(-most, most)
    near = (operand.double() - want).abs() <= (e + 2.0 ** -24 * (4 * 30 + 2)) * want.abs()
    assert bool(near[held].all())
    packed = torch.randint(0, 256, (32, 8), generator=torch.Generator(device=DEV).manual_seed(1), device=DEV, dtype=torch.uint8)
    payload = torch.full((m, 8), 255, dtype=torch.uint8, device=DEV)
    finite = held.all(0)
    assert bool(finite.any())
    evidence = kernels.gated_backward(dh, g, u, payload, torch.zeros(m, device=DEV), xs, packed,
                                      torch.ones(32, device=DEV), 64)[1]
    assert bool(torch.isfinite(evidence[finite]).all())


@pytest.mark.parametrize("cols", [64, 63])  # the wide pass, and an element a thread
def test_fp32_gradients_of_a_checkpoint(cols):
    """dg and du in fp32 at gates of -80 to 80.

    In units of 2^-24, relative: 2 for e^-g, 1 for 1 + e^-g and 1 for the division, so s has 4 (e^-g's share in the sum
    is at most all of it), 3 where g > 0 (at most half), 6 + 1 for e^-g s and its product.  For g > 3 the sum 1 + g e^-g s,
    whose second term is at most 0.28 of the first, has 0.28 * 7 + 1 < 3, times s 4 + 1, times dh u 1 + 1: 10 in all.  For
    g of 0 to 3 the exact difference 1 - s is off by 3 s, 1 + g (1 - s), which is at least 1.14 from g = 1 on and 1 below,
    by 3 * 3 * 0.96 + 1 < 10 of 1, below 9 of itself, and 15 in all.  For g < 0 the difference is off by 4 s + 1 units of
    1, s at most 1/2: 3 units, and 1 + g (1 - s) by 3 |g| + 1 of 1: (3 |g| + 1) of dh u s beside the 7 of dg.  du: 4 for s
    and 1 for each of two products."""

    from qste_amd import kernels

    rows = 4096
    g = torch.linspace(-80, 80, rows * cols, device=DEV).view(rows, cols)
    u, dh = (_randn((rows, cols), torch.float32, seed) for seed in (1, 2))
    kept = kernels.quantize_blocks(g), kernels.quantize_blocks(u)
    a, b = (kernels.dequantize_blocks(t).double() for t in kept)
    dg, du = kernels.swiglu_backward_blocks(dh, *kept)
    s, unit = torch.sigmoid(a), 2.0 ** -24
    one = dh.double() * b * s
    want = one * (1 + a * (1 - s))
    off = torch.where(a > 0, torch.where(a > 3, 10, 15) * want.abs(), 7 * want.abs() + (3 * a.abs() + 1) * one.abs()) * unit + 1e-37
    assert bool(((dg.double() - want).abs() <= off).all())
    want = dh.double() * a * s
    assert bool(((du.double() - want).abs() <= 6 * unit * want.abs() + 1e-37).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("m", [1, 65])  # the kernel for few rows, and the tiles
def test_the_gate_at_every_value(m, dtype):
    """silu(g) u at every 16-bit g, from layers whose values are their biases.

    For g > -87 in units of 2^-24, relative: e^-g has -g for its argument's rounding, which counts where g < 0, and 2; 1
    for the addition, 2 for the reciprocal, 1 for each of two products and 4 for the constant's rounding: max(-g, 0) +
    10, and below 1 for the argument where g > 0.  Then half a step of the type, relative or of its least one.  Below
    -87 |silu(g)| is under 2^-118 and may go to 0."""

    from qste_amd import kernels
    from qste_amd.kernels import _lib

    e, most = torch.finfo(dtype).eps / 2, torch.finfo(dtype).max
    tiny = 2.0 ** -25 if dtype == torch.float16 else 2.0 ** -126
    every = torch.arange(-32768, 32768, dtype=torch.int32, device=DEV).to(torch.int16).view(dtype)
    every = every[torch.isfinite(every)]
    gate, features = every.float(), every.numel()
    assert _lib.load().qste_gated_route(m, features, 1024, {torch.float16: 1, torch.bfloat16: 2}[dtype], 0) == (1 if m == 1 else 2)
    x = torch.zeros(m, 1024, dtype=dtype, device=DEV)
    bits = torch.full((features, 128), 255, dtype=torch.uint8, device=DEV)
    scale = torch.ones(features, device=DEV)
    for value in (1.0, -0.75, 1000.0 if dtype == torch.float16 else 1e30):
        up = torch.full((features,), value, device=DEV).to(dtype).float()
        h = kernels.gated_forward(x, bits, scale, gate, bits, scale, up, 1024)[0]
        assert torch.equal(h[-1], h[0])
        g, got = gate.double(), h[0].double()
        want = g * torch.sigmoid(g) * up.double()
        past = want.abs() * (1 - 2 * e) > most
        inside = ~past & (want.abs() * (1 + 2 * e) < most)
        assert bool(torch.isinf(h[0])[past].all()) and bool(torch.isfinite(h[0])[inside].all())
        off = 2.0 ** -24 * ((-g).clamp(min=0) + 11) * want.abs()
        bound = torch.where(g > -87, off + e * (want.abs() + off), want.abs() * (1 + e)) + tiny
        assert bool(((got - want).abs() <= bound)[inside].all())
        assert bool((got * want >= 0)[inside].all())  # of want's sign, or 0


def test_scales_and_biases_in_a_column():
    """Packed layers whose scale or bias is a column, which the layers themselves take."""

    import qste_amd as qste

    gen = torch.Generator(device=DEV).manual_seed(1)
    x = _randn((5, 64), torch.bfloat16, 2)
    bits = [torch.randint(0, 256, (40, 8), generator=gen, device=DEV, dtype=torch.uint8) for _ in range(2)]
    scale, bias = (torch.rand(40, generator=gen, device=DEV) for _ in range(2))
    flat = [qste.PackedLinear(b, scale, 64, bias) for b in bits]
    column = [qste.PackedLinear(b, scale[:, None], 64, bias[:, None]) for b in bits]
    assert torch.equal(column[0](x), flat[0](x))
    assert torch.equal(qste.nn.gated(x, *column), qste.nn.gated(x, *flat))


@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("m,d,ffn", [(70, 128, 192), (300, 256, 640), (5, 64, 64)])
def test_checkpointed_mlp_piece_by_piece(m, d, ffn, bias):
    """Output, input gradient, evidence, scale and bias gradients of the three layers, bit for bit those of the kernels
    that the node stands for."""

    import qste_amd as qste
    from qste_amd import kernels

    gate, up, down = layers = _layer(ffn, d, m + 1, bias), _layer(ffn, d, m + 2, bias), _layer(d, ffn, m + 3, bias)
    up.surface.log_scale.data = up.surface.log_scale.data.bfloat16()
    x = (_randn((m, d), torch.bfloat16, 4) + 0.1).requires_grad_()
    w = _randn((m, d), torch.bfloat16, 5)
    y = qste.nn.swiglu_mlp(x, *layers, checkpoint=True)
    y.backward(w)
    sides = [[None if t is None else t.detach() for t in (layer.surface.packed_sign, layer.scale, layer.bias)]
             for layer in layers]
    flat = x.detach()
    h, g, u = kernels.gated_forward(flat, *sides[0], *sides[1], d, keep="values")
    assert torch.equal(y.detach(), kernels.packed_linear_affine(h, *sides[2], ffn))
    dh, evidence_d, scale_d, bias_d = kernels.linear_backward(w, *kernels.pack_affine_rows(h), sides[2][0], sides[2][1], ffn,
                                                              need_bias=bias)
    dx, evidence, scales, biases = kernels.gated_backward(
        dh, kernels.quantize_blocks(g), kernels.quantize_blocks(u), *kernels.pack_affine_rows(flat),
        torch.cat((sides[0][0], sides[1][0])), torch.cat((sides[0][1].float(), sides[1][1].float())), d, need_bias=bias)
    assert torch.equal(x.grad, dx)
    parts = [(evidence[:ffn], scales[:ffn], biases[:ffn] if bias else None),
             (evidence[ffn:], scales[ffn:], biases[ffn:] if bias else None), (evidence_d, scale_d, bias_d)]
    for layer, (e, grad_scale, grad_bias) in zip(layers, parts):
        log_scale = layer.surface.log_scale
        assert len(layer.evidence) == 1 and torch.equal(layer.evidence[0], e)
        # (the scale's gradient in the log-scale's type, times exp's value in it)
        want = grad_scale.to(log_scale.dtype).float() * log_scale.detach().exp().float()
        assert log_scale.grad.dtype == log_scale.dtype and torch.equal(log_scale.grad, want.to(log_scale.dtype))
        if bias:
            assert torch.equal(layer.bias.grad, grad_bias)
    assert not torch.equal(gate.evidence[0], up.evidence[0])


def test_signs_off_16_byte_steps():
    from qste_amd import kernels

    gen = torch.Generator(device=DEV).manual_seed(1)
    scale = torch.rand(40, generator=gen, device=DEV)
    for m in (3, 90):
        x = _randn((m, 128), torch.bfloat16, 2)
        bits = [torch.randint(0, 256, (40, 16), generator=gen, device=DEV, dtype=torch.uint8) for _ in range(2)]
        moved = []
        for b in bits:
            room = torch.empty(b.numel() + 3, dtype=torch.uint8, device=DEV)
            moved.append(room[3:].view(40, 16).copy_(b))
            assert moved[-1].is_contiguous() and moved[-1].data_ptr() % 16
        got = kernels.gated_forward(x, moved[0], scale, None, moved[1], scale, None, 128)[0]
        assert torch.equal(got, kernels.gated_forward(x, bits[0], scale, None, bits[1], scale, None, 128)[0])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_in_inference_mode(dtype):
    """Training layers on inference tensors, as one node and one by one, give what they give without gradients."""

    import qste_amd as qste

    layers = _layer(192, 64, 1), _layer(192, 64, 2), _layer(64, 192, 3)
    x = _randn((10, 64), dtype, 4)
    for checkpoint in (False, True):
        calls = (lambda t: qste.nn.gated(t, *layers[:2], checkpoint=checkpoint),
                 lambda t: qste.nn.swiglu_mlp(t, *layers, checkpoint=checkpoint), lambda t: layers[2](layers[0](t)))
        for call in calls:
            with torch.no_grad():
                want = call(x)
            with torch.inference_mode():
                assert torch.equal(call(x * 1), want)
    assert all(layer.surface.ledger.open_uses == 0 for layer in layers)
