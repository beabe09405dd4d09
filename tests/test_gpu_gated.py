"""The gated feed-forward block in one kernel.

Values: against the definition in 64 bits, with the bound that the roundings
give; gate's and up's bit for bit against the layers called one by one where
the sums run in the same order.  The backward: bit for bit against the layers' own
backward calls at the values that were kept, and against differences.
"""

from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda"
CODES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}


@pytest.fixture(autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    from qste_amd import kernels

    assert kernels.native_available(), kernels.status()


def _bits(t):
    return t.contiguous().view({1: torch.int8, 2: torch.int16, 4: torch.int32}[t.element_size()])


def _operands(m, rows, cols, dtype, seed=0, bias=False):
    g = torch.Generator(device=DEV).manual_seed(seed + m + 3 * rows + 7 * cols)
    x = (torch.randn(m, cols, generator=g, device=DEV) + 0.1).to(dtype)
    layers = []
    for _ in range(2):
        bits = torch.randint(0, 256, (rows, -(-cols // 8)), generator=g, device=DEV, dtype=torch.uint8)
        if cols % 8:
            bits[:, -1] &= (1 << (cols % 8)) - 1
        scale = (torch.rand(rows, generator=g, device=DEV) + 0.2) / math.sqrt(max(cols, 1))
        layers += [bits, scale, torch.randn(rows, generator=g, device=DEV) * 0.1 if bias else None]
    return x, layers


def _route(m, rows, cols, dtype, keep=0):
    from qste_amd.kernels import _lib

    return _lib.load().qste_gated_route(m, rows, cols, CODES[dtype], keep)


def _within_roundings(h, x, layers, dtype):
    """Whether h is silu(g) u in 64 bits but for the roundings.

    e: half a step of the type, relative.  A sum of K terms in fp32 is off by at most K 2^-24 times the sum of their
    magnitudes, and scale and bias round twice more; g and u are then rounded (e).  silu's slope is at most 1.1; its
    value is computed in fp32 (16 units of 2^-24 for the exponential and the division) and rounded (e), and so is the
    product (e).  Subnormal fp16 values are rounded to 2^-25 at most."""

    e, tiny = torch.finfo(dtype).eps / 2, (2.0 ** -24 if dtype == torch.float16 else 1e-36)
    cols = x.shape[1]
    place = torch.arange(cols, device=DEV)
    values, errors = [], []
    for bits, scale, bias in (layers[:3], layers[3:]):
        sign = ((bits[:, place // 8].int() >> (place % 8)) & 1).double() * 2 - 1
        y = x.double() @ sign.t() * scale.double()
        if bias is not None:
            y = y + bias.double()
        size = x.double().abs().sum(1, keepdim=True) * scale.double()
        errors.append((cols + 2) * 2.0 ** -24 * size + (2.0 ** -23 + e) * y.abs() + tiny)
        values.append(y)
    g, u = values
    a = g * torch.sigmoid(g)
    error_a = 1.1 * errors[0] + (16 * 2.0 ** -24 + e) * (a.abs() + 1.1 * errors[0]) + tiny
    bound = error_a * (u.abs() + errors[1]) + a.abs() * errors[1]
    bound = bound + e * ((a * u).abs() + bound) + tiny
    return bool(((h.double() - a * u).abs() <= bound).all())


def _gate_of(h, g, u):
    """Whether h is silu(g) u at these g and u, rounded once.

    In units of 2^-24, relative: |g| for the exponential's argument, two each for it and the reciprocal, one each for an
    addition and three products, 10 in all; then half a step of the type, or of its least one."""

    e, tiny = torch.finfo(h.dtype).eps / 2, (2.0 ** -25 if h.dtype == torch.float16 else 1e-37)
    want = g.double() * torch.sigmoid(g.double()) * u.double()
    off = 2.0 ** -24 * (g.double().abs() + 10) * want.abs()
    return bool(((h.double() - want).abs() <= off + e * (want.abs() + off) + tiny).all())


# sizes of each way, with ends inside every unit: 16-row blocks, 512-column chunks, 128- and 256-row and
# 128-feature tiles, K in ranges
FEW = [(1, 16, 128), (1, 8, 256), (2, 24, 384), (3, 999, 128), (4, 4096, 1024), (5, 1000, 640), (7, 2816, 1024),
       (16, 5480, 2048), (17, 136, 4096), (21, 512, 2048), (31, 640, 512), (33, 5480, 2048), (48, 1000, 8192),
       (49, 77, 1024), (64, 256, 4096), (1, 14336, 4096)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("m,rows,cols", FEW)
def test_few_rows(m, rows, cols, dtype):
    from qste_amd import kernels

    if dtype == torch.float32 and m > 21:
        m = m % 21 + 1
    print(f"gated {m} x {rows} x {cols} {dtype}", flush=True)
    for bias in (False, True):
        x, layers = _operands(m, rows, cols, dtype, bias=bias)
        h, g, u = kernels.gated_forward(x, *layers, cols)
        assert g is None and u is None and h.dtype == dtype and h.shape == (m, rows)
        assert _within_roundings(h, x, layers, dtype)
    again = kernels.gated_forward(x, *layers, cols)[0]
    assert torch.equal(_bits(again), _bits(h))


def test_few_rows_take_their_kernel():
    assert _route(1, 14336, 4096, torch.bfloat16) == 1
    assert _route(3, 999, 128, torch.float16) == 1 and _route(21, 512, 2048, torch.float32) == 1
    assert _route(131, 999, 2048, torch.bfloat16) == 2 and _route(200, 1000, 512, torch.float32) == 2
    assert _route(100, 63, 60, torch.bfloat16) == 0


def test_a_row_is_the_same_beside_others():
    """Up to 16 rows a row's bits do not depend on how many there are."""

    from qste_amd import kernels

    for dtype in (torch.bfloat16, torch.float32):
        x, layers = _operands(16, 1000, 1024, dtype)
        whole = kernels.gated_forward(x, *layers, 1024)[0]
        for m in (1, 4, 5, 11):
            part = kernels.gated_forward(x[:m], *layers, 1024)[0]
            assert torch.equal(_bits(part), _bits(whole[:m]))


TILES = [(65, 8, 64), (100, 1024, 4096), (128, 120, 64), (129, 136, 128), (250, 2048, 768), (300, 264, 1024),
         (500, 8192, 2048), (513, 1000, 192), (2048, 4096, 1024), (2050, 16384, 256), (70, 4104, 8192)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("m,rows,cols", TILES)
def test_tiles(m, rows, cols, dtype):
    from qste_amd import kernels

    print(f"gated {m} x {rows} x {cols} {dtype}", flush=True)
    assert _route(m, rows, cols, dtype) == 2
    x, layers = _operands(m, rows, cols, dtype, bias=rows % 16 == 8)
    h = kernels.gated_forward(x, *layers, cols)[0]
    assert _within_roundings(h, x, layers, dtype)
    # what is kept changes nothing, and is what the values' blocks are
    h1, g, u = kernels.gated_forward(x, *layers, cols, keep="values")
    h2, g8, u8 = kernels.gated_forward(x, *layers, cols, keep="blocks")
    assert torch.equal(_bits(h1), _bits(h)) and torch.equal(_bits(h2), _bits(h))
    assert _gate_of(h, g, u)
    for kept, t in ((g8, g), (u8, u)):
        want = kernels.quantize_blocks(t)
        assert torch.equal(kept.payload, want.payload) and torch.equal(kept.codes, want.codes)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("m,rows,cols", [(2048, 4096, 1024), (4096, 8192, 512), (8192, 1000, 256)])
def test_the_same_bits_as_the_layers_one_by_one(m, rows, cols, dtype):
    """Products whose K is not cut, alone or together, sum in one order."""

    from qste_amd import kernels

    x, layers = _operands(m, rows, cols, dtype, bias=True)
    h, g, u = kernels.gated_forward(x, *layers, cols, keep="values")
    want = [kernels.packed_linear_affine(x, *layer, cols) for layer in (layers[:3], layers[3:])]
    assert torch.equal(_bits(g), _bits(want[0])) and torch.equal(_bits(u), _bits(want[1]))
    assert _gate_of(h, g, u)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("m,rows,cols", [(100, 63, 64), (70, 1000, 100), (3, 33, 65), (1, 1, 1), (80, 264, 7),
                                         (30, 128, 256), (5, 24, 0), (300, 1001, 200), (129, 77, 1000), (513, 264, 333),
                                         (40, 1000, 200), (1, 3000, 1000), (22, 300, 256), (200, 1000, 512),
                                         (512, 4416, 1712), (131, 999, 2048)])
def test_ragged_sizes(m, rows, cols, dtype):
    from qste_amd import kernels

    x, layers = _operands(m, rows, cols, dtype, bias=True)
    for keep in ("", "values", "blocks"):
        h, g, u = kernels.gated_forward(x, *layers, cols, keep=keep)
        assert _within_roundings(h, x, layers, dtype)
        if keep == "values" and _route(m, rows, cols, dtype, 1) == 0:
            assert torch.equal(_bits(kernels.swiglu_forward(g, u)[0]), _bits(h))
        if keep == "blocks":
            assert g.payload.shape == h.shape


def test_special_values():
    """Infinities and NaN in a row stay in it and give what the layers one by one give.

    Row 4 holds finite values whose sums pass the end of fp32: 3e38 - 3e38 + 3e38 + 3e38 is finite up to its third
    term and infinite from its fourth on, 3e38 + 3e38 - 3e38 - 3e38 from its second, and with sums of either sign
    in a tree inf - inf is NaN; which of them a sum meets is a matter of its order alone, which two layers in one
    kernel need not share with two kernels.  What it gives is not compared, that it stays in its row is."""

    from qste_amd import kernels

    same = [0, 1, 2, 3, 5]
    for m in (6, 300):
        x, layers = _operands(m, 256, 512, torch.bfloat16)
        clean = kernels.gated_forward(x, *layers, 512)[0]
        x[1, 5], x[2, 7], x[4] = math.inf, math.nan, 3e38
        h, g8, u8 = kernels.gated_forward(x, *layers, 512, keep="blocks")
        want = [kernels.packed_linear_affine(x, *layer, 512) for layer in (layers[:3], layers[3:])]
        plain = kernels.swiglu_forward(*want)[0]
        assert torch.equal(torch.isnan(h[same]), torch.isnan(plain[same]))
        assert torch.equal(torch.isinf(h[same]), torch.isinf(plain[same]))
        assert bool((g8.codes[1] == 255).all()) and bool((u8.codes[2] == 255).all())
        few = kernels.gated_forward(x, *layers, 512)[0]
        assert torch.equal(torch.isnan(few[same]), torch.isnan(plain[same]))
        for row in (0, 3, 5):
            assert torch.equal(_bits(few[row]), _bits(clean[row]))


def test_empty_and_shaped_inputs():
    from qste_amd import kernels

    x, layers = _operands(12, 64, 128, torch.bfloat16)
    flat = kernels.gated_forward(x, *layers, 128)[0]
    assert torch.equal(kernels.gated_forward(x.view(3, 4, 128), *layers, 128)[0], flat.view(3, 4, 64))
    assert kernels.gated_forward(x[:0], *layers, 128)[0].shape == (0, 64)
    wide = torch.zeros(12, 137, dtype=torch.bfloat16, device=DEV)
    wide[:, 9:] = x
    assert torch.equal(kernels.gated_forward(wide[:, 9:], *layers, 128)[0], flat)  # strided, off 16-byte steps
    assert torch.equal(kernels.gated_forward(x[0], *layers, 128)[0], flat[0])


def test_refusals():
    from qste_amd import kernels

    x, layers = _operands(4, 64, 128, torch.bfloat16)
    bits, scale = layers[:2]
    with pytest.raises(TypeError):
        kernels.gated_forward(x.double(), *layers, 128)
    with pytest.raises(ValueError, match="columns"):
        kernels.gated_forward(x[:, :64], *layers, 128)
    with pytest.raises(ValueError, match="rows"):
        kernels.gated_forward(x, bits, scale, None, bits[:32], scale[:32], None, 128)
    with pytest.raises(ValueError, match="scale"):
        kernels.gated_forward(x, bits, scale[:3], None, bits, scale, None, 128)
    with pytest.raises(ValueError, match="bias"):
        kernels.gated_forward(x, bits, scale, scale[:3], bits, scale, None, 128)
    with pytest.raises(ValueError, match="keep"):
        kernels.gated_forward(x, *layers, 128, keep="all")


# ---------------------------------------------------------------------------
# layers
# ---------------------------------------------------------------------------


def _pair(rows, cols, seed, bias=False, dtype=torch.float32):
    import qste_amd as qste

    g = torch.Generator(device=DEV).manual_seed(seed)
    layers = []
    for _ in range(2):
        coordinate = torch.randint(-127, 128, (rows, cols), generator=g, device=DEV, dtype=torch.int8)
        log_scale = torch.randn(rows, generator=g, device=DEV) * 0.1 - 0.5 * math.log(cols)
        layer = qste.QSTELinear(qste.Surface.from_state(coordinate, log_scale),
                                torch.randn(rows, generator=g, device=DEV) * 0.1 if bias else None).to(DEV)
        layer.surface.log_scale.data = log_scale.to(dtype)
        layer.evidence = []
        layer.surface.route_evidence(lambda s, e, to=layer.evidence: to.append(e.clone()))
        layers.append(layer)
    return layers


@pytest.mark.parametrize("checkpoint", [False, True])
@pytest.mark.parametrize("dtype,bias", [(torch.bfloat16, False), (torch.float16, True)])
@pytest.mark.parametrize("m,rows,cols", [(3, 64, 64), (250, 2048, 768), (300, 264, 128), (1030, 1000, 512), (70, 64, 72),
                                         (300, 264, 333), (600, 1000, 1000), (5, 8, 3), (70, 33, 64), (200, 1001, 128)])
def test_training_node(m, rows, cols, dtype, bias, checkpoint):
    """Values and gradients are those of the kernels that the node stands for, at the g and u it kept."""

    import qste_amd as qste
    from qste_amd import kernels

    print(f"gated node {m} x {rows} x {cols} {dtype} {checkpoint}", flush=True)
    gate, up = _pair(rows, cols, m, bias, torch.bfloat16)
    gen = torch.Generator(device=DEV).manual_seed(m)
    x = (torch.randn(m, cols, generator=gen, device=DEV) + 0.1).to(dtype).requires_grad_()
    grad = torch.randn(m, rows, generator=gen, device=DEV).to(dtype)
    h = qste.nn.gated(x, gate, up, checkpoint=checkpoint)
    h.backward(grad)
    # piece by piece
    flat, whole = x.detach(), -(-rows // 8) * 8

    def padded(t, dim=0):  # rows in whole eights, zeros behind
        more = whole - rows
        return t if t is None else torch.cat((t, t.new_zeros(*t.shape[:dim], more, *t.shape[dim + 1:])), dim)

    sides = [[padded(t if t is None else t.detach()) for t in (layer.surface.packed_sign, layer.scale, layer.bias)]
             for layer in (gate, up)]
    want, g, u = kernels.gated_forward(flat, *sides[0], *sides[1], cols, keep="values")
    assert torch.equal(_bits(h.detach()), _bits(want[:, :rows]))
    payload, offset, xscale = kernels.pack_affine_rows(flat)
    if checkpoint:
        g, u = kernels.quantize_blocks(g), kernels.quantize_blocks(u)
    dx, evidence, grad_scale, grad_bias = kernels.gated_backward(
        padded(grad, 1), g, u, payload, offset, xscale, torch.cat((sides[0][0], sides[1][0])),
        torch.cat((sides[0][1].float(), sides[1][1].float())), cols, need_bias=bias)
    assert torch.equal(_bits(x.grad), _bits(dx))
    for i, layer in enumerate((gate, up)):
        part = slice(i * whole, i * whole + rows)
        assert len(layer.evidence) == 1 and torch.equal(layer.evidence[0], evidence[part])
        # exp's value in the log-scale's type times the scale's gradient, rounded once
        log_scale = layer.surface.log_scale
        want = (log_scale.detach().exp().float() * grad_scale[part]).to(log_scale.dtype)
        assert torch.equal(log_scale.grad, want)
        if bias:
            assert torch.equal(layer.bias.grad, grad_bias[part])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("m,rows,cols", [(1, 8, 64), (70, 40, 64), (250, 2048, 768), (513, 264, 128), (33, 1000, 192),
                                         (2000, 512, 320), (70, 64, 72), (600, 1000, 1001), (5, 8, 3)])
@pytest.mark.parametrize("kept", ["values", "blocks"])
def test_backward_kernels(m, rows, cols, dtype, kept):
    """dx, evidence, scale and bias gradients against the formulas in 64 bits at the kept g and u.

    e: half a step of the type, relative.  dg and du are within e of theirs (fp32 before that: 2^-24 times a few tens,
    within another e / 16), the row scales are exact in the type here.  A sum in fp32 adds 2^-24 of its terms' magnitudes
    for each of its terms, and dx is rounded again.  So every element is within e (1 + 1/16) of the sum of its terms'
    magnitudes and that.  Over a tensor the errors are of random sign: a rounding is off by 0.42 e in the root mean
    square for values spread evenly over a binade's logarithm, so evidence with one rounding in its terms is off by
    0.42 e of itself, with two by 0.59 e: half of e is between them."""

    from qste_amd import kernels

    print(f"gated backward {m} x {rows} x {cols} {dtype} {kept}", flush=True)
    e = torch.finfo(dtype).eps / 2
    gen = torch.Generator(device=DEV).manual_seed(m + rows)
    x = (torch.randn(m, cols, generator=gen, device=DEV) + 0.1).to(dtype)
    x *= torch.rand(m, 1, generator=gen, device=DEV).add(0.5).to(dtype)
    g, u, dh = (torch.randn(m, rows, generator=gen, device=DEV).to(dtype) for _ in range(3))
    packed = torch.randint(0, 256, (2 * rows, -(-cols // 8)), generator=gen, device=DEV, dtype=torch.uint8)
    if cols % 8:
        packed[:, -1] &= (1 << (cols % 8)) - 1
    scale = (torch.rand(2 * rows, generator=gen, device=DEV) + 0.2).to(dtype).float()
    payload, offset, xs = kernels.pack_affine_rows(x)
    operands = [kernels.quantize_blocks(t) if kept == "blocks" else t for t in (g, u)]
    dx, evidence, grad_scale, grad_bias = kernels.gated_backward(dh, *operands, payload, offset, xs, packed, scale, cols,
                                                                 need_bias=True)
    if kept == "blocks":
        g, u = (kernels.dequantize_blocks(t) for t in operands)
    a, b, d = g.double(), u.double(), dh.double()
    s = torch.sigmoid(a)
    dy = torch.cat((d * b * s * (1 + a * (1 - s)), d * a * s), 1)
    place = torch.arange(cols, device=DEV)
    sign = ((packed[:, place // 8].int() >> (place % 8)) & 1).double() * 2 - 1
    x_sign = ((payload[:, place // 8].int() >> (place % 8)) & 1).double() * 2 - 1
    seen, wide = offset.double()[:, None] + xs.double()[:, None] * x_sign, scale.double()[:, None]
    term = e * (1 + 1 / 16)
    tiny = 2.0 ** -24 if dtype == torch.float16 else 1e-30

    def close(got, want, sizes, terms, rounded=0.0):
        bound = (term + terms * 2.0 ** -24) * sizes + rounded * (want.abs() + term * sizes) + tiny * (1 + terms)
        assert bool(((got.double() - want).abs() <= bound).all())

    close(dx, dy @ (sign * wide), dy.abs() @ wide.expand(-1, cols), 2 * rows, e)
    whole = dy.t() @ seen
    sizes = dy.abs().t() @ (offset.double().abs() + xs.double())[:, None].expand(-1, cols)
    close(evidence, whole * wide, sizes * wide, m)
    close(grad_scale, (whole * sign).sum(1), sizes.sum(1), m + cols)
    close(grad_bias, dy.sum(0), dy.abs().sum(0), m)
    if m * rows > 100000:
        assert float((evidence.double() - whole * wide).norm() / (whole * wide).norm()) <= 0.5 * e
    no_input = kernels.gated_backward(dh, *operands, payload, offset, xs, packed, scale, cols, need_input=False)
    assert no_input[0] is None and no_input[3] is None
    again = kernels.gated_backward(dh, *operands, payload, offset, xs, packed, scale, cols)
    assert torch.equal(again[1], evidence) and torch.equal(_bits(again[0]), _bits(dx))


@pytest.mark.parametrize("kept", ["values", "blocks"])
def test_past_32_bit_offsets(kept):
    """Outputs of 4.6 GB and gradients of 9.2: rows that repeat have results that repeat, bit for bit, wherever they lie
    (256 rows are whole tiles, and whole rounds of the backward's waves)."""

    from qste_amd import kernels

    repeats, features = 625, 14336
    x, layers = _operands(256, features, 64, torch.bfloat16)
    h, g, u = kernels.gated_forward(x.repeat(repeats, 1), *layers, 64, keep=kept)
    assert h.numel() * 2 > 1 << 32
    parts = (h, g, u) if kept == "values" else (h, g.payload, g.codes, u.payload, u.codes)
    for t in parts:
        assert torch.equal(t[-256:], t[:256])
    _, offset, scale = kernels.pack_affine_rows(x)
    grads, evidence, _ = kernels._gated_grads(h, g, u, offset.repeat(repeats), scale.repeat(repeats))
    for t in (grads, evidence):
        assert torch.equal(t[-256:], t[:256]) and bool(t[:256].any())
    small = (g[:256], u[:256]) if kept == "values" else [type(b)(b.payload[:256], b.codes[:256], b.dtype) for b in (g, u)]
    want = kernels._gated_grads(h[:256].contiguous(), *small, offset, scale)
    assert torch.equal(grads[:256], want[0]) and torch.equal(evidence[:256], want[1])


def test_scales_that_the_type_does_not_hold():
    """A sample whose scale is past fp16's range, or below its least, has evidence of infinities and of zeros, as the
    operand of that scale gives; the others' stay what they are."""

    from qste_amd import kernels

    gen = torch.Generator(device=DEV).manual_seed(5)
    g, u, dh = (torch.randn(40, 32, generator=gen, device=DEV).half() for _ in range(3))
    x, layers = _operands(40, 32, 64, torch.float16)
    packed, scale = torch.cat((layers[0], layers[3])), torch.cat((layers[1], layers[4]))
    payload, offset, xs = kernels.pack_affine_rows(x)
    dh[3] = 0
    want = kernels.gated_backward(dh, g, u, payload, offset, xs, packed, scale, 64)
    xs[3] = 1e-12  # of no gradient: nothing changes
    assert torch.equal(kernels.gated_backward(dh, g, u, payload, offset, xs, packed, scale, 64)[1], want[1])
    xs[4] = 1e6
    large = kernels.gated_backward(dh, g, u, payload, offset, xs, packed, scale, 64)
    assert torch.equal(_bits(large[0]), _bits(want[0])) and not bool(torch.isfinite(large[1]).any())


def test_backward_refusals():
    from qste_amd import kernels

    x, layers = _operands(6, 32, 64, torch.bfloat16)
    g = torch.zeros(6, 32, dtype=torch.bfloat16, device=DEV)
    payload, offset, xs = kernels.pack_affine_rows(x)
    packed, scale = torch.cat((layers[0], layers[3])), torch.cat((layers[1], layers[4]))
    good = [g, g, g, payload, offset, xs, packed, scale, 64]
    kernels.gated_backward(*good)
    for at, bad, error in ((0, g.float(), TypeError), (0, g[:, :31].contiguous(), ValueError), (0, g[:0], ValueError),
                           (1, g[:5], ValueError), (2, g.half(), ValueError), (3, payload[:5], ValueError),
                           (4, offset[:5], ValueError), (5, xs[:5], ValueError), (6, layers[0], ValueError),
                           (7, layers[1], ValueError), (1, kernels.quantize_blocks(g), TypeError)):
        with pytest.raises(error):
            kernels.gated_backward(*good[:at], bad, *good[at + 1:])


def test_node_against_the_layers_one_by_one():
    """Output, input gradient, evidence and scale gradients of the composition with the plain gate.

    The composition rounds dg (or du), twice on its way, and x's scale in the evidence's operand, the node dg and its
    scale together: four roundings' root of squares, 0.42 e each (see above), bounds the evidence's difference by e."""

    import qste_amd as qste

    gate, up = _pair(4096, 1024, 5)
    x = (torch.randn(2048, 1024, device=DEV, generator=torch.Generator(device=DEV).manual_seed(1)) + 0.1).bfloat16()
    grad = torch.randn(2048, 4096, device=DEV, generator=torch.Generator(device=DEV).manual_seed(2)).bfloat16()
    results = []
    for call in (lambda t: qste.nn.gated(t, gate, up), lambda t: qste.nn.swiglu(gate(t), up(t))):
        t = x.clone().requires_grad_()
        h = call(t)
        h.backward(grad)
        results.append((h.detach(), t.grad, gate.evidence.pop(), up.evidence.pop(), gate.surface.log_scale.grad,
                        up.surface.log_scale.grad))
        gate.surface.log_scale.grad = up.surface.log_scale.grad = None
    one, other = results
    # the output is rounded once and not twice; the input gradient once rather than twice with a sum in between; the
    # others may sum in another order
    e = 2.0 ** -8
    assert float((one[0].double() - other[0].double()).norm() / other[0].double().norm()) <= 2 * e
    assert float((one[1].double() - other[1].double()).norm() / other[1].double().norm()) <= 2 * e
    for a, b in zip(one[2:], other[2:]):
        assert float((a - b).norm() / b.norm()) <= e


def test_node_against_differences():
    """The input gradient along a direction against differences of the definition in 64 bits.

    dx is rounded to bf16, dg and du before it, and the row scales: each 2^-9 of a term at most, of random sign over
    thousands of terms; the direction's sum is within 4 2^-9 of the terms' root sum of squares, far above the
    difference's own error."""

    import qste_amd as qste

    m, rows, cols = 64, 512, 256
    gate, up = _pair(rows, cols, 9, dtype=torch.bfloat16)
    gen = torch.Generator(device=DEV).manual_seed(4)
    x = torch.randn(m, cols, generator=gen, device=DEV).bfloat16().requires_grad_()
    w = torch.randn(m, rows, generator=gen, device=DEV).bfloat16()
    v = torch.randn(m, cols, generator=gen, device=DEV).double()
    qste.nn.gated(x, gate, up).backward(w)
    signs = [layer.surface.sign.double() * layer.scale.detach().double()[:, None] for layer in (gate, up)]

    def value(t):
        g, u = t @ signs[0].t(), t @ signs[1].t()
        return (w.double() * g * torch.sigmoid(g) * u).sum()

    step = 2.0 ** -14
    slope = float((value(x.detach().double() + step * v) - value(x.detach().double() - step * v)) / (2 * step))
    terms = x.grad.double() * v
    assert abs(float(terms.sum()) - slope) <= 4 * 2.0 ** -9 * float(terms.norm()) * math.sqrt(8)


def test_log_scales_of_two_types_and_bounds():
    """Log-scales in different types, at and past the clamp, and surfaces with bounds of their own."""

    import qste_amd as qste
    from qste_amd import kernels

    x = torch.randn(40, 64, device=DEV, generator=torch.Generator(device=DEV).manual_seed(1)).bfloat16()
    w = torch.randn(40, 96, device=DEV, generator=torch.Generator(device=DEV).manual_seed(2)).bfloat16()
    for types, bounds in (((torch.float32, torch.bfloat16), (4.0, 4.0)), ((torch.bfloat16, torch.bfloat16), (4.0, 0.125)),
                          ((torch.float32, torch.float32), (0.125, 4.0))):
        gate, up = _pair(96, 64, 8)
        for layer, dtype, hi in zip((gate, up), types, bounds):
            layer.surface.cfg = qste.QSTEConfig(scale_max=hi)
            layer.surface.log_scale.data = layer.surface.log_scale.data.to(dtype)
        h = qste.nn.gated(x, gate, up)
        h.backward(w)
        scales = [layer.scale.detach().float() for layer in (gate, up)]
        assert all(float(s.max()) <= hi for s, hi in zip(scales, bounds))
        want, g, u = kernels.gated_forward(x, gate.packed_sign, scales[0], None, up.packed_sign, scales[1], None, 64,
                                           keep="values")
        assert torch.equal(h.detach(), want)
        grad_scale = kernels.gated_backward(w, g, u, *kernels.pack_affine_rows(x),
                                            torch.cat((gate.packed_sign.data, up.packed_sign.data)), torch.cat(scales),
                                            64)[2]
        for layer, part, hi in ((gate, grad_scale[:96], bounds[0]), (up, grad_scale[96:], bounds[1])):
            log_scale = layer.surface.log_scale
            e = log_scale.detach().exp()
            inside = (e.float() >= 1e-6) & (e.float() <= hi)
            assert log_scale.grad.dtype == log_scale.dtype
            assert torch.equal(log_scale.grad, torch.where(inside, e.float() * part, 0.0).to(log_scale.dtype))


def test_node_in_use():
    """Frozen inputs, gradients turned off, autocast, a pair of one layer, a strided and a broadcast gradient, a second
    backward through a kept graph, forward-mode refused."""

    import qste_amd as qste

    gate, up = _pair(128, 64, 3)
    x = torch.randn(10, 64, device=DEV, generator=torch.Generator(device=DEV).manual_seed(1)).bfloat16()
    with torch.no_grad():
        plain = qste.nn.gated(x, gate, up, checkpoint=True)
    assert not plain.requires_grad and gate.surface.ledger.open_uses == 0
    h = qste.nn.gated(x, gate, up, checkpoint=True)  # x is no leaf that wants a gradient
    assert torch.equal(h.detach(), plain)
    h.sum().backward()  # a broadcast gradient
    assert len(gate.evidence) == 1 and x.grad is None
    with torch.autocast("cuda", dtype=torch.bfloat16):
        assert torch.equal(qste.nn.gated(x.float(), gate, up).detach(), plain)
    gate.surface.reset_tracking(), up.surface.reset_tracking()
    gate.evidence.clear(), up.evidence.clear()
    t = x.clone().requires_grad_()
    h = qste.nn.gated(t, gate, up)
    wide = torch.randn(128, 10, device=DEV).bfloat16()
    h.backward(wide.t(), retain_graph=True)
    first = t.grad.clone()
    t.grad = None
    h.backward(wide.t().contiguous())
    assert torch.equal(t.grad, first)
    gate.evidence.clear()
    qste.nn.gated(x, gate, gate).sum().backward()  # one surface for both
    assert len(gate.evidence) == 1
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(x, torch.ones_like(x))
        with pytest.raises(NotImplementedError):
            qste.nn.gated(dual, gate, up)
        with pytest.raises(NotImplementedError):
            qste.nn.swiglu(dual, x, checkpoint=True)


@pytest.mark.parametrize("dtype,cols,rows", [(torch.float32, 64, 128), (torch.float32, 40, 33)])
def test_layers_that_the_node_does_not_take(dtype, cols, rows):
    import qste_amd as qste

    gate, up = _pair(rows, cols, 3)
    x = torch.randn(10, cols, device=DEV, generator=torch.Generator(device=DEV).manual_seed(1)).to(dtype)
    a, b = x.clone().requires_grad_(), x.clone().requires_grad_()
    one = qste.nn.gated(a, gate, up)
    one.sum().backward()  # (evidence is delivered when every forward has had its backward)
    evidence = gate.evidence.pop()
    other = qste.nn.swiglu(gate(b), up(b))
    other.sum().backward()
    assert torch.equal(one, other)
    assert torch.equal(a.grad, b.grad) and torch.equal(evidence, gate.evidence.pop())
    qste.nn.gated(a, gate, up, checkpoint=True).sum().backward()
    assert len(gate.evidence) == 1


def test_packed_layers():
    """As a model is served: exported layers, one token and many."""

    import qste_amd as qste

    for m, dtype in ((1, torch.bfloat16), (9, torch.float32), (200, torch.float16), (30, torch.float32)):
        x, layers = _operands(m, 1000, 256, dtype, bias=True)
        gate, up = qste.PackedLinear(*layers[:2], 256, layers[2]), qste.PackedLinear(*layers[3:5], 256, layers[5])
        h = qste.nn.gated(x.requires_grad_(), gate, up)
        assert not h.requires_grad and _within_roundings(h, x.detach(), layers, dtype)


def test_mlp_with_a_checkpoint():
    """swiglu_mlp with its gate and up kept in 8 bits: the output of the MLP without, gradients near its, and the steps
    that the coordinates take inside backward from them; a run of everything together."""

    import qste_amd as qste

    class MLP(torch.nn.Module):
        def __init__(self, checkpoint):
            super().__init__()
            gen = torch.Generator().manual_seed(0)
            self.gate, self.up = torch.nn.Linear(256, 640, bias=False), torch.nn.Linear(256, 640, bias=False)
            self.down = torch.nn.Linear(640, 256, bias=False)
            for p in self.parameters():
                p.data.copy_(torch.randn(p.shape, generator=gen) * 0.05)
            self.checkpoint = checkpoint

        def forward(self, x):
            return qste.nn.swiglu_mlp(x, self.gate, self.up, self.down, checkpoint=self.checkpoint)

    runs = []
    for checkpoint in (False, True):
        model = MLP(checkpoint)
        qste.convert(model, include=["*"])
        model.to(DEV)
        coords = qste.QSTEOptimizer(model)
        before = [s.coordinate.detach().clone() for s in qste.surfaces(model)]
        x = torch.randn(128, 256, device=DEV, generator=torch.Generator(device=DEV).manual_seed(1)).bfloat16().requires_grad_()
        w = torch.randn(128, 256, device=DEV, generator=torch.Generator(device=DEV).manual_seed(2)).bfloat16()
        y = model(x)
        y.backward(w)
        coords.step()
        moved = [float((s.coordinate.detach() != b).float().mean()) for s, b in zip(qste.surfaces(model), before)]
        runs.append((y.detach(), x.grad, moved))
    (y0, dx0, moved0), (y1, dx1, moved1) = runs
    assert float((y1.double() - y0.double()).norm() / y0.double().norm()) <= 2.0 ** -8
    # a kept value is off by up to a 128th of its block's largest, uniformly: about 1% of the gradient
    assert float((dx1.double() - dx0.double()).norm() / dx0.double().norm()) <= 0.05
    assert all(a > 0 and b > 0 for a, b in zip(moved0, moved1))


def test_trained_then_served():
    """One module whose block is a call of gated: trained by steps of both optimizers with its gate and up in 8 bits,
    exported, and served a prompt and then token by token."""

    import qste_amd as qste

    class Block(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.gate, self.up = torch.nn.Linear(192, 520), torch.nn.Linear(192, 520, bias=False)
            self.down = torch.nn.Linear(520, 192, bias=False)

        def forward(self, x):
            return self.down(qste.nn.gated(x, self.gate, self.up, checkpoint=True))

    torch.manual_seed(0)
    model = Block()
    qste.convert(model, include=["*"])
    model.to(DEV)
    optimizer = torch.optim.SGD(qste.continuous_parameters(model), lr=1e-3)
    coords = qste.QSTEOptimizer(model)
    x = torch.randn(2, 150, 192, device=DEV, generator=torch.Generator(device=DEV).manual_seed(1)).bfloat16()
    before = [s.coordinate.detach().clone() for s in qste.surfaces(model)]
    for _ in range(3):
        model(x).float().square().mean().backward()
        # (of a mean over 57600 outputs: times the learning rate far below half a unit, 2^-23, of a log-scale of -3.3,
        # so that they are looked at and not what the step makes of them)
        assert all(bool(torch.isfinite(p.grad).all()) and bool((p.grad != 0).any()) for p in optimizer.param_groups[0]["params"])
        optimizer.step(), optimizer.zero_grad()
        coords.step()
    for s, b in zip(qste.surfaces(model), before):
        assert bool((s.coordinate.detach() != b).any())
        assert torch.equal(s.packed_sign.data, qste.kernels.pack_coordinate(s.coordinate.data))
    with torch.no_grad():
        whole = model(x)
    served = qste.export_packed(model)
    assert isinstance(served.gate, qste.PackedLinear)
    prompt = served(x)
    # the same products; those of few tokens sum in another order, which g, u, h and the output's rounding show: four
    # roundings of half a step each
    assert torch.equal(prompt, whole)
    for t in (0, 7, 149):
        token = served(x[:, t])
        assert float((token.double() - whole[:, t].double()).norm() / whole[:, t].double().norm()) <= 4 * 2.0 ** -8


def test_streams_and_graphs():
    """On a side stream, and captured with two ways in one graph and replayed with eager work in between."""

    from qste_amd import kernels

    small, layers = _operands(3, 640, 512, torch.bfloat16)
    large = _operands(90, 640, 512, torch.bfloat16, seed=1)[0]  # K in ranges, with a workspace
    want = [kernels.gated_forward(t, *layers, 512)[0] for t in (small, large)]
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        got = [kernels.gated_forward(t, *layers, 512)[0] for t in (small, large)]
    stream.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = [kernels.gated_forward(t, *layers, 512)[0] for t in (small, large)]
        kept = kernels.gated_forward(large, *layers, 512, keep="blocks")
        encoding = kernels.pack_affine_rows(large)
        packed, scale = torch.cat((layers[0], layers[3])), torch.cat((layers[1], layers[4]))
        back = kernels.gated_backward(kept[0], *kept[1:], *encoding, packed, scale, 512, need_bias=True)
    for seed in (5, 6, 7):
        gen = torch.Generator(device=DEV).manual_seed(seed)
        for t in (small, large):
            t.copy_(torch.randn(t.shape, generator=gen, device=DEV))
        graph.replay()
        torch.cuda.synchronize()
        want = [kernels.gated_forward(t, *layers, 512)[0] for t in (small, large)]
        assert all(torch.equal(a, b) for a, b in zip(captured, want))
        eager = kernels.gated_forward(large, *layers, 512, keep="blocks")
        assert torch.equal(kept[0], eager[0]) and torch.equal(kept[1].payload, eager[1].payload)
        want = kernels.gated_backward(eager[0], *eager[1:], *kernels.pack_affine_rows(large), packed, scale, 512,
                                      need_bias=True)
        assert all(torch.equal(a, b) for a, b in zip(back, want))


@pytest.mark.parametrize("rows,checkpoint,dtype", [(192, True, torch.bfloat16), (203, True, torch.float16),
                                                   (192, False, torch.bfloat16)])
def test_node_captured(rows, checkpoint, dtype):
    """A training step of the block in a graph: every replay, with eager steps and synchronizations between, equals the
    eager step on what the inputs hold then."""

    import qste_amd as qste

    gate, up = _pair(rows, 96, 12, bias=True, dtype=dtype)
    x = torch.randn(70, 96, device=DEV, generator=torch.Generator(device=DEV).manual_seed(1)).to(dtype).requires_grad_()
    w = torch.randn(70, rows, device=DEV, generator=torch.Generator(device=DEV).manual_seed(2)).to(dtype)
    leaves = (x, gate.surface.log_scale, up.surface.log_scale, gate.bias, up.bias)

    def step():
        h = qste.nn.gated(x, gate, up, checkpoint=checkpoint)
        grads = torch.autograd.grad(h, leaves, w)
        return (h.detach(), *grads, gate.evidence.pop(), up.evidence.pop())

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for seed in (3, 4, 5, 6):
        gen = torch.Generator(device=DEV).manual_seed(seed)
        x.detach().copy_(torch.randn(70, 96, device=DEV, generator=gen))
        w.copy_(torch.randn(70, rows, device=DEV, generator=gen))
        graph.replay()
        torch.cuda.synchronize()
        kept = [t.clone() for t in captured]
        want = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(kept, want))
        assert bool(want[0].any()) and bool(want[-1].any())
