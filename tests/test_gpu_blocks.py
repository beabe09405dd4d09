"""8-bit blocks: the format against its definition in 64 bits, and the SwiGLU gate
that keeps its inputs in them.

Quantising and reading back have one right answer each (the scale is a power of
two, so nothing but the 8-bit value is rounded), and are compared bit for bit.
The gate with a checkpoint is compared bit for bit with the gate without one,
and its backward with the formula in 64 bits at the values that the blocks stand
for, and with differences of it.
"""

from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda"
DTYPES = [torch.bfloat16, torch.float16, torch.float32]
HALF_STEP = {t: torch.finfo(t).eps / 2 for t in DTYPES}


@pytest.fixture(autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    from qste_amd import kernels

    assert kernels.native_available(), kernels.status()


def _randn(shape, dtype, seed, std=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randn(shape, generator=g, device=DEV) * std).to(dtype)


def _bits(t):
    return t.contiguous().view({1: torch.int8, 2: torch.int16, 4: torch.int32}[t.element_size()])


def _reference(x):
    """(payload, codes) of x [rows, columns] by the definition, in 64 bits on the CPU."""

    x = x.detach().double().cpu()
    rows, cols = x.shape
    nblk = -(-cols // 32)
    padded = torch.zeros(rows, nblk * 32, dtype=torch.float64)
    padded[:, :cols] = x
    b = padded.view(rows, nblk, 32)
    bad = ~torch.isfinite(b).all(2)
    top = torch.where(bad, 1.0, b.abs().amax(2))
    _, e = torch.frexp(top)  # top = m 2^e, m in [1/2, 1): a biased exponent of e - 1 + 127
    codes = torch.where(top > 0, e + 126, 0).clamp(min=7)
    q = torch.round(torch.nan_to_num(b) * torch.exp2(133.0 - codes.double()).unsqueeze(2)).clamp(-127, 127)
    q = torch.where(bad.unsqueeze(2), 0.0, q)
    codes = torch.where(bad, 255, codes)
    return q.view(rows, -1)[:, :cols].to(torch.int8), codes.to(torch.uint8)


SHAPES = [(1, 1), (1, 7), (3, 8), (5, 31), (4, 32), (7, 33), (2, 40), (9, 96), (33, 1000), (2, 4099), (64, 4096),
          (300, 136)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_blocks_equal_the_definition(shape, dtype):
    from qste_amd import nn as qnn

    print(f"blocks {shape} {dtype}", flush=True)
    x = _randn(shape, dtype, sum(shape))
    x[:, ::5] *= 30.0
    x[0, 0] = 0.0
    b = qnn.quantize_blocks(x)
    payload, codes = _reference(x)
    assert b.payload.dtype == torch.int8 and b.codes.dtype == torch.uint8 and b.dtype == dtype
    assert torch.equal(b.codes.cpu(), codes) and torch.equal(b.payload.cpu(), payload)
    back = qnn.dequantize_blocks(b)
    want = payload.double() * torch.exp2(codes.double() - 133.0).repeat_interleave(32, 1)[:, :shape[1]]
    assert back.dtype == dtype and torch.equal(back.double().cpu(), want)  # exact in the type they came from
    # half a step for what is not clamped, a step for what is: magnitudes past 127.5 steps
    step = torch.exp2(codes.double() - 133.0).repeat_interleave(32, 1)[:, :shape[1]]
    clamped = x.double().cpu().abs() > 127.5 * step
    error = (back.double().cpu() - x.double().cpu()).abs()
    assert bool((error <= torch.where(clamped, step, step / 2)).all())


@pytest.mark.parametrize("dtype", DTYPES)
def test_blocks_of_every_value(dtype):
    """Every finite bf16 / fp16 value (and as many fp32 ones) as the largest of a block, the ends of the range and
    the subnormal ones among them."""

    from qste_amd import kernels

    if dtype == torch.float32:
        g = torch.Generator(device=DEV).manual_seed(3)
        x = torch.randint(-2**31, 2**31 - 1, (65536,), generator=g, device=DEV).to(torch.int32).view(torch.float32)
        x[:4] = torch.tensor([3.4028234663852886e38, -3.4028234663852886e38, 1.4e-45, -1.1754944e-38], device=DEV)
    else:
        x = torch.arange(-32768, 32768, device=DEV).to(torch.int16).view(dtype)
    x = torch.where(torch.isfinite(x), x, 0.0)
    rows = torch.zeros(65536, 33, dtype=dtype, device=DEV)
    rows[:, 3] = x
    rows[:, 20] = x * 0.37
    rows[:, 32] = -x  # a block of one
    b = kernels.quantize_blocks(rows)
    payload, codes = _reference(rows)
    assert torch.equal(b.codes.cpu(), codes) and torch.equal(b.payload.cpu(), payload)
    back = kernels.dequantize_blocks(b)
    assert bool(torch.isfinite(back).all())
    want = payload.double() * torch.exp2(codes.double() - 133.0).repeat_interleave(32, 1)[:, :33]
    assert torch.equal(back.double().cpu(), want)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("cols", [33, 64])
def test_blocks_of_what_is_not_finite(dtype, cols):
    from qste_amd import nn as qnn

    x = _randn((6, cols), dtype, 11)
    x[0, 4], x[1, 32], x[2, 31], x[3, :32] = math.inf, -math.inf, math.nan, 0.0
    b = qnn.quantize_blocks(x)
    payload, codes = _reference(x)
    assert torch.equal(b.codes.cpu(), codes) and torch.equal(b.payload.cpu(), payload)
    back = qnn.dequantize_blocks(b)
    bad = codes.repeat_interleave(32, 1)[:, :cols] == 255
    assert torch.equal(torch.isnan(back).cpu(), bad)
    assert bool((back[3, :32] == 0).all())


@pytest.mark.parametrize("dtype", DTYPES)
def test_blocks_of_views(dtype):
    """Strided, transposed and misaligned tensors, empty ones, and more dimensions."""

    from qste_amd import nn as qnn

    base = _randn((24, 520), dtype, 5)
    for x in (base[:, 3:99], base[::2], base.t()[:40], base[3:4, 1:], base.view(4, 6, 520), base[0]):
        b = qnn.quantize_blocks(x)
        flat = x.reshape(-1, x.shape[-1])
        payload, codes = _reference(flat)
        assert b.payload.shape == x.shape and b.codes.shape == (*x.shape[:-1], -(-x.shape[-1] // 32))
        assert torch.equal(b.payload.cpu().reshape(payload.shape), payload)
        assert torch.equal(b.codes.cpu().reshape(codes.shape), codes)
        again = qnn.dequantize_blocks(b, torch.float32)
        assert torch.equal(again.to(dtype), qnn.dequantize_blocks(b))
    for shape in ((0, 64), (3, 0), (2, 0, 5)):
        b = qnn.quantize_blocks(torch.empty(shape, dtype=dtype, device=DEV))
        assert qnn.dequantize_blocks(b).shape == shape


def test_blocks_past_32_bit_offsets():
    """A tensor of more than 2^32 bytes and more than 2^31 elements: its last rows."""

    from qste_amd import kernels

    rows, cols = (1 << 31) // 4104 + 5, 4104  # blocks that end inside a row
    x = torch.zeros(rows, cols, dtype=torch.bfloat16, device=DEV)
    x[-3:] = _randn((3, cols), torch.bfloat16, 1)
    b = kernels.quantize_blocks(x)
    payload, codes = _reference(x[-3:])
    assert torch.equal(b.payload[-3:].cpu(), payload) and torch.equal(b.codes[-3:].cpu(), codes)
    want = kernels.dequantize_blocks(kernels.quantize_blocks(x[-3:]))
    x.fill_(1.0)
    kernels.dequantize_blocks(b, torch.bfloat16)
    assert torch.equal(kernels.dequantize_blocks(b)[-3:], want)


# ---------------------------------------------------------------------------
# the gate with a checkpoint
# ---------------------------------------------------------------------------


def _as_kept(x):
    from qste_amd import kernels

    return kernels.dequantize_blocks(kernels.quantize_blocks(x))


def _exact_grads(grad, gate, up):
    """dg and du of silu(g) u at the blocks' values in 64 bits, and how far a kernel's may be off.

    In units of 2^-24, relative: the exponential's argument |g| log2(e) is rounded, |g| of them in e^-g, the exponential
    and the reciprocal are within two each, and the additions and products give one each: |g| + 10 of s, a = g s, du,
    and of 1 + g - a, whose terms are |g|, |a| and 1.  Then half a step of the type, relative or of its least one."""

    e, tiny = HALF_STEP[grad.dtype], (2.0 ** -25 if grad.dtype == torch.float16 else 1e-37)
    g, u, dh = _as_kept(gate).double(), _as_kept(up).double(), grad.double()
    s = torch.sigmoid(g)
    a, inner, unit = g * s, 1 + g * (1 - s), 2.0 ** -24 * (g.abs() + 10)
    dg, du = dh * u * s * inner, dh * a
    off = (dh * u * s).abs() * unit * (inner.abs() + a.abs() + g.abs() + 1)
    return dg, du, e * (dg.abs() + off) + off + tiny, (e + unit * (1 + e)) * du.abs() + tiny


def _near_exact(got, grad, gate, up):
    dg, du, off_g, off_u = _exact_grads(grad, gate, up)
    for x, want, off in ((got[0], dg, off_g), (got[1], du, off_u)):
        assert x.dtype == grad.dtype and torch.equal(torch.isnan(x), torch.isnan(want))
        assert bool(((x.double() - want).abs().nan_to_num(0.0) <= off.nan_to_num(0.0)).all())


GATES = [(1, 1), (2, 5), (7, 31), (5, 40), (33, 1000), (3, 17, 24), (6, 100), (64, 4096), (37, 14336), (5, 18000)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", GATES)
def test_gate_with_a_checkpoint(shape, dtype):
    from qste_amd import kernels, nn as qnn

    print(f"swiglu checkpoint {shape} {dtype}", flush=True)
    gate, up = _randn(shape, dtype, 1, 2.0), _randn(shape, dtype, 2)
    grad = _randn(shape, dtype, 3)
    g, u = gate.clone().requires_grad_(), up.clone().requires_grad_()
    h = qnn.swiglu(g, u, checkpoint=True)
    assert torch.equal(_bits(h.detach()), _bits(qnn.swiglu(gate, up)))
    h.backward(grad)
    _near_exact((g.grad, u.grad), grad, gate, up)
    # the encoding beside it, and the blocks
    flat_g, flat_u = gate.reshape(-1, shape[-1]), up.reshape(-1, shape[-1])
    out, encoding, kept_g, kept_u = kernels.swiglu_forward_blocks(flat_g, flat_u, encode=True)
    assert torch.equal(_bits(out), _bits(h.detach().reshape(out.shape)))
    for got, want in zip(encoding, kernels.pack_affine_rows(out)):
        assert torch.equal(_bits(got), _bits(want))
    for kept, t in ((kept_g, flat_g), (kept_u, flat_u)):
        want = kernels.quantize_blocks(t)
        assert torch.equal(kept.payload, want.payload) and torch.equal(kept.codes, want.codes)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(1, 8), (5, 40), (300, 1000), (513, 520), (9, 33), (5000, 1032),
                                   (40, 14336)])
def test_backward_sums_with_a_checkpoint(shape, dtype):
    from qste_amd import kernels

    print(f"swiglu sums {shape} {dtype}", flush=True)
    gate, up, grad = _randn(shape, dtype, 1, 2.0), _randn(shape, dtype, 2), _randn(shape, dtype, 3)
    off_g, off_u = _randn(shape[:1], torch.float32, 4), _randn(shape[:1], torch.float32, 5)
    kept = kernels.quantize_blocks(gate), kernels.quantize_blocks(up)
    got = kernels.swiglu_backward_blocks(grad, *kept, off_g, off_u)
    plain = kernels.swiglu_backward_blocks(grad, *kept)
    assert torch.equal(_bits(got[0]), _bits(plain[0])) and torch.equal(_bits(got[1]), _bits(plain[1]))
    _near_exact(got, grad, gate, up)
    # a sum of fp32 products in fp32: a unit of 2^-24 of the magnitudes' sum for each of its terms, beside the terms' own
    # errors (which are summed before or after they are rounded to the type, by the layout)
    for x, off, sums, error in zip(_exact_grads(grad, gate, up)[:2], (off_g, off_u), got[2], _exact_grads(grad, gate, up)[2:]):
        terms = x * off.double()[:, None]
        bound = (shape[0] + 4) * 2.0 ** -24 * terms.abs().sum(0) + (error * off.double().abs()[:, None]).sum(0)
        assert bool(((sums.double() - terms.sum(0)).abs() <= bound).all())
    if dtype != torch.float32 and shape[1] % 8 == 0:
        both, sums = kernels.swiglu_backward_blocks(grad, *kept, off_g, off_u, side_by_side=True)
        assert torch.equal(both, torch.cat(got[:2], 1)) and torch.equal(_bits(sums), _bits(got[2]))


def test_many_rows_take_the_tables():
    """Rows enough for the tabled passes, in both of their widths."""

    from qste_amd import kernels

    for shape in ((4100, 520), (4096, 4104)):
        gate, up, grad = (_randn(shape, torch.bfloat16, i, 2.0) for i in (1, 2, 3))
        gate[7, 3] = math.inf
        out, encoding, kept_g, kept_u = kernels.swiglu_forward_blocks(gate, up, encode=True)
        plain, plain_encoding = kernels.swiglu_forward(gate, up, encode=True)
        assert torch.equal(_bits(out), _bits(plain))
        for a, b in zip(encoding, plain_encoding):
            assert torch.equal(_bits(a), _bits(b))
        want = kernels.quantize_blocks(gate)
        assert torch.equal(kept_g.payload, want.payload) and torch.equal(kept_g.codes, want.codes)
        _near_exact(kernels.swiglu_backward_blocks(grad, kept_g, kept_u), grad, gate, up)


def test_gradients_against_differences():
    """The gradients are those of sum(w silu(g') u') at the blocks' values g', u', in 64 bits by central differences.

    fp32: a chain of a dozen operations on the values, each within a few units of 2^-24, against gradients that may
    cancel to a fraction of their terms: 2^-24 * 64 of the largest term.  Differences with a step of 2^-13: an error of
    step^2 / 6 times a third derivative below 1, and 2^-52 / step of rounding, both below 1e-8 of the terms."""

    from qste_amd import nn as qnn

    gate, up, w = _randn((9, 100), torch.float32, 1, 2.0), _randn((9, 100), torch.float32, 2), _randn((9, 100), torch.float32, 3)
    g, u = gate.clone().requires_grad_(), up.clone().requires_grad_()
    qnn.swiglu(g, u, checkpoint=True).backward(w)
    gd, ud, wd, step = _as_kept(gate).double(), _as_kept(up).double(), w.double(), 2.0 ** -13

    def value(a, b):
        return wd * a / (1 + torch.exp(-a)) * b

    slope_g = (value(gd + step, ud) - value(gd - step, ud)) / (2 * step)
    slope_u = (value(gd, ud + step) - value(gd, ud - step)) / (2 * step)
    bound = 64 * 2.0 ** -24 * (wd.abs() * (1 + ud.abs()) * (1 + gd.abs())) + 1e-7
    assert bool(((g.grad.double() - slope_g).abs() <= bound).all())
    assert bool(((u.grad.double() - slope_u).abs() <= bound).all())


def test_value_of_every_gate():
    """The value with a checkpoint is torch's, bit for bit, at every bf16 gate: each has a rounding of its own."""

    import torch.nn.functional as F

    from qste_amd import nn as qnn

    every = torch.arange(-32768, 32768, dtype=torch.int32, device=DEV).to(torch.int16)
    gate = every.view(torch.bfloat16).reshape(256, 256).requires_grad_()
    for seed in (1, 2):
        up = torch.ones_like(gate.detach()) if seed == 1 else _randn((256, 256), torch.bfloat16, seed)
        got, want = qnn.swiglu(gate, up, checkpoint=True).detach(), (F.silu(gate) * up).detach()
        number = ~torch.isnan(want)
        assert torch.equal(torch.isnan(got), ~number) and torch.equal(got[number].view(torch.int16),
                                                                      want[number].view(torch.int16))


def test_no_second_derivative():
    """A gradient that reached the node with a graph of its own is refused; one without any (a linear loss's) gives a
    gradient without one."""

    from qste_amd import nn as qnn

    gate, up = _randn((4, 64), torch.float32, 1).requires_grad_(), _randn((4, 64), torch.float32, 2)
    grad, = torch.autograd.grad(qnn.swiglu(gate, up, checkpoint=True).sum(), gate, create_graph=True)
    with pytest.raises(RuntimeError, match="does not require grad"):
        grad.sum().backward()
    loss = qnn.swiglu(gate, up, checkpoint=True).square().sum()
    grad, = torch.autograd.grad(loss, gate, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiate twice"):
        grad.sum().backward()


def test_codes_below_the_least_read_as_nothing():
    from qste_amd import nn as qnn

    payload = torch.full((2, 40), 100, dtype=torch.int8, device=DEV)
    codes = torch.tensor([[0, 6], [7, 133]], dtype=torch.uint8, device=DEV)
    for dtype in DTYPES:
        x = qnn.dequantize_blocks(qnn.Blocks8(payload, codes, dtype), torch.float32)
        assert bool((x[0] == 0).all()) and bool((x[1, :32] == 100 * 2.0 ** -126).all()) and bool((x[1, 32:] == 100).all())


def test_checkpoint_is_what_is_kept():
    """33 bytes for 32 elements, and nothing where no gradient is asked for."""

    from qste_amd import nn as qnn

    gate, up = _randn((64, 256), torch.bfloat16, 1).requires_grad_(), _randn((64, 256), torch.bfloat16, 2).requires_grad_()
    kept = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: kept.append(t.numel() * t.element_size()) or t, lambda t: t):
        h = qnn.swiglu(gate, up, checkpoint=True)
        assert sum(kept) == 2 * 64 * 256 * 33 // 32
        h.backward(torch.ones_like(h))
        kept.clear()
        with torch.no_grad():
            qnn.swiglu(gate, up, checkpoint=True)
        qnn.swiglu(gate.detach(), up.detach(), checkpoint=True)
        assert not kept


def test_captured():
    """Quantising, the gate and its backward in one graph, replayed with other values and eager work in between."""

    from qste_amd import kernels

    gate, up, grad = (_randn((40, 264), torch.bfloat16, i) for i in (1, 2, 3))
    off = _randn((40,), torch.float32, 4)

    def work():
        out, _, kept_g, kept_u = kernels.swiglu_forward_blocks(gate, up)
        both, sums = kernels.swiglu_backward_blocks(grad, kept_g, kept_u, off, off, side_by_side=True)
        return out, both, sums, kernels.dequantize_blocks(kept_g)

    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        work()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = work()
    for seed in (7, 8, 9):
        gate.copy_(_randn((40, 264), torch.bfloat16, seed))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(captured, work()):
            assert torch.equal(_bits(a), _bits(b))
