"""``qste_amd.nn.token_logprobs`` against its definition in 64 bits.

The plain form below works in float64 on the CPU from the logits' exact
values.  The bounds follow from the kernel's fp32 arithmetic: an exponential is
off by its argument's rounding, |z - m| log2(e) 2^-23 relative, and by two ulps;
a sum of V terms over the threads of a workgroup chains at most V / 256 + 16
additions, each 2^-24 relative, so over 131072 tokens ln S is within 528 * 2^-24
< 3.2e-5 in the worst case.  LOG below is that; an entropy adds the same for its
sum of e ln e over S, relative to the entropy.  A gradient's element carries
the relative error of p plus one rounding to the logits' dtype.
"""

from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda"
DTYPES = [torch.bfloat16, torch.float16, torch.float32]
LOG = 4e-5
ROUND = {torch.float32: 2.0 ** -23, torch.float16: 2.0 ** -10, torch.bfloat16: 2.0 ** -8}
LEAST = {torch.float32: 1e-37, torch.float16: 2.0 ** -24, torch.bfloat16: 1e-37}


@pytest.fixture(autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    from qste_amd import kernels

    assert kernels.native_available(), kernels.status()


def scores(logits, tokens, top=0, temperature=1.0):
    """The definition: (logprobs, entropy, top_logprobs, top_tokens) in float64 on the CPU."""

    z = logits.detach().cpu().double()
    lnp = torch.log_softmax(z / temperature, -1)
    lost = (z == -math.inf).all(-1)
    lnp = torch.where(lost.unsqueeze(-1), -math.inf, lnp)
    p = lnp.exp()
    entropy = -torch.where(p == 0, 0.0, p * lnp).sum(-1)
    entropy = torch.where(lost, 0.0, entropy)
    logprobs = None
    if tokens is not None:
        tokens = tokens.cpu().long()
        inside = tokens.clamp(0, z.shape[-1] - 1)
        logprobs = lnp.gather(-1, inside.unsqueeze(-1)).squeeze(-1)
        logprobs = torch.where(tokens >= z.shape[-1], math.nan, logprobs)
        logprobs = torch.where(tokens < 0, 0.0, logprobs)
        entropy = torch.where(tokens < 0, 0.0, entropy)
    values, places = torch.sort(z, dim=-1, descending=True, stable=True)
    places = places[..., :top]
    top_logprobs = lnp.gather(-1, places)
    if tokens is not None:
        unscored = (tokens < 0).unsqueeze(-1)
        places = torch.where(unscored, -1, places)
        top_logprobs = torch.where(unscored, -math.inf, top_logprobs)
    return logprobs, entropy, top_logprobs, places


def gradient(logits, tokens, g, h, temperature=1.0):
    """(dz, the size of the terms it is made of) in float64."""

    z = logits.detach().cpu().double()
    lnp = torch.log_softmax(z / temperature, -1)
    p = lnp.exp()
    lnp = torch.where(p == 0, 0.0, lnp)
    entropy = -(p * lnp).sum(-1, keepdim=True)
    g, h = (torch.zeros(z.shape[:-1]) if v is None else v.cpu() for v in (g, h))
    g, h = g.double().unsqueeze(-1), h.double().unsqueeze(-1)
    if tokens is not None:
        t = tokens.cpu().long().unsqueeze(-1)
        g, h = torch.where(t < 0, 0.0, g), torch.where(t < 0, 0.0, h)
        one = torch.zeros_like(z).scatter_(-1, t.clamp(min=0), 1.0)
    else:
        g, one = torch.zeros_like(g), torch.zeros_like(z)
    dz = (g * (one - p) - h * p * (lnp + entropy)) / temperature
    size = (g.abs() * (p + one) + h.abs() * p * (lnp.abs() + entropy)) / temperature
    return dz, size


def near(got, want, bound, what=""):
    """Within ``bound`` of ``want`` as fp32 can hold it; equal infinities and NaN where ``want`` has them."""

    got, want = got.detach().cpu().double(), want.float().double()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    same = (got == want) | (got.isnan() & want.isnan())
    off = torch.where(same, 0.0, (got - want).abs()).nan_to_num(nan=math.inf)
    bound = torch.as_tensor(bound).double().nan_to_num(nan=0.0, posinf=0.0)
    assert bool((off <= bound).all()), (what, float(off.max()), float((off - bound).max()))


def check(logits, tokens, top=0, temperature=1.0):
    import qste_amd as qste

    got = qste.nn.token_logprobs(logits, tokens, top=top, temperature=temperature)
    want = scores(logits, tokens, top, temperature)
    if tokens is None:
        assert got.logprobs is None
    else:
        near(got.logprobs, want[0], LOG + 1e-6 * want[0].abs(), "logprobs")
    near(got.entropy, want[1], LOG + LOG * want[1].abs(), "entropy")
    if top == 0:
        assert got.top_logprobs is None and got.top_tokens is None
    else:
        assert got.top_tokens.dtype == torch.int64
        assert torch.equal(got.top_tokens.cpu(), want[3])
        near(got.top_logprobs, want[2], LOG + 1e-6 * want[2].abs(), "top_logprobs")
    return got


def random_logits(shape, dtype, seed, spread=3.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randn(shape, generator=g, device=DEV) * spread).to(dtype)


def random_tokens(shape, vocab, seed):
    g = torch.Generator(device=DEV).manual_seed(seed + 1)
    return torch.randint(vocab, shape, generator=g, device=DEV)


SIZES = [(1, 1), (3, 2), (5, 7), (4, 8), (2, 9), (3, 63), (3, 64), (2, 129), (2, 511), (2, 513), (3, 1000), (2, 1024),
         (3, 2055), (2, 4099), (2, 8192), (2, 16391), (2, 32003), (2, 50257), (2, 65536), (1, 100003), (2, 131072),
         (1, 150001), (1, 300007)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,vocab", SIZES)
def test_scores(rows, vocab, dtype):
    print(f"scores {rows} x {vocab} {dtype}", flush=True)
    logits = random_logits((rows, vocab), dtype, vocab)
    tokens = random_tokens((rows,), vocab, vocab)
    check(logits, tokens, top=min(20, vocab))


@pytest.mark.parametrize("rows", [1, 2, 3, 16, 17, 255, 256, 257, 600])
def test_row_counts(rows):
    print(f"rows {rows}", flush=True)
    logits = random_logits((rows, 5003), torch.bfloat16, rows)
    check(logits, random_tokens((rows,), 5003, rows), top=3)


@pytest.mark.parametrize("top", [0, 1, 2, 63, 64, 65, 127, 128])
@pytest.mark.parametrize("vocab", [128, 600, 1030, 2000, 50257])
def test_top_counts(vocab, top):
    print(f"top {top} of {vocab}", flush=True)
    check(random_logits((3, vocab), torch.bfloat16, top), None, top=top)
    check(random_logits((3, vocab), torch.float32, top), None, top=top, temperature=0.5)


def test_top_of_the_whole_vocabulary():
    for vocab in (1, 5, 64, 128):
        check(random_logits((2, vocab), torch.float16, vocab), None, top=vocab)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab", [700, 9001, 50257, 131072])
def test_equal_and_ordered_logits(vocab, dtype):
    """Ties go to the lowest token: rows of one value, of a few values, in rising and falling order, and one
    where a long run of equals starts in the middle."""

    print(f"ties {vocab} {dtype}", flush=True)
    ramp = torch.arange(vocab, device=DEV).float() / vocab * 8
    few = torch.randint(0, 3, (vocab,), device=DEV, generator=torch.Generator(device=DEV).manual_seed(1)).float()
    step = (torch.arange(vocab, device=DEV) >= vocab // 2).float()
    zeros = torch.zeros(vocab, device=DEV)
    signed = torch.where(torch.arange(vocab, device=DEV) % 2 == 0, -0.0, 0.0)
    rows = torch.stack([zeros, zeros - 5, ramp, -ramp, few, step, signed]).to(dtype)
    for top in (1, 40, 128):
        check(rows, None, top=top)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab", [300, 5000, 50257, 140001])
def test_masked_rows(vocab, dtype):
    """-inf and the type's lowest value as masks: over most of a row, all but one token, and all of it."""

    print(f"masked {vocab} {dtype}", flush=True)
    lowest = torch.finfo(dtype).min
    g = torch.Generator(device=DEV).manual_seed(vocab)
    logits = random_logits((8, vocab), dtype, vocab)
    few = torch.rand(vocab, generator=g, device=DEV) > 7.0 / vocab
    logits[0].masked_fill_(few, -math.inf)
    logits[1].masked_fill_(few, lowest)
    logits[2] = -math.inf
    logits[3] = lowest
    logits[4, : vocab - 1] = -math.inf
    logits[5, 1:] = lowest
    logits[6, ::2] = -math.inf
    logits[7, vocab // 3:] = -math.inf
    tokens = torch.tensor([1, 2, 3, 4, vocab - 1, 0, 5, vocab - 1], device=DEV)
    want = scores(logits, tokens)
    assert float(want[0][2]) == -math.inf and abs(float(want[0][3]) + math.log(vocab)) < 1e-9
    check(logits, tokens, top=30)
    check(logits, tokens, top=2, temperature=0.7)


@pytest.mark.parametrize("dtype", DTYPES)
def test_infinite_and_nan_logits(dtype):
    vocab = 4097
    logits = random_logits((5, vocab), dtype, 3)
    logits[0, 17] = math.nan
    logits[1, 17] = math.inf
    logits[2, [5, 900]] = math.inf
    logits[3] = math.nan
    got = check(logits, torch.zeros(5, dtype=torch.long, device=DEV), top=4)
    assert got.logprobs[:4].isnan().all() and not got.logprobs[4].isnan()
    assert got.top_tokens[3].tolist() == [0, 1, 2, 3]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_huge_logits(dtype):
    """Near the end of fp32 the differences decide, not the scaled values."""

    for vocab in (9, 5000):
        logits = torch.full((4, vocab), -1e38, device=DEV)
        logits[0, 3] = 3e38
        logits[1, 2:6] = 3.3e38
        logits[2] = 2e38
        logits[3, 1] = -9e37
        check(logits.to(dtype), torch.tensor([3, 4, 0, 1], device=DEV), top=5)


@pytest.mark.parametrize("offset", [-3e4, 1e6, -2e7, 5e8, 1e12, -1e30])
@pytest.mark.parametrize("temperature", [1.0, 1e-3, 50.0])
def test_logits_far_from_zero(offset, temperature):
    """What a common offset leaves of the differences is what counts (fp32 logits: it leaves their rounding)."""

    logits = random_logits((4, 3001), torch.float32, 13) + offset
    check(logits, random_tokens((4,), 3001, 13), top=6, temperature=temperature)


def test_tokens_outside():
    vocab = 1000
    logits = random_logits((6, vocab), torch.bfloat16, 5)
    logits[1] = math.nan  # an unscored row is not read
    logits[4] = math.inf
    tokens = torch.tensor([3, -1, vocab, vocab - 1, -100, 1 << 40], device=DEV)
    got = check(logits, tokens, top=3)
    assert got.logprobs[2].isnan() and got.logprobs[5].isnan() and got.logprobs[1] == 0 and got.logprobs[4] == 0


@pytest.mark.parametrize("dtype", DTYPES)
def test_layouts(dtype):
    """Views are read in place: shifted sequences, padded vocabularies, swapped and broadcast dimensions, odd starts."""

    base = random_logits((3, 6, 1013), dtype, 11)
    tokens = random_tokens((3, 5), 900, 11)
    check(base[:, :-1], random_tokens((3, 5), 1013, 1), top=2)
    check(base[:, 1:, 3:903], tokens, top=2)
    check(base.transpose(0, 1)[1:, :, 1:], random_tokens((5, 3), 1012, 2), top=2)
    check(base[1:2, 2].expand(7, 1013), random_tokens((7,), 1013, 3), top=2)
    check(base[:, :, ::3], random_tokens((3, 6), 338, 4), top=2)
    check(base.view(3, 2, 3, 1013)[:, :, 1:], random_tokens((3, 2, 2), 1013, 5), top=2)
    check(base.view(3, 2, 3, 1013).permute(2, 0, 1, 3)[1:], random_tokens((2, 3, 2), 1013, 6), top=2)
    check(base[0, 0], torch.tensor(7, device=DEV), top=2)
    three = random_logits((2, 3, 4, 517), dtype, 12)[:, 1:, 1:]  # three strides: read through a copy
    check(three, random_tokens((2, 2, 3), 517, 12), top=2)
    flat = base.reshape(-1)[1:1 + 4 * 1013].view(4, 1013)
    check(flat, random_tokens((4,), 1013, 7).to(torch.int32), top=2)


@pytest.mark.parametrize("dtype,vocab", [(torch.bfloat16, 1_700_003), (torch.float32, 900_001), (torch.float16, 500_000)])
def test_very_long_rows(dtype, vocab):
    """In parts as long as registers hold, and past what so many parts hold."""

    print(f"long {vocab} {dtype}", flush=True)
    logits = random_logits((3, vocab), dtype, 14)
    logits[1] = torch.arange(vocab, device=DEV).float() / vocab  # in order, with long runs of equals
    logits[2, 5:] = -math.inf
    check(logits, torch.tensor([vocab - 1, 17, 3], device=DEV), top=100)


@pytest.mark.parametrize("rows,vocab", [(300, 32776), (150, 51200), (150, 51208), (1300, 65536)])
def test_many_long_rows(rows, vocab):
    """Both sides of where a row is cut, and of how many rows are cut into short parts."""

    print(f"many {rows} x {vocab}", flush=True)
    logits = random_logits((rows, vocab), torch.bfloat16, rows)
    tokens = random_tokens((rows,), vocab, rows)
    tokens[5] = -1
    check(logits, tokens, top=7)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,bytes_a_row", [(512, 32776), (512, 64006), (513, 64006), (512, 102400), (513, 102400),
                                              (512, 131086), (513, 131086), (512, 131088)])
def test_rows_around_the_wide_workgroups(rows, bytes_a_row, dtype):
    """Both sides of what a workgroup of more threads takes: by the number of rows, and by their length."""

    vocab = bytes_a_row // dtype.itemsize
    print(f"wide {rows} x {vocab} {dtype}", flush=True)
    logits = random_logits((rows, vocab), dtype, rows)
    logits[1] = torch.arange(vocab, device=DEV).float() / vocab
    logits[2, 5:] = -math.inf
    logits[3] = 1.5
    logits[4] = -math.inf
    tokens = random_tokens((rows,), vocab, rows)
    tokens[5] = -1
    check(logits, tokens, top=30)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("top", [1, 4, 8, 9, 16, 17])
def test_short_lists_of_parts(top, dtype):
    """Both sides of how the lists of a row's parts become one."""

    vocab = 131079
    logits = random_logits((7, vocab), dtype, top)
    logits[1] = torch.arange(vocab, device=DEV).float() / vocab
    logits[2, 5:] = -math.inf
    logits[3] = 1.5
    logits[4] = -math.inf
    logits[5, ::9001] = 60.0  # as the largest, some in every part
    check(logits, random_tokens((7,), vocab, top), top=top)
    check(logits, torch.full((7,), -1, device=DEV), top=top)


def test_rows_far_apart():
    """Offsets past 32 bits, in elements and in bytes."""

    stride, vocab = (1 << 31) + 12345, 4099
    buffer = torch.empty(stride + vocab, dtype=torch.bfloat16, device=DEV)
    logits = buffer.as_strided((2, vocab), (stride, 1))
    logits.copy_(random_logits((2, vocab), torch.bfloat16, 8))
    check(logits, torch.tensor([5, 4000], device=DEV), top=4)


def test_empty():
    import qste_amd as qste

    got = qste.nn.token_logprobs(torch.empty(0, 5, 100, device=DEV), torch.empty(0, 5, dtype=torch.long, device=DEV), top=3)
    assert got.logprobs.shape == (0, 5) and got.top_tokens.shape == (0, 5, 3)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("temperature", [1.0, 0.6, 2.5])
@pytest.mark.parametrize("rows,vocab", [(1, 1), (3, 5), (2, 8), (3, 1001), (2, 4104), (2, 50257), (1, 150001)])
def test_gradient(rows, vocab, temperature, dtype):
    import qste_amd as qste

    print(f"gradient {rows} x {vocab} {dtype} {temperature}", flush=True)
    gen = torch.Generator(device=DEV).manual_seed(rows + vocab)
    logits = random_logits((rows, vocab), dtype, vocab, 2.0).requires_grad_(True)
    tokens = random_tokens((rows,), vocab, vocab)
    if rows == 3:
        tokens[1] = -1
    g, h = torch.randn(2, rows, generator=gen, device=DEV)
    for weights in ((g, h), (g, None), (None, h)):
        s = qste.nn.token_logprobs(logits, tokens, temperature=temperature)
        total = sum((a * w).sum() for a, w in zip((s.logprobs, s.entropy), weights) if w is not None)
        got, = torch.autograd.grad(total, logits)
        want, size = gradient(logits, tokens, *weights, temperature)
        assert got.dtype == dtype and got.is_contiguous()
        near(got, want, ROUND[dtype] * want.abs() + LOG * size + LEAST[dtype], "grad")


def test_gradient_without_tokens_and_of_views():
    import qste_amd as qste

    base = random_logits((3, 4, 517), torch.float32, 2).requires_grad_(True)
    s = qste.nn.token_logprobs(base[:, :-1])
    s.entropy.sum().backward()  # a gradient that is one number, broadcast
    want, size = gradient(base[:, :-1], None, None, torch.ones(3, 3))
    near(base.grad[:, :-1], want, ROUND[torch.float32] * want.abs() + LOG * size + 1e-37)
    assert not base.grad[:, -1].any()
    shared = random_logits((517,), torch.float32, 3).requires_grad_(True)
    tokens = torch.tensor([1, 5, 5, 99], device=DEV)
    qste.nn.token_logprobs(shared.expand(4, 517), tokens).logprobs.sum().backward()
    want, size = gradient(shared.expand(4, 517), tokens, torch.ones(4), None)
    near(shared.grad, want.sum(0), LOG * size.sum(0) + 4e-7)


def test_gradient_of_masked_and_unscored_rows():
    """No gradient from rows of only -inf or unscored ones, none at masked tokens, NaN from a token past the end."""

    import qste_amd as qste

    vocab = 3001
    logits = random_logits((5, vocab), torch.bfloat16, 4)
    logits[0] = -math.inf
    logits[1] = math.nan
    logits[2, ::2] = -math.inf
    logits.requires_grad_(True)
    tokens = torch.tensor([4, -1, 5, vocab, 6], device=DEV)
    s = qste.nn.token_logprobs(logits, tokens)
    weight = torch.tensor([1.0, 1.0, 1.0, 1.0, 0.0], device=DEV)
    grad, = torch.autograd.grad((s.logprobs, s.entropy), logits, (weight, 0.5 * weight))
    assert not grad[0].any() and not grad[1].any() and not grad[4].any()
    assert not grad[2, ::2].any() and grad[2, 1::2].isfinite().all() and grad[3].isnan().all()
    want, size = gradient(logits[2:3], tokens[2:3], weight[2:3], 0.5 * weight[2:3])
    near(grad[2:3], want, ROUND[torch.bfloat16] * want.abs() + LOG * size + 1e-37)


def test_gradient_against_differences():
    """Central differences of the kernel's own forward: at 37 tokens its values are off by under 2e-6, over a step of
    1e-2 that is 2e-4; the third derivative of ln S in a direction of entries under 3 stays under 30, so the step
    itself adds 5e-4 (entropy: a few times that)."""

    import qste_amd as qste

    z = random_logits((6, 37), torch.float32, 9, 1.0)
    tokens = random_tokens((6,), 37, 9)
    v = random_logits((6, 37), torch.float32, 10, 1.0).clamp(-2.5, 2.5)

    def f(x):
        s = qste.nn.token_logprobs(x, tokens, temperature=1.3)
        return s.logprobs + 0.5 * s.entropy

    x = z.clone().requires_grad_(True)
    f(x).sum().backward()
    slope = (f(z + 1e-2 * v) - f(z - 1e-2 * v)) / 2e-2
    assert float((slope - (x.grad * v).sum(1)).abs().max()) < 4e-3


def test_same_bits_every_time_on_any_stream():
    import qste_amd as qste

    logits = random_logits((40, 50257), torch.bfloat16, 6).requires_grad_(True)
    tokens = random_tokens((40,), 50257, 6)

    def run():
        s = qste.nn.token_logprobs(logits, tokens, top=64)
        grad, = torch.autograd.grad((s.logprobs, s.entropy), logits, (torch.ones(40, device=DEV),) * 2)
        return [*(t.detach() for t in s), grad]

    first = run()
    side = torch.cuda.Stream()
    for _ in range(3):
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            again = run()
        torch.cuda.current_stream().wait_stream(side)
        assert all(torch.equal(a, b) for a, b in zip(first, again))


def test_in_a_graph():
    import qste_amd as qste

    logits = random_logits((3, 50257), torch.bfloat16, 1)
    tokens = random_tokens((3,), 50257, 1)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        qste.nn.token_logprobs(logits, tokens, top=8)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = qste.nn.token_logprobs(logits, tokens, top=8)
    for seed in range(4):
        logits.copy_(random_logits((3, 50257), torch.bfloat16, 20 + seed))
        tokens.copy_(random_tokens((3,), 50257, 20 + seed))
        graph.replay()
        torch.cuda.synchronize()
        eager = qste.nn.token_logprobs(logits, tokens, top=8)
        assert all(torch.equal(a, b) for a, b in zip(out, eager))


def test_refusals():
    import qste_amd as qste

    logits = torch.zeros(4, 100, device=DEV)
    tokens = torch.zeros(4, dtype=torch.long, device=DEV)
    f = qste.nn.token_logprobs
    for bad in (-1, 101, 129):
        with pytest.raises(ValueError, match="top must lie"):
            f(logits, tokens, top=bad)
    for bad in (0.0, -1.0, math.inf, math.nan):
        with pytest.raises(ValueError, match="temperature"):
            f(logits, tokens, temperature=bad)
    with pytest.raises(ValueError, match="tokens have shape"):
        f(logits, tokens[:3])
    with pytest.raises(TypeError, match="integers"):
        f(logits, tokens.float())
    with pytest.raises(TypeError, match="unsupported dtype"):
        f(logits.double(), tokens)
    with pytest.raises(ValueError, match="last dimension"):
        f(torch.zeros(4, 0, device=DEV), tokens)
    with pytest.raises(RuntimeError, match="GPU only"):
        f(logits.cpu(), tokens.cpu())
    with pytest.raises(RuntimeError, match="GPU only"):
        f(logits, tokens.cpu())
    x = logits.clone().requires_grad_(True)
    s = f(x, tokens, top=2)
    assert not s.top_logprobs.requires_grad and not s.top_tokens.requires_grad
    with torch.no_grad():
        assert not f(x, tokens).logprobs.requires_grad
