"""``qste_amd.nn.distillation_loss`` and ``distillation_loss_and_grad`` against their definition in 64 bits.

The plain form works in float64 on the CPU from the exact inputs.  The bounds
follow from the kernel's fp32 arithmetic: a log probability is within LOG (the
sum of up to 131072 exponentials chains at most 528 additions, 2^-24 relative
each), so a loss, an average of those, is within T^2 LOG and the rounding of its own sum of k
terms; the teacher's rest 1 - sum q is off by k 2^-23 at most, which its
logarithm's slope (under 20 for what is drawn here) turns into LOG again.  A
gradient's element carries the relative error of p (that of the sums) and
of its coefficient, plus one rounding to the logits' dtype.
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


def distilled(logits, tokens, values, weight, temperature=1.0, tail=False):
    """The definition, in float64 on the CPU: (losses, their terms' size, dz, its terms' size)."""

    z = logits.detach().cpu().double()
    shape, vocab = z.shape[:-1], z.shape[-1]
    k = tokens.shape[-1]
    z, tokens, v = z.reshape(-1, vocab), tokens.cpu().long().reshape(-1, k), values.cpu().double().reshape(-1, k)
    weight = weight.cpu().double().reshape(-1)
    losses, sizes = torch.zeros(len(z), dtype=torch.float64), torch.zeros(len(z), dtype=torch.float64)
    dz, dz_size = torch.zeros_like(z), torch.zeros_like(z)
    for r in range(len(z)):
        there = tokens[r] >= 0
        at, u = tokens[r][there], v[r][there]
        if len(at) == 0 or (not tail and bool((u == -math.inf).all())):
            continue
        if bool((z[r] == -math.inf).all()):
            losses[r] = math.inf
            continue
        lnp = torch.log_softmax(z[r] / temperature, 0)
        p = lnp.exp()
        ln_q = u if tail else torch.log_softmax(u, 0)
        q = ln_q.exp()
        terms = torch.where(q == 0, 0.0, q * (ln_q - lnp[at]))
        loss, size = terms.sum(), (q * (1 + (ln_q - lnp[at]).abs())).nan_to_num(nan=0.0, posinf=0.0).sum()
        teacher = torch.zeros_like(p).index_add_(0, at, q)
        listed = torch.zeros(vocab, dtype=torch.bool)
        listed[at] = True
        rest, p_rest = 0.0, 1.0
        if tail:
            p_rest = float(p[~listed].sum())
            rest = max(0.0, 1.0 - float(q.sum())) if p_rest > 0 else 0.0
            if rest > 0:
                loss = loss + rest * (math.log(rest) - math.log(p_rest))
                size = size + rest * (1 + abs(math.log(rest) - math.log(p_rest))) + 1
        s, ratio = float(q.sum()) + rest, rest / p_rest if rest > 0 else 0.0
        slope = torch.full_like(p, s - ratio)
        slope[listed] = s
        losses[r], sizes[r] = loss * temperature ** 2, size * temperature ** 2
        if weight[r] != 0:
            dz[r] = weight[r] * temperature * (p * slope - teacher)
            dz_size[r] = weight[r].abs() * temperature * (p * (s + ratio) + teacher)
    return (losses.reshape(shape), sizes.reshape(shape), dz.reshape(*shape, vocab), dz_size.reshape(*shape, vocab))


def near(got, want, bound, what=""):
    got, want = got.detach().cpu().double(), want.float().double()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    same = (got == want) | (got.isnan() & want.isnan())
    off = torch.where(same, 0.0, (got - want).abs()).nan_to_num(nan=math.inf)
    bound = torch.as_tensor(bound).double().nan_to_num(nan=0.0, posinf=0.0)
    assert bool((off <= bound).all()), (what, float(off.max()), float((off - bound).max()))


def check(logits, tokens, values, temperature=1.0, tail=False, weight=None):
    """Both forms against the definition; returns what they gave."""

    import qste_amd as qste

    dtype = logits.dtype
    if weight is None:
        g = torch.Generator(device=DEV).manual_seed(logits.shape[-1])
        weight = torch.randn(logits.shape[:-1], generator=g, device=DEV)
    want, size, dz, dz_size = distilled(logits, tokens, values, weight, temperature, tail)
    x = logits.detach().requires_grad_(True)
    losses = qste.nn.distillation_loss(x, tokens, values, temperature=temperature, tail=tail)
    grad, = torch.autograd.grad(losses, x, weight)
    assert losses.dtype == torch.float32 and grad.dtype == dtype and grad.is_contiguous()
    bound = ROUND[dtype] * dz.abs() + LOG * dz_size + LEAST[dtype]
    near(losses, want, LOG * size, "losses")
    near(grad, dz, bound, "grad")
    alone, once = qste.nn.distillation_loss_and_grad(logits.detach(), tokens, values, loss_grad=weight,
                                                     temperature=temperature, tail=tail)
    near(alone, want, LOG * size, "losses of the one pass")
    near(once, dz, bound, "grad of the one pass")
    assert not alone.requires_grad and once.dtype == dtype
    with torch.no_grad():
        plain = qste.nn.distillation_loss(logits, tokens, values, temperature=temperature, tail=tail)
    assert torch.equal(plain.isnan(), losses.isnan())
    return losses.detach(), grad


def random_logits(shape, dtype, seed, spread=2.5):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randn(shape, generator=g, device=DEV) * spread).to(dtype)


def random_teacher(shape, vocab, k, seed, mass=0.9):
    """k different tokens a row, their log probabilities in falling order, summing to ``mass``."""

    g = torch.Generator(device=DEV).manual_seed(seed + 1)
    first = torch.randint(vocab, (*shape, 1), generator=g, device=DEV)
    tokens = (first + torch.arange(k, device=DEV) * max(1, vocab // k)) % vocab
    values = torch.log_softmax(torch.randn(*shape, k, generator=g, device=DEV) * 1.5, -1).sort(-1, descending=True).values
    return tokens, values + math.log(mass)


SIZES = [(1, 2, 1), (3, 5, 2), (2, 8, 4), (3, 9, 3), (3, 64, 8), (2, 513, 20), (3, 1000, 1), (3, 2053, 64), (2, 4104, 128),
         (2, 16391, 100), (2, 50257, 64), (1, 65536, 513), (1, 131072, 1024), (1, 131079, 32), (1, 300007, 64)]


@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,vocab,k", SIZES)
def test_losses_and_gradients(rows, vocab, k, dtype, tail):
    print(f"distill {rows} x {vocab}, {k} entries, {dtype}, tail {tail}", flush=True)
    tokens, values = random_teacher((rows,), vocab, k, vocab)
    check(random_logits((rows, vocab), dtype, vocab), tokens, values, tail=tail)


@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("temperature", [0.5, 2.0, 8.0])
def test_temperatures(temperature, tail):
    tokens, values = random_teacher((4,), 3001, 32, 1)
    for dtype in DTYPES:
        check(random_logits((4, 3001), dtype, 2), tokens, values, temperature=temperature, tail=tail)


@pytest.mark.parametrize("rows", [1, 2, 3, 17, 255, 256, 257, 700])
def test_row_counts(rows):
    print(f"rows {rows}", flush=True)
    tokens, values = random_teacher((rows,), 2011, 16, rows)
    check(random_logits((rows, 2011), torch.bfloat16, rows), tokens, values, tail=True)


@pytest.mark.parametrize("tail", [False, True])
def test_ragged_entries(tail):
    """Rows with fewer entries, with none, with entries of no mass, and repeated tokens."""

    vocab, k = 4099, 40
    logits = random_logits((8, vocab), torch.float32, 3)
    tokens, values = random_teacher((8,), vocab, k, 3)
    tokens[0, 5:] = -1
    tokens[1] = -1
    tokens[2, ::2] = -7
    values[3, 10:] = -math.inf
    values[4] = -math.inf
    tokens[5, 20:] = tokens[5, :20]
    tokens[6] = 11
    tokens[7, 1:] = -1
    values[1] = math.nan  # of no entry
    losses, grad = check(logits, tokens, values, tail=tail)
    assert losses[1] == 0 and not grad[1].any()
    logits[1] = math.nan  # a row without entries is not read
    losses, grad = check(logits, tokens, values, tail=tail)
    assert losses[1] == 0 and not grad[1].any()
    check(logits.to(torch.bfloat16), tokens.to(torch.int32), values, tail=tail)


@pytest.mark.parametrize("dtype", DTYPES)
def test_a_student_sure_of_the_list(dtype):
    """A tail of little mass is summed, not taken as 1 less the rest."""

    vocab, k = 20011, 16
    logits = random_logits((3, vocab), dtype, 4, 1.0)
    tokens, values = random_teacher((3,), vocab, k, 4, mass=0.999)
    logits.scatter_(1, tokens, 24.0)  # the rest holds about 20000 e^-23.5 / 16 = 8e-8
    check(logits, tokens, values, tail=True)


def test_tails_that_vanish():
    """Down to 2^-100 of the mass the tail counts; below, it is left out."""

    vocab, k = 5003, 8
    tokens, values = random_teacher((3,), vocab, k, 15)
    logits = random_logits((3, vocab), torch.float32, 15, 1.0)
    rest = torch.ones(3, vocab, dtype=torch.bool, device=DEV).scatter_(1, tokens, False)
    logits[0, rest[0]] -= 60.0  # 5000 e^-60 = 2^-74
    logits[1, rest[1]] -= 85.0  # 2^-110
    logits[2, rest[2]] -= 1e4
    check(logits[:1], tokens[:1], values[:1], tail=True)
    import qste_amd as qste

    inside = values[1:] - values[1:].logsumexp(1, keepdim=True)
    for r in (1, 2):
        losses, grad = qste.nn.distillation_loss_and_grad(logits[r:r + 1], tokens[r:r + 1], values[r:r + 1], tail=True)
        # over the list alone the teacher is its mass times the same one renormalised
        mass = float(values[r].double().exp().sum())
        alone, _, _, _ = distilled(logits[r:r + 1], tokens[r:r + 1], inside[r - 1:r], torch.ones(1))
        assert abs(float(losses) - mass * (float(alone) + math.log(mass))) < 1e-4
        assert grad.isfinite().all() and float(grad[0, rest[r]].abs().max()) < 1e-30


@pytest.mark.parametrize("tail", [False, True])
def test_masked_students(tail):
    vocab, k = 1500, 12
    logits = random_logits((6, vocab), torch.float32, 5)
    tokens, values = random_teacher((6,), vocab, k, 5)
    keep = torch.zeros(6, vocab, dtype=torch.bool, device=DEV).scatter_(1, tokens, True)
    logits[0].masked_fill_(~keep[0], -math.inf)  # no mass outside the list: no tail term
    logits[1].masked_fill_(keep[1], -math.inf)  # none in it: an infinite loss, a finite gradient
    logits[2] = -math.inf
    logits[3] = torch.finfo(torch.float32).min
    logits[4, ::2] = torch.finfo(torch.float32).min
    logits[5, tokens[5, 0]] = -math.inf
    values[5, 0] = -math.inf  # the teacher has none there either
    losses, grad = check(logits, tokens, values, tail=tail)
    assert losses[1] == math.inf and grad[1].isfinite().all() and losses[2] == math.inf and not grad[2].any()
    assert losses[[0, 3, 5]].isfinite().all()


@pytest.mark.parametrize("tail", [False, True])
def test_nan_infinity_and_tokens_outside(tail):
    import qste_amd as qste

    vocab, k = 999, 6
    logits = random_logits((5, vocab), torch.bfloat16, 6)
    tokens, values = random_teacher((5,), vocab, k, 6)
    logits[0, 500] = math.nan
    logits[1, 500] = math.inf
    tokens[2, 3] = vocab
    values[3, 2] = math.nan
    weight = torch.ones(5, device=DEV)
    x = logits.clone().requires_grad_(True)
    losses = qste.nn.distillation_loss(x, tokens, values, tail=tail)
    grad, = torch.autograd.grad(losses, x, weight)
    alone, once = qste.nn.distillation_loss_and_grad(logits, tokens, values, tail=tail)
    for lo, gr in ((losses, grad), (alone, once)):
        assert lo[:4].isnan().all() and lo[4].isfinite()
        assert gr[:3].isnan().all() and gr[4].isfinite().all()
    # positions of weight 0 get zeros whatever they hold
    weight[:4] = 0
    grad, = torch.autograd.grad(qste.nn.distillation_loss(x, tokens, values, tail=tail), x, weight)
    _, once = qste.nn.distillation_loss_and_grad(logits, tokens, values, loss_grad=weight, tail=tail)
    assert not grad[:4].any() and not once[:4].any() and grad[4].any() and once[4].any()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tail", [False, True])
def test_layouts(dtype, tail):
    base = random_logits((3, 6, 1013), dtype, 7)
    tokens, values = random_teacher((3, 5), 900, 9, 7)
    check(base[:, :-1, :900], tokens, values, tail=tail)
    check(base[:, 1:, 113:], tokens, values, tail=tail)
    tokens, values = random_teacher((6, 3), 1012, 9, 8)
    check(base.transpose(0, 1)[:, :, 1:], tokens, values, tail=tail)
    check(base[:, :, ::2].transpose(0, 1), tokens % 507, values, tail=tail)
    check(base.transpose(0, 1), tokens.transpose(0, 1).contiguous().transpose(0, 1), values.to(torch.bfloat16), tail=tail)
    tokens, values = random_teacher((), 1013, 9, 9)
    check(base[0, 0], tokens, values, tail=tail)


def test_broadcast_weights():
    """A mean's gradient is one number for every position."""

    import qste_amd as qste

    logits = random_logits((2, 5, 777), torch.float32, 10).requires_grad_(True)
    tokens, values = random_teacher((2, 5), 777, 7, 10)
    qste.nn.distillation_loss(logits, tokens, values, tail=True).mean().backward()
    _, _, dz, size = distilled(logits, tokens, values, torch.full((2, 5), 0.1), tail=True)
    near(logits.grad, dz, LOG * size + 2.0 ** -23 * dz.abs())
    for weight in (0.1, torch.tensor(0.1, device=DEV), torch.full((5,), 0.1, device=DEV), torch.full((2, 1), 0.1, device=DEV)):
        _, grad = qste.nn.distillation_loss_and_grad(logits.detach(), tokens, values, loss_grad=weight, tail=True)
        near(grad, dz, LOG * size + 2.0 ** -23 * dz.abs())


@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("dtype,rows,vocab", [(torch.bfloat16, 1, 1_700_003), (torch.float32, 2, 900_001),
                                              (torch.float16, 300, 32776), (torch.bfloat16, 60, 51200),
                                              (torch.bfloat16, 60, 51208), (torch.bfloat16, 40, 102407),
                                              (torch.bfloat16, 160, 131079), (torch.float32, 170, 65537),
                                              (torch.float16, 165, 110001), (torch.bfloat16, 170, 131080)])
def test_long_rows(dtype, rows, vocab, tail):
    """Past what registers hold in one workgroup, and past what they hold in parts."""

    print(f"long {rows} x {vocab} {dtype}", flush=True)
    tokens, values = random_teacher((rows,), vocab, 40, 16)
    tokens[-1, 20:] = -1
    check(random_logits((rows, vocab), dtype, 16), tokens, values, tail=tail)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,vocab,k", [(5, 90, 90), (5, 2053, 1024), (4, 12291, 300), (4, 20013, 200), (3, 45003, 1024),
                                          (2, 131075, 1024), (161, 120003, 1024), (1, 530003, 600)])
def test_lists_at_the_ends(rows, vocab, k, dtype):
    """Entries side by side at a row's first and last columns, in every run's place and
    beside the runs; the widest lists on each way that a row is held."""

    print(f"ends {rows} x {vocab}, {k} entries, {dtype}", flush=True)
    _, values = random_teacher((rows,), vocab, k, 17)
    g = torch.Generator().manual_seed(vocab)
    ends = torch.cat([torch.arange(k // 2), torch.arange(vocab - (k + 1) // 2, vocab)])
    tokens = torch.stack([ends[torch.randperm(k, generator=g)] for _ in range(rows)])
    tokens[0, :k // 3] = -1
    # with all of a vocabulary listed there is no tail
    check(random_logits((rows, vocab), dtype, 17), tokens.to(DEV), values, tail=k < vocab)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,bytes_a_row", [(512, 32784), (512, 64006), (513, 64006), (513, 102400), (512, 131086),
                                              (513, 131086), (512, 131088)])
def test_rows_around_the_wide_workgroups(rows, bytes_a_row, dtype):
    """Both sides of what a workgroup of more threads takes: by the number of rows, and by their length."""

    vocab = bytes_a_row // dtype.itemsize
    print(f"wide {rows} x {vocab} {dtype}", flush=True)
    tokens, values = random_teacher((rows,), vocab, 50, 18)
    tokens[3, 10:] = -1
    tokens[4] = -1
    logits = random_logits((rows, vocab), dtype, 18)
    logits[5, 1000:] = -math.inf
    check(logits, tokens, values, tail=rows % 2 == 0)


def test_rows_far_apart():
    """Offsets past 32 bits in the logits and in the gradient."""

    import qste_amd as qste

    stride, vocab = (1 << 31) + 777, 4099
    buffer = torch.empty(stride + vocab, dtype=torch.bfloat16, device=DEV)
    logits = buffer.as_strided((2, vocab), (stride, 1))
    logits.copy_(random_logits((2, vocab), torch.bfloat16, 8))
    tokens, values = random_teacher((2,), vocab, 30, 8)
    check(logits, tokens, values, tail=True)
    del buffer, logits
    rows, vocab = 33000, 131072  # 2^32 elements; the last rows against the same rows alone
    row = random_logits((3, vocab), torch.bfloat16, 9)
    tokens, values = random_teacher((3,), vocab, 8, 9)
    many = torch.empty(rows, vocab, dtype=torch.bfloat16, device=DEV)
    many.view(rows // 3, 3, vocab).copy_(row)
    losses, grad = qste.nn.distillation_loss_and_grad(many, tokens.repeat(rows // 3, 1), values.repeat(rows // 3, 1))
    alone, once = qste.nn.distillation_loss_and_grad(row, tokens, values)
    near(losses[-3:], alone.cpu().double(), 1e-5)
    near(grad[-3:].float(), once.cpu().double(), 2.0 ** -8 * once.abs().cpu().double() + 1e-6)


def test_gradient_against_differences():
    """Central differences of the kernel's own forward (as for the token scores: 2e-4 from the values' rounding, 5e-4
    from the step, times T^2 = 1.7)."""

    import qste_amd as qste

    z = random_logits((6, 37), torch.float32, 9, 1.0)
    tokens, values = random_teacher((6,), 37, 5, 9)
    v = random_logits((6, 37), torch.float32, 10, 1.0).clamp(-2.5, 2.5)
    for tail in (False, True):
        def f(x):
            return qste.nn.distillation_loss(x, tokens, values, temperature=1.3, tail=tail)

        x = z.clone().requires_grad_(True)
        f(x).sum().backward()
        slope = (f(z + 1e-2 * v) - f(z - 1e-2 * v)) / 2e-2
        assert float((slope - (x.grad * v).sum(1)).abs().max()) < 4e-3


def test_scores_of_a_teacher_are_targets():
    """token_logprobs lists what distillation_loss takes: a student equal to the teacher has no loss and no gradient; unscored
    positions of the teacher are positions without entries."""

    import qste_amd as qste

    logits = random_logits((7, 5003), torch.float32, 12)
    marks = torch.zeros(7, dtype=torch.long, device=DEV)
    marks[3] = -1
    for temperature in (1.0, 2.0):
        s = qste.nn.token_logprobs(logits, marks, top=50, temperature=temperature)
        x = logits.clone().requires_grad_(True)
        losses = qste.nn.distillation_loss(x, s.top_tokens, s.top_logprobs, temperature=temperature, tail=True)
        losses.sum().backward()
        assert losses[3] == 0 and not x.grad[3].any()
        assert float(losses.abs().max()) < 8 * LOG and float(x.grad.abs().max()) < 8 * LOG


def test_same_bits_every_time_on_any_stream():
    import qste_amd as qste

    logits = random_logits((40, 50257), torch.bfloat16, 6).requires_grad_(True)
    tokens, values = random_teacher((40,), 50257, 64, 6)
    tokens[:, 40:] = tokens[:, :24]  # repeated ones too

    def run():
        losses = qste.nn.distillation_loss(logits, tokens, values, tail=True)
        grad, = torch.autograd.grad(losses.sum(), logits)
        return [losses.detach(), grad, *qste.nn.distillation_loss_and_grad(logits.detach(), tokens, values, tail=True)]

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

    logits = random_logits((5, 9001), torch.bfloat16, 1)
    tokens, values = random_teacher((5,), 9001, 20, 1)
    weight = torch.ones(5, device=DEV)

    def run():
        x = logits.detach().requires_grad_(True)
        losses = qste.nn.distillation_loss(x, tokens, values, tail=True)
        grad, = torch.autograd.grad(losses, x, weight)
        return [losses, grad, *qste.nn.distillation_loss_and_grad(logits, tokens, values, loss_grad=weight)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run()
    for seed in range(4):
        logits.copy_(random_logits((5, 9001), torch.bfloat16, 20 + seed))
        weight.fill_(1.0 + seed)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, run()))


def test_empty():
    import qste_amd as qste

    losses, grad = qste.nn.distillation_loss_and_grad(
        torch.empty(0, 100, device=DEV), torch.empty(0, 4, dtype=torch.long, device=DEV), torch.empty(0, 4, device=DEV))
    assert losses.shape == (0,) and grad.shape == (0, 100)


def test_refusals():
    import qste_amd as qste

    logits = torch.zeros(4, 100, device=DEV)
    tokens = torch.zeros(4, 3, dtype=torch.long, device=DEV)
    values = torch.zeros(4, 3, device=DEV)
    for f in (qste.nn.distillation_loss, qste.nn.distillation_loss_and_grad):
        with pytest.raises(ValueError, match="top_tokens"):
            f(logits, tokens[:3], values)
        with pytest.raises(ValueError, match="top_logprobs"):
            f(logits, tokens, values[:, :2])
        with pytest.raises(ValueError, match="entries"):
            f(logits, tokens[:, :0], values[:, :0])
        with pytest.raises(ValueError, match="entries"):
            f(logits, tokens.repeat(1, 400), values.repeat(1, 400))
        with pytest.raises(ValueError, match="entries"):
            f(logits, tokens[0], values[0])
        with pytest.raises(TypeError, match="integers"):
            f(logits, tokens.float(), values)
        with pytest.raises(TypeError, match="floating"):
            f(logits, tokens, tokens)
        with pytest.raises(TypeError, match="unsupported dtype"):
            f(logits.double(), tokens, values)
        with pytest.raises(ValueError, match="temperature"):
            f(logits, tokens, values, temperature=0.0)
        with pytest.raises(ValueError, match="detach"):
            f(logits, tokens, values.clone().requires_grad_(True))
        with pytest.raises(RuntimeError, match="GPU only"):
            f(logits.cpu(), tokens.cpu(), values.cpu())
    with pytest.raises(RuntimeError):
        qste.nn.distillation_loss_and_grad(logits, tokens, values, loss_grad=torch.ones(3, device=DEV))
    with pytest.raises(RuntimeError, match="GPU only"):
        qste.nn.distillation_loss_and_grad(logits, tokens, values, loss_grad=torch.ones(4))
