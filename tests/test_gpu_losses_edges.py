"""Token scores and distillation at the ends of what they accept.

Bounds as in test_gpu_scores.py and test_gpu_distill.py: a log probability is within LOG = 4e-5 (the sums' chain of
additions) and 1e-6 of itself (its three roundings).
"""

from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda"
LOG = 4e-5
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


@pytest.fixture(autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    from qste_amd import kernels

    assert kernels.native_available(), kernels.status()


def near(got, want, bound):
    got, want = got.detach().cpu().double(), want.cpu().double()
    assert got.shape == want.shape
    same = (got == want) | (got.isnan() & want.isnan())
    off = torch.where(same, 0.0, (got - want).abs()).nan_to_num(nan=math.inf)
    bound = torch.as_tensor(bound).double().cpu().nan_to_num(nan=0.0, posinf=0.0)
    assert bool((off <= bound).all()), (float(off.max()), float((off - bound).max()))


# ---------------------------------------------------------------------------
# a token past the vocabulary
# ---------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("weighted", [False, True])
def test_entropy_gradient_beside_a_token_outside(weighted, dtype):
    """The entropy does not depend on the token: its gradient is the formula's, unless a NaN log probability has a
    weight."""

    import qste_amd as qste

    vocab = 3001
    g = torch.Generator(device=DEV).manual_seed(5)
    logits = (torch.randn(3, vocab, generator=g, device=DEV) * 2).to(dtype).requires_grad_(True)
    tokens = torch.tensor([7, vocab, 1 << 40], device=DEV)
    s = qste.nn.token_logprobs(logits, tokens)
    h = torch.tensor([0.5, -1.0, 2.0], device=DEV)
    if weighted:
        grad, = torch.autograd.grad((s.logprobs, s.entropy), logits, (torch.zeros(3, device=DEV), h))
    else:
        grad, = torch.autograd.grad(s.entropy, logits, h)
    lnp = torch.log_softmax(logits.detach().cpu().double(), 1)
    p = lnp.exp()
    entropy = -(p * lnp).sum(1, keepdim=True)
    want = -h.cpu().double()[:, None] * p * (lnp + entropy)
    size = h.cpu().double().abs()[:, None] * p * (lnp.abs() + entropy)
    rounding = {torch.float32: 2.0 ** -23, torch.float16: 2.0 ** -10, torch.bfloat16: 2.0 ** -8}[dtype]
    near(grad, want, rounding * want.abs() + LOG * size + (2.0 ** -24 if dtype == torch.float16 else 1e-37))
    s = qste.nn.token_logprobs(logits, tokens)
    grad, = torch.autograd.grad(s.logprobs, logits, torch.tensor([1.0, 0.0, 1.0], device=DEV))
    assert grad[0].isfinite().all() and not grad[1].any() and grad[2].isnan().all()


# ---------------------------------------------------------------------------
# logits further apart than fp32's largest number
# ---------------------------------------------------------------------------


def far_apart(vocab, dtype):
    """Three rows of logits, two tokens of each further below its largest than fp32 reaches."""

    logits = torch.full((3, vocab), -1e38, device=DEV)
    logits[0, 3] = 3e38
    logits[1, 2:6] = 3.3e38
    logits[1, 8] = -3.3e38
    logits[2, 0] = torch.finfo(dtype).max
    logits[2, 7] = torch.finfo(dtype).min
    return logits.to(dtype), torch.tensor([[4, 5], [8, 0], [7, 8]], device=DEV)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("temperature", [2.5, 50.0, 1e20])
@pytest.mark.parametrize("vocab", [9, 5000, 60000, 150001])
def test_log_probabilities_of_differences_past_fp32(vocab, temperature, dtype):
    """Finite at a temperature that brings the differences back."""

    import qste_amd as qste

    logits, tokens = far_apart(vocab, dtype)
    z = logits.cpu().double()
    lnp = torch.log_softmax(z / temperature, 1)
    got = qste.nn.token_logprobs(logits, tokens[:, 0], top=9, temperature=temperature)
    want = lnp.gather(1, tokens.cpu())[:, 0]
    assert got.logprobs.isfinite().all()
    near(got.logprobs, want, LOG + 1e-6 * want.abs())
    places = torch.sort(z, dim=1, descending=True, stable=True).indices[:, :9]
    assert torch.equal(got.top_tokens.cpu(), places)
    want = lnp.gather(1, places)
    near(got.top_logprobs, want, LOG + 1e-6 * want.abs())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("temperature", [0.01, 0.25, 50.0])
@pytest.mark.parametrize("vocab", [9, 5000, 60000, 150001])
def test_losses_of_differences_past_fp32(vocab, temperature, dtype):
    """About temperature times a difference: finite where that fits, though the log probabilities in it do not."""

    import qste_amd as qste

    logits, tokens = far_apart(vocab, dtype)
    values = torch.tensor([0.75, 0.25], device=DEV).log().expand(3, 2)
    lnp = torch.log_softmax(logits.cpu().double() / temperature, 1).gather(1, tokens.cpu())
    q = torch.tensor([0.75, 0.25]).double()
    want = temperature ** 2 * (q * (q.log() - lnp)).sum(1)
    want = torch.where(want > torch.finfo(torch.float32).max, math.inf, want)
    assert want.isfinite().all() if temperature < 1 else want.isinf().all()
    losses, grad = qste.nn.distillation_loss_and_grad(logits, tokens, values, temperature=temperature)
    near(losses, want, 2e-6 * want)
    near(qste.nn.distillation_loss(logits, tokens, values, temperature=temperature), want, 2e-6 * want)
    assert grad.isfinite().all()


# ---------------------------------------------------------------------------
# a student and a list without mass
# ---------------------------------------------------------------------------


@pytest.mark.parametrize("vocab", [700, 60000, 150001])
def test_a_masked_student_against_a_list_without_mass(vocab):
    """With the tail all of the teacher's mass is outside the list: entries there are, and a row of only -inf has an
    infinite loss as with any others; without the tail it is a row without entries of mass."""

    import qste_amd as qste

    logits = torch.full((3, vocab), -math.inf, device=DEV)
    logits[2] = 0.0
    tokens = torch.tensor([[4, 5], [-1, -1], [4, 5]], device=DEV)
    values = torch.full((3, 2), -math.inf, device=DEV)
    for tail, first in ((True, math.inf), (False, 0.0)):
        losses, grad = qste.nn.distillation_loss_and_grad(logits, tokens, values, tail=tail)
        alone = qste.nn.distillation_loss(logits, tokens, values, tail=tail)
        for got in (losses, alone):
            assert got[0] == first and got[1] == 0
            # a flat student has all but 2 / vocab of its mass outside the list
            near(got[2:], torch.tensor([-math.log1p(-2 / vocab) if tail else 0.0]), LOG)
        assert not grad[:2].any() and grad.isfinite().all()


# ---------------------------------------------------------------------------
# more rows than one launch has workgroups for (2^32 threads of 256 a row)
# ---------------------------------------------------------------------------


def repeated(rows, want, got):
    """Every ``len(want)`` rows of ``got`` are ``want``."""

    n = len(want)
    whole = rows // n * n
    assert torch.equal(got[:whole].view(rows // n, n, *want.shape[1:]), want.expand(rows // n, *want.shape))
    assert torch.equal(got[whole:], want[: rows - whole])


@pytest.mark.parametrize("rows", [(1 << 24) - 1, 1 << 24, (1 << 24) + 21])
def test_scores_of_many_rows(rows):
    """Every row as the same ones alone, in both directions."""

    import qste_amd as qste

    n, vocab = 11, 8
    g = torch.Generator(device=DEV).manual_seed(1)
    base = torch.randn(n, vocab, generator=g, device=DEV, dtype=torch.bfloat16)
    marks = torch.randint(-1, vocab, (n,), generator=g, device=DEV)
    logits = base.repeat(-(-rows // n), 1)[:rows].requires_grad_(True)
    tokens = marks.repeat(-(-rows // n))[:rows]
    print(f"scores of {rows} rows", flush=True)
    few = base.clone().requires_grad_(True)
    want, got = (qste.nn.token_logprobs(x, t, top=2) for x, t in ((few, marks), (logits, tokens)))
    for a, b in zip(want, got):
        repeated(rows, a.detach(), b.detach())
    ones = torch.ones(rows, device=DEV)
    want, = torch.autograd.grad((want.logprobs, want.entropy), few, (ones[:n], ones[:n]))
    got, = torch.autograd.grad((got.logprobs, got.entropy), logits, (ones, ones))
    repeated(rows, want, got)


@pytest.mark.parametrize("rows", [(1 << 24) - 1, 1 << 24, (1 << 24) + 21])
def test_distillation_of_many_rows(rows):
    import qste_amd as qste

    n, vocab = 11, 8
    g = torch.Generator(device=DEV).manual_seed(2)
    base = torch.randn(n, vocab, generator=g, device=DEV, dtype=torch.bfloat16)
    entries = torch.stack([torch.arange(n, device=DEV) % 5, torch.arange(n, device=DEV) % 3 + 5], 1)
    entries[4] = -1
    values = torch.log_softmax(torch.randn(n, 2, generator=g, device=DEV), 1) - 0.1
    logits = base.repeat(-(-rows // n), 1)[:rows].requires_grad_(True)
    tokens, mass = (t.repeat(-(-rows // n), 1)[:rows] for t in (entries, values))
    print(f"distillation of {rows} rows", flush=True)
    few = base.clone().requires_grad_(True)
    want = qste.nn.distillation_loss(few, entries, values, tail=True)
    got = qste.nn.distillation_loss(logits, tokens, mass, tail=True)
    repeated(rows, want.detach(), got.detach())
    ones = torch.ones(rows, device=DEV)
    a, = torch.autograd.grad(want, few, ones[:n])
    b, = torch.autograd.grad(got, logits, ones)
    repeated(rows, a, b)
    losses, grad = qste.nn.distillation_loss_and_grad(logits.detach(), tokens, mass, tail=True)
    # a row's sums are ordered by where its gradient lies in a line of 128 bytes: as alone in the same eight places
    want, a = qste.nn.distillation_loss_and_grad(*(t.repeat(8, 1) for t in (base, entries, values)), tail=True)
    repeated(rows, want, losses)
    repeated(rows, a, grad)


def test_many_rows_in_parts():
    """Two parts a row, one physical row read for all: the parts pass the limit before the rows do."""

    import qste_amd as qste

    rows, vocab = (1 << 23) + 5, 51208
    g = torch.Generator(device=DEV).manual_seed(3)
    row = torch.randn(vocab, generator=g, device=DEV, dtype=torch.bfloat16)
    tokens = torch.arange(rows, device=DEV) % 997 - 1
    print(f"parts of {rows} rows", flush=True)
    want = qste.nn.token_logprobs(row.expand(997 + 512, vocab), tokens[: 997 + 512], top=1)
    got = qste.nn.token_logprobs(row.expand(rows, vocab), tokens, top=1)
    for a, b in zip(want, got):
        repeated(rows, a[:997], b)
    values = torch.zeros(rows, 1, device=DEV)
    want = qste.nn.distillation_loss(row.expand(997 + 512, vocab), tokens[: 997 + 512, None], values[: 997 + 512])
    got = qste.nn.distillation_loss(row.expand(rows, vocab), tokens[:, None], values)
    repeated(rows, want[:997], got)
