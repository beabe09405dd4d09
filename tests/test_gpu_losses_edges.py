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
