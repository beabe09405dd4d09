"""Scoring tokens, and distilling a student from a teacher's top tokens.

Both work on a model's logits, ``[..., vocab]`` in fp32, fp16 or bf16 on the GPU,
in any layout whose columns are adjacent (``logits[:, :-1]`` is read in place).
Softmax, sums and losses are fp32; a gradient is rounded once, to the
logits' dtype.  Forward-mode differentiation is refused.  The kernels are
``csrc/scores.hip`` and ``csrc/distill.hip``; the reference ends at the logits and
has no counterparts.

    with torch.no_grad():                    # the teacher, and what it thinks likely
        scores = qste.nn.token_logprobs(teacher(ids), top=64)
    losses = qste.nn.distillation_loss(student(ids), scores.top_tokens, scores.top_logprobs, tail=True)
    losses.mean().backward()
"""

from __future__ import annotations

from typing import NamedTuple, Optional

import torch
from torch import Tensor
from torch.autograd import Function, forward_ad
from torch.autograd.function import once_differentiable

from . import kernels


class TokenScores(NamedTuple):
    """What ``token_logprobs`` returns; every field has the logits' leading shape."""

    logprobs: Optional[Tensor]  # ln p of the given tokens; None without tokens
    entropy: Tensor  # -sum p ln p, in nats
    top_logprobs: Optional[Tensor]  # [..., top]; None for top = 0
    top_tokens: Optional[Tensor]  # int64 [..., top]; None for top = 0


class TokenLogprobsFn(Function):
    """``token_logprobs`` with the logits' gradient; keeps the logits, their rows'
    maxima and sums, and the entropies."""

    @staticmethod
    def forward(ctx, logits, tokens, top, temperature):
        ctx.set_materialize_grads(False)
        checked = kernels._check_scores(logits, tokens, top, temperature)
        logprobs, entropy, top_logprobs, top_tokens, stats = kernels._call_scores(*checked, True)
        rows, ctx.layout, tokens_i64, _, ctx.temperature = checked
        ctx.save_for_backward(rows, tokens_i64, entropy, stats)
        if top_tokens is not None:
            ctx.mark_non_differentiable(top_logprobs, top_tokens)
        return logprobs, entropy, top_logprobs, top_tokens

    @staticmethod
    @once_differentiable
    def backward(ctx, logprob_grad, entropy_grad, *_):
        if logprob_grad is None and entropy_grad is None:
            return None, None, None, None
        rows, tokens, entropy, stats = ctx.saved_tensors
        g = None if logprob_grad is None else logprob_grad.contiguous()
        h = None if entropy_grad is None else entropy_grad.contiguous()
        return (kernels._call_scores_backward(rows, ctx.layout, tokens, ctx.temperature, g, h, entropy, stats),
                None, None, None)


def _no_tangent(what: str, *tensors: Tensor) -> None:
    """Refuses forward-mode differentiation.  A dual tensor need not have
    ``requires_grad``, so it can reach the kernels' calls, which would take its
    values and lose its tangent."""

    for t in tensors:
        if forward_ad.unpack_dual(t).tangent is not None:
            raise NotImplementedError(f"{what} has no forward-mode derivative")


def token_logprobs(logits: Tensor, tokens: Optional[Tensor] = None, *, top: int = 0,
                   temperature: float = 1.0) -> TokenScores:
    """Log probabilities of ``tokens`` under ``softmax(logits / temperature)``, each
    row's entropy, and its ``top`` likeliest tokens with their log probabilities.

    ``tokens`` are integers of the logits' leading shape, or None.  A negative
    token marks a position that is not scored (padding): logprob and entropy
    0, top tokens -1 with -inf, no gradient, its logits not read.  A token past
    the vocabulary gives a NaN log probability, and NaN where a gradient flows back
    through it.  Equal logits are listed by the lowest token; ``top`` is
    at most 128.  Differentiable in ``logprobs`` and ``entropy``; the top
    log probabilities carry no gradient.
    """

    _no_tangent("token_logprobs", logits)
    if torch.is_grad_enabled() and logits.requires_grad:
        return TokenScores(*TokenLogprobsFn.apply(logits, tokens, top, temperature))
    return TokenScores(*kernels.token_logprobs_forward(logits, tokens, top=top, temperature=temperature)[:4])


class DistillationFn(Function):
    """``distillation_loss`` with the logits' gradient; keeps the logits, the
    teacher's entries and six floats a row."""

    @staticmethod
    def forward(ctx, logits, top_tokens, top_logprobs, temperature, tail):
        checked = kernels._check_distill(logits, top_tokens, top_logprobs, temperature, tail)
        losses, stats, _ = kernels._call_distill(*checked, None, True)
        rows, ctx.layout, tokens_i64, values, ctx.temperature, ctx.tail = checked
        ctx.save_for_backward(rows, tokens_i64, values, stats)
        return losses

    @staticmethod
    @once_differentiable
    def backward(ctx, loss_grad):
        rows, tokens, values, stats = ctx.saved_tensors
        return (kernels._call_distill_backward(rows, ctx.layout, tokens, values, ctx.temperature, ctx.tail,
                                               loss_grad.contiguous(), stats), None, None, None, None)


def _constant(top_logprobs: Tensor) -> None:
    if torch.is_grad_enabled() and top_logprobs.requires_grad:
        raise ValueError("the teacher's log probabilities are constants here: detach them")


def distillation_loss(logits: Tensor, top_tokens: Tensor, top_logprobs: Tensor, *, temperature: float = 1.0,
                      tail: bool = False) -> Tensor:
    """Per position the divergence KL(teacher || student), times ``temperature ** 2``,
    of a teacher known by its top tokens; differentiable in ``logits``.

    ``top_tokens`` and ``top_logprobs`` ``[..., k]`` (k at most 1024) are what
    ``token_logprobs(teacher_logits, top=k, temperature=temperature)`` lists: log
    probabilities at the same temperature as the student's here.  Without
    ``tail`` the teacher is renormalised over its list (any logits, already over the
    temperature, will do); with it the mass that the list leaves is one more
    outcome, set against all the student's mass outside the list.  A negative
    token is no entry; a position with none has the loss 0 and no gradient.  A
    token listed twice has a term for each entry in the loss, and their sum as its
    probability in the gradient.
    """

    _no_tangent("distillation_loss", logits, top_logprobs)
    _constant(top_logprobs)
    if torch.is_grad_enabled() and logits.requires_grad:
        return DistillationFn.apply(logits, top_tokens, top_logprobs, temperature, tail)
    return kernels.distill_forward(logits, top_tokens, top_logprobs, temperature=temperature, tail=tail)[0]


def distillation_loss_and_grad(logits: Tensor, top_tokens: Tensor, top_logprobs: Tensor, *,
                               loss_grad: Tensor | float = 1.0, temperature: float = 1.0,
                               tail: bool = False) -> tuple[Tensor, Tensor]:
    """``distillation_loss`` and the logits' gradient for the weights ``loss_grad`` (a
    number, or a tensor that broadcasts to the losses' shape) from one pass
    over the logits, where the autograd form reads them twice::

        losses, grad = distillation_loss_and_grad(logits, top_tokens, top_logprobs, loss_grad=mask / mask.sum())
        logits.backward(grad)

    Positions of weight 0 get zeros, whatever their logits hold.  Neither result
    carries a graph, also where ``logits`` or ``loss_grad`` require gradients.
    """

    _no_tangent("distillation_loss_and_grad", logits, top_logprobs)
    _constant(top_logprobs)
    shape = logits.shape[:-1]
    if isinstance(loss_grad, Tensor):
        _no_tangent("distillation_loss_and_grad", loss_grad)
        weights = loss_grad if loss_grad.shape == shape else loss_grad.expand(shape)
    else:
        weights = torch.full(shape, float(loss_grad), dtype=torch.float32, device=logits.device)
    losses, _, grad = kernels.distill_forward(logits, top_tokens, top_logprobs, temperature=temperature, tail=tail,
                                              loss_grad=weights)
    return losses, grad
