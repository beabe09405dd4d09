"""Token scores and distillation have no forward-mode derivatives: a tangent is refused, never dropped."""

from __future__ import annotations

import pytest
import torch
from torch.autograd import forward_ad

LOGITS, TOKENS, VALUES = torch.randn(3, 8), torch.zeros(3, 2, dtype=torch.long), torch.randn(3, 2)


@pytest.fixture
def called(monkeypatch):
    """The kernels' calls replaced: what arrives there has lost its tangent."""

    from qste_amd import kernels

    calls = []

    def scores(logits, *_, **__):
        calls.append("scores")
        return None, logits.new_zeros(logits.shape[:-1]), None, None, None

    def distill(logits, *_, **__):
        calls.append("distill")
        return logits.new_zeros(logits.shape[:-1]), None, logits

    monkeypatch.setattr(kernels, "token_logprobs_forward", scores)
    monkeypatch.setattr(kernels, "distill_forward", distill)
    return calls


def _calls(logits=LOGITS, values=VALUES, weight=1.0):
    import qste_amd as qste

    return {
        "token_logprobs": lambda: qste.nn.token_logprobs(logits),
        "distillation_loss": lambda: qste.nn.distillation_loss(logits, TOKENS, values),
        "distillation_loss_and_grad": lambda: qste.nn.distillation_loss_and_grad(logits, TOKENS, values,
                                                                                 loss_grad=weight),
    }


def _dual(t):
    return forward_ad.make_dual(t, torch.ones_like(t))


@pytest.mark.parametrize("grad_mode", [True, False])
@pytest.mark.parametrize("name,what", [("token_logprobs", "logits"), ("distillation_loss", "logits"),
                                       ("distillation_loss", "values"), ("distillation_loss_and_grad", "logits"),
                                       ("distillation_loss_and_grad", "values"),
                                       ("distillation_loss_and_grad", "weight")])
def test_a_tangent_is_refused(name, what, grad_mode, called):
    with forward_ad.dual_level(), torch.set_grad_enabled(grad_mode):
        dual = _dual({"logits": LOGITS, "values": VALUES, "weight": torch.ones(3)}[what])
        with pytest.raises(NotImplementedError, match="forward-mode"):
            _calls(**{what: dual})[name]()
    assert not called


@pytest.mark.parametrize("what", ["logits", "values", "weight"])
def test_a_tangent_beside_a_gradient_is_refused(what, called):
    with forward_ad.dual_level():
        args = {"logits": LOGITS.clone().requires_grad_(True), "values": VALUES, "weight": torch.ones(3)}
        args[what] = _dual(args[what])
        for name, call in _calls(**args).items():
            if what == "logits" or (what == "values" and name != "token_logprobs") or name.endswith("_and_grad"):
                with pytest.raises(NotImplementedError, match="forward-mode"):
                    call()


def test_plain_tensors_are_taken_inside_a_dual_level(called):
    with forward_ad.dual_level():
        for call in _calls().values():
            call()
    for call in _calls(weight=torch.ones(3)).values():
        call()
    assert called == ["scores", "distill", "distill"] * 2
