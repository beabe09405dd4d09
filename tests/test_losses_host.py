"""Token scores and distillation without a GPU: what the C entry points refuse, and how rows of logits are laid out."""

from __future__ import annotations

import pytest
import torch


def _args(dtype=0, outer=1, inner=1, vocab=8, logits=16):
    return (logits, dtype, outer, inner, vocab, vocab, vocab)


def test_c_entry_points_refuse_before_any_launch():
    from qste_amd.kernels import _lib

    lib = _lib.load()
    assert b"temperature" in lib.qste_error_string(-8)

    def score(*logits, temperature=1.0, top=0, entropy=16):
        return lib.qste_token_logprobs(*logits, None, temperature, top, None, entropy, None, None, None, None, 0, None)

    def score_back(*logits, temperature=1.0, grad=16):
        return lib.qste_token_logprobs_backward(*logits, None, temperature, None, None, 16, 16, grad, None)

    def distill(*logits, temperature=1.0, k=4, losses=16):
        return lib.qste_distill(*logits, 16, 16, k, temperature, 0, losses, None, None, None, None, 0, None)

    def distill_back(*logits, temperature=1.0, k=4, grad=16):
        return lib.qste_distill_backward(*logits, 16, 16, k, temperature, 0, 16, 16, grad, None)

    for entry in (score, score_back, distill, distill_back):
        assert entry(*_args(dtype=3)) == -1
        assert entry(*_args(vocab=0)) == -2
        assert entry(*_args(vocab=(1 << 30) + 1)) == -2
        assert entry(*_args(outer=-1)) == -2
        assert entry(*_args(outer=1 << 20, inner=1 << 20)) == -2
        assert entry(*_args(logits=None)) == -3
        assert entry(*_args(logits=17)) == -6
        assert entry(*_args(dtype=0, logits=18)) == -6
        for temperature in (0.0, -1.0, float("inf"), float("nan")):
            assert entry(*_args(), temperature=temperature) == -8
        assert entry(*_args(outer=0)) == 0  # nothing to do
    assert score(*_args(), top=9) == -2 and score(*_args(vocab=500), top=129) == -2 and score(*_args(), top=-1) == -2
    assert score(*_args(), top=2) == -3 and score(*_args(), entropy=None) == -3
    assert score_back(*_args(), grad=None) == -3 and score_back(*_args(), grad=24) == -6
    for entry in (distill, distill_back):
        assert entry(*_args(), k=0) == -2 and entry(*_args(), k=1025) == -2
    assert distill(*_args(), losses=None) == -3
    assert distill_back(*_args(), grad=None) == -3 and distill_back(*_args(), grad=8) == -6


def _addresses(rows, layout):
    outer, inner, outer_stride, inner_stride, _ = layout
    start = rows.storage_offset()
    return [start + o * outer_stride + i * inner_stride for o in range(outer) for i in range(inner)]


@pytest.mark.parametrize("view", [
    lambda t: t, lambda t: t[:, :-1], lambda t: t[:, 1:, 2:], lambda t: t[1], lambda t: t[1, 2], lambda t: t[1:2, 2:3],
    lambda t: t.transpose(0, 1), lambda t: t[:, ::2], lambda t: t[0, 0].expand(5, 7), lambda t: t[:, :1].expand(3, 4, 7),
    lambda t: t.view(3, 2, 2, 7)[:, :, 1:], lambda t: t.view(3, 2, 2, 7).permute(1, 2, 0, 3), lambda t: t[..., :1],
])
def test_rows_of_views_are_read_in_place(view):
    from qste_amd.kernels import _logit_rows

    t = view(torch.arange(3 * 4 * 7, dtype=torch.float32).view(3, 4, 7))
    rows, layout = _logit_rows(t)
    assert rows.data_ptr() == t.data_ptr() and layout[4] == t.shape[-1]
    # arange: a row's first value is where it starts
    assert _addresses(rows, layout) == t[..., 0].reshape(-1).int().tolist()


def test_other_layouts_are_copied():
    from qste_amd.kernels import _logit_rows

    t = torch.arange(2 * 3 * 4 * 5, dtype=torch.float32).view(2, 3, 4, 5)
    for view in (t[:, 1:, 1:], t[..., ::2], t.transpose(2, 3)):
        rows, layout = _logit_rows(view)
        assert rows.is_contiguous() and torch.equal(rows, view)
        assert _addresses(rows, layout) == [i * view.shape[-1] for i in range(view[..., 0].numel())]
    empty, layout = _logit_rows(torch.empty(0, 3, 5))
    assert layout == (0, 0, 0, 0, 5)
    with pytest.raises(ValueError):
        _logit_rows(torch.tensor(1.0))
    with pytest.raises(ValueError):
        _logit_rows(torch.empty(3, 0))


def test_public_names():
    import qste_amd as qste

    for name in ("TokenScores", "token_logprobs", "distillation_loss", "distillation_loss_and_grad"):
        assert name in qste.nn.__all__ and hasattr(qste.nn, name)
