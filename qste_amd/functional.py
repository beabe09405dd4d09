"""Autograd for binary linear layers on the gfx950 kernels.

Forward (``QSTELinearFn``, reference ``src/qste/functional.py:153-171``):
``y = (x @ sign^T) * scale + bias`` and, for backward, the input kept as one
bit per element plus two floats per sample (``encode_activation``,
functional.py:98-115): ``x ~ offset + xscale * sign(x - offset)``.

Backward (functional.py:173-194) is one library call, ``linear_backward``:
the input gradient, the decoded evidence with its rank-one offset correction,
the scale gradient, the evidence times the row scale, and the bias gradient.
The evidence goes to the surface -- usually straight into the coordinate step,
inside ``loss.backward()``.
"""

from __future__ import annotations

import weakref

import torch
from torch import Tensor
from torch.autograd import Function
from torch.autograd.function import once_differentiable

from . import kernels
from .losses import _no_tangent
from .surface import Surface


def _autocast(value: Tensor) -> Tensor:
    """Cast like autocast would cast a native GEMM input (functional.py:39-53)."""

    device = value.device.type
    if device not in ("cuda", "cpu") or not torch.is_autocast_enabled(device):
        return value
    return value.to(dtype=torch.get_autocast_dtype(device))


def encode_activation(flat: Tensor) -> tuple[Tensor, Tensor]:
    """``(bits, aux)`` with ``aux = stack(offset, scale)`` fp32 [2, samples]."""

    packed, offset, scale = kernels.pack_affine_rows(flat)
    return packed, kernels.stacked_pair(offset, scale)


# Layers that read the same input in one forward (a SwiGLU's gate and up
# projections) share its encoding: the last input encoded, held weakly, with
# its version counter and address.  Any backward clears it, so a reuse never
# spans a training step; and it is of one graph capture, or of none: an encoding
# recorded into a graph has not run yet, and a graph that read one from before
# it would not follow its input.
_last_encoding: tuple | None = None


def _encoding_of(inputs: Tensor, flat: Tensor, columns: int) -> tuple[Tensor, Tensor]:
    global _last_encoding
    if inputs.is_inference():  # has no version to be remembered by
        return encode_activation(flat)
    key = (inputs._version, inputs.data_ptr(), tuple(inputs.shape), inputs.dtype, columns, kernels.capture_id(inputs))
    if _last_encoding is not None:
        ref, last_key, payload, aux = _last_encoding
        if ref() is inputs and last_key == key:
            return payload, aux
    payload, aux = encode_activation(flat)
    _last_encoding = (weakref.ref(inputs), key, payload, aux)
    return payload, aux


def forget_encodings() -> None:
    global _last_encoding
    _last_encoding = None


def remember_encoding(value: Tensor, payload: Tensor, aux: Tensor) -> None:
    """Offer ``value``'s encoding (over its last dimension) to the next binary
    layer that reads ``value``, as if that layer had encoded it itself."""

    global _last_encoding
    columns = int(value.shape[-1])
    key = (value._version, value.data_ptr(), tuple(value.shape), value.dtype, columns, kernels.capture_id(value))
    _last_encoding = (weakref.ref(value), key, payload, aux)


# A binary layer's output carries, as an attribute, the encoding aux of the
# input it was computed from: a SwiGLU gate that reads two such outputs sums
# its gradients against those inputs' offsets while it writes them
# (swiglu_backward_sums), and offers each sum to the layer whose output it
# was.  An offer names the gradient tensor it belongs to (held, with its
# version) and the aux it was summed against; a layer takes it only when
# autograd hands it exactly that gradient, unchanged, and it saved that aux.
# Offers live for one backward pass: one that no layer took (a gradient that
# autograd summed with another use of the same output) is dropped when the
# pass ends, so it holds no gradient past it.
_AUX_ATTR = "_qste_input_aux"
_offers: dict[int, tuple] = {}


def _offer_offset_dot(grad: Tensor, aux: Tensor, offset_dot: Tensor) -> None:
    _offers[grad.data_ptr()] = (grad, grad._version, aux, offset_dot)


def _take_offset_dot(grad2: Tensor, aux: Tensor) -> Tensor | None:
    offer = _offers.pop(grad2.data_ptr(), None)
    if offer is None:
        return None
    grad, version, offered_aux, offset_dot = offer
    same = (offered_aux is aux and grad._version == version and grad.numel() == grad2.numel()
            and grad.dtype == grad2.dtype and grad.is_contiguous() and grad2.is_contiguous()
            and grad.untyped_storage().data_ptr() == grad2.untyped_storage().data_ptr())
    return offset_dot if same else None


def forget_offers() -> None:
    _offers.clear()


class QSTELinearFn(Function):
    @staticmethod
    def forward(ctx, inputs, packed, scale, bias, surface: Surface):
        columns = surface.columns
        output = kernels.packed_linear_affine(inputs, packed, scale, bias, columns)
        flat = inputs.reshape(-1, columns)
        payload, aux = _encoding_of(inputs, flat, columns)
        ctx.save_for_backward(payload, aux, packed, scale)
        ctx.surface = surface
        ctx.columns = columns
        ctx.input_shape = inputs.shape
        ctx.input_dtype = inputs.dtype
        ctx.bias_dtype = None if bias is None else bias.dtype
        output = output.to(inputs.dtype)
        setattr(output, _AUX_ATTR, aux)
        return output

    @staticmethod
    def backward(ctx, grad_output):
        forget_encodings()
        payload, aux, packed, scale = ctx.saved_tensors
        grad2 = grad_output.reshape(-1, grad_output.shape[-1])
        offset_dot = _take_offset_dot(grad2, aux)
        # the input-gradient product only when autograd wants that gradient
        # (the reference always forms it, functional.py:180-183)
        grad_inputs, evidence, grad_scale, grad_bias = kernels.linear_backward(
            grad2, payload, aux[0], aux[1], packed, scale.detach(), ctx.columns,
            need_bias=ctx.bias_dtype is not None, need_input=ctx.needs_input_grad[0],
            offset_dot=offset_dot)
        ctx.surface.consume_evidence(evidence)
        if grad_inputs is not None:
            grad_inputs = grad_inputs.reshape(ctx.input_shape).to(ctx.input_dtype)
        if grad_bias is not None:
            grad_bias = grad_bias.to(ctx.bias_dtype)
        return grad_inputs, None, grad_scale.to(scale.dtype), grad_bias, None


def qste_linear(inputs: Tensor, surface: Surface, bias: Tensor | None = None) -> Tensor:
    """Functional binary linear (functional.py:197-205)."""

    surface.note_forward()
    return QSTELinearFn.apply(_autocast(inputs), surface.packed_sign, surface.scale, bias, surface)


class QSTEWeightFn(Function):
    """Differentiable dense ``sign * scale`` for code that reads ``.weight``.

    functional.py:213-245: the gradient of the dense matrix becomes the
    surface's evidence, and its row inner product with the signs the scale
    gradient.
    """

    @staticmethod
    def forward(ctx, packed, scale, surface: Surface):
        ctx.save_for_backward(packed, scale)
        ctx.surface = surface
        sign = kernels.unpack_rows(packed, surface.columns, dtype=torch.float32)
        return sign.mul_(scale.detach().float().unsqueeze(1)).to(scale.dtype)

    @staticmethod
    def backward(ctx, grad_weight):
        packed, scale = ctx.saved_tensors
        surface = ctx.surface
        grad_weight = grad_weight.float().contiguous()
        grad_scale = kernels.packed_row_inner(grad_weight, packed, surface.columns)
        evidence = grad_weight.mul_(scale.detach().float().unsqueeze(1))
        surface.consume_evidence(evidence)
        return None, grad_scale.to(scale.dtype), None


def _save_kept(ctx, gate: kernels.Blocks8, up: kernels.Blocks8, *more: Tensor) -> None:
    """Saves gate's and up's 8-bit blocks, and ``more`` after them."""

    ctx.kept_dtype = gate.dtype
    ctx.save_for_backward(gate.payload, gate.codes, up.payload, up.codes, *more)


def _kept(ctx, saved) -> tuple:
    """g and u as a forward saved them: two tensors, or with a checkpoint the first four as two ``Blocks8``."""

    if not ctx.checkpoint:
        return saved[:2]
    gate_payload, gate_codes, up_payload, up_codes = saved[:4]
    return (kernels.Blocks8(gate_payload, gate_codes, ctx.kept_dtype),
            kernels.Blocks8(up_payload, up_codes, ctx.kept_dtype))


def _flat_blocks(b: kernels.Blocks8) -> kernels.Blocks8:
    """Blocks of a tensor as those of its rows."""

    return kernels.Blocks8(b.payload.reshape(-1, b.payload.shape[-1]), b.codes.reshape(-1, b.codes.shape[-1]), b.dtype)


class SwiGLUFn(Function):
    """``silu(gate) * up`` in one kernel each way, rounded as torch's
    ``F.silu(gate) * up`` and its autograd round, keeping ``gate`` and ``up``
    for backward.  With ``encode`` the forward also encodes the output's rows
    for the binary layer that reads it next (a SwiGLU MLP's down
    projection), which then does not read the output again to encode it.  With
    ``checkpoint`` gate and up are kept in 8-bit blocks, and the gradients are
    those at the values that the blocks stand for."""

    @staticmethod
    def forward(ctx, gate, up, encode: bool, checkpoint: bool):
        forget_offers()
        ctx.checkpoint = checkpoint
        # the encodings of the inputs of the binary layers that produced gate
        # and up (one [2, tokens] aux each), when both did
        aux_g, aux_u = getattr(gate, _AUX_ATTR, None), getattr(up, _AUX_ATTR, None)
        if checkpoint:
            # (over other layers than binary ones the next is taken to be no binary one either)
            encode = encode and aux_g is not None and aux_u is not None
            out, encoding, *kept = kernels.swiglu_forward_blocks(gate, up, encode=encode)
            _save_kept(ctx, *kept)
        else:
            out, encoding = kernels.swiglu_forward(gate, up, encode=encode)
            ctx.save_for_backward(gate, up)
        if encoding is not None:
            packed, offset, scale = encoding
            remember_encoding(out, packed, kernels.stacked_pair(offset, scale))
        ctx.auxes = None
        tokens = gate.numel() // gate.shape[-1] if gate.dim() and gate.shape[-1] else 0
        if (aux_g is not None and aux_u is not None and tokens and aux_g.shape == (2, tokens)
                and aux_u.shape == (2, tokens)):
            ctx.auxes = (aux_g, aux_u)
        return out

    @staticmethod
    def backward(ctx, grad_output):
        forget_offers()
        gate, up = _kept(ctx, ctx.saved_tensors)
        if ctx.auxes is None:
            backward = kernels.swiglu_backward_blocks if ctx.checkpoint else kernels.swiglu_backward
            grad_gate, grad_up = backward(grad_output.contiguous(), gate, up)
            return grad_gate, grad_up, None, None
        # the gradients and, for the two layers' backward, their offset sums
        aux_g, aux_u = ctx.auxes
        shape = grad_output.shape
        flat = grad_output.reshape(-1, shape[-1])
        if ctx.checkpoint:
            grad_gate, grad_up, sums = kernels.swiglu_backward_blocks(
                flat, _flat_blocks(gate), _flat_blocks(up), aux_g[0], aux_u[0])
        else:
            grad_gate, grad_up, sums = kernels.swiglu_backward_sums(
                flat, gate.reshape(flat.shape), up.reshape(flat.shape), aux_g[0], aux_u[0])
        grad_gate, grad_up = grad_gate.view(shape), grad_up.view(shape)
        _offer_offset_dot(grad_gate, aux_g, sums[0])
        _offer_offset_dot(grad_up, aux_u, sums[1])
        torch.autograd.Variable._execution_engine.queue_callback(forget_offers)
        return grad_gate, grad_up, None, None


class SwiGLUKeptFn(SwiGLUFn):
    """SwiGLUFn with a checkpoint: its gradients have none of their own."""

    backward = staticmethod(once_differentiable(SwiGLUFn.backward))


def _cast(grad: Tensor | None, dtype: torch.dtype | None) -> Tensor | None:
    return None if grad is None or dtype is None else grad.to(dtype)


def _through_scale(grad_scale: Tensor, e: Tensor, surface: Surface) -> Tensor:
    """The scale's gradient carried to the log-scale, as RowScaleFn does."""

    return kernels.row_scale_backward(e, grad_scale.to(e.dtype), surface.cfg.scale_min, surface.cfg.scale_max)


def _gate_up_backward(ctx, dh: list, kept: tuple, payload_x: Tensor, aux_x: Tensor, packed_g: Tensor, packed_u: Tensor,
                      scale_gu: Tensor, sg: Surface, su: Surface, plain: bool = False):
    """The gate's backward and that of the two layers before it as one layer of 2
    ffn rows, their evidence delivered: ``(dx, scale gradients [2 ffn], bias
    gradients [2 ffn] or None)``.  ``dh``: the gradient of h in a list, taken out of it
    so that it is free during the product; ``kept``: g and u, as tensors or ``Blocks8``;
    ``scale_gu``: both layers' scales, fp32; ``plain``: round as the gate and the
    layers one by one do, g and u being tensors.  ffn, the rows of ``packed_g`` and
    ``packed_u``, may be more than the surfaces have."""

    d, ffn = sg.columns, packed_g.shape[0]
    # (a copy of their signs: the deliveries below may rewrite them)
    packed_gu = torch.cat((packed_g, packed_u))
    need_bias = any(b is not None for b in ctx.bias_dtypes[:2])
    if plain:
        both, sums = kernels.swiglu_backward_sums(dh.pop(), *kept, aux_x[0], aux_x[0], side_by_side=True)
        dx, ev_gu, gs_gu, gb_gu = kernels.linear_backward(
            both, payload_x, aux_x[0], aux_x[1], packed_gu, scale_gu, d, need_bias=need_bias,
            need_input=ctx.needs_input_grad[0], offset_dot=sums.reshape(-1))
        del both
    else:
        grads = kernels._gated_grads(dh.pop(), *kept, aux_x[0], aux_x[1])
        dx, ev_gu, gs_gu, gb_gu = kernels._gated_products(*grads, payload_x, aux_x[1], packed_gu, scale_gu, d,
                                                          ctx.needs_input_grad[0], need_bias)
        del grads
    if dx is not None:
        dx = dx.reshape(ctx.input_shape)
    sg.consume_evidence(ev_gu[:sg.rows])
    su.consume_evidence(ev_gu[ffn:ffn + su.rows])
    return dx, gs_gu, gb_gu


def _halves(t: Tensor | None, rows: int) -> tuple:
    """A tensor of two layers' rows as the gate's and up's."""

    return (None, None) if t is None else (t[:rows], t[rows:])


def _eights(rows: int) -> int:
    return -(-rows // 8) * 8


def _in_eights(t: Tensor | None, dim: int = 0) -> Tensor | None:
    """``t`` with zeros behind it up to a whole number of eights along ``dim``."""

    more = 0 if t is None else -t.shape[dim] % 8
    return t if not more else torch.cat((t, t.new_zeros(*t.shape[:dim], more, *t.shape[dim + 1:])), dim)


def _bounds(surface: Surface) -> tuple[float, float]:
    return surface.cfg.scale_min, surface.cfg.scale_max


class GatedFn(Function):
    """``silu(gate(x)) * up(x)`` of two binary layers as one autograd node.

    The forward is one kernel over both layers' signs (``kernels.gated_forward``)
    and x's encoding; what it keeps of g and u is them, or with ``checkpoint``
    their 8-bit blocks.  The backward is ``kernels.gated_backward``.  Layers whose
    rows are no whole eights run with zero rows behind them."""

    @staticmethod
    def forward(ctx, inputs, packed_g, log_g, bias_g, packed_u, log_u, bias_u, surfaces, checkpoint: bool,
                grad_on: bool):
        sg, su = surfaces
        d, rows, ffn = sg.columns, sg.rows, _eights(sg.rows)
        flat = inputs.reshape(-1, d)
        scale_gu, e = kernels.pair_scale(log_g, _bounds(sg), log_u, _bounds(su), ffn)
        signs, biases, keep = (packed_g, packed_u), (bias_g, bias_u), ""
        scales = (scale_gu[:rows], scale_gu[ffn:ffn + rows])
        if grad_on:
            signs, biases = [_in_eights(t) for t in signs], [_in_eights(t) for t in biases]
            scales, keep = _halves(scale_gu, ffn), "blocks" if checkpoint else "values"
        h, g, u = kernels.gated_forward(flat, signs[0], scales[0], biases[0], signs[1], scales[1], biases[1], d, keep=keep)
        if grad_on:
            # encoded here, where both layers are: not what is remembered of a tensor by its identity, which a write
            # that its version does not count (a graph's replay, one through .data) would leave behind
            payload_x, aux_x = encode_activation(flat)
            more = (payload_x, aux_x, packed_g, packed_u, scale_gu, e)
            if checkpoint:
                _save_kept(ctx, g, u, *more)
            else:
                ctx.save_for_backward(g, u, *more)
            if rows != ffn:
                h = h[:, :rows].contiguous()
        ctx.checkpoint = checkpoint
        ctx.surfaces = surfaces
        ctx.input_shape = inputs.shape
        ctx.log_dtypes = (log_g.dtype, log_u.dtype)
        ctx.bias_dtypes = tuple(None if b is None else b.dtype for b in (bias_g, bias_u))
        return h.reshape(*inputs.shape[:-1], rows)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_output):
        forget_encodings()
        saved = ctx.saved_tensors
        payload_x, aux_x, packed_g, packed_u, scale_gu, e = saved[-6:]
        sg, su = ctx.surfaces
        dh = [_in_eights(grad_output.reshape(-1, sg.rows), 1)]
        dx, gs_gu, gb_gu = _gate_up_backward(ctx, dh, _kept(ctx, saved), payload_x, aux_x, _in_eights(packed_g),
                                             _in_eights(packed_u), scale_gu, sg, su)
        (dt_g, dt_u), rows = ctx.log_dtypes, sg.rows
        log_g, log_u = kernels.pair_scale_backward(e, gs_gu, dt_g, _bounds(sg), dt_u, _bounds(su), rows)
        gb_g, gb_u = _halves(gb_gu, _eights(rows))
        bg, bu = ctx.bias_dtypes
        if gb_gu is not None:
            gb_g, gb_u = gb_g[:rows], gb_u[:rows]
        return dx, None, log_g, _cast(gb_g, bg), None, log_u, _cast(gb_u, bu), None, None, None


class SwiGLUMLPFn(Function):
    """``down(swiglu(gate(x), up(x)))`` as one autograd node, bf16.

    The values are those of the three QSTELinearFn nodes and SwiGLUFn
    composed: the same products, the same gate arithmetic, the same
    encodings (x's shared by gate and up; h's from the gate kernel), and
    the row scales of the three surfaces from their log-scales with the
    kernels of ``surface.row_scale`` (inputs are the log-scales, so their
    gradients leave this node as RowScaleFn's would).  The
    backward runs the gate and up layers as one layer of 2 ffn rows: the
    gate's backward writes their gradients side by side into one [tokens,
    2 ffn] tensor (with the two layers' offset sums, in the order the layers
    would sum them), and one ``linear_backward`` over it and the two layers'
    concatenated signs and scales gives

    * their evidence and scale gradients as the row blocks of one product
      (each element as the layer's own product forms it; a split-K plan
      chosen for the longer product may sum some tiles in another order),
    * x's gradient as one product over K = 2 ffn, rounded once, where
      autograd rounds each layer's input gradient and then their sum --
      one launch and one pass over [tokens, d] tensors fewer.

    Evidence goes to each surface after every product that reads that
    surface's signs (a delivery may step the surface, rewriting them), as in
    QSTELinearFn: down first, then gate and up."""

    @staticmethod
    def forward(ctx, inputs, packed_g, log_g, bias_g, packed_u, log_u, bias_u, packed_d, log_d, bias_d,
                surfaces, checkpoint: bool, grad_on: bool):
        sg, su, sd = surfaces
        d, ffn = sg.columns, sg.rows
        flat = inputs.reshape(-1, d)
        # each layer's row scale (the kernel of surface.row_scale) right
        # before the product that needs it, so the first product is queued
        # after one small launch rather than three
        scale_g, e_g = kernels.row_scale(log_g, sg.cfg.scale_min, sg.cfg.scale_max)
        checkpoint = checkpoint and grad_on
        if checkpoint:
            scale_u, e_u = kernels.row_scale(log_u, su.cfg.scale_min, su.cfg.scale_max)
            h, g, u = kernels.gated_forward(flat, packed_g, scale_g, bias_g, packed_u, scale_u, bias_u, d, keep="blocks")
            enc = kernels.pack_affine_rows(h)
        else:
            g = kernels.packed_linear_affine(flat, packed_g, scale_g, bias_g, d)
            scale_u, e_u = kernels.row_scale(log_u, su.cfg.scale_min, su.cfg.scale_max)
            u = kernels.packed_linear_affine(flat, packed_u, scale_u, bias_u, d)
            h, enc = kernels.swiglu_forward(g, u, encode=grad_on)
        scale_d, e_d = kernels.row_scale(log_d, sd.cfg.scale_min, sd.cfg.scale_max)
        y = kernels.packed_linear_affine(h, packed_d, scale_d, bias_d, ffn)
        if grad_on:
            # (with a checkpoint as GatedFn does)
            payload_x, aux_x = encode_activation(flat) if checkpoint else _encoding_of(inputs, flat, d)
            aux_h = kernels.stacked_pair(enc[1], enc[2])
            more = (payload_x, aux_x, enc[0], aux_h, packed_g, scale_g, packed_u, scale_u, packed_d, scale_d, e_g, e_u,
                    e_d)
            if checkpoint:
                _save_kept(ctx, g, u, *more)
            else:
                ctx.save_for_backward(g, u, *more)
        ctx.checkpoint = checkpoint
        ctx.surfaces = surfaces
        ctx.input_shape = inputs.shape
        ctx.bias_dtypes = tuple(None if b is None else b.dtype for b in (bias_g, bias_u, bias_d))
        return y.reshape(*inputs.shape[:-1], d)

    @staticmethod
    def backward(ctx, grad_output):
        forget_encodings()
        saved = ctx.saved_tensors
        kept = _kept(ctx, saved)
        (payload_x, aux_x, payload_h, aux_h, packed_g, scale_g, packed_u, scale_u, packed_d, scale_d, e_g, e_u,
         e_d) = saved[-13:]
        sg, su, sd = ctx.surfaces
        d, ffn = sg.columns, sg.rows
        bg, bu, bd = ctx.bias_dtypes
        dy = grad_output.reshape(-1, d)
        # A surface's evidence may step it on delivery, rewriting its packed
        # signs in place; every product that multiplies by a layer's signs
        # runs before that layer's evidence is delivered, as in QSTELinearFn
        # (whose one call forms the input gradient before the delivery).
        dh, ev_d, gs_d, gb_d = kernels.linear_backward(
            dy, payload_h, aux_h[0], aux_h[1], packed_d, scale_d.detach(), ffn, need_bias=bd is not None)
        sd.consume_evidence(ev_d)
        del ev_d
        dh = [dh]
        scale_gu = torch.cat((scale_g.detach().float(), scale_u.detach().float()))
        dx, gs_gu, gb_gu = _gate_up_backward(ctx, dh, kept, payload_x, aux_x, packed_g, packed_u, scale_gu, sg, su,
                                             plain=not ctx.checkpoint)
        (gs_g, gs_u), (gb_g, gb_u) = _halves(gs_gu, ffn), _halves(gb_gu, ffn)

        return (dx, None, _through_scale(gs_g, e_g, sg), _cast(gb_g, bg), None, _through_scale(gs_u, e_u, su),
                _cast(gb_u, bu), None, _through_scale(gs_d, e_d, sd), _cast(gb_d, bd), None, None, None)


class SwiGLUMLPKeptFn(SwiGLUMLPFn):
    """SwiGLUMLPFn with a checkpoint: its gradients have none of their own."""

    backward = staticmethod(once_differentiable(SwiGLUMLPFn.backward))


# log-scale dtypes the row-scale kernels take (surface.row_scale)
_SCALE_DTYPES = (torch.float32, torch.float16, torch.bfloat16)


def swiglu_mlp_fusable(inputs: Tensor, gate, up, down) -> bool:
    """Whether ``SwiGLUMLPFn`` takes this MLP: training layers (packed ones have
    no surface), bf16 input on the GPU, the gate and up layers d -> ffn and the
    down layer ffn -> d, d and ffn multiples of 64."""

    sg, su, sd = (getattr(m, "surface", None) for m in (gate, up, down))
    if sg is None or su is None or sd is None:
        return False
    d, ffn = sg.columns, sg.rows
    return (inputs.is_cuda and inputs.dtype == torch.bfloat16 and inputs.dim() >= 1 and inputs.shape[-1] == d
            and su.columns == d and su.rows == ffn and sd.columns == ffn and sd.rows == d
            and d % 64 == 0 and ffn % 64 == 0 and inputs.numel() > 0
            and all(s.log_scale.is_cuda and s.log_scale.dtype in _SCALE_DTYPES for s in (sg, su, sd)))


def gated_fusable(inputs: Tensor, gate, up) -> bool:
    """Whether ``GatedFn`` takes this block: a bf16 or fp16 input on the GPU, both
    layers' gradients side by side within the matrix kernels' 32-bit offsets."""

    sg, su = gate.surface, up.surface
    tokens = inputs.numel() // max(sg.columns, 1)
    return (inputs.is_cuda and inputs.dtype in (torch.bfloat16, torch.float16) and inputs.dim() >= 1
            and tokens * 4 * _eights(sg.rows) < 1 << 32 and inputs.shape[-1] == sg.columns == su.columns and sg.rows == su.rows
            and inputs.numel() > 0 and all(s.log_scale.is_cuda and s.log_scale.dtype in _SCALE_DTYPES for s in (sg, su)))


def swiglu(gate: Tensor, up: Tensor, *, checkpoint: bool = False) -> Tensor:
    """The SwiGLU gate ``F.silu(gate) * up`` (same values and gradients), fused.

    No counterpart in the reference; a SwiGLU MLP written
    ``down(swiglu(gate(x), up(x)))`` computes what
    ``down(F.silu(gate(x)) * up(x))`` computes, with two elementwise passes
    instead of five and the down projection's activation encoding produced
    with its input.

    With ``checkpoint`` what is kept of gate and up for the backward are 8-bit
    blocks of 32 columns, 33 bytes for 32 elements: the value is the same, the
    gradients are those at the blocks' values (``nn.quantize_blocks``)."""

    grad_on = torch.is_grad_enabled()
    if checkpoint:
        _no_tangent("swiglu with a checkpoint", gate, up)
        if grad_on and (gate.requires_grad or up.requires_grad):
            return SwiGLUKeptFn.apply(gate, up, True, True)
    return SwiGLUFn.apply(gate, up, grad_on, False)


def qste_weight(surface: Surface) -> Tensor:
    surface.note_forward()
    return QSTEWeightFn.apply(surface.packed_sign, surface.scale, surface)


class QSTEEmbeddingFn(Function):
    """Binary embedding lookup; its backward is the surface's evidence (functional.py:260-282)."""

    @staticmethod
    def forward(ctx, ids, packed, scale, surface: Surface):
        output = kernels.packed_embedding(ids, packed, scale, surface.columns)
        ctx.save_for_backward(ids, packed, scale)
        ctx.surface = surface
        return output

    @staticmethod
    def backward(ctx, grad_output):
        ids, packed, scale = ctx.saved_tensors
        evidence, grad_scale = kernels.embedding_backward(
            ids, grad_output, packed, scale.detach(), ctx.surface.columns)
        ctx.surface.consume_evidence(evidence)
        return None, None, grad_scale.to(scale.dtype), None


def qste_embedding(ids: Tensor, surface: Surface) -> Tensor:
    """Functional binary embedding (functional.py:285-287)."""

    surface.note_forward()
    return QSTEEmbeddingFn.apply(ids, surface.packed_sign, surface.scale, surface)
