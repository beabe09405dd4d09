"""The gated feed-forward block and its 8-bit checkpoints, as cases to time.

Each case is a dict of plain values; ``prepare`` makes what a program holds
before the call, ``run`` is one pass through one operator: in its plain form
(elementary torch operations in 32 bits) or, with ``own`` set, through
``qste_amd.nn``.  Kinds:

``gated``   silu(gate(x)) * up(x) of two packed layers, as a model is served
``train``   the block of two training layers and its gradients, gate and up kept in 8 bits in between
``swiglu``  silu(gate) * up and its gradients, gate and up kept in 8 bits in between
``blocks``  a tensor brought to 8 bits, a power of two for each block of 32, and read back
"""

import math

import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BLOCK = 32


def listed():
    return [
        # one generated token of a 7-billion-parameter model
        {"name": "gated_token", "kind": "gated", "rows": 1, "width": 4096, "ffn": 14336, "dtype": "bf16"},
        # a decode batch in fp16, layers with a bias and a hidden size of no particular grain
        {"name": "gated_rows", "kind": "gated", "rows": 37, "width": 2048, "ffn": 5480, "dtype": "fp16", "bias": True},
        # a few tokens in 32 bits
        {"name": "gated_fp32", "kind": "gated", "rows": 5, "width": 1024, "ffn": 2816, "dtype": "fp32"},
        # one prompt
        {"name": "gated_prompt", "kind": "gated", "rows": 500, "width": 2048, "ffn": 8192, "dtype": "bf16"},
        # a batch of prompts through a large layer
        {"name": "gated_prompts", "kind": "gated", "rows": 8190, "width": 4096, "ffn": 14336, "dtype": "bf16"},
        # the smallest training step: one short sequence in fp16 under a loss scale
        {"name": "train_small", "kind": "train", "rows": 250, "width": 768, "ffn": 2048, "dtype": "fp16"},
        # a training step of a small model, layers with a bias
        {"name": "train_step", "kind": "train", "rows": 4096, "width": 1024, "ffn": 4096, "dtype": "bf16", "bias": True},
        # a training step of a large layer
        {"name": "train_large", "kind": "train", "rows": 8192, "width": 4096, "ffn": 14336, "dtype": "bf16"},
        # the gate alone over layers of the user's own, a small step in 32 bits, blocks that end inside a row
        {"name": "swiglu_small", "kind": "swiglu", "rows": 96, "ffn": 1000, "dtype": "fp32"},
        # the gate alone in a training step of a large layer
        {"name": "swiglu_large", "kind": "swiglu", "rows": 16384, "ffn": 14336, "dtype": "bf16"},
        # a small saved activation of odd width
        {"name": "blocks_small", "kind": "blocks", "rows": 37, "ffn": 4099, "dtype": "fp32"},
        # a layer's activation of a whole batch
        {"name": "blocks_large", "kind": "blocks", "rows": 16384, "ffn": 4096, "dtype": "bf16"},
    ]


def draw(rng):
    kind = rng.choice(["gated", "gated", "gated", "train", "train", "swiglu", "blocks"])
    ffn = _log(rng, 512, 14336)
    grain = rng.choice([64, 32, 8, 8, 1])  # most hidden sizes have a grain; odd ones among them
    ffn = max(1, ffn // grain) * grain
    case = {"kind": kind, "dtype": rng.choice(["bf16", "bf16", "fp16", "fp32"])}
    if kind in ("swiglu", "blocks"):
        case.update(rows=_log(rng, 1, 16384), ffn=ffn)
        return case
    width = _log(rng, 256, 4096)
    grain = rng.choice([128, 64, 64, 8, 1])
    width = width // grain * grain
    rows = _log(rng, 1, 8192) if kind == "gated" else _log(rng, 64, 4096)
    if case["dtype"] == "fp32":
        if kind == "train":
            case["dtype"] = "bf16"
        rows = min(rows, 512) if kind == "gated" else rows
    case.update(rows=rows, width=width, ffn=ffn, bias=rng.random() < 0.3)
    return case


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def work(case):
    """Inputs read once, outputs and what is kept for the backward written once and read once; the products' operations."""
    rows, ffn, kind = case["rows"], case["ffn"], case["kind"]
    size = 4 if case["dtype"] == "fp32" else 2
    hidden = rows * ffn
    kept = hidden + rows * -(-ffn // BLOCK)  # bytes of one tensor in 8 bits
    if kind == "blocks":
        return {"bytes": 2 * hidden * size + 2 * kept, "flops": 6 * hidden}
    if kind == "swiglu":
        return {"bytes": 6 * hidden * size + 4 * kept, "flops": 40 * hidden}
    signs = 2 * ffn * (-(-case["width"] // 8))
    flat = rows * case["width"]
    forward = flat * size + signs + 8 * ffn + hidden * size
    if kind == "gated":
        return {"bytes": forward, "flops": 4 * flat * ffn}
    encoding = flat // 8 + 8 * rows
    backward = hidden * size + 2 * kept + encoding + signs + flat * size + 2 * ffn * case["width"] * size
    return {"bytes": forward + 2 * kept + encoding + backward, "flops": 12 * flat * ffn}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    rows, ffn, kind, dtype = case["rows"], case["ffn"], case["kind"], DTYPES[case["dtype"]]
    state = {"case": dict(case)}

    def randn(*shape, std=1.0, to=dtype):
        return torch.randn(*shape, generator=g, device=DEV, dtype=to).mul_(std)

    if kind == "blocks":
        # activations: a few columns far above the others
        state["x"] = randn(rows, ffn) * (1.0 + 20.0 * (torch.rand(ffn, generator=g, device=DEV) < 0.01)).to(dtype)
        return state
    # fp16 trains under a loss scale; gradients of a mean over many tokens are small
    grad_std = 2.0 if dtype == torch.float16 else 1e-3
    if kind == "swiglu":
        state["gate"], state["up"] = randn(rows, ffn, std=1.2).requires_grad_(), randn(rows, ffn).requires_grad_()
        state["grad"] = randn(rows, ffn, std=grad_std)
        return state
    width = case["width"]
    # normalised inputs with an offset for each row, row scales about 1 / sqrt(width)
    state["x"] = randn(rows, width) + randn(rows, 1, std=0.2)
    for name in ("gate", "up"):
        log_scale = randn(ffn, std=0.2, to=torch.float32) - 0.5 * math.log(width)
        if kind == "gated":
            state[name + "_bits"] = torch.randint(0, 256, (ffn, -(-width // 8)), generator=g, device=DEV,
                                                  dtype=torch.uint8)
            state[name + "_scale"] = log_scale.exp()
        else:
            state[name + "_coordinate"] = torch.randint(-127, 128, (ffn, width), generator=g, device=DEV,
                                                        dtype=torch.int8)
            state[name + "_log_scale"] = log_scale.to(dtype)  # the model is kept in the inputs' type
        if case.get("bias"):
            state[name + "_bias"] = randn(ffn, std=0.1).float()
    if kind == "train":
        state["x"].requires_grad_()
        state["grad"] = randn(rows, ffn, std=grad_std)
    return state


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------


def run(state):
    return _run_own(state) if own else _run_plain(state)


def _layers(state):
    """The two layers, made once, as a program's model holds them."""
    import qste_amd as qste

    case = state["case"]
    layers = []
    for name in ("gate", "up"):
        bias = state.get(name + "_bias")
        if case["kind"] == "gated":
            layers.append(qste.PackedLinear(state[name + "_bits"], state[name + "_scale"], case["width"], bias))
            continue
        surface = qste.Surface.from_state(state[name + "_coordinate"], state[name + "_log_scale"])
        layer = qste.QSTELinear(surface, bias).to(DEV)
        surface.log_scale.data = state[name + "_log_scale"]
        # what a data-parallel program hands on to be summed over the ranks, in the model's type
        surface.route_evidence(lambda s, evidence: state.__setitem__(id(s), evidence.to(s.log_scale.dtype)))
        layers.append(layer)
    return layers


def _run_own(state):
    import qste_amd as qste

    case = state["case"]
    if case["kind"] == "blocks":
        return {"values": qste.nn.dequantize_blocks(qste.nn.quantize_blocks(state["x"]))}
    if case["kind"] == "swiglu":
        h = qste.nn.swiglu(state["gate"], state["up"], checkpoint=True)
        gate_grad, up_grad = torch.autograd.grad(h, (state["gate"], state["up"]), state["grad"])
        return {"h": h.detach(), "gate_grad": gate_grad, "up_grad": up_grad}
    if "layers" not in state:
        state["layers"] = _layers(state)
    gate, up = state["layers"]
    if case["kind"] == "gated":
        with torch.no_grad():
            return {"h": qste.nn.gated(state["x"], gate, up)}
    h = qste.nn.gated(state["x"], gate, up, checkpoint=True)
    leaves = [state["x"], gate.surface.log_scale, up.surface.log_scale]
    if case.get("bias"):
        leaves += [gate.bias, up.bias]
    grads = torch.autograd.grad(h, leaves, state["grad"])
    out = {"h": h.detach(), "x_grad": grads[0], "gate_scale_grad": grads[1], "up_scale_grad": grads[2],
           "gate_evidence": state.pop(id(gate.surface)), "up_evidence": state.pop(id(up.surface))}
    if case.get("bias"):
        out["gate_bias_grad"], out["up_bias_grad"] = (b.to(state["x"].dtype) for b in grads[3:])
    return out


def _signs(bits, width):
    """+-1 in 32 bits from signs packed eight to a byte, the lowest bit first."""
    shifts = torch.arange(8, device=DEV, dtype=torch.uint8)
    unpacked = (bits.unsqueeze(2) >> shifts) & 1
    return unpacked.reshape(bits.shape[0], -1)[:, :width].float() * 2 - 1


def _in_blocks(x):
    """(x in blocks of 32, the last one filled with zeros, as [rows, blocks, 32])"""
    columns = x.shape[-1]
    more = -columns % BLOCK
    if more:
        x = torch.cat((x, x.new_zeros(x.shape[0], more)), 1)
    return x.reshape(x.shape[0], -1, BLOCK)


def _eight_bits(x):
    """What x [rows, columns], in 32 bits, is in 8: a power of two for each block of 32, 6 bits and a sign above it."""
    whole = _in_blocks(x)
    top = whole.abs().amax(2, keepdim=True)
    _, exponent = torch.frexp(top.clamp(min=2.0 ** -120))  # top = mantissa in [1/2, 1) times 2^exponent
    step = torch.ldexp(torch.ones_like(top), exponent - 7)
    q = (whole / step).round().clamp(-127, 127)
    return (q * step).reshape(x.shape[0], -1)[:, :x.shape[1]]


def _run_plain(state):
    case = state["case"]
    kind, dtype = case["kind"], DTYPES[case["dtype"]]
    if kind == "blocks":
        return {"values": _eight_bits(state["x"].float()).to(dtype)}
    if kind == "swiglu":
        gate, up = state["gate"].detach().float(), state["up"].detach().float()
        h = gate / (1 + (-gate).exp()) * up
        gate_grad, up_grad = _swiglu_grads(state["grad"].float(), _eight_bits(gate), _eight_bits(up))
        return {"h": h.to(dtype), "gate_grad": gate_grad.to(dtype), "up_grad": up_grad.to(dtype)}
    x = state["x"].detach().float()
    signs, scales, hidden = {}, {}, {}
    for name in ("gate", "up"):
        if kind == "gated":
            signs[name], scales[name] = _signs(state[name + "_bits"], case["width"]), state[name + "_scale"]
        else:
            signs[name] = (state[name + "_coordinate"] >= 0).float() * 2 - 1
            scales[name] = state[name + "_log_scale"].float().exp().to(dtype).float()
        y = torch.mm(x, signs[name].t()) * scales[name]
        if case.get("bias"):
            y = y + state[name + "_bias"]
        hidden[name] = y.to(dtype).float()  # the layers' outputs are of the inputs' type
    gate, up = hidden["gate"], hidden["up"]
    h = gate / (1 + (-gate).exp()) * up
    if kind == "gated":
        return {"h": h.to(dtype)}
    grads = dict(zip(("gate", "up"), _swiglu_grads(state["grad"].float(), _eight_bits(gate), _eight_bits(up))))
    # what the layers keep of their input: its mean, its mean distance from that, and a sign for each element
    offset = x.mean(1, keepdim=True, dtype=torch.float64).float()
    away = x - offset
    kept = offset + away.abs().mean(1, keepdim=True, dtype=torch.float64).float() * ((away >= 0).float() * 2 - 1)
    x_grad = torch.zeros_like(x)
    out = {"h": h.to(dtype)}
    for name in ("gate", "up"):
        x_grad += torch.mm(grads[name] * scales[name], signs[name])
        evidence = torch.mm(grads[name].t(), kept)
        out[name + "_scale_grad"] = ((evidence * signs[name]).sum(1) * scales[name]).to(dtype)
        out[name + "_evidence"] = (evidence * scales[name].unsqueeze(1)).to(dtype)
        if case.get("bias"):
            out[name + "_bias_grad"] = grads[name].sum(0).to(dtype)
    out["x_grad"] = x_grad.to(dtype)
    order = ("h", "x_grad", "gate_scale_grad", "up_scale_grad", "gate_evidence", "up_evidence", "gate_bias_grad",
             "up_bias_grad")
    return {k: out[k] for k in order if k in out}


def _swiglu_grads(grad, gate, up):
    s = 1 / (1 + (-gate).exp())
    return grad * up * s * (1 + gate * (1 - s)), grad * gate * s


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------


def exact(case, seed):
    state = prepare(case, seed)
    kind, dtype = case["kind"], DTYPES[case["dtype"]]
    if kind == "blocks":
        return {"values": _exact_eight_bits(state["x"].double())}
    if kind == "swiglu":
        return _exact_swiglu(state["gate"].detach().double(), state["up"].detach().double(), state["grad"].double())
    x = state["x"].detach().double()
    weights, hidden = {}, {}
    for name in ("gate", "up"):
        if kind == "gated":
            place = torch.arange(case["width"], device=DEV)
            positive = state[name + "_bits"][:, place // 8].int().bitwise_right_shift(place % 8) % 2 == 1
            scale = state[name + "_scale"].double()
        else:
            positive = state[name + "_coordinate"] >= 0
            scale = state[name + "_log_scale"].double().exp().to(dtype).double()
        weights[name] = torch.where(positive, 1.0, -1.0).double(), scale
        y = x @ weights[name][0].T * scale
        if case.get("bias"):
            y += state[name + "_bias"].double()
        hidden[name] = y.to(dtype).double() if kind == "train" or dtype != torch.float32 else y
    if kind == "gated":
        return {"h": hidden["gate"].sigmoid() * hidden["gate"] * hidden["up"]}
    both = _exact_swiglu(hidden["gate"], hidden["up"], state["grad"].double())
    del hidden
    mean = x.mean(1, keepdim=True)
    spread = (x - mean).abs().mean(1, keepdim=True)
    kept = torch.where(state["x"].detach().float() >= mean.float(), mean + spread, mean - spread)
    out = {"h": both["h"], "x_grad": 0.0}
    late = {}
    for name in ("gate", "up"):
        sign, scale = weights.pop(name)
        grad = both.pop(name + "_grad")
        out["x_grad"] = out["x_grad"] + grad @ (sign * scale[:, None])
        evidence = grad.T @ kept
        out[name + "_scale_grad"] = (evidence * sign).sum(1) * scale
        late[name + "_evidence"] = evidence.mul_(scale[:, None])
        if case.get("bias"):
            late[name + "_bias_grad"] = grad.sum(0)
    out.update({k: late[k] for k in ("gate_evidence", "up_evidence", "gate_bias_grad", "up_bias_grad") if k in late})
    return out


def _exact_eight_bits(x):
    """Each block's values to the nearest multiple of the 64th part of the power of two under its largest one."""
    rows, columns = x.shape
    blocks = torch.nn.functional.pad(x, (0, -columns % BLOCK)).unflatten(1, (-1, BLOCK))
    largest = blocks.abs().amax(2, keepdim=True).clamp(min=2.0 ** -120)
    power = 2.0 ** torch.floor(torch.log2(largest))
    # log2 may round up to the next whole number just below it
    power = torch.where(power > largest, power / 2, power)
    parts = torch.clamp(torch.round(blocks / power * 64), -127, 127)
    return (parts * power / 64).flatten(1)[:, :columns]


def _exact_swiglu(gate, up, grad):
    h = gate.sigmoid() * gate * up
    gate, up = _exact_eight_bits(gate), _exact_eight_bits(up)
    s = gate.sigmoid()
    return {"h": h, "gate_grad": grad * up * (s + gate * s * (1 - s)), "up_grad": grad * gate * s}
