"""Scoring tokens and distilling from a teacher's top tokens, as cases to time.

Each case is a dict of plain values; ``prepare`` makes what a program holds
before the call, ``run`` is one pass through one operator: in its plain form
(elementary torch operations in 32 bits) or, with ``own`` set, through
``qste_amd.nn``.  Kinds:

``score``         log probabilities of given tokens, each row's entropy and its ``top`` likeliest tokens
``score_grad``    the log probabilities and entropies, and the logits' gradient for weights on both
``distill``       the distillation loss of a student's logits against a teacher's top tokens
``distill_grad``  that loss and the logits' gradient, as a training step takes them through autograd
``distill_pass``  that loss and the gradient for row weights known beforehand, from one call
"""

import math

import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def listed():
    return [
        # one generated token, reported with its alternatives, over GPT-2's vocabulary
        {"name": "score_token", "kind": "score", "batch": 1, "seq": 1, "vocab": 50257, "dtype": "bf16", "top": 20},
        # a decode batch over a large vocabulary, logits kept in 32 bits
        {"name": "score_batch", "kind": "score", "batch": 40, "seq": 1, "vocab": 131072, "dtype": "fp32", "top": 5},
        # constrained decoding: most of the vocabulary masked with -inf, fewer tokens left than asked for in some rows
        {"name": "score_masked", "kind": "score", "batch": 300, "seq": 1, "vocab": 32003, "dtype": "fp16", "top": 10,
         "temperature": 0.7, "masked": True},
        # perplexity of prompts: position t predicts token t + 1, so the logits are a view without each last position
        {"name": "score_prompts", "kind": "score", "batch": 4, "seq": 1023, "vocab": 50257, "dtype": "bf16", "top": 0,
         "view": True},
        # a teacher over a GPT-2 training batch (8 sequences of 1023 predicted tokens): the targets of a distillation
        {"name": "score_teacher", "kind": "score", "batch": 8, "seq": 1023, "vocab": 50257, "dtype": "bf16", "top": 64,
         "view": True},
        # a policy gradient with an entropy bonus on sampled tokens, two sequences, padding at the end of each
        {"name": "score_policy", "kind": "score_grad", "batch": 2, "seq": 1023, "vocab": 50257, "dtype": "bf16",
         "padded": True},
        # likelihood training of a small model with a byte-pair vocabulary of no particular size
        {"name": "score_small", "kind": "score_grad", "batch": 16, "seq": 64, "vocab": 4099, "dtype": "fp32"},
        # the smallest distillation step: a few dozen tokens of a small model
        {"name": "distill_small", "kind": "distill_grad", "batch": 1, "seq": 48, "vocab": 2053, "dtype": "fp32", "k": 8,
         "tail": False, "temperature": 2.0},
        # validation loss of a student against stored targets
        {"name": "distill_eval", "kind": "distill", "batch": 2, "seq": 1023, "vocab": 50257, "dtype": "fp32", "k": 64,
         "tail": True},
        # the training step of a GPT-2-sized student: 8 sequences of 1023 predicted tokens, some positions padded
        {"name": "distill_train", "kind": "distill_grad", "batch": 8, "seq": 1023, "vocab": 50257, "dtype": "bf16",
         "k": 64, "tail": True, "padded": True},
        # a micro-batch under loss scaling in fp16, the gradient from one call
        {"name": "distill_fp16", "kind": "distill_pass", "batch": 3, "seq": 511, "vocab": 32003, "dtype": "fp16", "k": 20,
         "tail": True, "temperature": 1.5},
        # the largest: a long batch over a large vocabulary, the gradient from one call
        {"name": "distill_large", "kind": "distill_pass", "batch": 4, "seq": 2048, "vocab": 131072, "dtype": "bf16",
         "k": 32, "tail": False},
    ]


def draw(rng):
    kind = rng.choice(["score", "score", "score", "score_grad", "distill", "distill_grad", "distill_pass"])
    vocab = _log(rng, 512, 131072)
    if rng.random() < 0.6:  # a grain of eight, as padded vocabularies have; else as it comes, odd ones among them
        vocab = vocab // 8 * 8
    rows = _log(rng, 1, min(8192, (1 << 28) // vocab))
    batch = rng.choice([1, 1, 2, 3, 4, 8])
    case = {"kind": kind, "batch": min(batch, rows), "seq": max(1, rows // batch), "vocab": vocab,
            "dtype": rng.choice(["bf16", "bf16", "fp16", "fp32"]), "temperature": rng.choice([1.0, 1.0, 0.7, 2.0]),
            "view": rng.random() < 0.4}
    if kind == "score":
        case["top"] = rng.choice([0, 1, 5, 20, 64, 128])
        case["masked"] = rng.random() < 0.2
    else:
        case["padded"] = rng.random() < 0.4
    if kind.startswith("distill"):
        case["k"] = _log(rng, 4, 128)
        case["tail"] = rng.random() < 0.5
    return case


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def work(case):
    """Logits read once and each output written once; per logit an exponential and a handful of operations."""
    rows, vocab = case["batch"] * case["seq"], case["vocab"]
    logits = rows * vocab * (4 if case["dtype"] == "fp32" else 2)
    grad = case["kind"] in ("score_grad", "distill_grad", "distill_pass")
    per_row = 12 * case["k"] + 8 if "k" in case else 16 + 12 * case.get("top", 0)
    return {"bytes": logits * (2 if grad else 1) + rows * per_row, "flops": rows * vocab * (16 if grad else 8)}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    batch, seq, vocab, kind = case["batch"], case["seq"], case["vocab"], case["kind"]
    dtype, view = DTYPES[case["dtype"]], case.get("view", False)
    full = seq + 1 if view else seq
    logits = torch.randn(batch, full, vocab, generator=g, device=DEV, dtype=dtype).mul_(2.5)
    # a language model's rows have a few likely tokens above the rest, spread over the vocabulary
    count = case.get("k", min(32, vocab // 8))
    likely = torch.randint(vocab, (batch, full, 1), generator=g, device=DEV)
    likely = (likely + torch.arange(count, device=DEV) * (vocab // count)) % vocab
    peak = 14.0 - 1.6 * torch.arange(1, count + 1, device=DEV).float().log()
    peak = peak + torch.randn(batch, full, count, generator=g, device=DEV)
    logits.scatter_(2, likely, peak.to(dtype))
    if case.get("masked"):
        # each row allows its own share of the vocabulary, from a handful of tokens to all of it
        share = torch.rand(batch, full, 1, generator=g, device=DEV).pow(3)
        share[::7] = 2.0 / vocab
        blocked = torch.rand(batch, full, vocab, generator=g, device=DEV) > share
        blocked.scatter_(2, likely[..., :1], False)
        logits.masked_fill_(blocked, -math.inf)
    state = {"case": dict(case), "logits": logits[:, :-1] if view else logits}
    likely = likely[:, :-1] if view else likely
    live = torch.ones(batch, seq, dtype=torch.bool, device=DEV)
    if case.get("padded"):
        ends = (seq * (0.5 + 0.5 * torch.rand(batch, 1, generator=g, device=DEV))).long()
        live = torch.arange(seq, device=DEV) < ends.clamp(min=1)
    if kind.startswith("score"):
        # a token among the likely ones, at padded positions the usual negative mark
        pick = torch.randint(count, (batch, seq, 1), generator=g, device=DEV)
        tokens = likely.gather(2, pick).squeeze(2)
        state["tokens"] = torch.where(live, tokens, -100)
    else:
        # the teacher's log probabilities: it puts most of its mass on these tokens, and no two of them apart by much
        fall = 1.1 * torch.arange(1, count + 1, device=DEV).float().log()
        value = torch.log_softmax(torch.randn(batch, seq, count, generator=g, device=DEV) - fall, 2)
        value, _ = value.sort(dim=2, descending=True)
        kept = 0.6 + 0.35 * torch.rand(batch, seq, 1, generator=g, device=DEV)
        state["top_logprobs"] = value + kept.log()
        # some rows hold fewer entries than the others: the rest are marked -1
        fewer = torch.rand(batch, seq, 1, generator=g, device=DEV) < 0.1
        drop = fewer & (torch.arange(count, device=DEV) >= (count + 1) // 2)
        state["top_tokens"] = torch.where(drop, -1, likely)
    if kind in ("score_grad", "distill_grad", "distill_pass"):
        # weights of the mean over the tokens that count; fp16 trains under a loss scale
        weight = torch.where(live, (2.0 ** 14 if dtype == torch.float16 else 1.0) / live.sum(), 0.0)
        if kind == "score_grad":
            state["logprob_grad"] = weight * torch.randn(batch, seq, generator=g, device=DEV)
            state["entropy_grad"] = -0.01 * weight
        else:
            state["loss_grad"] = weight
        if kind != "distill_pass":
            state["logits"].requires_grad_(True)
    return state


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------


def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(state):
    import qste_amd as qste

    case, logits = state["case"], state["logits"]
    kind, temperature = case["kind"], case.get("temperature", 1.0)
    if kind == "score":
        s = qste.nn.token_logprobs(logits, state["tokens"], top=case["top"], temperature=temperature)
        out = {"logprobs": s.logprobs, "entropy": s.entropy}
        if case["top"]:
            out.update(top_logprobs=s.top_logprobs, top_tokens=s.top_tokens)
        return out
    if kind == "score_grad":
        s = qste.nn.token_logprobs(logits, state["tokens"], temperature=temperature)
        grad, = torch.autograd.grad((s.logprobs, s.entropy), logits, (state["logprob_grad"], state["entropy_grad"]))
        return {"logprobs": s.logprobs.detach(), "entropy": s.entropy.detach(), "grad": grad}
    target = (state["top_tokens"], state["top_logprobs"])
    if kind == "distill":
        return {"losses": qste.nn.distillation_loss(logits, *target, temperature=temperature, tail=case["tail"])}
    if kind == "distill_grad":
        losses = qste.nn.distillation_loss(logits, *target, temperature=temperature, tail=case["tail"])
        grad, = torch.autograd.grad(losses, logits, state["loss_grad"])
        return {"losses": losses.detach(), "grad": grad}
    losses, grad = qste.nn.distillation_loss_and_grad(logits, *target, loss_grad=state["loss_grad"],
                                                      temperature=temperature, tail=case["tail"])
    return {"losses": losses, "grad": grad}


def _softmax_parts(logits, temperature):
    """(d, e, total): (z - max) / temperature, its exponential and the exponentials' sum, in 32 bits."""
    z = logits.detach().float()
    d = (z - z.amax(-1, keepdim=True)) / temperature
    e = d.exp()
    return d, e, e.sum(-1, keepdim=True)


def _run_plain(state):
    case = state["case"]
    if case["kind"].startswith("score"):
        return _score_plain(state, case)
    return _distill_plain(state, case)


def _score_plain(state, case):
    logits, tokens = state["logits"], state["tokens"]
    d, e, total = _softmax_parts(logits, case.get("temperature", 1.0))
    lnp, p = d - total.log(), e / total
    del d, e
    entropy = -torch.where(p > 0, p * lnp, 0.0).sum(-1)
    live = tokens >= 0
    logprobs = torch.where(live, lnp.gather(2, tokens.clamp(min=0).unsqueeze(2)).squeeze(2), 0.0)
    out = {"logprobs": logprobs, "entropy": torch.where(live, entropy, 0.0)}
    if case.get("top"):
        # values that order as the logits do (-0 as 0) above the places in reverse: equal logits go to the lowest token
        bits = (logits.float() + 0.0).view(torch.int32)
        order = (bits ^ ((bits >> 31) & 0x7FFFFFFF)).long()
        del bits
        order = (order << 32) + (0xFFFFFFFF - torch.arange(case["vocab"], device=DEV))
        places = 0xFFFFFFFF - (order.topk(case["top"], dim=2).values & 0xFFFFFFFF)
        out["top_logprobs"], out["top_tokens"] = lnp.gather(2, places), places
    if case["kind"] == "score_grad":
        a = torch.where(live, state["logprob_grad"], 0.0).unsqueeze(2)
        h = torch.where(live, state["entropy_grad"], 0.0).unsqueeze(2)
        grad = -p * (a + h * torch.where(p > 0, lnp + entropy.unsqueeze(2), 0.0))
        grad.scatter_add_(2, tokens.clamp(min=0).unsqueeze(2), a)
        out["grad"] = (grad / case.get("temperature", 1.0)).to(logits.dtype)
    return out


def _distill_plain(state, case):
    logits, tokens, values = state["logits"], state["top_tokens"], state["top_logprobs"].float()
    temperature, vocab = case.get("temperature", 1.0), case["vocab"]
    d, e, total = _softmax_parts(logits, temperature)
    there = tokens >= 0
    place = torch.where(there, tokens, vocab)  # one column past the vocabulary takes the entries that are not there
    values = torch.where(there, values, -math.inf)
    if case["tail"]:
        q = values.exp()
        rest = (1.0 - q.sum(2, keepdim=True)).clamp(min=0.0)
    else:
        q = (values - values.amax(2, keepdim=True)).exp()
        q = q / q.sum(2, keepdim=True)
        rest = torch.zeros_like(q[..., :1])
    lnp = d.gather(2, place.clamp(max=vocab - 1)) - total.log()
    losses = torch.where(q > 0, q * (q.log() - lnp), 0.0).sum(2)
    weight = q.sum(2, keepdim=True) + rest
    del d
    if case["tail"]:
        listed_ = torch.zeros(*q.shape[:2], vocab + 1, dtype=torch.bool, device=DEV).scatter_(2, place, True)[..., :vocab]
        p_rest = torch.where(listed_, 0.0, e).sum(2, keepdim=True) / total
        losses = losses + torch.where(rest > 0, rest * (rest.log() - p_rest.log()), 0.0).squeeze(2)
        weight = torch.where(listed_, weight, weight - rest / p_rest)
    losses = losses * temperature ** 2
    if case["kind"] == "distill":
        return {"losses": losses}
    grad = e.div_(total).mul_(weight)
    target = torch.zeros(*q.shape[:2], vocab + 1, device=DEV).scatter_add_(2, place, q)[..., :vocab]
    grad = grad.sub_(target).mul_(state["loss_grad"].unsqueeze(2) * temperature)
    return {"losses": losses, "grad": grad.to(logits.dtype)}


# ---------------------------------------------------------------------------
# the definitions in 64 bits, a few rows at a time
# ---------------------------------------------------------------------------


def exact(case, seed):
    state = prepare(case, seed)
    rows, vocab = case["batch"] * case["seq"], case["vocab"]
    flat = {k: v.detach().reshape(rows, *v.shape[2:]) for k, v in state.items() if k != "case"}
    step = max(1, (1 << 26) // vocab)
    parts = []
    for at in range(0, rows, step):
        part = {k: v[at:at + step] for k, v in flat.items()}
        parts.append(_exact_score(case, part) if case["kind"].startswith("score") else _exact_distill(case, part))
    whole = {k: torch.cat([p[k] for p in parts]) for k in parts[0]}
    return {k: v.reshape(case["batch"], case["seq"], *v.shape[1:]) for k, v in whole.items()}


def _exact_score(case, part):
    z, tokens = part["logits"].double(), part["tokens"]
    lnp = torch.log_softmax(z / case.get("temperature", 1.0), 1)
    p = lnp.exp()
    live = (tokens >= 0).double()
    entropy = -torch.special.xlogy(p, p).sum(1)
    row = torch.arange(len(z), device=DEV)
    out = {"logprobs": torch.where(live > 0, lnp[row, tokens.clamp(min=0)], 0.0), "entropy": entropy * live}
    if case.get("top"):
        _, places = torch.sort(z, dim=1, descending=True, stable=True)
        out["top_tokens"] = places[:, :case["top"]].contiguous()
        out["top_logprobs"] = lnp.gather(1, out["top_tokens"])
    if case["kind"] == "score_grad":
        a, h = part["logprob_grad"].double() * live, part["entropy_grad"].double() * live
        grad = -a[:, None] * p - h[:, None] * (torch.special.xlogy(p, p) + p * entropy[:, None])
        grad[row, tokens.clamp(min=0)] += a
        out["grad"] = grad / case.get("temperature", 1.0)
    return out


def _exact_distill(case, part):
    temperature, tail = case.get("temperature", 1.0), case["tail"]
    z, tokens, v = part["logits"].double() / temperature, part["top_tokens"], part["top_logprobs"].double()
    v = v.masked_fill(tokens < 0, -math.inf)
    q = v.exp() if tail else torch.softmax(v, 1)
    p = torch.softmax(z, 1)
    teacher = torch.zeros_like(p)
    teacher.scatter_add_(1, tokens.clamp(min=0), q)
    named = torch.zeros_like(p).scatter_add_(1, tokens.clamp(min=0), (tokens >= 0).double()) > 0
    # sum q ln q - q ln p over the named tokens
    cross = torch.special.xlogy(teacher, teacher).sum(1) - (teacher * torch.log_softmax(z, 1)).sum(1)
    slope = p - teacher
    if tail:
        rest, left = 1.0 - q.sum(1), p.masked_fill(named, 0.0).sum(1)
        cross = cross + torch.special.xlogy(rest, rest / left)
        slope = torch.where(named, slope, p * (1.0 - rest / left)[:, None])
    out = {"losses": cross * temperature ** 2}
    if case["kind"] != "distill":
        out["grad"] = slope * (part["loss_grad"].double() * temperature)[:, None]
    return out
