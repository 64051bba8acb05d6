"""The losses over the vocabulary's logits, as a training or serving program calls them: one dict per case.

``listed()`` names the measured cases, ``draw()`` gives more of the same ranges; ``prepare()`` makes
what a program holds before the call, ``run()`` is one pass through one operator, ``exact()`` the same
values in 64 bits.

Four kinds of pass, over logits ``[sequences, tokens, vocabulary]``:

* ``logprobs``: the log-probability of each token's label; in training also the logits' gradient.
* ``preference``: paired log ratios of chosen and rejected answers (the first and the second half of the
  sequences) against a reference model, and the logits' gradient.
* ``policy``: the clipped policy loss with a KL term, and the logits' gradient.
* ``distill``: the divergence from a teacher's top logits, and the logits' gradient.
"""
import math

import torch

own = False  # True: run() calls the framework's operators instead of their plain forms

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _case(kind, name=None, **kw):
    c = {"kind": kind, "dtype": "bf16", "temperature": 1.0, "padded": False, "padded_vocab": 0, **kw}
    return c if name is None else {"name": name, **c}


def listed():
    return [
        # serving: the log-probability of one sampled token
        _case("logprobs", "logprobs_1_token", seqs=1, tokens=1, vocab=128000, train=False),
        # serving: a decode step's batch, an odd vocabulary, sampled at a temperature, fp16 model
        _case("logprobs", "logprobs_37_tokens", seqs=37, tokens=1, vocab=50257, train=False, dtype="fp16",
              temperature=0.7),
        # training on two long answers of different lengths, fp32 logits
        _case("logprobs", "logprobs_train_1531", seqs=2, tokens=1531, vocab=32000, train=True, dtype="fp32", padded=True),
        # one short pair of answers
        _case("preference", "preference_1_pair", seqs=2, tokens=61, vocab=32000, loss="sigmoid", smoothing=0.0,
              average=False, beta=0.1),
        # a micro-batch of four pairs of full length behind prompts, a vocabulary with unused columns at its end
        _case("preference", "preference_4_pairs", seqs=8, tokens=1024, vocab=128000, loss="sigmoid", smoothing=0.1,
              average=False, beta=0.1, padded=True, padded_vocab=61),
        # length-normalised answers of an odd length and vocabulary
        _case("preference", "preference_odd", seqs=6, tokens=251, vocab=50257, loss="ipo", smoothing=0.0, average=True,
              beta=0.2, padded=True),
        # the first steps on a small model: four short completions, no reference model
        _case("policy", "policy_4_short", seqs=4, tokens=63, vocab=50257, kl=0.0, reduction="mean", steps=1),
        # a group of sixteen completions of different lengths, with the KL term
        _case("policy", "policy_16_long", seqs=16, tokens=512, vocab=128000, kl=0.04, reduction="mean", steps=1,
              padded=True),
        # a mean for each sequence, fp32 logits
        _case("policy", "policy_8_sequences", seqs=8, tokens=257, vocab=65536, kl=0.04, reduction="sequence", steps=1,
              dtype="fp32", padded=True),
        # a short answer and a teacher's eight best
        _case("distill", "distill_37_tokens", seqs=1, tokens=37, vocab=32000, top=8, reduction="mean", steps=1),
        # two answers of odd length, an odd vocabulary, fp16 logits, a mean for each
        _case("distill", "distill_2_odd", seqs=2, tokens=777, vocab=50257, top=20, reduction="sequence", steps=1,
              dtype="fp16", padded=True),
        # a training micro-batch at a temperature
        _case("distill", "distill_4_long", seqs=4, tokens=1024, vocab=128000, top=64, reduction="mean", steps=1,
              temperature=2.0),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("logprobs", "preference", "policy", "distill"))
    vocab = _log_int(rng, 1000, 152000)
    seqs = _log_int(rng, 1, 16)
    if kind == "preference":
        seqs = 2 * _log_int(rng, 1, 8)
    tokens = min(_log_int(rng, 1, 2048), max(1, 700000000 // (vocab * seqs)))
    dtype = rng.choice(("bf16", "bf16", "fp16", "fp32"))
    common = dict(seqs=seqs, tokens=tokens, vocab=vocab, dtype=dtype, padded=tokens > 1 and rng.random() < 0.6,
                  padded_vocab=rng.choice((0, 0, 0, rng.randint(1, 100))))
    if kind == "preference":
        loss = rng.choice(("sigmoid", "sigmoid", "hinge", "ipo"))
        return _case(kind, loss=loss, smoothing=rng.choice((0.0, 0.1)) if loss == "sigmoid" else 0.0,
                     average=rng.random() < 0.3, beta=rng.choice((0.05, 0.1, 0.3)), **common)
    common["temperature"] = rng.choice((1.0, 1.0, 0.7, 2.0))
    if kind == "logprobs":
        return _case(kind, train=rng.random() < 0.5, **common)
    # steps: micro-batches whose gradients are accumulated; each one's loss is divided by them
    common.update(reduction=rng.choice(("mean", "mean", "sequence", "none")), steps=rng.choice((1, 1, 4)))
    if kind == "policy":
        return _case(kind, kl=rng.choice((0.0, 0.02, 0.1)), **common)
    return _case(kind, top=_log_int(rng, 1, 128), **common)


# ------------------------------------------------------------------------------ inputs


def _gen(seed, part=0):
    return torch.Generator(device=DEV).manual_seed(1000 * seed + part)


def _spans(case):
    """(first, last + 1) counted token of each sequence: behind its prompt, before its padding."""
    T = case["tokens"]
    if not case["padded"]:
        return [(0, T)] * case["seqs"]
    return [(T // 5, T - (i * 37) % (T // 3 + 1)) for i in range(case["seqs"])]


def _counted(case, seed):
    spans = _spans(case)
    spans = spans[seed % len(spans):] + spans[:seed % len(spans)]  # the sequences in another order
    at = torch.arange(case["tokens"], device=DEV)
    return torch.stack([(at >= a) & (at < b) for a, b in spans])


def _log_softmax64(z, temperature):
    y = z.double() / temperature
    y = y - y.amax(-1, keepdim=True)
    return y - torch.exp(y).sum(-1, keepdim=True).log()


def _loss_scale(case):
    """What a program with fp16 logits multiplies its loss by, so that the gradient stays above the type's smallest values."""
    if case["dtype"] != "fp16":
        return 1.0
    return 128.0 if case["kind"] == "preference" else 4096.0


def prepare(case, seed):
    N, T, V, kind = case["seqs"], case["tokens"], case["vocab"], case["kind"]
    used = V - case["padded_vocab"]
    dtype, g = DTYPES[case["dtype"]], _gen(seed)
    counted = _counted(case, seed)
    labels = torch.randint(0, used, (N, T), generator=g, device=DEV)
    # a model's logits: the answer's token well above the others at most places, a few others near it
    logits = torch.empty(N, T, V, dtype=dtype, device=DEV)
    for i in range(N):
        z = 2.0 * torch.randn(T, V, generator=g, device=DEV)
        z.scatter_add_(-1, labels[i].unsqueeze(-1), 16.0 * torch.rand(T, 1, generator=g, device=DEV))
        z[:, used:] = -float("inf")
        logits[i] = z
    state = {"case": case, "labels": labels}
    train = kind != "logprobs" or case["train"]
    state["logits"] = logits.requires_grad_(train)
    if kind in ("logprobs", "preference"):
        state["labels"] = torch.where(counted, labels, -100)
    else:
        state["mask"] = counted if case["padded"] else None
    if kind == "logprobs":
        state["grad"] = _loss_scale(case) * torch.randn(N, T, generator=g, device=DEV)
        return state
    if kind == "preference":
        state["ref"] = torch.empty(N, T, device=DEV)
        state["grad"] = torch.full((N // 2,), 2.0 / N * _loss_scale(case), device=DEV)
    if kind == "policy":
        state["old"], state["ref"] = torch.empty(N, T, device=DEV), None
        state["advantages"] = torch.randn(N, generator=g, device=DEV)
        if case["kl"]:
            state["ref"] = torch.empty(N, T, device=DEV)
    if kind == "distill":
        k = min(case["top"], used)
        state["index"] = torch.empty(N, T, k, dtype=torch.int64, device=DEV)
        state["teacher"] = torch.empty(N, T, k, device=DEV)
        for i in range(N):  # a teacher that differs from the student by about one unit
            z = logits[i].detach().float()
            z = z + torch.randn(T, V, generator=g, device=DEV)
            state["teacher"][i], state["index"][i] = torch.topk(z, k, dim=-1)
    if kind in ("policy", "preference"):
        for i in range(N):
            lp = _log_softmax64(logits[i].detach(), case["temperature"]).gather(-1, labels[i].unsqueeze(-1)).squeeze(-1)
            if kind == "policy":
                # the policy a few updates ago; no ratio lies so near to a clipping border that 32 bits cannot say on
                # which side
                ratio = 0.2 * torch.randn(T, generator=g, device=DEV).double()
                for border in (math.log(0.8), math.log(1.2)):
                    near = (ratio - border).abs() < 1e-3
                    ratio = torch.where(near, border + torch.where(ratio >= border, 1e-3, -1e-3), ratio)
                state["old"][i] = (lp - ratio).float()
            if state["ref"] is not None:
                state["ref"][i] = (lp + 0.3 * torch.randn(T, generator=g, device=DEV)).float()
    if kind != "preference":
        shape = {"none": (N, T), "sequence": (N,), "mean": ()}[case["reduction"]]
        per = {"none": N * T, "sequence": N, "mean": 1}[case["reduction"]] * case["steps"]
        state["grad"] = torch.full(shape, _loss_scale(case) / per, device=DEV)
    return state


# ------------------------------------------------------------------------- plain forms


def _rows(state):
    """exp((z - max) / temperature) and its sum, (z - max) / temperature, all in 32 bits."""
    y = state["logits"].detach().float()
    y = (y - y.amax(-1, keepdim=True)) / state["case"]["temperature"]
    e = torch.exp(y)
    return y, e, e.sum(-1, keepdim=True)


def _logps(y, total, labels):
    """(log-probability of each label in total's type, which of them count, the labels with 0 in the place of others)"""
    counted = (labels >= 0) & (labels < y.shape[-1])
    at = torch.where(counted, labels, 0)
    lp = y.gather(-1, at.unsqueeze(-1)).squeeze(-1).to(total.dtype) - torch.log(total).squeeze(-1)
    return torch.where(counted, lp, 0.0), counted, at


def _logps_grad(state, e, total, at, coef):
    """coef [N, T]: the loss's derivative by each label's log-probability."""
    grad = e * (-coef.unsqueeze(-1) / total)
    grad.scatter_add_(-1, at.unsqueeze(-1), coef.unsqueeze(-1))
    return (grad / state["case"]["temperature"]).to(state["logits"].dtype)


def _plain_logprobs(state):
    y, e, total = _rows(state)
    lp, counted, at = _logps(y, total, state["labels"])
    if not state["case"]["train"]:
        return lp
    return {"logps": lp, "logits_grad": _logps_grad(state, e, total, at, torch.where(counted, state["grad"], 0.0))}


def _plain_preference(state):
    case = state["case"]
    y, e, total = _rows(state)
    # in 64 bits: the differences of long sums are small beside the sums
    lp, counted, at = _logps(y, e.sum(-1, keepdim=True, dtype=torch.float64), state["labels"])
    each = counted.double().sum(-1).clamp(min=1) if case["average"] else torch.ones(lp.shape[0], device=DEV).double()
    ratio = torch.where(counted, lp - state["ref"].double(), 0.0).sum(-1) / each
    B, beta = lp.shape[0] // 2, case["beta"]
    d = ratio[:B] - ratio[B:]
    h = beta * d
    if case["loss"] == "sigmoid":
        loss = (1 - case["smoothing"]) * torch.log1p(torch.exp(-h)) + case["smoothing"] * torch.log1p(torch.exp(h))
        slope = beta * (case["smoothing"] / (1 + torch.exp(-h)) - (1 - case["smoothing"]) / (1 + torch.exp(h)))
    elif case["loss"] == "hinge":
        loss = (1 - h).clamp(min=0)
        slope = torch.where(h < 1, -beta, 0.0)
    else:
        loss = (d - 1 / (2 * beta)) ** 2
        slope = 2 * (d - 1 / (2 * beta))
    slope = slope * state["grad"].double()
    coef = (torch.cat([slope, -slope]) / each).float().unsqueeze(-1) * counted
    return {"loss": loss.float(), "rewards": (beta * ratio).float(),
            "logits_grad": _logps_grad(state, e, total, at, coef)}


def _reduced(state, each, counted):
    """(the reduced loss, the derivative of what is differentiated by each token's loss)"""
    reduction, grad = state["case"]["reduction"], state["grad"]
    each = torch.where(counted, each, 0.0)
    if reduction == "none":
        return each, grad * counted
    if reduction == "sequence":
        n = counted.sum(-1).clamp(min=1)
        return (each.double().sum(-1) / n).float(), (grad / n).unsqueeze(-1) * counted
    n = counted.sum().clamp(min=1)
    return (each.double().sum() / n).float(), grad / n * counted


def _plain_policy(state):
    case = state["case"]
    y, e, total = _rows(state)
    labels = state["labels"] if state["mask"] is None else torch.where(state["mask"], state["labels"], -1)
    lp, counted, at = _logps(y, total, labels)
    ratio = torch.exp(lp - state["old"])
    adv = state["advantages"].unsqueeze(-1)
    clipped = ratio.clamp(0.8, 1.2)
    each = -torch.minimum(ratio * adv, clipped * adv)
    slope = torch.where(ratio * adv <= clipped * adv, -adv * ratio, 0.0)
    if case["kl"]:
        away = state["ref"] - lp
        each = each + case["kl"] * (torch.exp(away) - away - 1)
        slope = slope + case["kl"] * (1 - torch.exp(away))
    loss, by = _reduced(state, each, counted)
    return {"loss": loss, "logps": lp, "logits_grad": _logps_grad(state, e, total, at, slope * by)}


def _plain_distill(state):
    t = state["case"]["temperature"]
    y, e, total = _rows(state)
    counted = torch.ones(y.shape[:2], dtype=torch.bool, device=DEV) if state["mask"] is None else state["mask"]
    w = state["teacher"]
    w = (w - w.amax(-1, keepdim=True)) / t
    p = torch.exp(w)
    norm = p.sum(-1, keepdim=True)
    p = p / norm
    away = (w - torch.log(norm)) - (y.gather(-1, state["index"]) - torch.log(total))
    each = t * t * torch.where(p > 0, p * away, 0.0).sum(-1)
    loss, by = _reduced(state, each, counted)
    by = by.unsqueeze(-1)
    grad = torch.where(counted.unsqueeze(-1), e * (t * by / total), 0.0)
    grad.scatter_add_(-1, state["index"], -t * by * p)
    return {"loss": loss, "logits_grad": grad.to(state["logits"].dtype)}


_PLAIN = {"logprobs": _plain_logprobs, "preference": _plain_preference, "policy": _plain_policy, "distill": _plain_distill}


def run(state):
    case = state["case"]
    kind = case["kind"]
    if not own:
        with torch.no_grad():
            return _PLAIN[kind](state)
    import experts4bit_qlora_amd as e4b

    logits, t = state["logits"], case["temperature"]
    if kind == "logprobs":
        logps = e4b.token_logprobs(logits, state["labels"], temperature=t)
        if not case["train"]:
            return logps
        (grad,) = torch.autograd.grad(logps, logits, state["grad"])
        return {"logps": logps.detach(), "logits_grad": grad}
    if kind == "preference":
        loss, rewards = e4b.preference_loss(logits, state["labels"], state["ref"], beta=case["beta"],
                                            loss_type=case["loss"], label_smoothing=case["smoothing"],
                                            average=case["average"])
        (grad,) = torch.autograd.grad(loss, logits, state["grad"])
        return {"loss": loss.detach(), "rewards": rewards, "logits_grad": grad}
    if kind == "policy":
        loss, logps = e4b.policy_loss(logits, state["labels"], state["old"], state["advantages"], ref_logps=state["ref"],
                                      clip=(0.2, 0.2), kl_coef=case["kl"], mask=state["mask"], temperature=t,
                                      reduction=case["reduction"])
        (grad,) = torch.autograd.grad(loss, logits, state["grad"])
        return {"loss": loss.detach(), "logps": logps, "logits_grad": grad}
    loss = e4b.distill_loss(logits, state["teacher"], state["index"], mask=state["mask"], temperature=t,
                            reduction=case["reduction"])
    (grad,) = torch.autograd.grad(loss, logits, state["grad"])
    return {"loss": loss.detach(), "logits_grad": grad}


def work(case):
    N, T, V = case["seqs"], case["tokens"], case["vocab"]
    rows = sum(b - a for a, b in _spans(case))
    b = DTYPES[case["dtype"]].itemsize
    train = case["kind"] != "logprobs" or case["train"]
    # the counted rows' logits in, every row's gradient out; what a token has beside its logits
    beside = {"logprobs": 8 + 4 + (4 if train else 0), "preference": 12, "policy": 8 + 4 + 4 + (4 if case.get("kl") else 0),
              "distill": 12 * case.get("top", 0)}[case["kind"]]
    return {"bytes": float(rows * V * b + (N * T * V * b if train else 0) + N * T * beside),
            "flops": (8.0 if train else 4.0) * rows * V}


# ----------------------------------------------------------------------- 64-bit results


def _exact_terms(case, state, i, z, counted):
    """(each token's log-probability or loss, its loss) of sequence i as differentiable functions of z."""
    lsm = torch.log_softmax(z / case["temperature"], -1)
    if case["kind"] == "distill":
        t = case["temperature"]
        p = torch.softmax(state["teacher"][i].double() / t, -1)
        cross = -(p * lsm.gather(-1, state["index"][i])).sum(-1)
        entropy = -(p * torch.log(p.clamp(min=1e-300))).sum(-1)
        return None, torch.where(counted, t * t * (cross - entropy), 0.0)
    at = torch.where(counted, state["labels"][i], 0)
    lp = torch.where(counted, lsm.gather(-1, at[:, None])[:, 0], 0.0)
    if case["kind"] != "policy":
        return lp, lp
    a = state["advantages"][i].double()
    r = torch.exp(lp - state["old"][i].double())
    lower, upper = 0.8, 1.2
    gain = a * r.clamp(max=upper) if float(a) >= 0 else a * r.clamp(min=lower)
    each = -gain
    if case["kl"]:
        x = state["ref"][i].double() - lp
        each = each + case["kl"] * (torch.expm1(x) - x)
    return lp.detach(), torch.where(counted, each, 0.0)


def exact(case, seed):
    state = prepare(case, seed)
    N, T, kind = case["seqs"], case["tokens"], case["kind"]
    counted = _counted(case, seed)
    train = kind != "logprobs" or case["train"]
    grads = torch.empty(state["logits"].shape, dtype=torch.float64 if N * T * case["vocab"] < 2 ** 31 else torch.float32,
                        device=DEV) if train else None
    n = counted.double().sum(-1)
    slope = None
    if kind == "preference":  # first every sequence's sum, then its gradient
        each = n.clamp(min=1) if case["average"] else torch.ones_like(n)
        with torch.no_grad():
            sums = torch.stack([_exact_terms(case, state, i, state["logits"][i].double(), counted[i])[0].sum()
                                for i in range(N)])
        ratio = ((sums - (state["ref"].double() * counted).sum(-1)) / each).requires_grad_()
        d = ratio[:N // 2] - ratio[N // 2:]
        if case["loss"] == "sigmoid":
            ls = torch.nn.functional.logsigmoid
            loss = -(1 - case["smoothing"]) * ls(case["beta"] * d) - case["smoothing"] * ls(-case["beta"] * d)
        elif case["loss"] == "hinge":
            loss = torch.relu(1 - case["beta"] * d)
        else:
            loss = (d - 0.5 / case["beta"]).square()
        (slope,) = torch.autograd.grad(loss, ratio, state["grad"].double())
        slope = slope / each
    tokens, logps = [], []
    for i in range(N):
        z = state["logits"][i].detach().double().requires_grad_(train)
        lp, each_token = _exact_terms(case, state, i, z, counted[i])
        if train:
            if kind == "preference":
                by = slope[i].expand(T)
            elif kind == "logprobs" or case["reduction"] == "none":
                by = state["grad"][i].double()
            elif case["reduction"] == "sequence":
                by = (state["grad"][i].double() / n[i].clamp(min=1)).expand(T)
            else:
                by = (state["grad"].double() / n.sum().clamp(min=1)).expand(T)
            (grads[i],) = torch.autograd.grad(each_token, z, by * counted[i])
        tokens.append(each_token.detach())
        logps.append(lp if lp is None else lp.detach())
    if kind == "logprobs":
        return {"logps": torch.stack(logps), "logits_grad": grads} if train else torch.stack(logps)
    if kind == "preference":
        return {"loss": loss.detach(), "rewards": case["beta"] * ratio.detach(), "logits_grad": grads}
    tokens = torch.stack(tokens)
    loss = {"none": tokens, "sequence": tokens.sum(-1) / n.clamp(min=1), "mean": tokens.sum() / n.sum().clamp(min=1)}
    out = {"loss": loss[case["reduction"]], "logps": torch.stack(logps) if kind == "policy" else None, "logits_grad": grads}
    return out if kind == "policy" else {"loss": out["loss"], "logits_grad": grads}
