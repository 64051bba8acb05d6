"""The operators around the expert products, as a user's program calls them: one dict per case.

``listed()`` names the measured cases, ``draw()`` gives more of the same ranges; ``prepare()`` makes
what a program holds before the call, ``run()`` is one pass through one operator, ``exact()`` the same
values in 64 bits.

Four kinds of pass:

* ``quantize``: dense rows to microscaled 4-bit floating point (e2m1 values, one e8m0 scale per 32),
  returned as the values that the codes and scales stand for.
* ``product``: rows of 16-bit activations, grouped by expert, quantised the same way and multiplied by
  the experts' microscaled weights.
* ``gate``: router logits to the chosen experts and their weights; in training also the logits' gradient.
* ``balance``: the load-balance loss and the per-expert counts, and the logits' gradient.
"""
import math

import torch

own = False  # True: run() calls the framework's operators instead of their plain forms

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _case(kind, name=None, **kw):
    c = {"kind": kind, "dtype": "bf16", **kw}
    return c if name is None else {"name": name, **c}


def listed():
    return [
        # the hidden states of five sequences in a decode step
        _case("quantize", "quantize_5_rows", rows=5, k=2880),
        # loading: one layer's dense gate and up projections of 32 experts
        _case("quantize", "quantize_experts", rows=32 * 5760, k=2880),
        # one token's four experts, gate and up: a decode step, bound by the weights
        _case("product", "product_1_token", tokens=1, top_k=4, experts=32, n=5760, k=2880, zipf=0.0),
        # a serving batch of an odd size through the down projections, fp16 model
        _case("product", "product_37_tokens", tokens=37, top_k=4, experts=32, n=2880, k=2880, zipf=0.0, dtype="fp16"),
        # a prompt of odd length, skewed expert popularity, a small layer whose sizes are not whole tiles
        _case("product", "product_1531_tokens", tokens=1531, top_k=4, experts=16, n=1408, k=1216, zipf=1.1),
        # a long prompt through gate and up
        _case("product", "product_4096_tokens", tokens=4096, top_k=4, experts=32, n=5760, k=2880, zipf=0.0),
        # one token's router: top-k, then the softmax over the chosen logits
        _case("gate", "gate_1_token", tokens=1, experts=32, top_k=4, scoring="topk_then_softmax", renorm=False,
              train=False),
        # a prompt of odd length, fp32 logits
        _case("gate", "gate_1531_tokens", tokens=1531, experts=64, top_k=8, scoring="softmax_then_topk", renorm=False,
              train=False, dtype="fp32"),
        # one training micro-batch: renormalised weights and the logits' gradient
        _case("gate", "gate_train_8192", tokens=8192, experts=128, top_k=8, scoring="softmax_then_topk", renorm=True,
              train=True),
        # one layer of a short padded batch
        _case("balance", "balance_509_tokens", layers=1, tokens=509, experts=128, top_k=8, padded=True),
        # the 16 layers of a training step
        _case("balance", "balance_16_layers", layers=16, tokens=8192, experts=64, top_k=8, padded=False),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("quantize", "product", "product", "gate", "balance"))
    if kind == "quantize":
        return _case(kind, rows=_log_int(rng, 1, 100000), k=64 * _log_int(rng, 1, 64),
                     dtype=rng.choice(("bf16", "bf16", "fp16", "fp32")))
    if kind == "product":
        experts = rng.choice((4, 8, 16, 32))
        return _case(kind, tokens=_log_int(rng, 1, 4096), top_k=rng.randint(1, 4), experts=experts,
                     n=_log_int(rng, 48, 5760), k=32 * _log_int(rng, 2, 90), zipf=rng.choice((0.0, 0.6, 1.1)),
                     dtype=rng.choice(("bf16", "bf16", "fp16")))
    experts = rng.choice((8, 16, 32, 60, 64, 96, 128, 256))
    if kind == "gate":
        scoring = rng.choice(("softmax_then_topk", "softmax_then_topk", "topk_then_softmax"))
        return _case(kind, tokens=_log_int(rng, 1, 16384), experts=experts, top_k=rng.randint(1, 8), scoring=scoring,
                     renorm=scoring == "softmax_then_topk" and rng.random() < 0.5, train=rng.random() < 0.6,
                     dtype=rng.choice(("bf16", "bf16", "fp16", "fp32")))
    return _case(kind, layers=rng.randint(1, 16), tokens=_log_int(rng, 16, 8192), experts=min(experts, 128),
                 top_k=rng.randint(1, 8), padded=rng.random() < 0.5, dtype=rng.choice(("bf16", "bf16", "fp32")))


# ------------------------------------------------------------------------------ inputs


def _gen(seed, part=0):
    return torch.Generator(device=DEV).manual_seed(1000 * seed + part)


def _rows(rows, k, dtype, g):
    """Hidden states: normal values, a few channels much larger than the rest, rows of different size."""
    channel = torch.where(torch.rand(k, generator=g, device=DEV) < 0.01, 8.0, 1.0)
    size = torch.exp(0.5 * torch.randn(rows, 1, generator=g, device=DEV))
    return (torch.randn(rows, k, generator=g, device=DEV) * channel * size).to(DTYPES[dtype])


def _group_sizes(case, seed):
    """Rows per expert of a batch whose tokens each choose top_k different experts (host integers)."""
    E, T, k = case["experts"], case["tokens"], case["top_k"]
    g = torch.Generator().manual_seed(1000 * seed + 1)
    popular = -case["zipf"] * torch.log((torch.randperm(E, generator=g) + 1).float())
    noise = -torch.log(-torch.log(torch.rand(T, E, generator=g).clamp(1e-9, 1 - 1e-7)))
    chosen = torch.topk(popular + noise, k, dim=-1).indices
    counts = torch.bincount(chosen.reshape(-1), minlength=E).tolist()
    ids = [e for e in range(E) if counts[e]]
    return [counts[e] for e in ids], ids


def _stored_weights(case, seed):
    """e2m1 bytes ``[E, n, k/2]`` (low nibble first) and e8m0 scales ``[E, n, k/32]`` of normal weights."""
    E, n, k = case["experts"], case["n"], case["k"]
    mids = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], device=DEV)
    blocks = torch.empty(E, n, k // 2, dtype=torch.uint8, device=DEV)
    scales = torch.empty(E, n, k // 32, dtype=torch.uint8, device=DEV)
    g = _gen(seed, 2)
    for e0 in range(0, E, 8):
        w = torch.randn(min(8, E - e0), n, k // 32, 32, generator=g, device=DEV) * 0.02
        x = torch.floor(torch.log2(w.abs().amax(-1))) - 2
        w = torch.ldexp(w, -x.unsqueeze(-1))
        q = torch.bucketize(w.abs(), mids, out_int32=True).to(torch.uint8) | ((w < 0).to(torch.uint8) << 3)
        blocks[e0:e0 + 8] = ((q[..., 1::2] << 4) | q[..., 0::2]).reshape(-1, n, k // 2)
        scales[e0:e0 + 8] = (x + 127).to(torch.uint8)
    return blocks, scales


def _logits(case, shape, seed):
    """Router logits: a popularity of each expert, the token's own part."""
    g = _gen(seed, 3)
    popular = 0.7 * torch.randn(*shape[:-2], 1, shape[-1], generator=g, device=DEV)
    return (popular + torch.randn(*shape, generator=g, device=DEV)).to(DTYPES[case["dtype"]])


def _chosen(z, k):
    """The k largest of each row, in descending order, ties to the lower index."""
    return torch.sort(z, dim=-1, descending=True, stable=True).indices[..., :k]


def prepare(case, seed):
    state = {"case": case}
    if case["kind"] == "quantize":
        state["x"] = _rows(case["rows"], case["k"], case["dtype"], _gen(seed))
    elif case["kind"] == "product":
        sizes, ids = _group_sizes(case, seed)
        state["sizes"], state["ids"] = sizes, torch.tensor(ids, device=DEV)
        state["x"] = _rows(sum(sizes), case["k"], case["dtype"], _gen(seed))
        state["blocks"], state["scales"] = _stored_weights(case, seed)
    elif case["kind"] == "gate":
        state["logits"] = _logits(case, (case["tokens"], case["experts"]), seed).requires_grad_(case["train"])
        state["grad"] = torch.randn(case["tokens"], case["top_k"], generator=_gen(seed, 4), device=DEV).to(
            DTYPES[case["dtype"]])
    else:
        L, T = case["layers"], case["tokens"]
        logits = _logits(case, (L, T, case["experts"]), seed)
        state["logits"] = logits.requires_grad_()
        state["index"] = _chosen(logits.detach().float(), case["top_k"])
        state["mask"] = torch.arange(T, device=DEV) < T - T // 5 if case["padded"] else None
        state["grad"] = torch.rand(L, generator=_gen(seed, 4), device=DEV) + 0.5
    return state


# ------------------------------------------------------------------------- plain forms


def _e2m1(x, wide):
    """Rows ``[..., k]`` as the microscaled values they round to (in ``wide``'s type) and their scales."""
    v = x.to(wide).reshape(*x.shape[:-1], -1, 32)
    amax = v.abs().amax(-1, keepdim=True)
    exponent = (torch.frexp(amax).exponent - 3).clamp(-127, 127)
    exponent = torch.where(amax > 0, exponent, torch.full_like(exponent, -127))
    v = torch.ldexp(v, -exponent)
    a = v.abs()
    # the grid's step is 0.5 up to 2, then 1 up to 4, then 2 up to its largest value, 6
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0)).to(wide)
    a = (torch.round(a / step) * step).clamp(max=6)
    return torch.ldexp(torch.copysign(a, v), exponent).reshape(x.shape)


def _weights32(blocks, scales):
    table = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0],
                         device=blocks.device)
    codes = torch.stack([blocks & 15, blocks >> 4], -1).int()
    v = table[codes].reshape(*scales.shape, 32)
    return torch.ldexp(v, (scales.int() - 127).unsqueeze(-1)).reshape(*scales.shape[:-1], -1)


def _product(state):
    """Every group padded to the longest: one product over (group, row)."""
    x, sizes = state["x"], torch.tensor(state["sizes"], device=DEV)
    a = _e2m1(x, torch.float32)
    w = _weights32(state["blocks"][state["ids"]], state["scales"][state["ids"]])
    first = torch.cumsum(sizes, 0) - sizes
    at = torch.arange(max(state["sizes"]), device=DEV)
    rows = first[:, None] + at[None, :]
    held = at[None, :] < sizes[:, None]
    padded = a[torch.where(held, rows, 0)]
    return torch.matmul(padded, w.transpose(1, 2).contiguous())[held].to(x.dtype)


def _softmax(z):
    e = torch.exp(z - z.amax(-1, keepdim=True))
    return e / e.sum(-1, keepdim=True)


def _gate(state):
    case, logits = state["case"], state["logits"].detach()
    z = logits.float()
    index = _chosen(z, case["top_k"])
    over_chosen = case["renorm"] or case["scoring"] == "topk_then_softmax"
    if over_chosen:
        w = _softmax(torch.gather(z, -1, index))
    else:
        p = _softmax(z)
        w = torch.gather(p, -1, index)
    if not case["train"]:
        return {"index": index, "weights": w.to(logits.dtype)}
    g = state["grad"].float()
    mean = (g * w).sum(-1, keepdim=True)
    if over_chosen:
        grad = torch.zeros_like(z).scatter(-1, index, w * (g - mean))
    else:
        grad = p * (torch.zeros_like(z).scatter(-1, index, g) - mean)
    return {"index": index, "weights": w.to(logits.dtype), "logits_grad": grad.to(logits.dtype)}


def _balance(state):
    logits, index, mask = state["logits"].detach(), state["index"], state["mask"]
    L, T, E = logits.shape
    p = _softmax(logits.float())
    m = torch.ones(T, device=DEV) if mask is None else mask.float()
    n = m.sum()
    each = m.long()[None, :, None].expand(index.shape).reshape(L, -1)
    counts = torch.zeros(L, E, dtype=torch.int64, device=DEV).scatter_add(1, index.reshape(L, -1), each)
    share = (p * m[:, None]).sum(1)
    loss = E * (counts / n * (share / n)).sum(-1)
    c = counts.float()[:, None, :]
    grad = state["grad"][:, None, None] * m[:, None] * (E / (n * n)) * p * (c - (c * p).sum(-1, keepdim=True))
    return {"loss": loss, "counts": counts, "logits_grad": grad.to(logits.dtype)}


def run(state):
    case = state["case"]
    kind = case["kind"]
    if own:
        import experts4bit_qlora_amd as e4b
        from experts4bit_qlora_amd import ops

        if kind == "quantize":
            rows, k = case["rows"], case["k"]
            blocks, scales = e4b.quantize_mxfp4(state["x"])
            return ops.dequant(ops.mxfp4_qweight(blocks, scales, rows, k, num_experts=1), dtype=state["x"].dtype)[0]
        if kind == "product":
            return e4b.gemm_mxfp4_grouped(state["x"], state["blocks"], state["scales"], state["sizes"], state["ids"],
                                          act_quant="mxfp4")
        if kind == "gate":
            index, weights = e4b.router_topk(state["logits"], case["top_k"], scoring=case["scoring"],
                                             renorm=case["renorm"])
            if not case["train"]:
                return {"index": index, "weights": weights}
            (grad,) = torch.autograd.grad(weights, state["logits"], state["grad"])
            return {"index": index, "weights": weights.detach(), "logits_grad": grad}
        loss, counts = e4b.balance_loss(state["logits"], state["index"], mask=state["mask"])
        (grad,) = torch.autograd.grad(loss, state["logits"], state["grad"])
        return {"loss": loss.detach(), "counts": counts, "logits_grad": grad}
    with torch.no_grad():
        if kind == "quantize":
            return _e2m1(state["x"], torch.float32).to(state["x"].dtype)
        if kind == "product":
            return _product(state)
        return _gate(state) if kind == "gate" else _balance(state)


def work(case):
    b = DTYPES[case["dtype"]].itemsize
    if case["kind"] == "quantize":  # the rows in, the values out
        n = case["rows"] * case["k"]
        return {"bytes": 2.0 * n * b, "flops": 3.0 * n}
    if case["kind"] == "product":  # rows in and out, the chosen experts' stored weights
        E, k, T = case["experts"], case["top_k"], case["tokens"]
        p = [1.0 / (e + 1) ** case["zipf"] for e in range(E)]
        hit = sum(1 - (1 - min(1.0, k * v / sum(p))) ** T for v in p)
        rows = T * k
        return {"bytes": hit * case["n"] * case["k"] * 17 / 32 + rows * (case["k"] + case["n"]) * b,
                "flops": 2.0 * rows * case["n"] * case["k"]}
    E, k = case["experts"], case["top_k"]
    if case["kind"] == "gate":
        T = case["tokens"]
        once = T * E * b + T * k * (8 + b)  # logits and the chosen experts with their weights
        # the gradient's pass has the weights' gradient and the index in, the logits' gradient out
        return {"bytes": once + (2 * T * E * b + T * k * (8 + b) if case["train"] else 0),
                "flops": (10.0 if case["train"] else 5.0) * T * E}
    T = case["layers"] * case["tokens"]
    return {"bytes": 3 * T * E * b + T * k * 8, "flops": 12.0 * T * E}


# ----------------------------------------------------------------------- 64-bit results


def _round64(x):
    """A row's microscaled values by the nearest entry of the grid (its even one at a tie), in 64 bits."""
    v = x.double().reshape(-1, 32)
    amax = v.abs().amax(-1)
    top = torch.where(amax > 0, amax, 1.0)
    power = torch.pow(2.0, torch.floor(torch.log2(top)))
    power = torch.where(power > top, power / 2, torch.where(2 * power <= top, 2 * power, power))  # log2 rounds
    scale = torch.where(amax > 0, (power / 4).clamp(2.0 ** -127, 2.0 ** 127), 1.0)[:, None]
    v = v / scale
    grid = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64, device=x.device)
    best = torch.zeros_like(v)
    for i in range(1, 8):
        middle = (grid[i - 1] + grid[i]) / 2
        up = (v.abs() >= middle) if i % 2 == 0 else (v.abs() > middle)
        best = torch.where(up, grid[i], best)
    return (torch.sign(v) * best * scale).reshape(x.shape)


def _weights64(blocks, scales):
    """[n, k] from an expert's bytes: sign, two exponent bits, one bit of fraction."""
    c = torch.stack([blocks & 15, blocks >> 4], -1).reshape(blocks.shape[0], -1).double()
    sign = 1 - 2 * torch.floor(c / 8)
    e, f = torch.floor(c / 2) % 4, c % 2
    v = sign * torch.where(e > 0, torch.pow(2.0, e - 1) * (1 + f / 2), f / 2)
    return v * torch.pow(2.0, scales.double() - 127).repeat_interleave(32, dim=1)


def exact(case, seed):
    state = prepare(case, seed)
    with torch.no_grad():
        if case["kind"] == "quantize":
            return torch.cat([_round64(x) for x in state["x"].split(32768)])
        if case["kind"] == "product":
            out = []
            for x, e in zip(state["x"].split(state["sizes"]), state["ids"].tolist()):
                out.append(_round64(x) @ _weights64(state["blocks"][e], state["scales"][e]).T)
            return torch.cat(out)
        z = state["logits"].detach().double()
        p = torch.softmax(z, -1)
        if case["kind"] == "gate":
            index = torch.argsort(-z, dim=-1, stable=True)[:, :case["top_k"]]
            picked = torch.zeros_like(z).scatter(-1, index, 1.0)
            over_chosen = case["renorm"] or case["scoring"] == "topk_then_softmax"
            q = p * picked / (p * picked).sum(-1, keepdim=True) if over_chosen else p
            w = q.gather(-1, index)
            if not case["train"]:
                return {"index": index, "weights": w}
            g = state["grad"].double()
            toward = torch.zeros_like(z).scatter(-1, index, g)
            # the softmax's derivative, diag(q) - q q^T, applied to the weights' gradient
            grad = q * toward - q * (q * toward).sum(-1, keepdim=True)
            return {"index": index, "weights": w, "logits_grad": grad}
        L, T, E = z.shape
        valid = torch.ones(T, dtype=torch.bool, device=DEV) if state["mask"] is None else state["mask"]
        n = int(valid.sum())
        counts = torch.stack([torch.bincount(i[valid].reshape(-1), minlength=E) for i in state["index"]])
        f = counts.double() / n
        loss = E * (f * p[:, valid].mean(1)).sum(-1)
        f = f[:, None, :]
        grad = E / n * p * (f - (f * p).sum(-1, keepdim=True)) * valid[:, None] * state["grad"].double()[:, None, None]
        return {"loss": loss, "counts": counts, "logits_grad": grad}
