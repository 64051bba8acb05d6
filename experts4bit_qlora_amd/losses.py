"""Losses over the vocabulary's logits, with gradients: what the adapters of a training lane learn from.

``token_logprobs`` (the log-probability of each label: what serving reports for a generated token, and what the losses take
from an older or a reference model), ``preference_loss`` (paired log ratios of chosen and rejected answers),
``policy_loss`` (clipped ratios with a KL term) and ``distill_loss`` (divergence from a teacher's top logits). On a HIP
device each reads the logits once forward and once backward (``csrc/losses.h``) and keeps a few floats per token
between; tensors elsewhere, other dtypes, sizes beyond the kernels' limits, tensors that a trace or forward-mode differentiation
follows, and all calls inside a transform (``torch.func``) or a recording (``make_fx``) take the torch formulation, which is
the definition.

Logits are ``[..., tokens, vocab]``; the leading axes are sequences. They may be a view whose rows lie at any stride
(``logits[:, :-1]`` is not copied). The gradient of such a view is copied into the whole's by autograd: shifting the
labels instead (the last one ``-100``) saves that. A token counts iff its mask is nonzero (where a mask is given) and, in
the three losses with labels, its label is inside ``[0, vocab)``; other tokens' logits have no influence, whatever they
are, and get a zero gradient. A row whose logits are all ``-inf`` gives every label probability 0 and gets a zero
gradient. Everything but the logits is a constant to the gradient. A backward pass is captured into a graph like any other of
torch's: with no eager graph of the same leaves alive.

The reference has no losses of its own (its training lane starts at a model's, ``experts4bit_qlora/engines/fast.py:453-674``).
"""
from __future__ import annotations

import math

import torch

from . import _native as N
from . import ops
from .quant import _forward_ad
from .router import _on_kernel

_PREFERENCE = {"sigmoid": N.PREFERENCE_SIGMOID, "hinge": N.PREFERENCE_HINGE, "ipo": N.PREFERENCE_IPO}
_REDUCTION = {"none": N.REDUCE_NONE, "sequence": N.REDUCE_SEQUENCE, "mean": N.REDUCE_MEAN}
_MAX_TOP = 1024


# ------------------------------------------------------------------------------- arguments


def _sequences(logits: torch.Tensor):
    """(logits as ``[seqs, tokens, vocab]``, their shape up to the vocabulary)"""
    shape = logits.shape
    if len(shape) < 2 or not shape[-1] or not logits.is_floating_point():
        raise ValueError("logits must be a floating-point tensor [..., tokens, vocab]")
    if len(shape) == 3:
        return logits, shape[:2]
    z = logits.unsqueeze(0) if len(shape) == 2 else logits.reshape(shape[:-2].numel(), *shape[-2:])
    return z, shape[:-1]


def _integers(name: str, t: torch.Tensor, logits: torch.Tensor, shape) -> None:
    if t.shape != shape or t.is_floating_point() or t.is_complex() or t.dtype == torch.bool:
        raise ValueError(f"{name} must be integers {list(shape)}, got {t.dtype} {list(t.shape)}")
    if t.device != logits.device:
        raise ValueError(f"logits and {name} must be on one device")


def _floats(name: str, t: torch.Tensor, logits: torch.Tensor, *shapes) -> None:
    if t.shape not in shapes or not t.is_floating_point():
        raise ValueError(f"{name} must be floating-point {' or '.join(str(list(s)) for s in shapes)}, got {t.dtype} "
                         f"{list(t.shape)}")
    if t.device != logits.device:
        raise ValueError(f"logits and {name} must be on one device")


def _mask(mask, logits: torch.Tensor, shape):
    """The mask as bool ``[tokens]`` or ``[seqs, tokens]``, or None."""
    if mask is None:
        return None
    if mask.shape != shape and mask.shape != shape[-1:]:
        raise ValueError(f"mask must be {list(shape[-1:])} or {list(shape)}, got {list(mask.shape)}")
    if mask.device != logits.device:
        raise ValueError("logits and mask must be on one device")
    if mask.dtype != torch.bool:
        mask = mask != 0
    return mask if mask.dim() <= 2 else mask.reshape(shape[:-1].numel(), shape[-1])


def _temperature(t: float, logits: torch.Tensor) -> float:
    if not (t > 0 and math.isfinite(t)):
        raise ValueError(f"temperature={t} is not positive and finite")
    if not 2.0 ** -126 <= t <= 2.0 ** 126 and logits.dtype != torch.float64:  # rows are divided by it in fp32
        raise ValueError(f"temperature={t}: it or its inverse is not a normal fp32 number")
    return float(t)


def _reduction(name: str) -> int:
    if name not in _REDUCTION:
        raise ValueError(f"reduction must be one of {sorted(_REDUCTION)}, got {name!r}")
    return _REDUCTION[name]


_MODE = torch._C._TorchDispatchModeKey


def _recorded() -> bool:
    """Whether torch's operators are recorded or stood in for, which leaves out what a kernel does."""
    mode = torch._C._get_dispatch_mode
    return torch._C._len_torch_dispatch_stack() > 0 and any(mode(k) is not None for k in (_MODE.PROXY, _MODE.FAKE,
                                                                                         _MODE.FUNCTIONAL))


def _fits(z: torch.Tensor, temperature: float, *others) -> bool:
    """Whether the kernels may take these: plain device tensors, in memory as they are to be read, within the limits of
    ``e4b_logits``."""
    if not _on_kernel(z) or z.is_neg():
        return False
    # transforms admit no autograd function of the extension, whatever it is given
    if torch._C._are_functorch_transforms_active() or _recorded():
        return False
    wrapped = torch._C._functorch.is_functorch_wrapped_tensor
    for t in others:
        if t is not None and (wrapped(t) or t.is_neg()):
            return False
    seqs, tokens, vocab = z.shape
    return seqs <= 2 ** 21 and seqs * tokens < 2 ** 31 and vocab <= 2 ** 30 and 1e-30 < temperature < 1e30


def _rows(z: torch.Tensor) -> torch.Tensor:
    return z if z.stride(2) == 1 or z.shape[2] == 1 else z.contiguous()


def _contiguous(mask):
    return mask if mask is None or mask.is_contiguous() else mask.contiguous()


def _constant(t, dtype, shape):
    """A constant of the gradient, contiguous and of one dtype (or None)."""
    if t is None:
        return None
    if t.requires_grad or _forward_ad._current_level >= 0:
        t = t.detach()
    if t.dtype != dtype:
        t = t.to(dtype)
    if t.shape != shape:
        t = t.reshape(shape)
    return t if t.is_contiguous() else t.contiguous()


# ----------------------------------------------------------------------- log-probabilities


def token_logprobs(logits: torch.Tensor, labels: torch.Tensor, mask: torch.Tensor | None = None,
                   temperature: float = 1.0) -> torch.Tensor:
    """Log-probability of each label under ``softmax(logits / temperature)``: logits ``[..., T, V]``, labels ``[..., T]``
    integers, mask ``[T]`` or ``[..., T]`` -> fp32 ``[..., T]`` (fp64 for fp64 logits), 0 where a token does not count.
    The temperature and its inverse are normal fp32 numbers (for fp64 logits: any positive finite one).
    Differentiable with respect to the logits (once)."""
    z, shape = _sequences(logits)
    _integers("labels", labels, logits, shape)
    m, t = _mask(mask, logits, shape), _temperature(temperature, logits)
    flat = z.shape[:2]
    if _fits(z, t, labels, m):
        logps = N.torch_lib().token_logprobs(_rows(z), _constant(labels, torch.int64, flat), _contiguous(m), t)
    else:
        logps = _token_logprobs_torch(z, labels.reshape(flat), m, t)[0]
    return logps if len(shape) == 2 else logps.view(shape)


def _wide(z: torch.Tensor) -> torch.Tensor:
    return z if z.dtype == torch.float64 else z.float()


def _log_softmax(z: torch.Tensor, counted: torch.Tensor, temperature: float) -> torch.Tensor:
    """Of rows that count, -inf throughout where all logits are; zeros' elsewhere."""
    z = torch.where(counted.unsqueeze(-1), _wide(z), 0.0)
    empty = (z == -math.inf).all(-1, keepdim=True)
    y = torch.where(empty, 0.0, z)
    y = (y - y.detach().amax(-1, keepdim=True)) / temperature
    return torch.log_softmax(y, -1).masked_fill(empty, -math.inf)


def _token_logprobs_torch(z, labels, mask, temperature):
    labels = labels.to(torch.int64)  # the vocabulary's size may lie outside their own type, where it would wrap
    counted = (labels >= 0) & (labels < z.shape[-1])
    if mask is not None:
        counted = counted & mask
    at = torch.where(counted, labels, 0).unsqueeze(-1)
    logps = _log_softmax(z, counted, temperature).gather(-1, at).squeeze(-1)
    return torch.where(counted, logps, 0.0), counted


# ------------------------------------------------------------------------------ preference


def preference_loss(logits: torch.Tensor, labels: torch.Tensor, ref_logps: torch.Tensor | None = None, beta: float = 0.1,
                    loss_type: str = "sigmoid", label_smoothing: float = 0.0, average: bool = False,
                    mask: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Preference loss of pairs: logits ``[2B, T, V]`` and labels ``[2B, T]``, the chosen answers in the first half and the
    rejected ones in the second -> ``(loss fp32 [B], rewards fp32 [2B])``.

    With ``S`` the sum of an answer's counted log-probabilities (``average``: their mean) and ``r`` the same under the
    reference model, ``d = (S_c - r_c) - (S_r - r_r)`` and ``h = beta d``: ``"sigmoid"`` ``-(1 - e) log sigmoid(h) - e
    log sigmoid(-h)`` with ``e = label_smoothing``, ``"hinge"`` ``max(0, 1 - h)``, ``"ipo"`` ``(d - 1 / (2 beta))^2``.
    ``ref_logps``: per token ``[2B, T]`` as ``token_logprobs`` gives them (the difference is then summed in 64 bits
    token by token), or the answers' sums (means) ``[2B]``, fp64 ones as they are; None: zeros. ``rewards = beta (S - r)``,
    constants to the gradient. The loss is differentiable with respect to the logits (once)."""
    if logits.dim() != 3 or logits.shape[0] % 2:
        raise ValueError(f"logits must be [2 * pairs, tokens, vocab], got {list(logits.shape)}")
    z, shape = _sequences(logits)
    _integers("labels", labels, logits, shape)
    if ref_logps is not None:
        _floats("ref_logps", ref_logps, logits, shape, shape[:1])
    if loss_type not in _PREFERENCE:
        raise ValueError(f"loss_type must be one of {sorted(_PREFERENCE)}, got {loss_type!r}")
    if not (beta > 0 and math.isfinite(beta)):
        raise ValueError(f"beta={beta} is not positive and finite")
    if not 0 <= label_smoothing <= 1:
        raise ValueError(f"label_smoothing={label_smoothing} outside [0, 1]")
    if label_smoothing and loss_type != "sigmoid":
        raise ValueError("label_smoothing belongs to loss_type='sigmoid'")
    m = _mask(mask, logits, shape)
    kind = _PREFERENCE[loss_type]
    if not (_fits(z, 1.0, labels, m, ref_logps) and 1e-30 < beta < 1e30):
        return _preference_loss_torch(z, labels, m, ref_logps, kind, beta, label_smoothing, average)
    ref = ref_logps
    if ref is not None:
        ref = _constant(ref, ref.dtype if ref.dtype == torch.float64 else torch.float32, ref.shape)
    return N.torch_lib().preference_loss(_rows(z), _constant(labels, torch.int64, shape), _contiguous(m), ref, kind, beta,
                                         label_smoothing, average)


def _preference_loss_torch(z, labels, mask, ref, kind, beta, smoothing, average):
    lp, counted = _token_logprobs_torch(z, labels, mask, 1.0)
    lp = lp.double()
    if ref is not None and ref.dim() == 2:
        lp = lp - torch.where(counted, ref.detach(), 0.0).double()
    ratio = lp.sum(-1)
    if average:
        ratio = ratio / counted.sum(-1).clamp(min=1)
    if ref is not None and ref.dim() == 1:
        ratio = ratio - ref.detach().double()
    d = ratio[:len(ratio) // 2] - ratio[len(ratio) // 2:]
    h = beta * d
    if kind == N.PREFERENCE_SIGMOID:
        loss = -(1 - smoothing) * torch.nn.functional.logsigmoid(h)
        if smoothing:
            loss = loss - smoothing * torch.nn.functional.logsigmoid(-h)
    elif kind == N.PREFERENCE_HINGE:
        loss = torch.relu(1 - h)
    else:
        loss = (d - 1 / (2 * beta)) ** 2
    dtype = _wide(z[:0]).dtype
    return loss.to(dtype), (beta * ratio).detach().to(dtype)


# ---------------------------------------------------------------------------------- policy


def policy_loss(logits: torch.Tensor, labels: torch.Tensor, old_logps: torch.Tensor, advantages: torch.Tensor,
                ref_logps: torch.Tensor | None = None, clip: tuple[float, float] = (0.2, 0.2), kl_coef: float = 0.0,
                mask: torch.Tensor | None = None, temperature: float = 1.0,
                reduction: str = "mean") -> tuple[torch.Tensor, torch.Tensor]:
    """Clipped policy loss: logits ``[..., T, V]``, labels (the sampled tokens) and ``old_logps`` ``[..., T]``, ``advantages``
    ``[...]`` or ``[..., T]`` -> ``(loss fp32, logps fp32 [..., T])``.

    With ``lp`` a token's log-probability at the temperature, ``r = exp(lp - old_logps)`` and ``x = ref_logps - lp``, a
    counted token's loss is ``-min(r A, clamp(r, 1 - clip[0], 1 + clip[1]) A) + kl_coef (e^x - x - 1)``; the KL term
    needs ``ref_logps``. ``reduction``: ``"mean"`` over all counted tokens (one value), ``"sequence"`` over
    each sequence's ``[...]``, ``"none"`` each token's ``[..., T]``; 0 where nothing counts. ``old_logps``,
    ``advantages`` and ``ref_logps`` are taken in fp32 (fp64 for fp64 logits). ``logps`` are constants to the gradient. The
    loss is differentiable with respect to the logits (once)."""
    z, shape = _sequences(logits)
    _integers("labels", labels, logits, shape)
    _floats("old_logps", old_logps, logits, shape)
    _floats("advantages", advantages, logits, shape[:-1], shape)
    if ref_logps is not None:
        _floats("ref_logps", ref_logps, logits, shape)
    elif kl_coef:
        raise ValueError("kl_coef needs ref_logps")
    if not math.isfinite(kl_coef):
        raise ValueError(f"kl_coef={kl_coef} is not finite")
    lo, hi = clip
    if not (0 <= lo <= 1 and 0 <= hi and math.isfinite(hi)):
        raise ValueError(f"clip={tuple(clip)}: below in [0, 1], above not negative")
    m, t, red = _mask(mask, logits, shape), _temperature(temperature, logits), _reduction(reduction)
    ref, flat = ref_logps if kl_coef else None, z.shape[:2]
    of_advantages = flat if advantages.dim() == len(shape) else flat[:1]
    if _fits(z, t, labels, m, old_logps, advantages, ref):
        loss, logps = N.torch_lib().policy_loss(
            _rows(z), _constant(labels, torch.int64, flat), _contiguous(m), _constant(old_logps, torch.float32, flat),
            _constant(advantages, torch.float32, of_advantages), _constant(ref, torch.float32, flat), 1 - lo, 1 + hi, kl_coef, t,
            red)
    else:
        loss, logps = _policy_loss_torch(z, labels.reshape(flat), m, old_logps.reshape(flat), advantages.reshape(of_advantages),
                                         None if ref is None else ref.reshape(flat), 1 - lo, 1 + hi, kl_coef, t, red)
    return (loss, logps) if len(shape) == 2 else (_unflatten(loss, shape, red), logps.view(shape))


def _unflatten(loss: torch.Tensor, shape, reduction: int) -> torch.Tensor:
    if reduction == N.REDUCE_MEAN or len(shape) == 2:
        return loss
    return loss.view(shape[:-1] if reduction == N.REDUCE_SEQUENCE else shape)


def _reduce_torch(each, counted, reduction):
    if reduction == N.REDUCE_NONE:
        return each
    if reduction == N.REDUCE_SEQUENCE:
        return (each.double().sum(-1) / counted.sum(-1).clamp(min=1)).to(each.dtype)
    return (each.double().sum() / counted.sum().clamp(min=1)).to(each.dtype)


def _policy_loss_torch(z, labels, mask, old, advantages, ref, clip_lo, clip_hi, kl_coef, temperature, reduction):
    lp, counted = _token_logprobs_torch(z, labels, mask, temperature)
    held = [torch.where(counted, t.detach().to(lp.dtype), 0.0) for t in
            (old, advantages if advantages.dim() == 2 else advantages.unsqueeze(-1).expand_as(lp))]
    ratio = torch.exp(lp - held[0])
    # a minimum whose two sides are equal takes the unclipped side's derivative
    free, kept = ratio * held[1], ratio.detach().clamp(clip_lo, clip_hi) * held[1]
    each = -torch.where(free <= kept, free, torch.where(free.isnan(), free, kept))
    if ref is not None:
        x = torch.where(counted, ref.detach().to(lp.dtype), 0.0) - lp
        e = torch.expm1(x)
        each = each + kl_coef * torch.where(e == math.inf, e, e - x)
    return _reduce_torch(torch.where(counted, each, 0.0), counted, reduction), lp.detach()


# ---------------------------------------------------------------------------- distillation


def distill_loss(logits: torch.Tensor, teacher_logits: torch.Tensor, teacher_index: torch.Tensor,
                 mask: torch.Tensor | None = None, temperature: float = 1.0, reduction: str = "mean") -> torch.Tensor:
    """Distillation from a teacher's top logits: logits ``[..., T, V]``, ``teacher_logits`` and ``teacher_index`` ``[..., T,
    K]`` (values, or log-probabilities, and where in the vocabulary they belong) -> loss fp32.

    With ``p = softmax(teacher_logits / temperature)`` over a token's K entries and ``q = softmax(logits /
    temperature)`` over the vocabulary, a counted token's loss is ``temperature^2 sum_k p_k (log p_k - log q[index_k])``.
    Entries whose index is outside ``[0, V)`` or whose value is ``-inf`` have no probability; a token without any has
    loss 0 (and counts, if its mask says so). ``reduction`` as in ``policy_loss``. Differentiable with respect to
    the logits (once)."""
    z, shape = _sequences(logits)
    if teacher_index.dim() != len(shape) + 1 or not teacher_index.shape[-1]:
        raise ValueError(f"teacher_index must be {list(shape)} and at least one entry, got {list(teacher_index.shape)}")
    K = teacher_index.shape[-1]
    _integers("teacher_index", teacher_index, logits, (*shape, K))
    _floats("teacher_logits", teacher_logits, logits, (*shape, K))
    m, t, red = _mask(mask, logits, shape), _temperature(temperature, logits), _reduction(reduction)
    flat = (*z.shape[:2], K)
    if _fits(z, t, m, teacher_logits, teacher_index) and K <= _MAX_TOP and teacher_logits.dtype in ops._DT:
        loss = N.torch_lib().distill_loss(_rows(z), _contiguous(m), _constant(teacher_logits, teacher_logits.dtype, flat),
                                          _constant(teacher_index, torch.int64, flat), t, red)
    else:
        loss = _distill_loss_torch(z, m, teacher_logits.reshape(flat), teacher_index.reshape(flat), t, red)
    return _unflatten(loss, shape, red)


def _distill_loss_torch(z, mask, teacher, index, temperature, reduction):
    counted = torch.ones(z.shape[:2], dtype=torch.bool, device=z.device) if mask is None else mask.expand(z.shape[:2])
    index = index.to(torch.int64)
    log_q = _log_softmax(z, counted, temperature)
    w = teacher.detach().to(log_q.dtype)
    usable = (index >= 0) & (index < z.shape[-1]) & counted.unsqueeze(-1)
    w = torch.where(usable, w, -math.inf)
    none = (w == -math.inf).all(-1, keepdim=True)
    top = torch.where(none, 0.0, w.amax(-1, keepdim=True))
    y = (w - top) / temperature
    log_p = torch.log_softmax(torch.where(none, 0.0, y), -1)
    p = torch.exp(log_p).masked_fill(none, 0.0)
    away = log_p - log_q.gather(-1, torch.where(usable, index, 0))
    each = temperature ** 2 * torch.where(p == 0, 0.0, p * torch.where(p == 0, 0.0, away)).sum(-1)
    return _reduce_torch(torch.where(counted, each, 0.0), counted, reduction)
