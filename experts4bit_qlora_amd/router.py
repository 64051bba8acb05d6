"""The router beside the expert layers: the top-k gate and the load-balance loss, both with gradients.

``router_topk`` turns a router's logits into the ``(top_k_index, top_k_weights)`` that ``route`` and the
expert modules take; ``balance_loss`` gives the auxiliary loss that keeps the experts in use, and the
per-expert counts. On a HIP device each is a kernel each way (``csrc/gate.h``); tensors elsewhere, other
dtypes, more than 1,024 experts or 64 choices, rows (or a layer's choices) from 2^31 on, and tensors that a
transform, a trace or forward-mode differentiation follows take the torch formulation, which is the definition.

The reference leaves both to the models (its CPU engine restates the gate,
``experts4bit_qlora/engines/cpu_router.py:100-120``).
"""
from __future__ import annotations

import torch

from . import _native as N
from . import ops
from .quant import _forward_ad

_SCORING = {"softmax_then_topk": N.SCORE_ALL, "topk_then_softmax": N.SCORE_CHOSEN}


def _on_kernel(t: torch.Tensor) -> bool:
    """Whether the kernels may take ``t``: a plain device tensor; autograd is served by the Functions below."""
    return (t.is_cuda and t.dtype in ops._DT and type(t) in (torch.Tensor, torch.nn.Parameter)
            and not torch._C._functorch.is_functorch_wrapped_tensor(t) and not torch._C._is_tracing()
            and (_forward_ad._current_level < 0 or _forward_ad.unpack_dual(t).tangent is None))


def _aligned(t: torch.Tensor) -> torch.Tensor:
    return t if t.is_contiguous() else t.contiguous()


def _once():
    """Refuse a backward that is itself to be differentiated (torch's ``once_differentiable`` does it at
    ~10 us a call)."""
    if torch.is_grad_enabled():
        raise RuntimeError("router_topk and balance_loss are differentiable once: no create_graph=True on the device")


# -------------------------------------------------------------------------------- gate


class _Gate(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, top_k, scoring, weight_dtype):
        index, weights = ops.router_topk(logits, top_k, scoring, weight_dtype)
        ctx.save_for_backward(logits, index)
        ctx.scoring = scoring
        ctx.mark_non_differentiable(index)
        ctx.set_materialize_grads(False)  # no zeros in the place of the index's gradient
        return index, weights

    @staticmethod
    def backward(ctx, _, grad):
        if grad is None:
            return None, None, None, None
        _once()
        logits, index = ctx.saved_tensors
        return ops.router_topk_backward(logits, index, _aligned(grad), ctx.scoring), None, None, None


def router_topk(logits: torch.Tensor, top_k: int, scoring: str = "softmax_then_topk", renorm: bool = False,
                weight_dtype: torch.dtype | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Router logits ``[..., E]`` -> ``(top_k_index int64 [..., k], top_k_weights [..., k])``.

    The ``top_k`` largest logits of each row in descending order, ties to the lower index. Their weights:
    ``"softmax_then_topk"`` the softmax over all logits (``renorm``: divided by their sum),
    ``"topk_then_softmax"`` the softmax over the chosen logits; fp32, rounded once into ``weight_dtype``
    (default: the logits' dtype). A row whose logits are all ``-inf`` gets zero weights. The weights are
    differentiable with respect to the logits (once). A backward pass is captured into a graph like any other
    of torch's: with no eager graph of the same leaves alive."""
    if scoring not in _SCORING:
        raise ValueError(f"scoring must be one of {sorted(_SCORING)}, got {scoring!r}")
    if logits.dim() < 1 or not logits.is_floating_point():
        raise ValueError("logits must be a floating-point tensor [..., num_experts]")
    E = logits.shape[-1]
    if not 1 <= top_k <= E:
        raise ValueError(f"top_k={top_k} outside [1, {E}]")
    wd = logits.dtype if weight_dtype is None else weight_dtype
    code = N.SCORE_CHOSEN if renorm else _SCORING[scoring]
    if not (E <= 1024 and top_k <= 64 and logits.numel() < E << 31 and wd in ops._DT and _on_kernel(logits)):
        return _router_topk_torch(logits, top_k, code, wd)
    z = _aligned(logits) if logits.dim() == 2 else logits.reshape(-1, E).contiguous()
    if z.requires_grad and torch.is_grad_enabled():
        index, weights = _Gate.apply(z, top_k, code, wd)
    else:
        index, weights = ops.router_topk(z, top_k, code, wd)
    if logits.dim() == 2:
        return index, weights
    return index.view(*logits.shape[:-1], top_k), weights.view(*logits.shape[:-1], top_k)


def _softmax_or_zero(z: torch.Tensor) -> torch.Tensor:
    """The softmax over the last axis; zeros where every entry is -inf."""
    empty = (z == -float("inf")).all(-1, keepdim=True)
    return torch.softmax(torch.where(empty, 0.0, z), -1).masked_fill(empty, 0.0)


def _router_topk_torch(logits, top_k, scoring, weight_dtype):
    z = logits if logits.dtype == torch.float64 else logits.float()
    index = torch.sort(z.detach(), dim=-1, descending=True, stable=True).indices[..., :top_k]
    if scoring == N.SCORE_CHOSEN:
        weights = _softmax_or_zero(z.gather(-1, index))
    else:
        weights = _softmax_or_zero(z).gather(-1, index)
    return index, weights.to(weight_dtype)


# --------------------------------------------------------------------------- balance loss


class _Balance(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, index, mask):
        # The backward reads the counts that the workspace begins with: a collective may reduce the public ones over
        # ranks meanwhile without raising autograd's version. They are saved so that an ordinary change is refused.
        loss, counts, valid, kept = ops.balance_loss(logits, index, mask)
        ctx.save_for_backward(logits, mask, counts, kept, valid)
        ctx.mark_non_differentiable(counts)
        ctx.set_materialize_grads(False)
        return loss, counts

    @staticmethod
    def backward(ctx, grad, _):
        if grad is None:
            return None, None, None
        _once()
        logits, mask, _, kept, valid = ctx.saved_tensors
        return ops.balance_loss_backward(logits, mask, kept, valid, _aligned(grad)), None, None


def balance_loss(logits: torch.Tensor, top_k_index: torch.Tensor,
                 mask: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Load-balance loss of router logits ``[..., T, E]`` (leading axes: layers, or sequences) and the choices
    ``top_k_index [..., T, k]`` -> ``(loss fp32 [...], counts int64 [..., E])``.

    Over the valid tokens, N of them (``mask [T]`` or ``[..., T]``: nonzero is valid): ``counts[e]`` the choices
    of expert e (ids outside ``[0, E)`` count nowhere), ``P[e]`` the mean of the softmax probabilities, ``loss = E
    * sum_e counts[e] / N * P[e]``, 0 where N is 0. For one loss over several
    layers' tokens together, pass them as one axis. The loss is
    differentiable with respect to the logits (once), the counts are constants to it: the gradient is that of this
    call's own tokens also where a collective (``torch.distributed.all_reduce``) has summed ``counts`` over the ranks
    before the backward. An ordinary change of ``counts`` in place before the backward goes to a copy (on the device
    autograd refuses it)."""
    if logits.dim() < 2 or not logits.is_floating_point():
        raise ValueError("logits must be a floating-point tensor [..., tokens, num_experts]")
    lead, (T, E) = logits.shape[:-2], logits.shape[-2:]
    if top_k_index.shape[:-1] != logits.shape[:-1] or top_k_index.is_floating_point() or not top_k_index.shape[-1]:
        raise ValueError(f"top_k_index must be integers [{', '.join(map(str, logits.shape[:-1]))}, k], got "
                         f"{top_k_index.dtype} {list(top_k_index.shape)}")
    if mask is not None and mask.shape != logits.shape[:-1] and mask.shape != (T,):
        raise ValueError(f"mask must be [{T}] or {list(logits.shape[:-1])}, got {list(mask.shape)}")
    if not all(t is None or t.device == logits.device for t in (top_k_index, mask)):
        raise ValueError("logits, top_k_index and mask must be on one device")
    if mask is not None and mask.dtype != torch.bool:
        mask = mask != 0
    layers = lead.numel()
    if not (1 <= E <= 1024 and layers <= 65535 and T * top_k_index.shape[-1] < 2 ** 31 and _on_kernel(logits)
            and _on_kernel_index(top_k_index, mask)):
        return _balance_loss_torch(logits, top_k_index, mask)
    z = _aligned(logits) if len(lead) == 1 else logits.reshape(layers, T, E).contiguous()
    index = top_k_index if top_k_index.dtype == torch.int64 else top_k_index.to(torch.int64)
    index = _aligned(index) if len(lead) == 1 else index.reshape(layers, T, -1).contiguous()
    if mask is not None:
        mask = _aligned(mask) if mask.dim() == 1 else mask.reshape(layers, T).contiguous()
    if z.requires_grad and torch.is_grad_enabled():
        loss, counts = _Balance.apply(z, index, mask)
    else:
        loss, counts, _, _ = ops.balance_loss(z, index, mask)
    return (loss, counts) if len(lead) == 1 else (loss.view(lead), counts.view(*lead, E))


def _on_kernel_index(index: torch.Tensor, mask) -> bool:
    plain = torch._C._functorch.is_functorch_wrapped_tensor
    return not plain(index) and (mask is None or not plain(mask))


def _balance_loss_torch(logits, top_k_index, mask):
    z = logits if logits.dtype == torch.float64 else logits.float()
    T, E = z.shape[-2:]
    valid = torch.ones(z.shape[:-1], dtype=torch.bool, device=z.device) if mask is None else mask.expand(z.shape[:-1])
    if mask is not None:  # before the softmax, whose gradient at a NaN or an infinity is NaN whatever it is multiplied by
        z = torch.where(valid.unsqueeze(-1), z, 0.0)
    p = _softmax_or_zero(z)
    n = valid.sum(-1)
    i = top_k_index.to(torch.int64)
    held = valid.unsqueeze(-1) & (i >= 0) & (i < E)
    each = held.to(torch.int64).flatten(-2)
    counts = torch.zeros(*z.shape[:-2], E, dtype=torch.int64, device=z.device)
    counts = counts.scatter_add(-1, torch.where(held, i, 0).flatten(-2), each)
    share = torch.where(valid.unsqueeze(-1), p, 0.0).sum(-2)
    some = n.clamp(min=1).to(z.dtype).unsqueeze(-1)
    loss = E * ((counts.to(z.dtype) / some) * (share / some)).sum(-1)
    return loss.float(), counts
