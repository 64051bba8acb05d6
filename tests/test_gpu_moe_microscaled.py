"""A MoE layer of the device operators, as a model runs it: ``quantize_mxfp4`` for the expert weights,
``router_topk`` and ``balance_loss`` on the router's logits, the rows sorted by expert, two products of
microscaled operands around the activation, and the weighted sum.

Quantization rounds to few values, so a reference that ran on its own from the start could part from the
kernels by a whole step wherever a value lies near a tie. Each stage is therefore checked in 64 bits from the
inputs that the kernels gave it. Tolerances: the products' as derived in test_gpu_mx_gemm.py; router weights and
loss a few fp32 roundings (2^-20 relative is eight of them); the weighted sum is torch's own, not under test."""
import pytest
import torch

import experts4bit_qlora_amd as e4b
from experts4bit_qlora_amd import quant as Q

from test_gpu_mx_gemm import _check

pytestmark = pytest.mark.gpu
DEV = "cuda"


class _Layer:
    def __init__(self, E, hidden, inter, k, dtype, seed):
        g = torch.Generator(device=DEV).manual_seed(seed)
        self.E, self.k = E, k
        self.router = (torch.randn(E, hidden, generator=g, device=DEV) * hidden ** -0.5).requires_grad_()
        self.gu = torch.randn(E, 2 * inter, hidden, generator=g, device=DEV, dtype=dtype)
        self.dn = torch.randn(E, hidden, inter, generator=g, device=DEV, dtype=dtype)
        self.gu_q, self.dn_q = e4b.quantize_mxfp4(self.gu), e4b.quantize_mxfp4(self.dn)
        self.ids = torch.arange(E, device=DEV)

    def route(self, x, mask=None):
        logits = torch.nn.functional.linear(x.float(), self.router)
        index, weights = e4b.router_topk(logits, self.k, renorm=True)
        loss, counts = e4b.balance_loss(logits[None], index[None], None if mask is None else mask)
        return logits, index, weights, loss[0], counts[0]

    def experts(self, x, index, weights, sizes, seen=None):
        flat = index.flatten()
        order = torch.sort(flat, stable=True).indices
        a = x[order // self.k].contiguous()
        h = e4b.gemm_mxfp4_grouped(a, *self.gu_q, sizes, self.ids, act_quant="mxfp4")
        gate, up = h.float().chunk(2, -1)
        act = (torch.nn.functional.silu(gate) * up).to(x.dtype)
        down = e4b.gemm_mxfp4_grouped(act, *self.dn_q, sizes, self.ids, act_quant="mxfp4")
        if seen is not None:
            seen += [(a, h, self.gu_q), (act, down, self.dn_q)]
        each = torch.zeros(flat.numel(), x.shape[-1], device=DEV).index_copy(0, order, down.float())
        return (each.view(*index.shape, -1) * weights.float().unsqueeze(-1)).sum(-2)


@pytest.mark.parametrize("dtype", (torch.bfloat16, torch.float16))
@pytest.mark.parametrize("tokens,E,k,hidden,inter", [(1, 8, 2, 128, 96), (7, 5, 3, 96, 160), (150, 4, 2, 288, 128)])
def test_layer(tokens, E, k, hidden, inter, dtype):
    layer = _Layer(E, hidden, inter, k, dtype, tokens)
    for dense, q in ((layer.gu, layer.gu_q), (layer.dn, layer.dn_q)):
        for got, want in zip(q, Q._quantize_mxfp4_torch(dense.cpu())):
            assert torch.equal(got.cpu(), want)
    g = torch.Generator(device=DEV).manual_seed(tokens + 1)
    x = torch.randn(tokens, hidden, generator=g, device=DEV).to(dtype)
    mask = torch.rand(tokens, generator=g, device=DEV) < 0.8
    logits, index, weights, loss, counts = layer.route(x, mask)
    sizes = torch.bincount(index.flatten(), minlength=E).tolist()
    seen = []
    out = layer.experts(x, index, weights, sizes, seen)

    z = logits.detach().double().cpu()
    p = torch.softmax(z, -1)
    chosen = torch.sort(z, dim=-1, descending=True, stable=True).indices[:, :k]
    assert torch.equal(index.cpu(), chosen)
    w = p.gather(-1, chosen)
    w = w / w.sum(-1, keepdim=True)
    assert torch.allclose(weights.detach().double().cpu(), w, rtol=2.0 ** -20, atol=0)
    valid = mask.cpu()
    held = torch.bincount(chosen[valid].flatten(), minlength=E)
    assert torch.equal(counts.cpu(), held)
    n = max(int(valid.sum()), 1)
    want = E * ((held.double() / n) * (p[valid].sum(0) / n)).sum()
    assert abs(loss.item() - want.item()) <= 2.0 ** -20 * want.item()
    for a, got, q in seen:
        _check(a.cpu(), q[0].cpu(), q[1].cpu(), sizes, list(range(E)), got)

    # the router's gradient from both uses of its logits
    grad = torch.autograd.grad((out * out.detach()).sum() + loss, layer.router)[0]
    each = torch.zeros(tokens * k, hidden, dtype=torch.float64)
    order = torch.sort(chosen.flatten(), stable=True).indices
    each[order] = seen[1][1].double().cpu()
    r = layer.router.detach().double().cpu().requires_grad_()
    zr = x.double().cpu() @ r.T
    pr = torch.softmax(zr, -1)
    wr = pr.gather(-1, chosen)
    wr = wr / wr.sum(-1, keepdim=True)
    o = (each.view(tokens, k, hidden) * wr.unsqueeze(-1)).sum(1)
    lr = E * ((held.double() / n) * (pr[valid].sum(0) / n)).sum()
    want = torch.autograd.grad((o * o.detach()).sum() + lr, r)[0]
    # fp32 all along, the rows' dot products of `hidden` terms: hidden * 2^-23 of the largest terms, with the
    # logits' own error of the same kind passing through the exponential
    top = (each.view(tokens, k, hidden).abs().sum(-1).amax() * o.detach().abs().amax() + 1) * x.double().abs().amax().cpu()
    assert (grad.double().cpu() - want).abs().max() <= 4 * hidden * tokens * 2.0 ** -23 * top


@pytest.mark.parametrize("dtype", (torch.bfloat16, torch.float16))
@pytest.mark.parametrize("tokens,E,k,hidden,inter", [(1, 8, 2, 128, 96), (7, 5, 3, 96, 160), (150, 4, 2, 288, 128)])
def test_layer_gradients_of_gate_and_loss(tokens, E, k, hidden, inter, dtype):
    """The logits' gradient through the experts' weighted sum, through the balance loss and through both, against the
    formulas in 64 bits on the same logits and expert outputs, element by element; the loss is weighted (by a power of
    two) so that either part is far above the bound of their sum, so a sum without one of them, or with its sign
    changed, is refused.

    Bounds, with u = 2^-24 and `reach` the relative error of a probability, (largest distance from a row's maximum + E
    + 8) u: a weight's gradient is torch's sum of `hidden` rounded products, (hidden + 1) u of their magnitudes (dg);
    the gate turns it into w (g - mean), off by w (dg + mean of dg) and by w (|g| + mean of |g|) (3 reach + (k + 4) u);
    the loss's part f p (c - dot) is off by f p (c + dot) (3 reach + 8 u). Each is rounded once, their sum once more;
    products of these errors are below 2^-10 of them."""
    layer = _Layer(E, hidden, inter, k, dtype, tokens + 40)
    g = torch.Generator(device=DEV).manual_seed(tokens + 41)
    x = torch.randn(tokens, hidden, generator=g, device=DEV).to(dtype)
    mask = torch.rand(tokens, generator=g, device=DEV) < 0.8
    mask[0] = True
    logits = torch.nn.functional.linear(x.float(), layer.router).detach().requires_grad_()
    index, weights = e4b.router_topk(logits, k, renorm=True)
    loss, counts = e4b.balance_loss(logits[None], index[None], mask)
    sizes, seen = torch.bincount(index.flatten(), minlength=E).tolist(), []
    out = layer.experts(x, index, weights, sizes, seen)
    down = seen[1][1]
    into = torch.randn(tokens, hidden, generator=g, device=DEV) / down.float().square().mean().sqrt()

    u = 2.0 ** -24
    z = logits.detach().double().cpu()
    chosen = torch.sort(z, dim=-1, descending=True, stable=True).indices[:, :k]
    each = torch.zeros(tokens * k, hidden, dtype=torch.float64)
    each[torch.sort(chosen.flatten(), stable=True).indices] = down.double().cpu()
    terms = each.view(tokens, k, hidden) * into.double().cpu().unsqueeze(1)
    gw, dg = terms.sum(-1), (hidden + 1) * u * terms.abs().sum(-1)
    p = torch.softmax(z, -1)
    w = p.gather(-1, chosen)
    w = w / w.sum(-1, keepdim=True)
    reach = ((z.amax(-1, keepdim=True) - z).amax() + E + 8) * u
    on = lambda v: torch.zeros_like(z).scatter(-1, chosen, v)
    mean = lambda v: (w * v).sum(-1, keepdim=True)
    gate = on(w * (gw - mean(gw)))
    gate_off = on(w * (dg + mean(dg)) + w * (gw.abs() + mean(gw.abs())) * (3 * reach + (k + 4) * u)) + u * gate.abs()
    valid = mask.cpu()
    n, c = valid.sum().double(), torch.bincount(chosen[valid].flatten(), minlength=E).double()
    dot = (p * c).sum(-1, keepdim=True)
    f = E / n ** 2 * valid.double().unsqueeze(-1)
    balance = f * p * (c - dot)
    alpha = 2.0 ** round(torch.log2(gate.abs().max() / balance.abs().max()).item())
    balance = alpha * balance
    balance_off = alpha * f * p * (c + dot) * (3 * reach + 8 * u) + u * balance.abs()

    def off(want, bound):  # whether an element is further off than its bound (2^-149: below fp32's normal range)
        return ((got.double().cpu() - want).abs() > bound * (1 + 2.0 ** -10) + 2.0 ** -149).any()

    (got,) = torch.autograd.grad(out, logits, into, retain_graph=True)
    assert not off(gate, gate_off)
    (got,) = torch.autograd.grad(alpha * loss.sum(), logits, retain_graph=True)
    assert not off(balance, balance_off)
    (got,) = torch.autograd.grad([out, alpha * loss.sum()], logits, [into, torch.ones((), device=DEV)])
    bound = gate_off + balance_off + u * (gate + balance).abs()
    assert not off(gate + balance, bound)
    assert off(gate, bound) and off(balance, bound) and off(gate - balance, bound) and off(balance - gate, bound)
    assert off(gate + 1.01 * balance, bound) and off(1.01 * gate + balance, bound)


def test_layer_replayed():
    """The layer captured with fixed group sizes (every token to every expert), replayed on new inputs between
    eager runs."""
    layer = _Layer(4, 96, 64, 4, torch.bfloat16, 3)
    tokens, sizes = 9, [9] * 4
    x = torch.randn(tokens, 96, device=DEV, dtype=torch.bfloat16)

    def run(x):
        with torch.no_grad():
            logits, index, weights, loss, counts = layer.route(x)
            return layer.experts(x, index, weights, sizes), loss, counts

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run(x)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = run(x)
    for i in range(4):
        x.copy_(torch.randn(tokens, 96, device=DEV))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in held]
        for a, b in zip(got, run(x)):
            assert torch.equal(a, b)
