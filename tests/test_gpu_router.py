"""The router's kernels against 64-bit plain torch on the CPU.

Tolerances, with u = 2^-24 and R the largest finite distance of a logit from its row's maximum: an exponential
is off by (R + 3) u relative (its argument's rounding, the function's ulp), a sum of E positive terms by E u
more, each product or quotient by u; a result rounded into a 16-bit type by half a step of it (eps / 2), or half
a subnormal step. A gradient p (g - mean) is off by that share of p (|g| + mean of |g|)."""
import pytest
import torch

import experts4bit_qlora_amd as e4b
from experts4bit_qlora_amd import router as R

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24
DTYPES = (torch.float32, torch.bfloat16, torch.float16)
KINDS = (("softmax_then_topk", False), ("softmax_then_topk", True), ("topk_then_softmax", False))
# both sides of every number of lanes per row, odd ones, the limits
EXPERTS = (1, 2, 7, 8, 9, 16, 17, 32, 60, 64, 65, 100, 128, 130, 256, 300, 512, 520, 1000, 1024)


def _logits(shape, dtype, seed, spread=2.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * spread).to(dtype)


def _step(dtype, value):
    """Half a step of dtype at a value."""
    f = torch.finfo(dtype)
    return f.eps / 2 * value.abs().clamp(min=f.smallest_normal)


def _reach(z):
    """(R + E + 8) u: the relative error of a probability."""
    d = (z.amax(-1, keepdim=True) - z).nan_to_num(0.0, 0.0, 0.0)
    return (d.amax().item() + z.shape[-1] + 8) * U


def _gate64(z, k, scoring, renorm):
    index = torch.sort(z, dim=-1, descending=True, stable=True).indices[..., :k]
    p = R._softmax_or_zero(z)
    if renorm or scoring == "topk_then_softmax":
        return index, R._softmax_or_zero(z.gather(-1, index)), p
    return index, p.gather(-1, index), p


def _check_gate(logits, k, scoring, renorm, weight_dtype=None, seed=0):
    z = logits.detach().cpu().double()
    leaf = logits.to(DEV).requires_grad_()
    index, weights = e4b.router_topk(leaf, k, scoring=scoring, renorm=renorm, weight_dtype=weight_dtype)
    want_i, want_w, p = _gate64(z, k, scoring, renorm)
    assert index.dtype == torch.int64 and torch.equal(index.cpu(), want_i)
    wd = weight_dtype or logits.dtype
    assert weights.dtype == wd
    err = (weights.detach().cpu().double() - want_w).abs()
    reach = _reach(z)
    assert (err <= reach * want_w + _step(wd, want_w) + 2.0 ** -150).all()
    with torch.no_grad():  # the call without a graph is the same kernel
        again = e4b.router_topk(leaf, k, scoring=scoring, renorm=renorm, weight_dtype=weight_dtype)
    assert torch.equal(again[0], index) and torch.equal(again[1], weights)
    grad = _logits(weights.shape, wd, seed + 1, 1.0)
    (got,) = torch.autograd.grad(weights, leaf, grad.to(DEV))
    g = torch.zeros_like(z).scatter(-1, want_i, grad.double())
    on = torch.zeros_like(z).scatter(-1, want_i, 1.0)
    q = on * p / (on * p).sum(-1, keepdim=True).clamp(min=1e-300) if renorm or scoring == "topk_then_softmax" else p
    mean, reaches = (q * g).sum(-1, keepdim=True), (q * g.abs()).sum(-1, keepdim=True)
    want = q * (g - mean)
    # below fp32's normal range a rounding is half a subnormal step, 2^-150, whatever the value: once for the
    # exponential and once for the probability, both times (|g| + mean of |g|), once for the product
    tiny = 2.0 ** -150 * (2 * (g.abs() + reaches) + 1)
    bound = q * (g.abs() + reaches) * (3 * reach + (k + 4) * U) + _step(logits.dtype, want) + tiny
    assert got.dtype == logits.dtype and got.shape == logits.shape
    assert ((got.cpu().double() - want).abs() <= bound).all()


@pytest.mark.parametrize("E", EXPERTS)
def test_gate_every_width(E):
    for i, (scoring, renorm) in enumerate(KINDS):
        for k in sorted({1, min(8, E), min(64, E)}):
            _check_gate(_logits((33, E), DTYPES[i], E + k), k, scoring, renorm, seed=k)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T", (1, 2, 31, 32, 33, 257, 1531))
def test_gate_every_length(T, dtype):
    _check_gate(_logits((T, 64), dtype, T), 8, "softmax_then_topk", False)
    _check_gate(_logits((T, 60), dtype, T), 4, "topk_then_softmax", False)


def test_gate_weight_dtypes_and_wide_ranges():
    for wd in DTYPES:
        _check_gate(_logits((20, 32), torch.bfloat16, 5), 4, "softmax_then_topk", True, weight_dtype=wd)
    for spread in (1e-3, 30.0, 1e4):
        _check_gate(_logits((64, 128), torch.float32, 6, spread), 8, "softmax_then_topk", False)


def test_gate_ties_zeros_and_order():
    """Equal logits in and across lanes, -0 beside 0, descending and ascending rows."""
    rows = [torch.zeros(128), torch.arange(128.0), -torch.arange(128.0), torch.arange(128.0) % 3,
            torch.where(torch.arange(128) % 2 == 0, -0.0, 0.0), torch.full((128,), -5.0)]
    for dtype in DTYPES:
        _check_gate(torch.stack(rows).to(dtype), 64, "softmax_then_topk", False)


@pytest.mark.parametrize("E,k", ((60, 8), (256, 8)))
def test_gate_minus_infinity_infinity_and_nan(E, k):
    z = _logits((8, E), torch.float32, 7)
    z[0] = -float("inf")  # nothing left
    z[1, 3:] = -float("inf")  # fewer finite logits than choices
    z[2] = torch.finfo(torch.float32).min  # the type's lowest value
    z[3, 5:] = torch.finfo(torch.float32).min
    for scoring, renorm in KINDS:
        _check_gate(z, k, scoring, renorm)
    z[4, 17], z[5, 9], z[6, 2] = float("nan"), float("inf"), -float("nan")
    for scoring, renorm in KINDS:
        index, weights = e4b.router_topk(z.to(DEV), k, scoring=scoring, renorm=renorm)
        assert index[4, 0] == 17 and index[5, 0] == 9 and index[6, 0] == 2
        assert weights[4:7].isnan().all() and torch.isfinite(weights[[0, 1, 2, 3, 7]]).all()
        assert ((index >= 0) & (index < E)).all()


def _valid(mask, shape):
    return torch.ones(shape, dtype=torch.bool) if mask is None else (mask != 0).expand(shape)


def _check_balance(logits, index, mask=None):
    z, i = logits.detach().cpu().double(), index.cpu()
    leaf = logits.to(DEV).requires_grad_()
    loss, counts = e4b.balance_loss(leaf, index.to(DEV), None if mask is None else mask.to(DEV))
    lead, (T, E) = z.shape[:-2], z.shape[-2:]
    valid = _valid(mask, z.shape[:-1])
    n = valid.sum(-1)
    held = (valid.unsqueeze(-1) & (i >= 0) & (i < E)).flatten(-2)
    c = torch.zeros(*lead, E, dtype=torch.int64).scatter_add(-1, torch.where(held, i.flatten(-2), 0), held.long())
    assert counts.dtype == torch.int64 and torch.equal(counts.cpu(), c)
    p = R._softmax_or_zero(z) * valid.unsqueeze(-1)
    some = n.clamp(min=1).double().unsqueeze(-1)
    want = E * (c / some * p.sum(-2) / some).sum(-1)
    reach = _reach(z)
    # a lane sums at most T rows, its group's sums are at most 256; one rounding at the end
    assert loss.shape == lead and loss.dtype == torch.float32
    assert ((loss.detach().cpu().double() - want).abs() <= want * (reach + (min(T, 1000) + 257) * U)).all()
    grad = torch.rand(lead, generator=torch.Generator().manual_seed(9)) + 0.5
    (got,) = torch.autograd.grad(loss, leaf, grad.to(DEV))
    cd = c.double().unsqueeze(-2)
    dot = (cd * p).sum(-1, keepdim=True)
    f = (grad.double() * E).reshape(*lead, 1, 1) / some.unsqueeze(-1) ** 2
    want = f * p * (cd - dot)
    bound = f * p * (cd + dot) * (3 * reach + 8 * U) + _step(logits.dtype, want)
    assert got.dtype == logits.dtype
    assert ((got.cpu().double() - want).abs() <= bound).all()
    assert not got.cpu()[~valid].any()


def _choices(logits, k):
    return torch.topk(logits.float(), k, dim=-1).indices


@pytest.mark.parametrize("E", EXPERTS)
def test_balance_every_width(E):
    z = _logits((2, 77, E), DTYPES[E % 3], E)
    _check_balance(z, _choices(z, min(E, 8)))


@pytest.mark.parametrize("L,T", ((1, 1), (1, 2), (3, 33), (1, 509), (16, 100), (2, 2049), (1200, 5)))
def test_balance_lengths_and_masks(L, T):
    z = _logits((L, T, 64), torch.bfloat16, T)
    index = _choices(z, 8)
    g = torch.Generator().manual_seed(T)
    one, each = torch.rand(T, generator=g) > 0.3, torch.rand(L, T, generator=g) > 0.5
    each[0] = False  # a layer without a valid token
    for mask in (None, one, each, each.int() * 3):
        _check_balance(z, index, mask)


def test_balance_leading_axes_and_one_layer():
    z = _logits((2, 3, 40, 32), torch.float32, 1)
    _check_balance(z, _choices(z, 4), torch.rand(2, 3, 40) > 0.5)
    _check_balance(z[0, 0], _choices(z[0, 0], 4))


def test_balance_ids_outside_and_repeated():
    z = _logits((1, 50, 16), torch.float32, 2)
    index = _choices(z, 4).clone()
    index[0, 3] = torch.tensor([-1, 16, 1 << 40, -(1 << 40)])
    index[0, 7] = 5  # one expert four times
    _check_balance(z, index)


def test_balance_masked_nan_and_empty_rows():
    """What a mask hides has no influence; a row of -inf adds no probability."""
    z = _logits((1, 20, 24), torch.float32, 3)
    index = _choices(z, 2)
    z[0, 4] = -float("inf")
    _check_balance(z, index)
    mask = torch.ones(20)
    mask[[1, 2]] = 0
    bad = z.clone()
    bad[0, 1], bad[0, 2, 3] = float("nan"), float("inf")
    outs = []
    for logits in (z, bad):
        leaf = logits.to(DEV).requires_grad_()
        loss, counts = e4b.balance_loss(leaf, index.to(DEV), mask.to(DEV))
        outs.append((loss, counts, torch.autograd.grad(loss.sum(), leaf)[0]))
    assert all(torch.equal(a, b) for a, b in zip(*outs))
    with torch.no_grad():
        assert e4b.balance_loss(bad.to(DEV), index.to(DEV))[0].isnan().all()


def test_views_and_broadcast_gradients():
    """Strided logits, a start inside another tensor, an expanded incoming gradient."""
    big = _logits((40, 70), torch.bfloat16, 4).to(DEV).requires_grad_()
    for view in (big[:, 3:63], big[::2, :64], big.t()[:60, :33]):
        index, weights = e4b.router_topk(view, 4)
        same = e4b.router_topk(view.detach().clone(), 4)
        assert torch.equal(index, same[0]) and torch.equal(weights, same[1])
        (got,) = torch.autograd.grad(weights.sum(), big, retain_graph=True)
        leaf = view.detach().clone().requires_grad_()
        _, w = e4b.router_topk(leaf, 4)
        (want,) = torch.autograd.grad(w, leaf, torch.ones_like(w))
        full = torch.zeros_like(big)
        (full[:, 3:63] if view.shape == (40, 60) else full[::2, :64] if view.shape == (20, 64) else
         full.t()[:60, :33]).copy_(want)
        assert torch.equal(got, full)
    z = big.detach()[None].expand(3, 40, 70).requires_grad_()
    loss, _ = e4b.balance_loss(z, _choices(z, 4))
    assert torch.equal(loss[0], loss[2])
    assert torch.autograd.grad(loss.sum(), z)[0].shape == (3, 40, 70)


def test_formulations_agree_where_the_kernel_does_not_reach():
    z = _logits((5, 1100), torch.float32, 5).to(DEV)
    index, weights = e4b.router_topk(z, 70)
    assert torch.equal(index, torch.sort(z, descending=True, stable=True).indices[:, :70]) and weights.shape == (5, 70)
    d = _logits((5, 32), torch.float32, 6).double().to(DEV).requires_grad_()
    assert torch.autograd.gradcheck(lambda a: e4b.router_topk(a, 4)[1], d)
    x, t = (_logits((6, 16), torch.float32, s).to(DEV) for s in (7, 8))
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(x, t)
        tangent = torch.autograd.forward_ad.unpack_dual(e4b.router_topk(dual, 4)[1]).tangent
    assert tangent is not None and tangent.any()
    one = torch.func.vmap(lambda r: e4b.router_topk(r, 4)[1])(x)
    assert torch.allclose(one, e4b.router_topk(x, 4)[1])


def test_second_derivatives_are_refused():
    z = _logits((4, 16), torch.float32, 9).to(DEV).requires_grad_()
    _, w = e4b.router_topk(z, 2)
    with pytest.raises(RuntimeError, match="once"):
        torch.autograd.grad(w.square().sum(), z, create_graph=True)
    loss, _ = e4b.balance_loss(z, _choices(z, 2))
    with pytest.raises(RuntimeError, match="once"):
        torch.autograd.grad(loss, z, create_graph=True)


def test_an_output_changed_in_place_is_refused():
    z = _logits((2, 4, 16), torch.float32, 9).to(DEV).requires_grad_()
    index, w = e4b.router_topk(z[0], 2)
    index.zero_()
    with pytest.raises(RuntimeError, match="inplace"):
        torch.autograd.grad(w.sum(), z)
    loss, counts = e4b.balance_loss(z, _choices(z, 2))
    counts.add_(1)
    with pytest.raises(RuntimeError, match="inplace"):
        torch.autograd.grad(loss.sum(), z)


def test_captured_and_replayed():
    """Gate, loss and both gradients in one graph, replayed on new logits, against the eager calls."""
    z = _logits((2, 300, 64), torch.float32, 10).to(DEV)
    gw = _logits((600, 8), torch.float32, 11).to(DEV)

    def step():
        leaf = z.detach().requires_grad_()
        index, weights = e4b.router_topk(leaf.view(600, 64), 8)
        loss, counts = e4b.balance_loss(leaf, index.view(2, 300, 8))
        (grad,) = torch.autograd.grad([weights, loss], leaf, [gw, torch.ones_like(loss)])
        return index, weights.detach(), loss.detach(), counts, grad

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for i in range(4):
        z.copy_(_logits((2, 300, 64), torch.float32, 20 + i))
        graph.replay()
        got = [o.clone() for o in outs]
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, step()))


def test_another_stream_repeats_and_no_synchronization():
    z = _logits((2000, 128), torch.bfloat16, 12).to(DEV)
    index, weights = e4b.router_topk(z * 2, 8)
    loss, counts = e4b.balance_loss(z * 2, index)
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    torch.cuda.set_sync_debug_mode("error")
    try:
        with torch.cuda.stream(stream):
            got = []
            for _ in range(5):
                doubled = z * 2
                i, w = e4b.router_topk(doubled, 8)
                got.append((i, w, *e4b.balance_loss(doubled, i)))
    finally:
        torch.cuda.set_sync_debug_mode("default")
    stream.synchronize()
    for i, w, l, c in got:
        assert torch.equal(i, index) and torch.equal(w, weights) and torch.equal(l, loss) and torch.equal(c, counts)


def test_no_tokens_on_the_device():
    z = torch.zeros(0, 8, device=DEV, requires_grad=True)
    index, weights = e4b.router_topk(z, 2)
    assert index.shape == weights.shape == (0, 2)
    assert torch.autograd.grad(weights.sum(), z)[0].shape == (0, 8)
    z = torch.zeros(3, 0, 8, device=DEV, requires_grad=True)
    loss, counts = e4b.balance_loss(z, torch.zeros(3, 0, 2, dtype=torch.int64, device=DEV))
    assert not loss.any() and not counts.any() and counts.shape == (3, 8)
    assert torch.autograd.grad(loss.sum(), z)[0].shape == (3, 0, 8)


@pytest.mark.parametrize("L,T,E,k,masked", ((1, 1, 8, 2, False), (3, 200, 60, 4, True), (2, 5000, 128, 8, False), (1200, 5, 16, 2, True)))
def test_counts_reduced_over_ranks_before_the_backward(L, T, E, k, masked):
    """A collective writes its sum into ``counts`` without raising autograd's version (``.data`` does the same here): the
    gradient is still that of this call's own tokens."""
    z = _logits((L, T, E), torch.bfloat16, T).to(DEV).requires_grad_()
    index, grad = _choices(z, k), torch.rand(L, generator=torch.Generator().manual_seed(T)).to(DEV)
    mask = torch.rand(L, T, generator=torch.Generator().manual_seed(E)).to(DEV) > 0.3 if masked else None
    loss, counts = e4b.balance_loss(z, index, mask)
    (want,) = torch.autograd.grad(loss, z, grad)
    loss, counts = e4b.balance_loss(z, index, mask)
    counts.data.mul_(3).add_(torch.arange(E, device=DEV))
    assert counts._version == 0
    (got,) = torch.autograd.grad(loss, z, grad)
    assert torch.equal(got, want)
