"""``router_topk`` and ``balance_loss`` off the device (the torch formulation, which is the kernels'
definition): values against numpy, gradients against differences, refusals."""
import numpy as np
import pytest
import torch

import experts4bit_qlora_amd as e4b
from oracle import routing


@pytest.mark.parametrize("renorm,scoring", ((False, "softmax_then_topk"), (True, "softmax_then_topk"),
                                            (False, "topk_then_softmax")))
def test_gate_equals_the_oracle(renorm, scoring):
    z = torch.randn(50, 24, generator=torch.Generator().manual_seed(1))
    z[7, 3] = z[7, 9] = z[7].max() + 1  # a tie for the first place
    index, weights = e4b.router_topk(z, 5, scoring=scoring, renorm=renorm)
    want_w, want_i = routing.router_topk(z.numpy(), 5, scoring, renorm)
    assert np.array_equal(index.numpy(), want_i) and index[7, :2].tolist() == [3, 9]
    np.testing.assert_allclose(weights.numpy(), want_w, rtol=1e-5)


@pytest.mark.parametrize("renorm,scoring", ((False, "softmax_then_topk"), (True, "softmax_then_topk"),
                                            (False, "topk_then_softmax")))
def test_gate_gradient_by_differences(renorm, scoring):
    z = torch.randn(2, 3, 9, dtype=torch.float64, generator=torch.Generator().manual_seed(2), requires_grad=True)
    assert torch.autograd.gradcheck(lambda a: e4b.router_topk(a, 4, scoring=scoring, renorm=renorm)[1], z)


def test_gate_rows_of_minus_infinity():
    z = torch.randn(3, 8, dtype=torch.float64)
    z[1] = -float("inf")
    z[2, 2:] = -float("inf")
    z.requires_grad_()
    for scoring in ("softmax_then_topk", "topk_then_softmax"):
        index, weights = e4b.router_topk(z, 4, scoring=scoring)
        assert index[1].tolist() == [0, 1, 2, 3] and not weights[1].any()
        assert sorted(index[2, :2].tolist()) == [0, 1] and index[2, 2:].tolist() == [2, 3] and not weights[2, 2:].any()
        (grad,) = torch.autograd.grad(weights.square().sum(), z)
        assert not grad[1].any() and torch.isfinite(grad).all()


def _plain_loss(z, index, valid):
    """The definition, one (token, choice) at a time."""
    T, E = z.shape
    p = np.exp(z - z.max(-1, keepdims=True))
    p /= p.sum(-1, keepdims=True)
    n, counts, share = 0, np.zeros(E, dtype=np.int64), np.zeros(E)
    for t in range(T):
        if valid[t]:
            n += 1
            share += p[t]
            for e in index[t]:
                if 0 <= e < E:
                    counts[e] += 1
    return (E * (counts / n * share / n).sum() if n else 0.0), counts


def test_balance_values_gradients_and_layers():
    g = torch.Generator().manual_seed(3)
    z = torch.randn(2, 3, 11, 6, dtype=torch.float64, generator=g)
    index, _ = e4b.router_topk(z, 3)
    index[0, 0, 2, 1] = -1
    index[1, 2, 5, 0] = 6
    mask = torch.rand(2, 3, 11, generator=g) > 0.4
    mask[0, 1] = False
    for m in (None, mask, mask[0, 0], mask.int() * 7):
        loss, counts = e4b.balance_loss(z, index, mask=m)
        assert loss.shape == (2, 3) and loss.dtype == torch.float32 and counts.dtype == torch.int64
        for i in range(2):
            for j in range(3):
                valid = torch.ones(11) if m is None else m if m.dim() == 1 else m[i, j]
                want, c = _plain_loss(z[i, j].numpy(), index[i, j].numpy(), valid.numpy())
                assert np.array_equal(counts[i, j].numpy(), c)
                assert abs(loss[i, j].item() - want) <= 2.0 ** -23 * want
    z.requires_grad_()
    loss, _ = e4b.balance_loss(z, index, mask=mask)
    (grad,) = torch.autograd.grad(loss.sum(), z)
    assert not grad[~mask].any() and not grad[0, 1].any() and grad[0, 0].any()
    # against differences of the 64-bit definition
    at = z.detach()[1, 0].clone().numpy()
    for t, e in ((0, 0), (4, 5), (10, 2)):
        ends = []
        for d in (1e-5, -1e-5):
            moved = at.copy()
            moved[t, e] += d
            ends.append(_plain_loss(moved, index[1, 0].numpy(), mask[1, 0].numpy())[0])
        # the loss is fp32 but its gradient fp64; a central difference is off by O(1e-10)
        assert abs((ends[0] - ends[1]) / 2e-5 - grad[1, 0, t, e].item()) < 1e-6


def test_balance_of_layers_as_one_axis():
    """Several layers' tokens passed as one axis: the loss of all of them together."""
    z = torch.randn(3, 40, 8, generator=torch.Generator().manual_seed(4))
    index, _ = e4b.router_topk(z, 2)
    loss, counts = e4b.balance_loss(z.reshape(120, 8), index.reshape(120, 2))
    p, each = torch.softmax(z.double(), -1), torch.zeros(8, dtype=torch.float64)
    for e in index.flatten():
        each[e] += 1
    want = 8 * ((each / 120) * p.mean((0, 1))).sum()
    assert loss.shape == () and abs(loss.item() - want.item()) <= 1e-5 * want.item()
    assert torch.equal(counts, each.long())


def test_no_tokens():
    index, weights = e4b.router_topk(torch.zeros(0, 8), 2)
    assert index.shape == weights.shape == (0, 2)
    loss, counts = e4b.balance_loss(torch.zeros(3, 0, 8), torch.zeros(3, 0, 2, dtype=torch.int64))
    assert not loss.any() and counts.shape == (3, 8) and not counts.any()


def test_refusals():
    z = torch.zeros(4, 8)
    index = torch.zeros(4, 2, dtype=torch.int64)
    with pytest.raises(ValueError, match="scoring"):
        e4b.router_topk(z, 2, scoring="sigmoid")
    for k in (0, 9):
        with pytest.raises(ValueError, match="top_k"):
            e4b.router_topk(z, k)
    with pytest.raises(ValueError, match="floating"):
        e4b.router_topk(z.long(), 2)
    with pytest.raises(ValueError, match="top_k_index"):
        e4b.balance_loss(z, index[:3])
    with pytest.raises(ValueError, match="top_k_index"):
        e4b.balance_loss(z, index.float())
    with pytest.raises(ValueError, match="mask"):
        e4b.balance_loss(z, index, mask=torch.ones(5))
    with pytest.raises(ValueError, match="logits"):
        e4b.balance_loss(z[0], index[0])


@pytest.mark.parametrize("dtype", (torch.float32, torch.float64))
def test_balance_values_behind_the_mask_have_no_influence(dtype):
    """NaN and infinities in masked tokens: loss, counts and gradient are those of finite values there, the masked
    tokens' gradient is zero."""
    z = torch.randn(2, 20, 24, dtype=dtype, generator=torch.Generator().manual_seed(5))
    index, _ = e4b.router_topk(z, 2)
    one = torch.ones(20)
    one[[1, 2, 5, 7]] = 0
    each = one.expand(2, 20).clone()
    each[1, 9] = 0
    bad = z.clone()
    bad[:, 1], bad[:, 2, 3], bad[:, 5], bad[:, 7, 4] = float("nan"), float("inf"), -float("inf"), torch.finfo(dtype).min
    for mask in (one, each):
        outs = []
        for logits in (z, bad):
            leaf = logits.clone().requires_grad_()
            loss, counts = e4b.balance_loss(leaf, index, mask)
            outs.append((loss, counts, torch.autograd.grad(loss.sum(), leaf)[0]))
        assert all(torch.equal(a, b) for a, b in zip(*outs))
        assert not outs[1][2][(mask == 0).expand(2, 20)].any() and outs[1][2].any()


def test_sizes_beyond_the_kernels_take_the_torch_formulation(monkeypatch):
    """Choices and tokens that pass the kernels' 32 bits: broadcast tensors of one element, seen as device tensors."""
    from experts4bit_qlora_amd import router as R

    seen = []
    monkeypatch.setattr(R, "_on_kernel", lambda t: True)
    monkeypatch.setattr(R, "_aligned", lambda t: t)  # nothing of this size is made
    monkeypatch.setattr(R.ops, "balance_loss", lambda *a: seen.append("kernel") or (torch.zeros(1), torch.zeros(1, 4), None, None))
    monkeypatch.setattr(R.ops, "router_topk", lambda *a: seen.append("kernel") or (torch.zeros(1, 1), torch.zeros(1, 1)))
    monkeypatch.setattr(R, "_balance_loss_torch", lambda *a: seen.append("torch"))
    monkeypatch.setattr(R, "_router_topk_torch", lambda *a: seen.append("torch"))
    z, index = torch.zeros(1, 1, 4), torch.zeros(1, 1, 1, dtype=torch.int64)
    e4b.balance_loss(z, index)
    e4b.balance_loss(z.expand(1, 1 << 29, 4), index.expand(1, 1 << 29, 4))
    e4b.balance_loss(z.expand(1, 1 << 31, 4), index.expand(1, 1 << 31, 1))
    e4b.router_topk(z[0], 1)
    e4b.router_topk(z[0].expand(1 << 31, 4), 1)
    assert seen == ["kernel", "torch", "torch", "kernel", "torch"]
