"""The losses over the vocabulary's logits off the device (the torch formulation, which is the kernels' definition): values
against numpy one token at a time, gradients against differences, masks, refusals."""
import math

import numpy as np
import pytest
import torch

import experts4bit_qlora_amd as e4b
from experts4bit_qlora_amd import losses as L

INF = float("inf")


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _batch(seqs=4, tokens=5, vocab=11, seed=1, dtype=torch.float64):
    g = _gen(seed)
    z = (2 * torch.randn(seqs, tokens, vocab, generator=g, dtype=torch.float64)).to(dtype)
    labels = torch.randint(0, vocab, (seqs, tokens), generator=g)
    labels[0, 0], labels[1, 2], labels[2, 1] = -100, vocab, -1
    mask = torch.rand(seqs, tokens, generator=g) > 0.2
    return z, labels, mask


def _plain_lp(row, label, tau):
    y = row / tau
    return y[label] - y.max() - math.log(np.exp(y - y.max()).sum())


def _plain_counted(labels, mask, vocab):
    return (labels >= 0) & (labels < vocab) & (np.ones(labels.shape, bool) if mask is None else mask)


def _plain_logprobs(z, labels, mask, tau):
    counted = _plain_counted(labels, mask, z.shape[-1])
    out = np.zeros(labels.shape)
    for n, t in zip(*np.nonzero(counted)):
        out[n, t] = _plain_lp(z[n, t], labels[n, t], tau)
    return out, counted


@pytest.mark.parametrize("tau", (0.5, 1.0, 3.0))
def test_logprobs(tau):
    z, labels, mask = _batch()
    for m in (None, mask, mask[0], mask.int() * 7):
        got = e4b.token_logprobs(z, labels, mask=m, temperature=tau)
        full = None if m is None else (m != 0).expand(4, 5).numpy()
        want, _ = _plain_logprobs(z.numpy(), labels.numpy(), full, tau)
        assert got.dtype == torch.float64 and got.shape == (4, 5)
        np.testing.assert_allclose(got.numpy(), want, rtol=1e-12, atol=1e-13)
    assert e4b.token_logprobs(z.bfloat16(), labels).dtype == torch.float32
    z.requires_grad_()
    assert torch.autograd.gradcheck(lambda a: e4b.token_logprobs(a, labels, mask, temperature=tau), z)


def test_leading_axes_and_label_types():
    z, labels, mask = _batch()
    want = e4b.token_logprobs(z, labels, mask)
    assert torch.equal(e4b.token_logprobs(z.view(2, 2, 5, 11), labels.view(2, 2, 5), mask.view(2, 2, 5)),
                       want.view(2, 2, 5))
    assert torch.equal(e4b.token_logprobs(z[1], labels[1], mask[1]), want[1])
    assert torch.equal(e4b.token_logprobs(z, labels.int(), mask), want)
    old, adv = torch.randn(4, 5, generator=_gen(2)) - 3, torch.randn(4, generator=_gen(3))
    for red, shape in (("none", (2, 2, 5)), ("sequence", (2, 2)), ("mean", ())):
        a, lp = e4b.policy_loss(z, labels, old, adv, mask=mask, reduction=red)
        b, lp2 = e4b.policy_loss(z.view(2, 2, 5, 11), labels.view(2, 2, 5), old.view(2, 2, 5), adv.view(2, 2),
                                 mask=mask.view(2, 2, 5), reduction=red)
        assert b.shape == shape and torch.equal(a.reshape(shape), b) and torch.equal(lp.view(2, 2, 5), lp2)


@pytest.mark.parametrize("loss_type,smoothing", (("sigmoid", 0.0), ("sigmoid", 0.1), ("hinge", 0.0), ("ipo", 0.0)))
@pytest.mark.parametrize("average", (False, True))
@pytest.mark.parametrize("ref_dim", (0, 1, 2))
def test_preference(loss_type, smoothing, average, ref_dim):
    z, labels, mask = _batch()
    ref = [None, torch.tensor([-3.0, -4.5, -2.0, -6.0]), torch.randn(4, 5, generator=_gen(4)) - 3][ref_dim]
    beta = 0.3
    loss, rewards = e4b.preference_loss(z, labels, ref, beta=beta, loss_type=loss_type, label_smoothing=smoothing,
                                        average=average, mask=mask)
    lp, counted = _plain_logprobs(z.numpy(), labels.numpy(), mask.numpy(), 1.0)
    S = []
    for n in range(4):
        c = counted[n]
        s = sum(lp[n][c]) - (sum(ref[n].numpy()[c].astype(np.float64)) if ref_dim == 2 else 0.0)
        s = s / max(1, c.sum()) if average else s
        S.append(s - (ref[n].item() if ref_dim == 1 else 0.0))
    np.testing.assert_allclose(rewards.numpy(), beta * np.array(S), rtol=1e-12)
    for b in range(2):
        d = S[b] - S[b + 2]
        h = beta * d
        sig = lambda x: 1 / (1 + math.exp(-x))  # noqa: E731
        want = {"sigmoid": -(1 - smoothing) * math.log(sig(h)) - smoothing * math.log(sig(-h)), "hinge": max(0.0, 1 - h),
                "ipo": (d - 1 / (2 * beta)) ** 2}[loss_type]
        assert abs(loss[b].item() - want) <= 1e-12 * max(1.0, abs(want))
    z.requires_grad_()
    assert torch.autograd.gradcheck(lambda a: e4b.preference_loss(
        a, labels, ref, beta=beta, loss_type=loss_type, label_smoothing=smoothing, average=average, mask=mask)[0], z)


@pytest.mark.parametrize("kl", (0.0, 0.1))
@pytest.mark.parametrize("per_token", (False, True))
def test_policy(kl, per_token):
    z, labels, mask = _batch()
    lp, counted = _plain_logprobs(z.numpy(), labels.numpy(), mask.numpy(), 0.8)
    g = _gen(5)
    old = torch.from_numpy(lp) - 0.4 * torch.randn(4, 5, generator=g, dtype=torch.float64)  # inside and outside the clip
    ref = torch.from_numpy(lp) + 0.3 * torch.randn(4, 5, generator=g, dtype=torch.float64)
    adv = torch.randn((4, 5) if per_token else (4,), generator=g, dtype=torch.float64)
    want = np.zeros((4, 5))
    for n, t in zip(*np.nonzero(counted)):
        a = adv[n, t].item() if per_token else adv[n].item()
        r = math.exp(lp[n, t] - old[n, t].item())
        want[n, t] = -min(r * a, min(max(r, 0.9), 1.3) * a)
        if kl:
            x = ref[n, t].item() - lp[n, t]
            want[n, t] += kl * (math.exp(x) - x - 1)
    call = lambda a, red: e4b.policy_loss(a, labels, old, adv, ref if kl else None, clip=(0.1, 0.3), kl_coef=kl,  # noqa: E731
                                          mask=mask, temperature=0.8, reduction=red)
    each, logps = call(z, "none")
    np.testing.assert_allclose(each.numpy(), want, rtol=1e-11, atol=1e-13)
    np.testing.assert_allclose(logps.numpy(), lp, rtol=1e-12, atol=1e-13)
    np.testing.assert_allclose(call(z, "sequence")[0].numpy(), want.sum(1) / counted.sum(1).clip(1), rtol=1e-11)
    np.testing.assert_allclose(call(z, "mean")[0].item(), want.sum() / counted.sum(), rtol=1e-11)
    z.requires_grad_()
    for red in ("none", "sequence", "mean"):
        assert torch.autograd.gradcheck(lambda a: call(a, red)[0], z)


@pytest.mark.parametrize("tau", (1.0, 2.0))
def test_distill(tau):
    z, _, mask = _batch()
    g = _gen(6)
    index = torch.randint(0, 11, (4, 5, 3), generator=g)
    index[0, 0, 1], index[0, 1, 0], index[2, 2] = -1, 11, torch.tensor([4, 4, 4])  # outside, outside, one entry thrice
    index[3, 3] = -5  # nothing usable
    mask[2, 2] = mask[3, 3] = mask[0, 0] = True
    teacher = torch.randn(4, 5, 3, generator=g, dtype=torch.float64)
    teacher[1, 1, 2] = -INF
    teacher[0, 0, 1] = float("nan")  # behind an index outside
    want = np.zeros((4, 5))
    for n, t in zip(*np.nonzero(mask.numpy())):
        y = z[n, t].numpy() / tau
        lq = y - y.max() - math.log(np.exp(y - y.max()).sum())
        use = [k for k in range(3) if 0 <= index[n, t, k] < 11 and teacher[n, t, k] > -INF]
        if use:
            w = np.array([teacher[n, t, k].item() for k in use]) / tau
            p = np.exp(w - w.max())
            p /= p.sum()
            want[n, t] = tau ** 2 * sum(p[i] * (math.log(p[i]) - lq[index[n, t, k]]) for i, k in enumerate(use))
    call = lambda a, red: e4b.distill_loss(a, teacher, index, mask=mask, temperature=tau, reduction=red)  # noqa: E731
    np.testing.assert_allclose(call(z, "none").numpy(), want, rtol=1e-11, atol=1e-13)
    n = mask.sum(1).numpy()
    np.testing.assert_allclose(call(z, "sequence").numpy(), want.sum(1) / n.clip(1), rtol=1e-11)
    np.testing.assert_allclose(call(z, "mean").item(), want.sum() / n.sum(), rtol=1e-11)
    z.requires_grad_()
    for red in ("none", "sequence", "mean"):
        assert torch.autograd.gradcheck(lambda a: call(a, red), z)
    (grad,) = torch.autograd.grad(call(z, "none").sum(), z)
    assert not grad[3, 3].any() and not grad[~mask].any() and grad[2, 2].any()


def _every_loss(z, labels, mask, ref=None):
    """(name, loss) of each with gradients, all tokens' mask applied."""
    old = torch.full(labels.shape, -2.0, device=z.device)
    index = torch.where((labels < 0) | (labels >= z.shape[-1]), 0, labels).unsqueeze(-1)
    yield "logprobs", e4b.token_logprobs(z, labels, mask)
    yield "preference", e4b.preference_loss(z, labels, ref, mask=mask)[0]
    yield "policy", e4b.policy_loss(z, labels, old, torch.ones(len(z), device=z.device), old, kl_coef=0.1, mask=mask)[0]
    yield "distill", e4b.distill_loss(z, torch.zeros(index.shape, device=z.device), index, mask=mask)


@pytest.mark.parametrize("dtype", (torch.float32, torch.float64))
def test_values_behind_the_mask_have_no_influence(dtype):
    z, labels, mask = _batch(dtype=dtype)
    mask[:, 1], mask[:, 3] = False, False
    mask[0, 2] = True
    bad = z.clone()
    bad[0, 1], bad[1, 1, 4], bad[2, 1], bad[3, 1, 5], bad[:, 3] = float("nan"), INF, -INF, torch.finfo(dtype).min, float("nan")
    outs = []
    for logits in (z, bad):
        leaf = logits.clone().requires_grad_()
        outs.append([(v.detach(), torch.autograd.grad(v.sum(), leaf)[0]) for _, v in _every_loss(leaf, labels, mask)])
    for (v, g), (bv, bg) in zip(*outs):
        assert torch.equal(v, bv) and torch.equal(g, bg) and not bg[~mask].any() and torch.isfinite(bg).all()


def test_masks_that_leave_nothing():
    z, labels, mask = _batch()
    mask[:] = False
    z.requires_grad_()
    for name, v in _every_loss(z, labels, mask):
        (grad,) = torch.autograd.grad(v.sum(), z)
        assert not grad.any() and torch.isfinite(v).all()
        if name == "preference":
            assert torch.allclose(v, torch.full_like(v, math.log(2)))
        else:
            assert not v.any()


def test_rows_without_a_finite_logit():
    """All -inf: every label has probability 0 and the gradient is zero; all the type's lowest: an even distribution."""
    z = torch.zeros(2, 2, 8)
    z[0, 0], z[0, 1] = -INF, torch.finfo(torch.float32).min
    z.requires_grad_()
    labels = torch.zeros(2, 2, dtype=torch.int64)
    lp = e4b.token_logprobs(z, labels)
    assert lp[0, 0] == -INF and torch.allclose(lp[0, 1], torch.tensor(-math.log(8)))
    (grad,) = torch.autograd.grad(lp, z, torch.ones_like(lp))
    assert not grad[0, 0].any() and torch.allclose(grad[0, 1], (torch.arange(8) == 0).float() - 1 / 8)
    v = e4b.distill_loss(z, torch.zeros(2, 2, 1), labels.unsqueeze(-1), reduction="none")
    assert v[0, 0] == INF and torch.allclose(v[0, 1], torch.tensor(math.log(8)))
    (grad,) = torch.autograd.grad(v, z, torch.ones_like(v))
    assert not grad[0, 0].any() and torch.isfinite(grad).all()
    v, _ = e4b.policy_loss(z, labels, torch.full((2, 2), -2.0), torch.ones(2), torch.full((2, 2), -2.0), kl_coef=0.1,
                           reduction="none")
    assert v[0, 0] == INF and torch.isfinite(v[0, 1])


def test_no_tokens():
    labels = torch.zeros(2, 0, dtype=torch.int64)
    for shape in ((2, 0, 8), (0, 3, 8)):
        z = torch.zeros(shape, requires_grad=True)
        labels = torch.zeros(shape[:2], dtype=torch.int64)
        for name, v in _every_loss(z, labels, None):
            assert torch.isfinite(v).all()
            assert torch.autograd.grad(v.sum(), z)[0].shape == shape
    z = torch.zeros(2, 3, 0, 8)
    labels = torch.zeros(2, 3, 0, dtype=torch.int64)
    assert e4b.token_logprobs(z, labels, torch.ones(2, 3, 0)).shape == (2, 3, 0)
    assert e4b.distill_loss(z, torch.zeros(2, 3, 0, 4), torch.zeros(2, 3, 0, 4).long(), reduction="sequence").shape == (2, 3)


def test_refusals():
    z, labels, mask = _batch()
    old, adv = torch.zeros(4, 5), torch.zeros(4)
    index, teacher = torch.zeros(4, 5, 2, dtype=torch.int64), torch.zeros(4, 5, 2)

    def refused(match, f, *a, **kw):
        with pytest.raises(ValueError, match=match):
            f(*a, **kw)

    for f, args in ((e4b.token_logprobs, (labels,)), (e4b.preference_loss, (labels,)), (e4b.policy_loss, (labels, old, adv)),
                    (e4b.distill_loss, (teacher, index))):
        refused("logits", f, z.long(), *args)
        refused("logits", f, z[0, 0], *args)
        refused("logits", f, z[..., :0], *args)
        refused("mask", f, z, *args, mask=torch.ones(4, 4))
        refused("mask", f, z, *args, mask=mask.to("meta"))
    for f, rest in ((e4b.token_logprobs, ()), (e4b.preference_loss, ()), (e4b.policy_loss, (old, adv))):
        for bad in (labels[:3], labels.float(), labels > 0, labels.to("meta")):
            refused("labels", f, z, bad, *rest)
    for t in (0.0, -1.0, INF, float("nan")):
        refused("temperature", e4b.token_logprobs, z, labels, temperature=t)
        refused("temperature", e4b.policy_loss, z, labels, old, adv, temperature=t)
        refused("temperature", e4b.distill_loss, z, teacher, index, temperature=t)
    for red in ("sum", None):
        refused("reduction", e4b.policy_loss, z, labels, old, adv, reduction=red)
        refused("reduction", e4b.distill_loss, z, teacher, index, reduction=red)
    refused("pairs", e4b.preference_loss, z[:3], labels[:3])
    refused("pairs", e4b.preference_loss, z[0], labels[0])
    refused("ref_logps", e4b.preference_loss, z, labels, old[:, :4])
    refused("ref_logps", e4b.preference_loss, z, labels, torch.zeros(2))
    refused("loss_type", e4b.preference_loss, z, labels, loss_type="kto")
    for beta in (0.0, -0.1, INF, float("nan")):
        refused("beta", e4b.preference_loss, z, labels, beta=beta)
    refused("label_smoothing", e4b.preference_loss, z, labels, label_smoothing=1.5)
    refused("label_smoothing", e4b.preference_loss, z, labels, loss_type="hinge", label_smoothing=0.1)
    refused("old_logps", e4b.policy_loss, z, labels, old[:2], adv)
    refused("old_logps", e4b.policy_loss, z, labels, old.long(), adv)
    refused("advantages", e4b.policy_loss, z, labels, old, adv[:2])
    refused("ref_logps", e4b.policy_loss, z, labels, old, adv, old[0])
    refused("kl_coef", e4b.policy_loss, z, labels, old, adv, kl_coef=0.1)
    refused("kl_coef", e4b.policy_loss, z, labels, old, adv, old, kl_coef=INF)
    for clip in ((-0.1, 0.2), (1.1, 0.2), (0.2, -0.1), (0.2, INF)):
        refused("clip", e4b.policy_loss, z, labels, old, adv, clip=clip)
    refused("teacher_index", e4b.distill_loss, z, teacher, index[0])
    refused("teacher_index", e4b.distill_loss, z, teacher[..., :0], index[..., :0])
    refused("teacher_index", e4b.distill_loss, z, teacher, teacher)
    refused("teacher_logits", e4b.distill_loss, z, teacher[..., :1], index)
    refused("teacher_logits", e4b.distill_loss, z, index, index)


def test_sizes_beyond_the_kernels_take_the_torch_formulation(monkeypatch):
    """Broadcast tensors of one element, seen as device tensors: nothing of these sizes is made."""
    seen = []
    monkeypatch.setattr(L, "_on_kernel", lambda t: True)
    monkeypatch.setattr(L, "_constant", lambda t, *a: t)

    class Kernels:
        token_logprobs = staticmethod(lambda z, *a: seen.append("kernel") or torch.zeros(1, 1).expand(z.shape[:2]))
        distill_loss = staticmethod(lambda *a: seen.append("kernel") or torch.zeros(()))

    monkeypatch.setattr(L.N, "torch_lib", lambda: Kernels)
    monkeypatch.setattr(L, "_token_logprobs_torch",
                        lambda z, *a: seen.append("torch") or (torch.zeros(1, 1).expand(z.shape[:2]), None))
    z, labels = torch.zeros(1, 1, 1), torch.zeros(1, 1, dtype=torch.int64)
    for shape in ((1, 5, 4), (1 << 21, 2, 4), (1, (1 << 31) - 1, 4), (1, 2, 1 << 30)):
        e4b.token_logprobs(z.expand(shape), labels.expand(shape[:2]))
    assert seen == ["kernel"] * 4
    for shape in ((1, 1 << 31, 4), ((1 << 21) + 1, 1, 4), (1 << 16, 1 << 15, 4), (1, 1, (1 << 30) + 1)):
        e4b.token_logprobs(z.expand(shape), labels.expand(shape[:2]))
    e4b.token_logprobs(z, labels, temperature=1e-31)
    assert seen[4:] == ["torch"] * 5
    monkeypatch.setattr(L, "_distill_loss_torch", lambda *a: seen.append("torch") or torch.zeros(()))
    for k, dtype in ((1024, torch.float32), (1025, torch.float32), (4, torch.float64)):
        e4b.distill_loss(z, torch.zeros(1, 1, 1, dtype=dtype).expand(1, 1, k), labels.unsqueeze(-1).expand(1, 1, k))
    assert seen[9:] == ["kernel", "torch", "torch"]


@pytest.mark.parametrize("vocab", (300, 50257))
@pytest.mark.parametrize("dtype", (torch.uint8, torch.int8, torch.int16, torch.int32, torch.uint16, torch.uint32, torch.uint64))
def test_narrow_and_unsigned_labels_and_indexes(dtype, vocab):
    """Integer types that do not hold the vocabulary's size, or that torch does not compare: as int64."""
    z = (2 * torch.randn(2, 4, vocab, generator=_gen(7))).requires_grad_()
    top = min(vocab, torch.iinfo(dtype).max + 1)
    labels = torch.randint(0, top, (2, 4), generator=_gen(8))
    labels[0, 0], labels[0, 1] = 0, top - 1
    if dtype.is_signed:
        labels[1, 0] = -100
    index = torch.randint(0, top, (2, 4, 3), generator=_gen(9))
    teacher = torch.randn(2, 4, 3, generator=_gen(10))
    old, adv = torch.full((2, 4), -9.0), torch.tensor([1.0, -1.0])
    for f, i in ((lambda i: e4b.token_logprobs(z, i), labels), (lambda i: e4b.preference_loss(z, i)[0], labels),
                 (lambda i: e4b.policy_loss(z, i, old, adv)[0], labels), (lambda i: e4b.distill_loss(z, teacher, i), index)):
        want, got = f(i), f(i.to(dtype))
        assert torch.equal(got, want) and want.any()
        ours, theirs = (torch.autograd.grad(v.sum(), z)[0] for v in (got, want))
        assert torch.equal(ours, theirs) and theirs.any()


def test_logits_that_a_transform_leaves_alone(monkeypatch):
    """Inside vmap, grad and jvp the kernels' autograd functions may not be called, whatever tensors they are given: logits that
    the transform does not follow (seen here as device tensors) take the torch formulation too."""
    z, labels, mask = _batch(dtype=torch.float32)
    ref = torch.randn(4, 5, generator=_gen(11)) - 3
    want = [v.detach() for _, v in _every_loss(z, labels, mask, ref)]
    monkeypatch.setattr(L, "_on_kernel", lambda t: True)
    monkeypatch.setattr(L.N, "torch_lib", None)
    w = torch.arange(1.0, 4.0)

    def scaled(a):
        return torch.stack([(a * v).sum() for _, v in _every_loss(z, labels, mask, ref)])

    sums = torch.stack([v.sum() for v in want])
    assert torch.allclose(torch.func.vmap(scaled)(w), w[:, None] * sums)
    assert torch.allclose(torch.func.jacrev(scaled)(w[0]), sums)
    assert torch.allclose(torch.func.jvp(scaled, (w[0],), (w[1],))[1], 2 * sums)


def test_complex_labels_are_refused():
    z, labels, mask = _batch()
    for f, args in ((e4b.token_logprobs, ()), (e4b.preference_loss, ()), (e4b.policy_loss, (torch.zeros(4, 5), torch.zeros(4)))):
        with pytest.raises(ValueError, match="labels must be integers"):
            f(z, labels.to(torch.complex64), *args)
    with pytest.raises(ValueError, match="teacher_index must be integers"):
        e4b.distill_loss(z, torch.zeros(4, 5, 2), torch.zeros(4, 5, 2, dtype=torch.complex64))


@pytest.mark.parametrize("dtype", (torch.float32, torch.bfloat16))
def test_temperatures_beyond_the_32_bits_of_the_logits_are_refused(dtype):
    """A temperature, or its inverse, that fp32 does not hold as a normal number divided rows into NaN; fp64 logits take it."""
    z, labels, _ = _batch(dtype=dtype)
    teacher, index = torch.zeros(4, 5, 2), torch.zeros(4, 5, 2, dtype=torch.int64)
    for t in (1e-46, 1e-39, 3e38, 1e39):
        for call in (lambda a: e4b.token_logprobs(a, labels, temperature=t),
                     lambda a: e4b.policy_loss(a, labels, torch.zeros(4, 5), torch.zeros(4), temperature=t),
                     lambda a: e4b.distill_loss(a, teacher, index, temperature=t)):
            with pytest.raises(ValueError, match="temperature"):
                call(z)
        assert torch.isfinite(e4b.token_logprobs(z.double(), labels, temperature=max(t, 1e-39))).any()
    for t in (1.2e-38, 8e37):
        assert not e4b.token_logprobs(z, labels, temperature=t).isnan().any()


def test_constants_with_a_tangent(monkeypatch):
    """Forward-mode tangents of what is a constant to the gradient do not reach the extension, whose functions refuse them."""
    import torch.autograd.forward_ad as fa

    z, labels, _ = _batch(dtype=torch.float32)
    old, adv, index = torch.randn(4, 5), torch.randn(4), torch.zeros(4, 5, 2, dtype=torch.int64)
    seen = []

    class Kernels:
        def __getattr__(self, name):
            def call(z, *args):
                seen.append((name, [fa.unpack_dual(t).tangent for t in args if isinstance(t, torch.Tensor)]))
                out = torch.zeros(())
                return (out, torch.zeros(4, 5)) if name in ("preference_loss", "policy_loss") else out
            return call

    monkeypatch.setattr(L, "_on_kernel", lambda t: True)
    monkeypatch.setattr(L.N, "torch_lib", lambda: Kernels())
    with fa.dual_level():
        dual = lambda t: fa.make_dual(t, torch.ones_like(t))  # noqa: E731
        e4b.preference_loss(z, labels, dual(old))
        e4b.policy_loss(z, labels, dual(old), dual(adv), dual(old), kl_coef=0.1)
        e4b.distill_loss(z, dual(torch.randn(4, 5, 2)), index)
    assert [n for n, _ in seen] == ["preference_loss", "policy_loss", "distill_loss"]
    assert all(t is None for _, ts in seen for t in ts)


def test_recorded_calls_take_the_torch_formulation(monkeypatch):
    """make_fx records torch's operators: what a kernel writes is not among them, and the recorded function would return
    memory that nothing fills. The logits are seen here as device tensors."""
    from torch.fx.experimental.proxy_tensor import make_fx

    z, labels, mask = _batch(dtype=torch.float32)
    other = z.flip(0) * 0.5
    want = [v for _, v in _every_loss(other, labels, mask)]
    monkeypatch.setattr(L, "_on_kernel", lambda t: True)
    monkeypatch.setattr(L.N, "torch_lib", None)
    for mode in ("real", "fake", "symbolic"):
        recorded = make_fx(lambda a: [v for _, v in _every_loss(a, labels, mask)], tracing_mode=mode,
                           _allow_non_fake_inputs=True)(z)
        assert all(torch.allclose(a, b, rtol=1e-5) for a, b in zip(recorded(other), want))
