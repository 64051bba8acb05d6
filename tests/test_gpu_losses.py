"""The kernels of the losses over the vocabulary's logits against 64-bit plain torch on the CPU.

Tolerances, with u = 2^-24, D = (max z - z_j) / temperature and R the row's largest D at most 104 (beyond, an exponential is
below fp32's smallest value and its error below 2^-149): a difference to the maximum, its factor log2(e) / temperature and
their product make an exponential's argument off by at most 4 u D, the exponential by 2 u more (where the difference is to
the label instead, two multiply-adds round an argument of at most D_j + D_l <= 2 R: 1.4 u of that, no more; and the first's result
may be larger than that by the product with the factor's small part, 2^-11 of at most 2^16: 22 u, which n has room for). A row's sum has
at most n = max(64, V / 256) + 40 additions one after the other, each of which may be followed by a rescaling of 3
roundings, so it is off by E = (4 R + 4 n) u relative. A log-probability D_l - log s is off by E + (3 D_l + 2 |log s| + |lp|) u; a
probability by E + (4 D + 8) u relative; a result rounded into a 16-bit type by half a step of it, or of its smallest
normal value."""
import pytest
import torch

import experts4bit_qlora_amd as e4b
from experts4bit_qlora_amd import _native as N
from experts4bit_qlora_amd import losses as L

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24
TINY = 2.0 ** -126  # exponentials and products below fp32's normal range
INF = float("inf")
DTYPES = (torch.float32, torch.bfloat16, torch.float16)
# both sides of a piece, a wave, a workgroup and its unrolled step, of a backward part; odd ones; large ones
VOCABS = (1, 2, 3, 7, 8, 9, 15, 17, 63, 64, 65, 129, 500, 1000, 1023, 2047, 2049, 4095, 4097, 8191, 8192, 8193, 8207, 16385,
          32000, 32769, 50257, 65537, 131075)


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _logits(shape, dtype, seed, spread=3.0):
    return (torch.randn(shape, generator=_gen(seed)) * spread).to(dtype)


def _half_step(dtype, value):
    f = torch.finfo(dtype)
    return f.eps / 2 * value.abs().clamp(min=f.smallest_normal)


class Row64:
    """Log-probabilities and probabilities of every entry in 64 bits, and how far the kernels may be off."""

    def __init__(self, logits, tau):
        z = logits.detach().cpu().double()
        V = z.shape[-1]
        self.tau, self.empty = tau, (z == -INF).all(-1, keepdim=True)
        z = torch.where(self.empty, 0.0, z)
        self.D = (z.amax(-1, keepdim=True) - z) / tau
        self.s = torch.exp(-self.D).sum(-1, keepdim=True)
        self.lp = (-self.D - self.s.log()).masked_fill(self.empty, -INF)
        self.q = torch.exp(-self.D) / self.s
        R = self.D.clamp(max=104).amax(-1, keepdim=True)
        self.E = (4 * R + 4 * (max(64, V / 256) + 40)) * U

    def lp_bound(self):
        return self.E + (3 * self.D.nan_to_num(0, 0, 0) + 2 * self.s.log() + self.lp.abs().nan_to_num(0, 0, 0)) * U + TINY

    def q_bound(self):
        return self.q * (self.E + (4 * self.D.clamp(max=1e4) + 8) * U) + TINY


def _labels_grad(r, at, w, dw, dtype):
    """(gradient, bound) of labels `at` whose log-probabilities have the derivatives w, known up to dw (both [N, T])."""
    w, dw = w.unsqueeze(-1), dw.unsqueeze(-1)
    hit = torch.zeros_like(r.q).scatter(-1, at.unsqueeze(-1), 1.0)
    want = torch.where(r.empty, 0.0, w / r.tau * (hit - r.q))
    bound = ((w.abs() * (r.q_bound() + 6 * U * (hit + r.q))) + dw * (hit + r.q)) / r.tau
    return want, torch.where(r.empty, 0.0, bound) + _half_step(dtype, want) + TINY


def _near(got, want, bound, what=""):
    out = got.detach().cpu()
    err = (out.double() - want).abs()
    # the want rounded into the result's type is right whatever the bound: beyond that type's range, an infinity
    same = (out == want.to(out.dtype)) | (err <= bound)
    assert same.all(), f"{what}: off by {err[~same].max().item():.3g}, {(err / bound)[~same].max().item():.3g} of the bound"


def _counted(labels, mask, shape, V):
    c = (labels >= 0) & (labels < V)
    return c if mask is None else c & (mask != 0).expand(shape)


def _check_logprobs(logits, labels, mask=None, tau=1.0, seed=0):
    leaf = logits.to(DEV).detach().requires_grad_()
    args = (labels.to(DEV), None if mask is None else mask.to(DEV))
    lp = e4b.token_logprobs(leaf, *args, temperature=tau)
    V, shape = logits.shape[-1], logits.shape[:-1]
    c = _counted(labels, mask, shape, V)
    r, at = Row64(logits, tau), torch.where(c, labels.long(), 0)
    want = r.lp.gather(-1, at.unsqueeze(-1)).squeeze(-1)
    bound = r.lp_bound().gather(-1, at.unsqueeze(-1)).squeeze(-1)
    assert lp.dtype == torch.float32 and lp.shape == shape
    _near(lp, torch.where(c, want, 0.0), torch.where(c, bound, 0.0), "logps")
    with torch.no_grad():
        assert torch.equal(e4b.token_logprobs(leaf, *args, temperature=tau), lp)
    g = torch.randn(shape, generator=_gen(seed))
    (got,) = torch.autograd.grad(lp, leaf, g.to(DEV))
    assert got.dtype == logits.dtype and got.shape == logits.shape
    w = torch.where(c, g.double(), 0.0)
    _near(got, *_labels_grad(r, at, w, torch.zeros_like(w), logits.dtype), "gradient")
    assert not got.cpu()[~c].any()


@pytest.mark.parametrize("V", VOCABS)
def test_logprobs_every_vocabulary(V):
    for i, dtype in enumerate(DTYPES):
        labels = torch.randint(0, V, (1, 3), generator=_gen(V))
        labels[0, 0], labels[0, 1] = 0, V - 1  # the first and the last entry
        _check_logprobs(_logits((1, 3, V), dtype, V + i), labels, tau=(1.0, 0.7, 2.0)[i], seed=V)


@pytest.mark.parametrize("seqs,tokens", ((1, 1), (2, 1), (1, 2), (37, 1), (3, 61), (5, 257), (700, 3)))
def test_logprobs_lengths_and_masks(seqs, tokens):
    g = _gen(seqs * tokens)
    V = 777
    labels = torch.randint(-3, V + 3, (seqs, tokens), generator=g)  # some outside
    one, each = torch.rand(tokens, generator=g) > 0.3, torch.rand(seqs, tokens, generator=g) > 0.5
    for i, mask in enumerate((None, one, each, each.int() * 3)):
        _check_logprobs(_logits((seqs, tokens, V), DTYPES[i % 3], i), labels, mask)


@pytest.mark.parametrize("V", (74999, 75000, 81920, 81921, 149999, 150000, 152064, 155648, 155649))
@pytest.mark.parametrize("rows", (1, 9, 64, 65))
def test_few_long_rows(rows, V):
    """Rows shared by several workgroups (from 300,000 bytes on), and one row or logit short of it; labels and the largest logit
    at the parts' borders, uncounted rows and ones of a very wide range between."""
    for i, dtype in enumerate(DTYPES):
        z = _logits((rows, 1, V), dtype, V + rows + i)
        edges = torch.tensor([0, 8191, 8192, 8193, V - 1, 65535 % V, 65536 % V, 16383, 3])
        labels = edges[torch.arange(rows) % 9].unsqueeze(-1)
        z[torch.arange(rows), 0, edges.flip(0)[torch.arange(rows) % 9]] += 12
        if rows > 4:
            labels[3], z[3] = -100, float("nan")
            z[4] *= 100
        if rows > 9:
            z[5] = -INF
        _check_logprobs(z.nan_to_num(0.0, posinf=INF, neginf=-INF), labels, tau=(1.0, 0.7, 2.0)[i])
        if rows > 4:
            pairs = z[:2 * (rows // 2)].clamp(min=-50, max=50).nan_to_num(0.0)
            _check_preference(pairs, labels[:len(pairs)], None, beta=0.01)
            _check_policy(pairs, labels[:len(pairs)].clamp(min=0), torch.ones(len(pairs)), kl=0.05)
        teacher, index = _teacher(z.nan_to_num(0.0, neginf=-INF)[:9], 6, V)
        _check_distill(z[:9].nan_to_num(0.0, neginf=-INF), teacher.clamp(min=-50), index, None, 1.0, "none")


def test_logprobs_label_types_and_far_labels():
    z = _logits((2, 5, 100), torch.float32, 1)
    labels = torch.tensor([[0, 99, 100, -1, 1 << 40], [-(1 << 40), 50, -100, 3, 2 ** 63 - 1]])
    _check_logprobs(z, labels)
    for dtype in (torch.int32, torch.int16, torch.uint8):
        _check_logprobs(z, labels.clamp(0, 99).to(dtype))


@pytest.mark.parametrize("dtype", DTYPES)
def test_logprobs_ranges_and_extremes(dtype):
    V = 3001
    labels = torch.randint(0, V, (1, 12), generator=_gen(3))
    low, high = torch.finfo(dtype).min, torch.finfo(dtype).max
    z = _logits((1, 12, V), dtype, 4)
    z[0, 0] = -INF
    z[0, 1] = low
    z[0, 2, 5:] = low
    z[0, 3, 1:] = -INF
    z[0, 4] = 0
    z[0, 5, :] = -1000.0
    z[0, 6, 17] = high
    z[0, 7] = high
    z[0, 8, 100:] = -INF
    z[0, 9, ::2] = low
    z[0, 10, 2000] = 60.0
    labels[0, :4] = torch.tensor([3, 5, 1, 0])
    labels[0, 8], labels[0, 10] = 99, 2000
    for tau in (1.0, 0.3, 5.0):
        _check_logprobs(z, labels, tau=tau)
    for spread in (1e-4, 30.0, 300.0):
        _check_logprobs(_logits((1, 12, V), dtype, 5, spread), labels)


@pytest.mark.parametrize("dtype", DTYPES)
def test_logits_far_from_zero(dtype):
    """The same rows moved up and down: on both sides of where the reference leaves fp32's room, and far behind it."""
    V = 5000
    z = _logits((2, 4, V), torch.float32, 81, 2.0)
    labels = torch.randint(0, V, (2, 4), generator=_gen(82))
    for off in (3e2, -3e3, 4e4, 4.5e4, -4.55e4, -4.6e4, 6e4, 1e6, -1e6, 1e10, -1e10):
        if dtype != torch.float16 or abs(off) <= 6e4:
            moved = (z + off).to(dtype)
            _check_logprobs(moved, labels)
            want = torch.log_softmax(moved.double(), -1).gather(-1, labels.unsqueeze(-1)).double()[..., 0]
            rewards = e4b.preference_loss(moved.to(DEV), labels.to(DEV), beta=1.0)[1].cpu()
            r = Row64(moved, 1.0)
            bound = r.lp_bound().gather(-1, labels.unsqueeze(-1))[..., 0]
            _near(rewards, want.sum(-1), bound.sum(-1) + 2 * U * want.sum(-1).abs(), f"rewards at {off}")


@pytest.mark.parametrize("dtype", (torch.float32, torch.bfloat16))
@pytest.mark.parametrize("V", (1000, 32000))
def test_rewards_errors_do_not_add_up(dtype, V):
    """A sequence's log-probabilities summed: rounded to the nearest, their errors are as often up as down. 2,048 of them are off
    by 2^-26 each in the mean at most, a quarter of the half step of one rounding that always goes the same way."""
    T = 2048
    z = _logits((2, T, V), dtype, 83, 2.0)
    labels = torch.randint(0, V, (2, T), generator=_gen(84))
    lp = torch.log_softmax(z.double(), -1).gather(-1, labels.unsqueeze(-1))[..., 0]
    ref = lp.float()
    rewards = e4b.preference_loss(z.to(DEV), labels.to(DEV), ref.to(DEV), beta=1.0)[1].cpu().double()
    off = rewards - (lp - ref.double()).sum(-1)
    assert (off.abs() <= T * 2.0 ** -26).all(), off / T


def test_temperatures_at_the_ends():
    """So low that a scaled logit leaves fp32, so high that all are alike."""
    z = _logits((1, 6, 300), torch.float32, 71, 1e9)
    labels = torch.randint(0, 300, (1, 6), generator=_gen(72))
    labels[0, :3] = z[0, :3].argmax(-1)
    lp = e4b.token_logprobs(z.to(DEV), labels.to(DEV), temperature=2e-30).cpu()
    # the largest logit has all the probability; the others' are -(max - z) / 2e-30, from 3.4e38 on an infinity
    away = (z.double().gather(-1, labels.unsqueeze(-1)).squeeze(-1) - z.double().amax(-1)) / 2e-30
    assert torch.equal(lp[0, :3], torch.zeros(3)) and (lp[0, 3:] < -1e36).all()
    assert torch.allclose(lp, away.float(), rtol=1e-6)
    lp = e4b.token_logprobs(z.to(DEV), labels.to(DEV), temperature=5e29)
    assert torch.allclose(lp.cpu(), torch.full((1, 6), -5.703782474656201))
    for tau in (1e-6, 1e6):
        _check_logprobs(_logits((1, 6, 300), torch.float32, 73, tau), labels, tau=tau)


def test_label_without_probability():
    """A label at -inf, beside finite logits: log-probability -inf, a finite gradient."""
    z = _logits((1, 2, 50), torch.float32, 6)
    z[0, 0, 7] = -INF
    leaf = z.to(DEV).requires_grad_()
    lp = e4b.token_logprobs(leaf, torch.tensor([[7, 7]], device=DEV))
    assert lp[0, 0] == -INF and torch.isfinite(lp[0, 1])
    (grad,) = torch.autograd.grad(lp.sum(), leaf)
    want = (torch.arange(50) == 7).double() - torch.softmax(z.double(), -1)
    assert torch.isfinite(grad).all() and (grad.cpu().double() - want).abs().max() < 1e-5


def test_nan_and_infinity_stay_in_their_rows():
    z = _logits((1, 5, 300), torch.float32, 7)
    z[0, 1, 30], z[0, 2, 40] = float("nan"), INF
    z[0, 3] = float("nan")
    leaf = z.to(DEV).requires_grad_()
    labels = torch.full((1, 5), 9, device=DEV)
    lp = e4b.token_logprobs(leaf, labels)
    assert lp[0, 1:4].isnan().all() and torch.isfinite(lp[0, [0, 4]]).all()
    at_label = z.clone()
    at_label[0, 0, 9], at_label[0, 4, 9] = INF, float("nan")
    got = e4b.token_logprobs(at_label.to(DEV), labels)
    assert got.isnan().all()
    (grad,) = torch.autograd.grad(lp.sum(), leaf)
    assert grad[0, 1].isnan().all() and torch.isfinite(grad[0, [0, 4]]).all() and grad[0, 3].isnan().all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_views(dtype):
    """Rows at other strides and addresses, transposed ones, broadcast ones; the gradient reaches the whole tensor."""
    V = 333
    big = _logits((4, 9, V + 10), dtype, 8).to(DEV).requires_grad_()
    labels = torch.randint(0, V, (4, 9), generator=_gen(9)).to(DEV)
    turned = _logits((V, 9, 4), dtype, 10).to(DEV).requires_grad_()
    cases = ((big, lambda t: t[:, :-1], labels[:, 1:]), (big, lambda t: t[:, 1:, 3:V], labels[:, 1:] % (V - 3)),
             (big, lambda t: t[::2, ::3, 1:V + 1], labels[::2, ::3]), (big, lambda t: t[2, :, 5:], labels[2]),
             (turned, lambda t: t.permute(2, 1, 0), labels), (big, lambda t: t[:1].expand(4, 9, V + 10), labels),
             (big, lambda t: t[:, :1].expand(4, 9, V + 10), labels))
    for leaf, view, lab in cases:
        v = view(leaf)
        lp = e4b.token_logprobs(v, lab)
        # the sums' order goes by the rows' addresses: each is held to the 64-bit values, not to a copy's
        r, at = Row64(v.contiguous(), 1.0), lab.cpu().unsqueeze(-1)
        _near(lp, *(t.gather(-1, at).squeeze(-1) for t in (r.lp, r.lp_bound())), "logps")
        (own,) = torch.autograd.grad(lp, v, torch.ones_like(lp), retain_graph=True)
        one = torch.ones(lab.shape, dtype=torch.float64)
        _near(own, *_labels_grad(r, lab.cpu(), one, 0 * one, dtype), "gradient")
        (got,) = torch.autograd.grad(lp, leaf, torch.ones_like(lp))
        second = leaf.detach().clone().requires_grad_()
        (want,) = torch.autograd.grad(view(second), second, own)
        assert torch.equal(got, want)


# ----------------------------------------------------------------------- the three losses


def _check_preference(logits, labels, ref, mask=None, beta=0.1, loss_type="sigmoid", smoothing=0.0, average=False):
    leaf = logits.to(DEV).detach().requires_grad_()
    on = lambda t: None if t is None else t.to(DEV)  # noqa: E731
    kw = dict(beta=beta, loss_type=loss_type, label_smoothing=smoothing, average=average, mask=on(mask))
    loss, rewards = e4b.preference_loss(leaf, labels.to(DEV), on(ref), **kw)
    c = _counted(labels, mask, labels.shape, logits.shape[-1])
    r, at = Row64(logits, 1.0), torch.where(c, labels, 0)
    lp = r.lp.gather(-1, at.unsqueeze(-1)).squeeze(-1)
    if ref is not None and ref.dim() == 2:
        lp = lp - ref.double()
    n = c.sum(-1).clamp(min=1).double() if average else torch.ones(len(c), dtype=torch.float64)
    # the sums are in 64 bits of log-probabilities whose own row sums are in 32
    dS = torch.where(c, r.E.squeeze(-1), 0.0).sum(-1) / n + 1e-12
    S = torch.where(c, lp, 0.0).sum(-1) / n
    if ref is not None and ref.dim() == 1:
        S = S - ref.double()
    S.requires_grad_()
    B = len(S) // 2
    d = S[:B] - S[B:]
    if loss_type == "sigmoid":
        ls = torch.nn.functional.logsigmoid
        want = -(1 - smoothing) * ls(beta * d) - smoothing * ls(-beta * d)
        steep, bend = beta, beta * beta / 4  # the largest slope and curvature by d
    elif loss_type == "hinge":
        want = torch.relu(1 - beta * d)
        steep, bend = beta, 0.0
        assert ((beta * d - 1).abs() > 1e-3).all()  # no pair where 32 bits may choose the other side
    else:
        want = (d - 0.5 / beta) ** 2
        steep, bend = 2 * (d.detach() - 0.5 / beta).abs() + 1e-3, 2.0
    dd = dS[:B] + dS[B:]
    assert loss.shape == (B,) and rewards.shape == (2 * B,) and loss.dtype == rewards.dtype == torch.float32
    # beta and the smoothing travel as fp32
    _near(loss, want.detach(), steep * dd + 8 * U * (want.detach() + steep * d.detach().abs()) + 1e-9, "loss")
    _near(rewards, beta * S.detach(), beta * dS + 4 * U * beta * S.detach().abs() + 1e-9, "rewards")
    up = torch.rand(B, generator=_gen(11)) + 0.5
    (got,) = torch.autograd.grad(loss, leaf, up.to(DEV))
    (w,) = torch.autograd.grad(want, S, up.double())
    w = (w / n).unsqueeze(-1) * c
    dw = ((bend * dd * up.double()).repeat(2) / n + 1e-12).unsqueeze(-1) + 8 * U * w.abs() + 4 * U * (
        steep * up.double()).repeat(2).unsqueeze(-1) / n.unsqueeze(-1)
    _near(got, *_labels_grad(r, at, w, torch.where(c, dw, 0.0), logits.dtype), "gradient")
    assert not got.cpu()[~c].any()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("loss_type,smoothing", (("sigmoid", 0.0), ("sigmoid", 0.2), ("hinge", 0.0), ("ipo", 0.0)))
def test_preference_kinds(dtype, loss_type, smoothing):
    z = _logits((6, 33, 1001), dtype, 12)
    labels = torch.randint(-20, 1001, (6, 33), generator=_gen(13))
    mask = torch.rand(6, 33, generator=_gen(14)) > 0.3
    per_token = torch.randn(6, 33, generator=_gen(15)) - 9
    for ref in (None, per_token, torch.tensor([-250.0, -200.0, -180.0, -160.0, -220.0, -210.0])):
        for average in (False, True):
            _check_preference(z, labels, ref, mask, 0.05, loss_type, smoothing, average)


@pytest.mark.parametrize("pairs,tokens,V", ((1, 1, 9), (1, 2, 5000), (3, 1025, 100), (40, 7, 300), (1, 5000, 64)))
def test_preference_lengths(pairs, tokens, V):
    z = _logits((2 * pairs, tokens, V), torch.float32, tokens)
    labels = torch.randint(0, V, (2 * pairs, tokens), generator=_gen(tokens))
    ref = Row64(z, 1.0).lp.gather(-1, labels.unsqueeze(-1)).squeeze(-1).float() + 0.3 * torch.randn(
        labels.shape, generator=_gen(16))
    _check_preference(z, labels, ref)


def test_preference_empty_answers_and_hidden_references():
    """An answer without a counted token has sum 0; reference values behind the mask have no influence."""
    z = _logits((4, 6, 50), torch.float32, 17)
    labels = torch.randint(0, 50, (4, 6), generator=_gen(18))
    labels[1] = -100
    mask = torch.ones(4, 6, dtype=torch.bool)
    mask[2] = False
    mask[0, 3] = False
    ref = torch.randn(4, 6, generator=_gen(19)) - 4
    for average in (False, True):
        _check_preference(z, labels, ref, mask, average=average)
    bad = ref.clone()
    bad[0, 3], bad[1], bad[2, 1] = float("nan"), INF, -INF
    for a, b in zip(*(e4b.preference_loss(z.to(DEV), labels.to(DEV), t.to(DEV), mask=mask.to(DEV)) for t in (ref, bad))):
        assert torch.equal(a, b)


def test_preference_far_apart():
    """Ratios of thousands either way: the loss grows like their difference, nothing overflows."""
    z = torch.zeros(2, 400, 20)
    z[0, :, 3], z[1, :, 3] = 20.0, -20.0
    labels = torch.full((2, 400), 3)
    for lab in (labels, labels):
        _check_preference(z, lab, None, beta=1.0)
        _check_preference(z.flip(0).contiguous(), lab, None, beta=1.0, smoothing=0.1)


def _reduced64(each, c, red):
    if red == "none":
        return each
    return each.sum(-1) / c.sum(-1).clamp(min=1) if red == "sequence" else each.sum() / c.sum().clamp(min=1)


def _upstream(red, shape, seed=20):
    lead = {"none": shape, "sequence": shape[:1], "mean": ()}[red]
    return torch.rand(lead, generator=_gen(seed)) + 0.5


def _by_token(up, c, red):
    if red == "none":
        return up.double() * c
    if red == "sequence":
        return (up.double() / c.sum(-1).clamp(min=1)).unsqueeze(-1) * c
    return up.double() / c.sum().clamp(min=1) * c


def _check_policy(logits, labels, adv, mask=None, kl=0.0, tau=1.0, red="mean", clip=(0.2, 0.2), seed=21):
    V, shape = logits.shape[-1], labels.shape
    c = _counted(labels, mask, shape, V)
    r, at = Row64(logits, tau), torch.where(c, labels, 0)
    pick = lambda t: t.gather(-1, at.unsqueeze(-1)).squeeze(-1)  # noqa: E731
    lp, dlp = pick(r.lp), pick(r.lp_bound())
    # ratios inside and outside, none so near a border that 32 bits may choose the other side
    x = 0.3 * torch.randn(shape, generator=_gen(seed), dtype=torch.float64)
    for b in (torch.tensor(1 - clip[0]).log(), torch.tensor(1 + clip[1]).log()):
        x = torch.where((x - b).abs() < 1e-2, b + 1e-2, x)
    old = (lp - x).float()
    ref = (lp + 0.3 * torch.randn(shape, generator=_gen(seed + 1), dtype=torch.float64)).float() if kl else None
    leaf = logits.to(DEV).detach().requires_grad_()
    on = lambda t: None if t is None else t.to(DEV)  # noqa: E731
    loss, logps = e4b.policy_loss(leaf, labels.to(DEV), on(old), on(adv), on(ref), clip=clip, kl_coef=kl, mask=on(mask),
                                  temperature=tau, reduction=red)
    _near(logps, torch.where(c, lp, 0.0), torch.where(c, dlp, 0.0), "logps")
    A = adv.double() if adv.dim() == 2 else adv.double().unsqueeze(-1)
    ratio = torch.exp(lp - old.double())
    held = ratio.clamp(1 - clip[0], 1 + clip[1])
    free = ratio * A <= held * A
    each = -torch.minimum(ratio * A, held * A)
    slope = torch.where(free, -A * ratio, 0.0)
    # the exponent is off by the log-probability's error and its own rounding, the ratio by that and 2 u
    dr = dlp + (lp - old.double()).abs() * U + 4 * U
    dslope, deach = A.abs() * ratio * dr, A.abs() * (ratio.clamp(max=2) + 2) * (dr + 4 * U)
    if kl:
        y = ref.double() - lp
        e = torch.expm1(y)
        each, slope = each + kl * (e - y), slope - kl * e
        dy = dlp + y.abs() * U
        deach = deach + kl * ((e.abs() + 1) * (dy + 4 * U) + dy + (e.abs() + y.abs()) * 4 * U)
        dslope = dslope + kl * (e.abs() + 1) * (dy + 6 * U)
    each, deach = torch.where(c, each, 0.0), torch.where(c, deach, 0.0)
    want = _reduced64(each, c, red)
    assert loss.shape == want.shape and loss.dtype == torch.float32
    _near(loss, want, _reduced64(deach + 4 * U * each.abs(), c, red) + 2 * U * want.abs(), "loss")
    up = _upstream(red, shape)
    (got,) = torch.autograd.grad(loss, leaf, up.to(DEV))
    by = _by_token(up, c, red)
    w = torch.where(c, slope, 0.0) * by
    dw = torch.where(c, dslope, 0.0) * by + 6 * U * w.abs()
    _near(got, *_labels_grad(r, at, w, dw, logits.dtype), "gradient")
    assert not got.cpu()[~c].any()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("red", ("none", "sequence", "mean"))
def test_policy_reductions_and_kinds(dtype, red):
    z = _logits((5, 41, 1003), dtype, 22)
    labels = torch.randint(-9, 1003, (5, 41), generator=_gen(23))
    mask = torch.rand(5, 41, generator=_gen(24)) > 0.3
    mask[3] = False  # a sequence without a counted token
    adv = torch.randn(5, generator=_gen(25))
    adv[1] = 0
    for kl in (0.0, 0.1):
        _check_policy(z, labels, adv, mask, kl, 1.0, red)
        _check_policy(z, labels, torch.randn(5, 41, generator=_gen(26)), mask[0], kl, 0.7, red, clip=(0.1, 0.4))


@pytest.mark.parametrize("seqs,tokens,V", ((1, 1, 5), (1, 1, 40000), (2, 1025, 65), (300, 3, 129), (1, 3000, 256)))
def test_policy_lengths(seqs, tokens, V):
    z = _logits((seqs, tokens, V), torch.bfloat16, tokens)
    labels = torch.randint(0, V, (seqs, tokens), generator=_gen(tokens))
    for red in ("mean", "sequence"):
        _check_policy(z, labels, torch.randn(seqs, generator=_gen(27)), None, 0.05, 2.0, red)


def test_policy_clipped_tokens_have_no_gradient():
    z = _logits((1, 4, 40), torch.float32, 28)
    labels = torch.randint(0, 40, (1, 4), generator=_gen(29))
    lp = torch.log_softmax(z, -1).gather(-1, labels.unsqueeze(-1)).squeeze(-1)
    old = lp - torch.tensor([[1.0, -1.0, 1.0, -1.0]])
    adv = torch.tensor([[1.0, 1.0, -1.0, -1.0]])  # clipped, free, free, clipped
    leaf = z.to(DEV).requires_grad_()
    loss, _ = e4b.policy_loss(leaf, labels.to(DEV), old.to(DEV), adv.to(DEV), reduction="none")
    (grad,) = torch.autograd.grad(loss.sum(), leaf)
    assert not grad[0, 0].any() and grad[0, 1].any() and grad[0, 2].any() and not grad[0, 3].any()
    assert torch.allclose(loss[0, [0, 3]].cpu(), torch.tensor([-1.2, 0.8]))


def test_policy_values_without_a_number():
    """A NaN advantage or old log-probability, a token of probability 0, an overflowing ratio: their own tokens alone, and as
    the formula has it."""
    z = _logits((1, 6, 40), torch.float32, 30)
    z[0, 2, 5] = -INF
    labels = torch.full((1, 6), 5)
    adv = torch.tensor([[float("nan"), 1.0, 1.0, -1.0, 1.0, 1.0]])
    old = torch.tensor([[-3.0, float("nan"), -3.0, -1000.0, -1000.0, -3.0]])
    outs = []
    for f, dev in ((e4b.policy_loss, DEV), (e4b.policy_loss, "cpu")):
        leaf = z.to(dev).requires_grad_()
        loss, _ = f(leaf, labels.to(dev), old.to(dev), adv.to(dev), torch.full((1, 6), -3.0, device=dev), kl_coef=0.1,
                    reduction="none")
        outs.append(loss.detach().cpu())
    assert torch.allclose(outs[0], outs[1], rtol=1e-5, equal_nan=True)
    assert outs[0][0, :2].isnan().all() and outs[0][0, 2] == INF and outs[0][0, 3] == INF and torch.isfinite(outs[0][0, 4:]).all()


def _check_distill(logits, teacher, index, mask=None, tau=1.0, red="mean"):
    V, shape = logits.shape[-1], logits.shape[:-1]
    c = torch.ones(shape, dtype=torch.bool) if mask is None else (mask != 0).expand(shape)
    r = Row64(logits, tau)
    w = teacher.double().masked_fill((index < 0) | (index >= V), -INF)
    none = (w == -INF).all(-1, keepdim=True)
    Dt = ((w.amax(-1, keepdim=True) - w) / tau).masked_fill(none, INF)
    p = torch.exp(-Dt)
    norm = p.sum(-1, keepdim=True)
    p = torch.where(none, 0.0, p / norm)
    lpt = torch.where(p > 0, -Dt - norm.log(), 0.0)
    at = torch.where((index >= 0) & (index < V), index, 0).long()
    pick = lambda t: t.gather(-1, at)  # noqa: E731
    lq, dlq = pick(r.lp), pick(r.lp_bound())
    K = index.shape[-1]
    dp = torch.where(p > 0, p * (4 * Dt.clamp(max=104) + 2 * K + 16) * U, 0.0) + TINY
    away = torch.where(p > 0, lpt - lq, 0.0)
    each = torch.where(c, tau ** 2 * (p * away).sum(-1), 0.0)
    # p and log p by the teacher's own row, log q by the student's; K additions
    dl = torch.where(p > 0, dlq + (3 * Dt.clamp(max=104) + 2 * norm.log().clamp(min=0) + lpt.abs() + 2 * K) * U, 0.0)
    deach = tau ** 2 * (dp * away.abs() + p * dl + (K + 8) * U * p * away.abs()).sum(-1)
    deach = torch.where(c, deach, 0.0)
    leaf = logits.to(DEV).detach().requires_grad_()
    on = lambda t: None if t is None else t.to(DEV)  # noqa: E731
    loss = e4b.distill_loss(leaf, on(teacher), on(index), mask=on(mask), temperature=tau, reduction=red)
    want = _reduced64(each, c, red)
    assert loss.shape == want.shape and loss.dtype == torch.float32
    _near(loss, want, _reduced64(deach + 4 * U * each.abs(), c, red) + 2 * U * want.abs(), "loss")
    up = _upstream(red, shape)
    (got,) = torch.autograd.grad(loss, leaf, up.to(DEV))
    by = (_by_token(up, c, red) * tau).unsqueeze(-1)
    by = torch.where(none | r.empty, 0.0, by)
    on_entries = torch.zeros_like(r.q).scatter_add(-1, at, p)
    slack = torch.zeros_like(r.q).scatter_add(-1, at, dp + (K + 8) * U * p)
    want = by * (r.q - on_entries)
    _near(got, want, by * (r.q_bound() + 6 * U * r.q + slack) + _half_step(logits.dtype, want) + TINY, "gradient")
    assert not got.cpu()[~c].any()


def _teacher(z, k, seed, dtype=torch.float32):
    values, index = torch.topk(z.float() + torch.randn(z.shape, generator=_gen(seed)), min(k, z.shape[-1]), dim=-1)
    return values.to(dtype), index


@pytest.mark.parametrize("K", (1, 2, 8, 63, 64, 65, 200, 1024))
def test_distill_entries(K):
    for i, dtype in enumerate(DTYPES):
        z = _logits((2, 5, 9000), dtype, K + i)
        teacher, index = _teacher(z, K, 31, DTYPES[(i + 1) % 3])
        _check_distill(z, teacher, index, None, (1.0, 2.0, 0.5)[i], ("none", "sequence", "mean")[i])


@pytest.mark.parametrize("V", (1, 2, 7, 9, 64, 1000, 2049, 8193, 16385, 50257))
def test_distill_every_vocabulary(V):
    for dtype in DTYPES:
        z = _logits((1, 3, V), dtype, V)
        _check_distill(z, *_teacher(z, 20, V), None, 1.5, "none")


@pytest.mark.parametrize("seqs,tokens", ((1, 1), (3, 61), (2, 1025), (300, 2)))
def test_distill_lengths_and_masks(seqs, tokens):
    z = _logits((seqs, tokens, 300), torch.bfloat16, tokens)
    teacher, index = _teacher(z, 5, 32)
    one, each = torch.rand(tokens, generator=_gen(33)) > 0.3, torch.rand(seqs, tokens, generator=_gen(34)) > 0.5
    for mask in (None, one, each, each.float()):
        for red in ("none", "sequence", "mean"):
            _check_distill(z, teacher, index, mask, 1.0, red)


def test_distill_entries_outside_repeated_and_empty():
    z = _logits((1, 8, 100), torch.float32, 35)
    teacher, index = _teacher(z, 6, 36)
    index = index.clone()
    index[0, 0, 2], index[0, 0, 3] = -1, 100
    index[0, 1] = torch.tensor([1 << 40, -(1 << 40), 2, 2, 2, 99])  # outside, one entry three times
    index[0, 2] = -1  # none usable
    index[0, 3] = 50  # one entry six times
    teacher[0, 0, 2] = float("nan")  # behind an index outside
    teacher[0, 4, 1:] = -INF
    teacher[0, 5] = -INF  # no value
    teacher[0, 6, 0] = 1e30
    z[0, 7] = -INF
    teacher[0, 7] = -INF
    for red in ("none", "mean"):
        _check_distill(z, teacher.nan_to_num(0.0, neginf=-INF), index, red=red)
    leaf = z.to(DEV).requires_grad_()
    a, b = (e4b.distill_loss(leaf, t.to(DEV), index.to(DEV), reduction="none")
            for t in (teacher, teacher.nan_to_num(0.0, neginf=-INF)))
    assert torch.equal(a, b)
    lone = z.to(DEV)
    teacher[0, 5, 3] = float("nan")
    got = e4b.distill_loss(lone, teacher.to(DEV), index.to(DEV), reduction="none")
    assert got[0, 5].isnan() and torch.isfinite(got[0, [0, 1, 2, 3, 4, 6, 7]]).all()


def test_distill_student_without_probability():
    """The student at -inf where the teacher has probability: an infinite loss, a finite gradient."""
    z = _logits((1, 2, 30), torch.float32, 37)
    z[0, 0, 4] = -INF
    z[0, 1] = -INF
    index = torch.tensor([[[4, 5], [4, 5]]])
    leaf = z.to(DEV).requires_grad_()
    loss = e4b.distill_loss(leaf, torch.zeros(1, 2, 2, device=DEV), index.to(DEV), reduction="none")
    assert (loss == INF).all()
    (grad,) = torch.autograd.grad(loss, leaf, torch.ones_like(loss))
    assert torch.isfinite(grad).all() and not grad[0, 1].any() and abs(grad[0, 0, 4].item() + 0.5) < 1e-6


# ------------------------------------------------------------------------------- behaviour


def _step(z, labels, mask, index, teacher, old):
    """Every loss and its gradient, through the public calls."""
    leaf = z.detach().requires_grad_()
    lp = e4b.token_logprobs(leaf, labels, mask)
    pair, rewards = e4b.preference_loss(leaf, labels, old, mask=mask)
    policy, logps = e4b.policy_loss(leaf, labels, old, old.sum(-1) + 9, old, kl_coef=0.1, mask=mask)
    each, _ = e4b.policy_loss(leaf, labels, old, old, mask=mask, reduction="sequence")
    away = e4b.distill_loss(leaf, teacher, index, mask=mask, temperature=2.0)
    outs = [lp, pair, policy, each, away]
    grads = [torch.autograd.grad(o, leaf, torch.ones_like(o))[0] for o in outs]
    return [o.detach() for o in outs] + [rewards, logps] + grads


def _inputs(dtype=torch.bfloat16, seqs=4, tokens=50, V=5000, seed=40):
    z = _logits((seqs, tokens, V), dtype, seed)
    teacher, index = _teacher(z, 8, seed)
    labels = torch.randint(-5, V, (seqs, tokens), generator=_gen(seed + 1))
    mask = torch.rand(seqs, tokens, generator=_gen(seed + 2)) > 0.2
    old = torch.randn(seqs, tokens, generator=_gen(seed + 3)) - 9
    return [t.to(DEV) for t in (z, labels, mask, index, teacher, old)]


def test_values_behind_the_mask_have_no_influence():
    z, labels, mask, index, teacher, old = _inputs()
    want = _step(z, labels, mask, index, teacher, old)
    hide = ~mask | (labels < 0)
    mask = ~hide
    want = _step(z, labels, mask, index, teacher, old)
    bad = [t.clone() for t in (z, old, teacher)]
    rows = hide.nonzero()
    for i, (n, t) in enumerate(rows.tolist()):
        bad[0][n, t] = (float("nan"), INF, -INF, torch.finfo(z.dtype).min)[i % 4]
    bad[2][hide] = float("nan")
    got = _step(bad[0], labels, mask, index, bad[2], old)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert all(torch.isfinite(t).all() for t in got)


def test_captured_and_replayed():
    """Everything in one graph, replayed on new inputs, against the eager calls."""
    data = _inputs()

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _step(*data)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = _step(*data)
    for i in range(4):
        for t, new in zip(data, _inputs(seed=50 + i)):
            t.copy_(new)
        graph.replay()
        got = [o.clone() for o in outs]
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, _step(*data)))


def test_another_stream_repeats_and_no_synchronization():
    data = _inputs(torch.float32)
    want = _step(data[0] * 2, *data[1:])
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    torch.cuda.set_sync_debug_mode("error")
    try:
        with torch.cuda.stream(stream):
            got = [_step(data[0] * 2, *data[1:]) for _ in range(4)]
    finally:
        torch.cuda.set_sync_debug_mode("default")
    stream.synchronize()
    for outs in got:
        assert all(torch.equal(a, b) for a, b in zip(outs, want))


def test_backward_twice_and_other_gradients():
    """The graph kept: the same gradient again, whatever became of the first one; a gradient of another size; a sum of two."""
    z, labels, mask, index, teacher, old = _inputs()
    for f in (lambda a: e4b.policy_loss(a, labels, old, old.sum(-1), mask=mask)[0],
              lambda a: e4b.distill_loss(a, teacher, index, mask=mask), lambda a: e4b.preference_loss(a, labels, old)[0].sum(),
              lambda a: e4b.token_logprobs(a, labels).sum()):
        leaf = z.detach().requires_grad_()
        loss = f(leaf)
        (one,) = torch.autograd.grad(loss, leaf, retain_graph=True)
        keep = one.clone()
        one.zero_()
        (two,) = torch.autograd.grad(loss, leaf, retain_graph=True)
        assert torch.equal(two, keep) and keep.any()
        (half,) = torch.autograd.grad(loss, leaf, torch.full_like(loss, 0.5), retain_graph=True)
        # half of every value, exactly, above the type's subnormal numbers
        assert torch.equal(half[keep.abs() > 1e-30], keep[keep.abs() > 1e-30] / 2)
        (zero,) = torch.autograd.grad(loss, leaf, torch.zeros_like(loss))
        assert not zero.any()


def test_gradients_by_differences():
    """Central differences of the kernels' own values along v in {-1, 1}^V, a token each. A row's log-probability moves along v
    with first to third derivatives of at most 2, 1 and 0.77 (mean, variance and third cumulant of values in [-1, 1]); a
    difference is off by h^2 / 6 of the loss's third derivative and by the values' own errors over h."""
    N_, V, h = 24, 50, 2.0 ** -5
    z = _logits((N_, 1, V), torch.float32, 90, 1.5)
    v = torch.where(torch.rand(N_, 1, V, generator=_gen(91)) < 0.5, -1.0, 1.0)
    labels = torch.randint(0, V, (N_, 1), generator=_gen(92)).to(DEV)
    adv = torch.randn(N_, generator=_gen(93)).to(DEV)
    teacher, index = (t.to(DEV) for t in _teacher(z, 5, 94))
    with torch.no_grad():
        start = e4b.token_logprobs(z.to(DEV), labels)
    # third derivatives: of A e^(lp - old) (r below 1.1 here: no ratio reaches the clip within h), |A| r (2^3 + 3 2 1 + 0.77),
    # of the KL term 0.1 e^x of the same (e^x below 2) and 0.1 0.77; of the pair's sigmoid at beta = 0.1, whose derivatives by d
    # are at most 0.1, 0.1^2 / 4 and 0.1^3 / 8, with d's at most 4, 2 and 1.54
    calls = (("logprobs", lambda a: e4b.token_logprobs(a, labels), 0.77),
             ("preference", lambda a: e4b.preference_loss(a, labels, start)[0], 0.008 + 0.06 + 0.154),
             ("policy", lambda a: e4b.policy_loss(a, labels, start, adv, start - 0.5, kl_coef=0.1, reduction="none")[0],
              1.1 * 14.8 * adv.abs().max().item() + 0.1 * (2 * 14.8 + 0.77)),
             ("distill", lambda a: e4b.distill_loss(a, teacher, index, temperature=2.0, reduction="none"), 0.77 / 2))
    for name, f, third in calls:
        leaf = z.to(DEV).requires_grad_()
        out = f(leaf)
        (grad,) = torch.autograd.grad(out, leaf, torch.ones_like(out))
        along = (grad.cpu().double() * v).sum((1, 2))
        with torch.no_grad():
            ends = [f((z + s * h * v).to(DEV)).cpu().double() for s in (1, -1)]
        diff = ((ends[0] - ends[1]) / (2 * h)).flatten()
        if name == "preference":
            along = along[:N_ // 2] + along[N_ // 2:]
        # a value's error: a row's (Row64's E at R = 10, twice in a pair), and z + h v's rounding, all times a slope of at most 4
        slack = 4 * 2 * ((40 + 4 * 104) + 60) * U / h + third * h * h / 6 + 1e-4
        assert ((along - diff).abs() <= slack).all(), (name, (along - diff).abs().max().item(), slack)


def test_saved_tensors_elsewhere_and_recomputed():
    """Saved tensors kept on the host between the passes, and a forward computed again in the backward."""
    from torch.utils.checkpoint import checkpoint

    z, labels, mask, index, teacher, old = _inputs()
    for f in (lambda a: e4b.token_logprobs(a, labels, mask).sum(), lambda a: e4b.preference_loss(a, labels, old)[0].sum(),
              lambda a: e4b.policy_loss(a, labels, old, old, mask=mask)[0], lambda a: e4b.distill_loss(a, teacher, index)):
        leaf = z.detach().requires_grad_()
        (want,) = torch.autograd.grad(f(leaf), leaf)
        with torch.autograd.graph.save_on_cpu():
            loss = f(leaf)
        assert torch.equal(torch.autograd.grad(loss, leaf)[0], want)
        assert torch.equal(torch.autograd.grad(checkpoint(f, leaf, use_reentrant=False), leaf)[0], want)
        with pytest.raises(RuntimeError, match="second time"):
            loss = f(leaf)
            torch.autograd.grad(loss, leaf)
            torch.autograd.grad(loss, leaf)


def test_leaf_gradients_accumulate():
    z, labels, mask, index, teacher, old = _inputs(torch.float32)
    leaf = z.detach().requires_grad_()
    parts = []
    for i in range(2):
        loss = e4b.distill_loss(leaf, teacher, index, mask=mask)
        parts.append(torch.autograd.grad(loss, leaf, retain_graph=True)[0])
        loss.backward()
    assert torch.equal(leaf.grad, parts[0] + parts[1])


def test_views_with_a_pending_sign():
    """Real tensors whose memory holds their negative (the imaginary part of a conjugate)."""
    z, labels = _logits((2, 5, 300), torch.float32, 91).to(DEV), torch.randint(0, 300, (2, 5), generator=_gen(92)).to(DEV)
    old, adv = _logits((2, 5), torch.float32, 93).to(DEV), _logits((2,), torch.float32, 94).to(DEV)
    index, teacher = torch.randint(0, 300, (2, 5, 7), generator=_gen(95)).to(DEV), _logits((2, 5, 7), torch.float32, 96).to(DEV)

    def negative(t):
        out = torch.complex(t, -t).conj().imag
        assert out.is_neg() and torch.equal(out, t)
        return out

    for a, b in ((e4b.token_logprobs(z, labels), e4b.token_logprobs(negative(z), labels)),
                 (e4b.policy_loss(z, labels, old, adv)[0], e4b.policy_loss(z, labels, negative(old), negative(adv))[0]),
                 (e4b.preference_loss(z, labels, old)[0], e4b.preference_loss(z, labels, negative(old))[0]),
                 (e4b.distill_loss(z, teacher, index), e4b.distill_loss(z, negative(teacher), index))):
        assert torch.allclose(a, b, rtol=1e-4, atol=1e-5)  # the wrong sign is off by the values themselves


def test_outputs_changed_in_place_leave_the_gradient():
    z, labels, mask, index, teacher, old = _inputs()
    leaf = z.detach().requires_grad_()
    loss, logps = e4b.policy_loss(leaf, labels, old, old.sum(-1), mask=mask, reduction="none")
    (want,) = torch.autograd.grad(loss, leaf, torch.ones_like(loss), retain_graph=True)
    logps.zero_()
    old.zero_()
    scaled = loss.mul_(2)
    (got,) = torch.autograd.grad(scaled, leaf, torch.full_like(loss, 0.5))
    assert torch.equal(got, want)
    leaf2 = (leaf.detach() * 1).requires_grad_()
    z2 = leaf2 * 1
    lp = e4b.token_logprobs(z2, labels)
    z2.zero_()  # the logits are needed again
    with pytest.raises(RuntimeError, match="inplace"):
        torch.autograd.grad(lp.sum(), leaf2)


def test_second_derivatives_are_refused():
    z, labels, mask, index, teacher, old = _inputs(torch.float32, 2, 3, 50)
    z.requires_grad_()
    for loss in (e4b.token_logprobs(z, labels).sum(), e4b.preference_loss(z, labels)[0].sum(),
                 e4b.policy_loss(z, labels, old, old)[0], e4b.distill_loss(z, teacher, index)):
        with pytest.raises(RuntimeError, match="once"):
            torch.autograd.grad(loss, z, create_graph=True)


def test_broadcast_and_strided_upstream_gradients():
    z, labels, mask, index, teacher, old = _inputs(torch.float32)
    leaf = z.requires_grad_()
    lp = e4b.token_logprobs(leaf, labels)
    w = torch.randn(lp.shape[1], lp.shape[0], device=DEV).t()
    (a,) = torch.autograd.grad(lp, leaf, w, retain_graph=True)
    (b,) = torch.autograd.grad(lp, leaf, w.contiguous(), retain_graph=True)
    (c,) = torch.autograd.grad(lp.sum(), leaf, retain_graph=True)
    (d,) = torch.autograd.grad(lp, leaf, torch.ones_like(lp))
    assert torch.equal(a, b) and torch.equal(c, d)
    each, _ = e4b.policy_loss(leaf, labels, old, old, reduction="sequence")
    (a,) = torch.autograd.grad(each.mean(), leaf, retain_graph=True)
    (b,) = torch.autograd.grad(each, leaf, torch.full_like(each, 0.25))
    assert torch.equal(a, b)


def test_formulations_agree_where_the_kernels_do_not_reach():
    z, labels, mask, index, teacher, old = _inputs(torch.float32, 2, 4, 2000)
    wide, many = torch.topk(z, 1100, dim=-1)
    ours = e4b.distill_loss(z, wide[..., :1024], many[..., :1024])
    assert torch.isfinite(e4b.distill_loss(z, wide, many)) and torch.isfinite(ours)
    d = z[:, :, :12].double().requires_grad_()
    few = labels % 12
    assert torch.autograd.gradcheck(lambda a: e4b.token_logprobs(a, few), d)
    single = e4b.token_logprobs(z, labels, mask)
    double = e4b.token_logprobs(z.double(), labels, mask)
    assert torch.allclose(single.double(), double, atol=1e-4)
    mapped = torch.func.vmap(lambda a, b: e4b.token_logprobs(a, b))(z, labels)
    assert torch.allclose(mapped, e4b.token_logprobs(z, labels), atol=1e-4)
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(z, torch.ones_like(z) * torch.arange(2000.0, device=DEV))
        tangent = torch.autograd.forward_ad.unpack_dual(e4b.token_logprobs(dual, labels)).tangent
    assert tangent is not None and tangent.any()


def test_no_tokens_on_the_device():
    for shape in ((2, 0, 8), (0, 3, 8)):
        z = torch.zeros(shape, device=DEV, requires_grad=True)
        labels = torch.zeros(shape[:2], dtype=torch.int64, device=DEV)
        ones = torch.zeros(shape[:2], device=DEV)
        outs = [e4b.token_logprobs(z, labels), e4b.preference_loss(z, labels, ones)[0],
                e4b.policy_loss(z, labels, ones, ones, ones, kl_coef=0.1)[0],
                e4b.policy_loss(z, labels, ones, ones, reduction="sequence")[0],
                e4b.distill_loss(z, torch.zeros(*shape[:2], 2, device=DEV), labels.unsqueeze(-1).expand(*shape[:2], 2))]
        for o in outs:
            assert torch.isfinite(o).all() and torch.autograd.grad(o.sum(), z)[0].shape == shape


def test_two_calls_at_once():
    """Host threads with a stream each."""
    import threading

    data = [_inputs(seed=60 + i) for i in range(3)]
    want = [_step(*d) for d in data]
    torch.cuda.synchronize()
    got, errors = [None] * 3, []

    def work(i):
        try:
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                for _ in range(5):
                    got[i] = _step(*data[i])
            stream.synchronize()
        except Exception as e:  # noqa: BLE001 - reported below
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(3)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert not errors
    for a, b in zip(got, want):
        assert all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize("dtype,V", ((torch.bfloat16, 131072), (torch.float32, 100003)))
def test_offsets_beyond_32_bits(dtype, V):
    """More than 2^31 logits (2^33 bytes in fp32): the last rows' values and gradients, zeros before them."""
    rows = 2 ** 31 // V + 40
    z = torch.zeros(1, rows, V, dtype=dtype, device=DEV)
    tail = _logits((1, 3, V), dtype, 70)
    z[:, -3:] = tail.to(DEV)
    z.requires_grad_()
    labels = torch.full((1, rows), -100, device=DEV)
    last = torch.tensor([[0, 12345, V - 1]])
    labels[:, -3:] = last.to(DEV)
    lp = e4b.token_logprobs(z, labels)
    (grad,) = torch.autograd.grad(lp.sum(), z)
    r, at, one = Row64(tail, 1.0), last.unsqueeze(-1), torch.ones(1, 3, dtype=torch.float64)
    _near(lp[:, -3:], *(t.gather(-1, at).squeeze(-1) for t in (r.lp, r.lp_bound())), "logps")
    _near(grad[:, -3:], *_labels_grad(r, last, one, 0 * one, dtype), "gradient")
    assert not lp[:, :-3].any() and not grad[:, -1000:-3].any() and not grad[:, :1000].any()
    index = torch.zeros(1, rows, 2, dtype=torch.int64, device=DEV)
    index[..., 1] = V - 1
    loss = e4b.distill_loss(z, torch.zeros(1, rows, 2, device=DEV), index, mask=labels[0] >= 0, reduction="none")
    (grad,) = torch.autograd.grad(loss.sum(), z)
    ends = torch.tensor([0, V - 1])
    away = -0.6931471805599453 - r.lp[..., ends]
    _near(loss[:, -3:], away.mean(-1), (r.lp_bound()[..., ends] + 16 * U * (1 + away.abs())).mean(-1), "loss")
    want = r.q.clone()
    want[..., ends] -= 0.5
    _near(grad[:, -3:], want, r.q_bound() + 8 * U + _half_step(dtype, want), "gradient")
    assert not loss[:, :-3].any() and not grad[:, -1000:-3].any() and not grad[:, :1000].any()


def test_a_training_step_with_the_adapters():
    """Expert layer with adapters (the training lane), head, and the losses in turn as a program trains: log-probabilities
    of the untrained model, then a step each on preference, policy and teacher; the adapters' gradients against the torch
    formulation's on the same logits."""
    E, H, I, k, N_, T, V = 4, 128, 64, 2, 4, 12, 301
    g = _gen(80)
    base = e4b.Experts4bit.from_float((torch.randn(E, 2 * I, H, generator=g) * 0.05).to(DEV),
                                      (torch.randn(E, H, I, generator=g) * 0.05).to(DEV), compute_dtype=torch.bfloat16)
    lora = e4b.ExpertsLoRA(base, r=4, alpha=8).to(DEV)
    with torch.no_grad():
        for p in (lora.gate_up_lora_B, lora.down_lora_B):
            p.copy_(torch.randn(p.shape, generator=g) * 0.05)
    assert e4b.enable_fast_train(lora) == 1
    x = torch.randn(N_ * T, H, generator=g).to(DEV, torch.bfloat16)
    gate = (torch.randn(H, E, generator=g) * 0.1).to(DEV, torch.bfloat16)
    head = (torch.randn(V, H, generator=g) * 0.3).to(DEV, torch.bfloat16)
    labels = torch.randint(0, V, (N_, T), generator=g).to(DEV)
    labels[:, :3] = -100
    adapters = [lora.gate_up_lora_A, lora.gate_up_lora_B, lora.down_lora_A, lora.down_lora_B]

    def logits():
        index, weights = e4b.router_topk(x @ gate, k, renorm=True)
        return torch.nn.functional.linear(x + lora(x, index, weights), head).view(N_, T, V)

    with torch.no_grad():
        z = logits()
        start = e4b.token_logprobs(z, labels)
        teacher, index = torch.topk(z.float() + torch.randn(z.shape, generator=g).to(DEV), 6, dim=-1)
    adv = torch.tensor([1.0, -0.5, 0.3, -1.0], device=DEV)
    losses = (lambda f, a: f.preference_loss(a, labels, start)[0].mean(),
              lambda f, a: f.policy_loss(a, labels, start - 0.05, adv, start, kl_coef=0.1)[0],
              lambda f, a: f.distill_loss(a, teacher, index, mask=labels >= 0, temperature=2.0))

    class Plain:  # the torch formulation of the same calls, in fp64
        preference_loss = staticmethod(lambda a, *r, **kw: L.preference_loss(a.double(), *r, **kw))
        policy_loss = staticmethod(lambda a, *r, **kw: L.policy_loss(a.double(), *r, **kw))
        distill_loss = staticmethod(lambda a, *r, **kw: L.distill_loss(a.double(), *r, **kw))

    for f in losses:
        z = logits()
        (through,) = torch.autograd.grad(f(e4b, z), z, retain_graph=True)
        ours = torch.autograd.grad(z, adapters, through, retain_graph=True)
        (plain,) = torch.autograd.grad(f(Plain, z), z, retain_graph=True)
        theirs = torch.autograd.grad(z, adapters, plain)
        # both gradients of the logits are fp64 values rounded to bf16 once, up to fp32's error: a step apart at most
        assert ((through.double() - plain.double()).abs() <= 2.0 ** -7 * plain.double().abs() + 1e-7).all()
        for a, b in zip(ours, theirs):
            assert torch.isfinite(a).all() and a.any()
            assert (a - b).norm() <= 2e-2 * b.norm()
    e4b.disable_fast_train(lora)


def _every_loss(labels, old, teacher, index):
    """The losses as functions of the logits, every reduction among them."""
    adv = old.sum(-1) + 9
    return {"logprobs": lambda a: e4b.token_logprobs(a, labels), "preference": lambda a: e4b.preference_loss(a, labels, old)[0],
            "policy, each": lambda a: e4b.policy_loss(a, labels, old, adv, old, kl_coef=0.1, reduction="none")[0],
            "policy, sequences": lambda a: e4b.policy_loss(a, labels, old, adv, reduction="sequence")[0],
            "distill, mean": lambda a: e4b.distill_loss(a, teacher, index),
            "distill, each": lambda a: e4b.distill_loss(a, teacher, index, reduction="none")}


@pytest.mark.parametrize("dtype", (torch.float32, torch.bfloat16))
def test_upstream_gradients_with_a_pending_sign(dtype):
    """Upstream gradients whose memory holds their negative: given by the caller, and as torch's complex products pass them."""
    z, labels, mask, index, teacher, old = _inputs(dtype, 4, 6, 300)
    for name, f in _every_loss(labels, old, teacher, index).items():
        leaf = z.detach().requires_grad_()
        loss = f(leaf)
        up = torch.randn(loss.shape, generator=_gen(97)).to(DEV)
        (want,) = torch.autograd.grad(loss, leaf, up, retain_graph=True)
        negative = torch.complex(up, -up).conj().imag
        assert negative.is_neg() and torch.equal(negative, up) and want.any()
        assert torch.equal(torch.autograd.grad(loss, leaf, negative)[0], want), name
        seen = []
        loss = f(leaf)
        loss.register_hook(lambda g: seen.append(g))
        w = torch.complex(up, up * 0.5 + 1)
        total = (torch.complex(torch.ones_like(loss), loss).conj() * w).sum().real
        (got,) = torch.autograd.grad(total, leaf)
        assert seen[0].is_neg(), name
        (want,) = torch.autograd.grad(f(leaf), leaf, seen[0].resolve_neg().clone())
        assert torch.equal(got, want), name


@pytest.mark.parametrize("loss_type", ("sigmoid", "ipo"))
def test_references_in_64_bits(loss_type, monkeypatch):
    """References whose values lie between fp32's: the rewards move by just what was added to an fp32 reference, up to their own
    rounding; per token and per sequence, without the torch formulation."""
    monkeypatch.setattr(L, "_preference_loss_torch", None)
    z = _logits((4, 1500, 500), torch.float32, 98).to(DEV)
    labels = torch.randint(0, 500, (4, 1500), generator=_gen(99)).to(DEV)
    lp = torch.log_softmax(z.cpu().double(), -1).gather(-1, labels.cpu().unsqueeze(-1))[..., 0]
    for ref, move in ((lp.float(), lp.abs() * 2.0 ** -26),  # a quarter of their spacing at most
                      (lp.sum(-1).float(), torch.tensor([2e-4, -1e-4, 3e-4, 1e-4], dtype=torch.float64))):
        fine = ref.double() + move
        assert torch.equal(fine.float(), ref)  # rounded to fp32, nothing of it is left
        kw = dict(beta=1.0, loss_type=loss_type)
        base = e4b.preference_loss(z, labels, ref.to(DEV), **kw)[1].cpu().double()
        leaf = z.detach().requires_grad_()
        loss, got = e4b.preference_loss(leaf, labels, fine.to(DEV), **kw)
        want = base - (move.sum(-1) if move.dim() == 2 else move)
        # the rewards' two roundings, and the 64-bit sums of 1,500 terms below 32
        assert ((got.cpu().double() - want).abs() <= U * (base.abs() + want.abs()) + 1500 * 1500 * 32 * 2.0 ** -53).all()
        d = want[:2] - want[2:]
        value = (d - 0.5) ** 2 if loss_type == "ipo" else -torch.nn.functional.logsigmoid(d)
        slope = 2 * (d - 0.5) if loss_type == "ipo" else -torch.sigmoid(-d)
        slack = U * (base.abs() + want.abs()).sum() + 1e-9
        assert ((loss.detach().cpu().double() - value).abs() <= 2 * U * value + 2 * slope.abs() * slack).all()
        # the gradients along the label's row are the slope's: their ratio to the slope is that of the fp32 reference's
        (grad,) = torch.autograd.grad(loss.sum(), leaf)
        q = torch.softmax(z.cpu().double(), -1)
        pull = torch.cat([slope, -slope])[:, None] * (1 - q.gather(-1, labels.cpu().unsqueeze(-1))[..., 0])
        r = Row64(z, 1.0)
        bound = r.q_bound().gather(-1, labels.cpu().unsqueeze(-1))[..., 0] * torch.cat([slope, slope]).abs()[:, None]
        _near(grad.gather(-1, labels.unsqueeze(-1))[..., 0], pull, bound + 8 * U * pull.abs() + 2 * slack, "gradient")


def test_references_in_64_bits_behind_the_mask():
    z, labels, mask, index, teacher, old = _inputs(torch.float32)
    counted = mask & (labels >= 0)
    bad = old.double().masked_fill(~counted, float("nan"))
    for average in (False, True):
        for a, b in zip(e4b.preference_loss(z, labels, old, mask=mask, average=average),
                        e4b.preference_loss(z, labels, bad, mask=mask, average=average)):
            assert torch.equal(a, b)
        sums = old.sum(-1)
        for a, b in zip(e4b.preference_loss(z, labels, sums, mask=mask, average=average),
                        e4b.preference_loss(z, labels, sums.double(), mask=mask, average=average)):
            assert torch.equal(a, b)


def test_batched_upstream_gradients():
    """Several upstream gradients at once (a vectorised Jacobian): each one's gradient as by itself."""
    z, labels, mask, index, teacher, old = _inputs(torch.float32, 4, 3, 120)
    for name, f in _every_loss(labels, old, teacher, index).items():
        leaf = z.detach().requires_grad_()
        loss = f(leaf)
        ups = torch.randn(5, *loss.shape, generator=_gen(100)).to(DEV)
        want = torch.stack([torch.autograd.grad(loss, leaf, u, retain_graph=True)[0] for u in ups])
        (got,) = torch.autograd.grad(loss, leaf, ups, is_grads_batched=True, retain_graph=True)
        assert torch.equal(got, want), name
        strided = ups.movedim(0, -1).contiguous().movedim(-1, 0)
        (got,) = torch.autograd.grad(loss, leaf, strided, is_grads_batched=True, retain_graph=True)
        assert torch.equal(got, want), name
        jacobian = torch.autograd.functional.jacobian(f, z.detach(), vectorize=True)
        ones = torch.autograd.functional.jacobian(f, z.detach())
        assert torch.equal(jacobian, ones) and ones.any(), name
    lp = e4b.token_logprobs(leaf, labels)
    one = torch.ones_like(lp)
    twice = torch.func.vmap(lambda a: torch.func.vmap(lambda b: torch.autograd.grad(lp, leaf, one * a * b, retain_graph=True)[0])(
        torch.arange(1.0, 4.0, device=DEV)))(torch.arange(1.0, 3.0, device=DEV))
    (base,) = torch.autograd.grad(lp, leaf, one * 2, retain_graph=True)
    assert torch.equal(twice[1, 0], base) and twice.shape == (2, 3, *leaf.shape)


def test_logits_that_a_transform_leaves_alone():
    """Inside vmap and grad, logits that the transform does not follow: the torch formulation, and no error."""
    z, labels, mask, index, teacher, old = _inputs(torch.float32, 4, 6, 300)
    for name, f in _every_loss(labels, old, teacher, index).items():
        leaf = z.detach().requires_grad_()
        for logits in (z, leaf):
            total = f(logits).detach().sum()
            got = torch.func.vmap(lambda a: a * f(logits).sum())(torch.arange(1.0, 4.0, device=DEV)).detach()
            assert torch.allclose(got, total * torch.arange(1.0, 4.0, device=DEV), rtol=1e-4), name
            assert torch.allclose(torch.func.grad(lambda a: a * f(logits).detach().sum())(torch.ones((), device=DEV)), total,
                                  rtol=1e-4), name


def test_tokens_and_teachers_made_in_inference_mode():
    """Sampled tokens, masks and a teacher's entries out of torch.inference_mode, logits that are trained."""
    z, labels, mask, index, teacher, old = _inputs(torch.float32)
    with torch.inference_mode():
        made = [t.clone() for t in (labels, mask, index, teacher, old)]
    assert all(t.is_inference() for t in made)
    want, got = _step(z, labels, mask, index, teacher, old), _step(z, *made)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    with torch.inference_mode():
        got = [e4b.token_logprobs(z, *made[:2]), e4b.preference_loss(z, made[0], made[4], mask=made[1])[0],
               e4b.policy_loss(z, made[0], made[4], made[4].sum(-1) + 9, made[4], kl_coef=0.1, mask=made[1])[0],
               e4b.policy_loss(z, made[0], made[4], made[4], mask=made[1], reduction="sequence")[0],
               e4b.distill_loss(z, made[3], made[2], mask=made[1], temperature=2.0)]
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    with torch.inference_mode():
        made_z = z.clone()
    got = [e4b.token_logprobs(made_z, *made[:2]), e4b.preference_loss(made_z, labels, old, mask=mask)[0]]
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_teacher_without_a_number_leaves_no_gradient_unmarked():
    """A teacher's NaN or +inf makes the token's loss NaN and its whole row's gradient, as the torch formulation has it."""
    z = _logits((1, 4, 3000), torch.float32, 101)
    teacher, index = _teacher(z, 5, 102)
    teacher[0, 0, 3], teacher[0, 1, 0], teacher[0, 2, 1] = float("nan"), INF, -INF
    outs = []
    for dev in (DEV, "cpu"):
        leaf = z.to(dev).requires_grad_()
        loss = e4b.distill_loss(leaf, teacher.to(dev), index.to(dev), reduction="none")
        (grad,) = torch.autograd.grad(loss, leaf, torch.ones_like(loss))
        outs.append((loss.detach().cpu().isnan(), grad.cpu().isnan()))
    for a, b in zip(*outs):
        assert torch.equal(a, b)
    assert outs[0][0].tolist() == [[True, True, False, False]] and outs[0][1][0, :2].all() and not outs[0][1][0, 2:].any()


@pytest.mark.parametrize("dtype,V", ((torch.bfloat16, 152064), (torch.float32, 100003)))
def test_parts_of_a_long_row_are_joined_in_64_bits(dtype, V):
    """A row of zeros with one logit v in each part of 8,192, e^v = 0.94 of 2^-12: a thread's 32 values keep it (their partial
    sums, below 32, round 13 times by 2^-20 or less: 1.3e-5), while beside a part's 8,191 ones it is less than half of fp32's
    last bit and would be lost, 2.3e-4 a part and 2.7e-8 of the row's sum. The ones themselves are exact."""
    per, v = 8192, -8.375
    z = torch.zeros(2, 1, V, dtype=dtype)
    parts = V // per  # whole ones
    for i in range(2):
        for p in range(parts):
            z[i, 0, p * per + (377 * p + 1023 * i + 100) % per] = v
    labels = torch.tensor([[5], [V - 1]])
    assert not z.gather(-1, labels.unsqueeze(-1)).any()
    few = z.double().exp().sum(-1) - 1
    assert ((z != 0).sum(-1) == parts).all()
    lp = -torch.log1p(few)
    ref = lp.float()
    rewards = e4b.preference_loss(z.to(DEV), labels.to(DEV), ref.to(DEV), beta=1.0)[1].cpu().double()
    want = (lp - ref.double())[:, 0]
    bound = parts * 13 * 2.0 ** -20 / few[:, 0] + 4 * U * want.abs() + parts * 2.3e-4 * 16 * U / few[:, 0]
    assert bound.max() < 2e-9
    assert ((rewards - want).abs() <= bound).all(), (rewards - want, bound)


def test_constants_with_a_tangent():
    """Inside forward-mode differentiation that follows everything but the logits: the values, without a tangent."""
    import torch.autograd.forward_ad as fa

    z, labels, mask, index, teacher, old = _inputs(torch.float32)
    want = [e4b.policy_loss(z, labels, old, old.sum(-1), old, kl_coef=0.1)[0], e4b.preference_loss(z, labels, old)[0],
            e4b.distill_loss(z, teacher, index)]
    with fa.dual_level():
        o, s, t = (fa.make_dual(v, torch.ones_like(v)) for v in (old, old.sum(-1), teacher))
        got = [e4b.policy_loss(z, labels, o, s, o, kl_coef=0.1)[0], e4b.preference_loss(z, labels, o)[0],
               e4b.distill_loss(z, t, index)]
        assert all(fa.unpack_dual(g).tangent is None for g in got)
    assert all(torch.equal(g, w) for g, w in zip(got, want))


def test_recorded_calls_take_the_torch_formulation():
    """A function that make_fx recorded, on other logits, forward and with its gradient."""
    from torch.fx.experimental.proxy_tensor import make_fx

    z, labels, mask, index, teacher, old = _inputs(torch.float32, 4, 6, 300)
    other = z.flip(0) * 0.5
    for name, f in _every_loss(labels, old, teacher, index).items():
        for g in (f, lambda a: torch.autograd.grad(f(a.requires_grad_()).sum(), a)[0]):
            assert torch.allclose(make_fx(g)(z.clone())(other.clone()), g(other.clone()), rtol=1e-4, atol=1e-6), name


def test_a_backward_recorded_by_itself_is_refused():
    """Of a loss that was computed before the recording: what the kernel writes would not be in it."""
    from torch.fx.experimental.proxy_tensor import make_fx

    z, labels, mask, index, teacher, old = _inputs(torch.float32, 4, 6, 300)
    for name, f in _every_loss(labels, old, teacher, index).items():
        leaf = z.detach().requires_grad_()
        loss = f(leaf)
        with pytest.raises(RuntimeError, match="recorded"):
            make_fx(lambda up: torch.autograd.grad(loss, leaf, up, retain_graph=True)[0])(torch.ones_like(loss))
        assert torch.autograd.grad(loss, leaf, torch.ones_like(loss))[0].any(), name


def test_upstream_gradients_with_a_tangent():
    """Forward-mode differentiation that follows the upstream gradient alone: the gradient is linear in it."""
    import torch.autograd.forward_ad as fa

    z, labels, mask, index, teacher, old = _inputs(torch.float32, 4, 6, 300)
    for name, f in _every_loss(labels, old, teacher, index).items():
        leaf = z.detach().requires_grad_()
        loss = f(leaf)
        up, along = (torch.randn(loss.shape, generator=_gen(103 + i)).to(DEV) for i in range(2))
        want = [torch.autograd.grad(loss, leaf, u, retain_graph=True)[0] for u in (up, along)]
        with fa.dual_level():
            got = fa.unpack_dual(torch.autograd.grad(loss, leaf, fa.make_dual(up, along), retain_graph=True)[0])
            assert torch.equal(got.primal, want[0]) and torch.equal(got.tangent, want[1]) and want[1].any(), name
            (plain,) = torch.autograd.grad(loss, leaf, up, retain_graph=True)
            assert fa.unpack_dual(plain).tangent is None and torch.equal(plain, want[0])
        (none,) = torch.autograd.grad(loss, leaf, torch._efficientzerotensor(loss.shape, device=DEV))
        assert none.shape == leaf.shape and not none.any(), name
