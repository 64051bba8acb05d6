"""The microscaled operators and the router on tensors whose offsets pass 32 bits: the last rows of a large call
equal the same rows in a call of their own."""
import pytest
import torch

import experts4bit_qlora_amd as e4b

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _bytes(*shape, lo=0, hi=256):
    return torch.randint(lo, hi, shape, dtype=torch.uint8, device=DEV)


@pytest.mark.parametrize("rows,n,k", [(300_001, 8200, 64), (280_001, 8200, 288)])
def test_product_outputs(rows, n, k):
    """More than 2^31 outputs, by 32-row tiles (K of one chunk) and by 256-row tiles."""
    assert rows * n > 2 ** 31
    b, s = _bytes(2, n, k // 2), _bytes(2, n, k // 32, lo=120, hi=130)
    a = torch.randn(rows, k, device=DEV, dtype=torch.bfloat16)
    ids = torch.tensor([1, 0], device=DEV)
    out = e4b.gemm_mxfp4_grouped(a, b, s, [100, rows - 100], ids, act_quant="mxfp4")
    part = e4b.gemm_mxfp4_grouped(a[-300:].contiguous(), b, s, [300], ids[1:], act_quant="mxfp4")
    assert torch.equal(out[-300:], part)


@pytest.mark.parametrize("size", (2, 9, 40, 200))
def test_product_weights(size):
    """A stack of more than 2^32 bytes: the last expert."""
    E, n, k = 33, 16384, 16384
    assert E * n * k // 2 > 2 ** 32
    b, s = _bytes(E, n, k // 2), _bytes(E, n, k // 32, lo=120, hi=130)
    a = torch.randn(size, k, device=DEV, dtype=torch.bfloat16)
    out = e4b.gemm_mxfp4_grouped(a, b, s, [size], torch.tensor([E - 1], device=DEV), act_quant="mxfp4")
    alone = e4b.gemm_mxfp4_grouped(a, b[-1:].clone(), s[-1:].clone(), [size], torch.tensor([0], device=DEV),
                                   act_quant="mxfp4")
    assert torch.equal(out, alone)


def test_quantize():
    x = torch.randn(70_000, 65_536, device=DEV, dtype=torch.bfloat16)
    assert x.numel() > 2 ** 32
    blocks, scales = e4b.quantize_mxfp4(x)
    last = e4b.quantize_mxfp4(x[-3:].clone())
    assert torch.equal(blocks[-3:], last[0]) and torch.equal(scales[-3:], last[1])


def test_router():
    T, E, k = 2_200_003, 1000, 2
    assert T * E > 2 ** 31
    z = torch.randn(T, E, device=DEV, dtype=torch.bfloat16).requires_grad_()
    index, weights = e4b.router_topk(z, k)
    (grad,) = torch.autograd.grad(weights, z, torch.ones_like(weights))
    tail = z.detach()[-5:].clone().requires_grad_()
    i, w = e4b.router_topk(tail, k)
    assert torch.equal(index[-5:], i) and torch.equal(weights[-5:], w)
    assert torch.equal(grad[-5:], torch.autograd.grad(w, tail, torch.ones_like(w))[0])
    del grad
    # only the last rows are valid: what the loss reads and writes lies past 2^31
    mask = torch.zeros(T, dtype=torch.bool, device=DEV)
    mask[-5:] = True
    loss, counts = e4b.balance_loss(z[None], index[None], mask)
    (grad,) = torch.autograd.grad(loss.sum(), z)
    own, each = e4b.balance_loss(tail[None], i[None])
    (want,) = torch.autograd.grad(own.sum(), tail)
    assert torch.equal(counts, each)
    # five probabilities per expert, summed in another order: 2^-20 is sixteen fp32 roundings
    assert torch.allclose(loss, own, rtol=2.0 ** -20, atol=0)
    assert torch.equal(grad[-5:], want) and not grad[:-5].any()


def test_gate_of_more_work_items_than_a_launch_holds():
    """2^26 rows of more than 256 experts (64 lanes each) in several launches: every row against one call of the rows
    that repeat, new rows where one launch may end and at the end."""
    E, k, rows = 257, 2, 1 << 16
    T = (1 << 26) + 5
    base = torch.randn(rows, E, device=DEV, dtype=torch.bfloat16)
    z = base.repeat(1025, 1)[:T]
    new = [slice(t - 2, t + 3) for t in (1 << 24, 1 << 25, (1 << 25) + (1 << 24))] + [slice(T - 5, T)]
    for s in new:
        z[s] = torch.randn(5, E, device=DEV, dtype=torch.bfloat16)
    z.requires_grad_()
    index, weights = e4b.router_topk(z, k)
    (grad,) = torch.autograd.grad(weights, z, torch.ones_like(weights))

    def own(t):
        t = t.detach().clone().requires_grad_()
        i, w = e4b.router_topk(t, k)
        return i, w.detach(), torch.autograd.grad(w, t, torch.ones_like(w))[0]

    for s in new:
        assert all(torch.equal(a, b) for a, b in zip((index[s], weights.detach()[s], grad[s]), own(z[s])))
    want = own(base)
    for lo in range(0, T - 5, rows):
        part = slice(lo, lo + rows)
        for got, each in zip((index[part], weights.detach()[part], grad[part]), want):
            other = (got != each).any(-1)
            for s in new:  # (rows of their own, compared above)
                other[max(s.start - lo, 0):max(s.stop - lo, 0)] = False
            assert not other.any()


def test_product_of_more_chunks_than_a_launch_quantizes():
    """2^27 chunks of 256 values and more (64 GiB of rows): every row against one call of the rows that repeat, new ones
    where one launch may end and at the end."""
    n, k, rows = 40, 32768, 1 << 12
    M = (1 << 20) + 77
    b, s = _bytes(1, n, k // 2), _bytes(1, n, k // 32, lo=120, hi=130)
    ids = torch.tensor([0], device=DEV)
    base = torch.randn(rows, k, device=DEV, dtype=torch.bfloat16)
    x = base.repeat(257, 1)[:M]
    new = [slice(r - 3, r + 4) for r in (1 << 18, 1 << 19, (1 << 19) + (1 << 18))] + [slice(M - 7, M)]
    for part in new:
        x[part] = torch.randn(7, k, device=DEV, dtype=torch.bfloat16)
    out = e4b.gemm_mxfp4_grouped(x, b, s, [M], ids, act_quant="mxfp4")

    def own(part):  # beside zero rows without an expert, enough for 256-row tiles, whose order of sums is the large call's
        more = torch.zeros(50_000, k, device=DEV, dtype=torch.bfloat16)
        return e4b.gemm_mxfp4_grouped(torch.cat([part, more]), b, s, [len(part), len(more)],
                                      torch.tensor([0, -1], device=DEV), act_quant="mxfp4")[:len(part)]

    want = own(base)
    for part in new:
        assert torch.equal(out[part], own(x[part.start - 300:part.stop])[300:])
    for lo in range(0, M, rows):
        got = out[lo:lo + rows]
        other = (got != want[:got.shape[0]]).any(-1)
        for part in new:
            other[max(part.start - lo, 0):max(part.stop - lo, 0)] = False
        assert not other.any()


@pytest.mark.parametrize("size", (1, 17))
def test_product_of_more_workgroups_than_a_launch_holds(size):
    """512 groups times 2^16 column blocks and more, rows quantized inside the tiles and before them: groups of one
    expert have the same rows and so the same outputs."""
    n, k = (1 << 21) + 40, 32
    b, s = _bytes(2, n, k // 2), _bytes(2, n, k // 32, lo=120, hi=130)
    rows = torch.randn(2, size, k, device=DEV, dtype=torch.bfloat16)
    ids = torch.arange(512, device=DEV) % 2
    ids[300] = 2
    sizes = [size] * 512
    sizes[255], sizes[256] = 0, 0  # beside a launch's last group
    x = torch.cat([rows[g % 2][:r] for g, r in enumerate(sizes)])
    out = e4b.gemm_mxfp4_grouped(x, b, s, sizes, ids, act_quant="mxfp4")
    want = e4b.gemm_mxfp4_grouped(rows.flatten(0, 1), b, s, [size] * 2, ids[:2], act_quant="mxfp4").view(2, size, n)
    assert out.shape[0] == 510 * size and want.any()
    at = 0
    for g, r in enumerate(sizes):
        got = out[at:at + r]
        at += r
        assert torch.equal(got, want[g % 2][:r]) if g != 300 else not got.any()


@pytest.mark.parametrize("k", (64, 288))
def test_product_outputs_of_small_groups(k):
    """More than 2^31 outputs with the last ones written by 32-row tiles: more than 32 small groups behind a large one
    take a launch of their own (in test_product_outputs the 256-row tiles take all rows)."""
    n, sizes = 8200, [280_000] + [30] * 33
    M = sum(sizes)
    assert 280_000 * n > 2 ** 31
    b, s = _bytes(2, n, k // 2), _bytes(2, n, k // 32, lo=120, hi=130)
    a = torch.randn(M, k, device=DEV, dtype=torch.bfloat16)
    ids = torch.arange(34, device=DEV) % 2
    out = e4b.gemm_mxfp4_grouped(a, b, s, sizes, ids, act_quant="mxfp4")
    part = e4b.gemm_mxfp4_grouped(a[280_000:].clone(), b, s, sizes[1:], ids[1:], act_quant="mxfp4")
    assert torch.equal(out[280_000:], part)
