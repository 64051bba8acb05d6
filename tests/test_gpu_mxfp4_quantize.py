"""``quantize_mxfp4`` on the device against the torch formulation in ``quant.py``, bit for bit: codes and
scales are the stored bytes, so nothing may differ."""
import pytest
import torch

import experts4bit_qlora_amd as e4b
from experts4bit_qlora_amd import quant as Q

pytestmark = pytest.mark.gpu
DEV = "cuda"
DTYPES = (torch.float32, torch.bfloat16, torch.float16)


def _same(w):
    got, want = e4b.quantize_mxfp4(w), Q._quantize_mxfp4_torch(w)
    assert all(a.shape == b.shape and a.dtype == b.dtype for a, b in zip(got, want))
    assert torch.equal(got[1], want[1])
    assert torch.equal(got[0], want[0])
    if w.dtype != torch.float32:  # (the CPU's and the device's fp32 log2 round differently near powers of two)
        host = Q._quantize_mxfp4_torch(w.cpu())
        assert all(torch.equal(a.cpu(), b) for a, b in zip(got, host))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", ((32,), (1, 64), (3, 32), (5, 2880), (255, 32), (256, 32), (257, 32), (7, 3, 1216)))
def test_random_rows(shape, dtype):
    g = torch.Generator().manual_seed(sum(shape))
    w = torch.randn(shape, generator=g) * torch.exp(3 * torch.randn(*shape[:-1], 1, generator=g))
    _same(w.to(dtype).to(DEV))


@pytest.mark.parametrize("dtype", DTYPES)
def test_every_code_midpoint_and_sign_at_many_scales(dtype):
    """The grid, the midpoints between its values and their neighbours, at every scale of the type."""
    grid = torch.tensor([0.0, 0.25, 0.5, 0.75, 1.0, 1.25, 1.5, 1.75, 2.0, 2.5, 3.0, 3.5, 4.0, 5.0, 6.0, 7.0])
    values = torch.cat([grid, -grid]).double()
    powers = torch.pow(2.0, torch.arange(-149, 127, dtype=torch.float64))
    rows = (values[None, :] * powers[:, None])
    for shift in (0.0, 2.0 ** -7, -(2.0 ** -7)):
        _same((rows * (1 + shift)).to(dtype).to(DEV))


@pytest.mark.parametrize("dtype", (torch.bfloat16, torch.float16))
def test_every_value_of_a_16_bit_type_as_the_largest(dtype):
    """All 65,536 patterns in one block each (infinities and NaN among them), smaller values beside them."""
    bits = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(dtype)
    block = torch.zeros(65536, 32, dtype=dtype)
    block[:, 5] = bits
    block[:, 6] = (bits.float() * -0.4).to(dtype)
    _same(block.to(DEV))


def test_fp32_maxima_near_powers_of_two():
    """The largest 512 and smallest 512 mantissas of every binade: fp32's log2 rounds some up."""
    exponent = torch.arange(0, 255, dtype=torch.int32)[:, None]
    mantissa = torch.cat([torch.arange(512, dtype=torch.int32), 0x7FFFFF - torch.arange(512, dtype=torch.int32)])
    top = ((exponent << 23) | mantissa[None, :]).reshape(-1).view(torch.float32)
    block = torch.zeros(top.numel(), 32)
    block[:, 31] = -top
    block[:, 0] = top * 0.55
    _same(block.to(DEV))


@pytest.mark.parametrize("dtype", DTYPES)
def test_blocks_of_zeros_infinities_and_nan(dtype):
    rows = [torch.zeros(32), -torch.zeros(32)]
    for special in (float("nan"), -float("nan"), float("inf"), -float("inf")):
        row = torch.linspace(-9, 9, 32)
        row[11] = special
        rows += [row, torch.where(torch.arange(32) == 3, torch.full((32,), special), torch.zeros(32))]
    _same(torch.stack(rows).to(dtype).to(DEV))


def test_views_other_dtypes_and_the_torch_route():
    w = torch.randn(64 * 64 + 2, device=DEV)
    for v in (w[2:].view(64, 64), w[:4096].view(64, 64).t(), w[:4096].view(64, 64).double(), w[1:4097]):
        got, want = e4b.quantize_mxfp4(v), Q._quantize_mxfp4_torch(v.float())
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert e4b.quantize_mxfp4(w[:0].view(0, 64))[0].shape == (0, 32)
    with pytest.raises(ValueError, match="multiple of 32"):
        e4b.quantize_mxfp4(w[:48])


def test_another_stream():
    """The kernel runs on the current stream: a product of that stream's own work."""
    s = torch.cuda.Stream()
    w = torch.randn(4096, 256, device=DEV)
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        doubled = w * 2
        got = e4b.quantize_mxfp4(doubled)
    s.synchronize()
    want = Q._quantize_mxfp4_torch(w * 2)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_fp32_blocks_equal_the_cpu_formulation():
    """Scale bytes are the floor of the exact logarithm on either side: maxima next to every power of two, random rows."""
    exponent = torch.arange(0, 255, dtype=torch.int32)[:, None]
    mantissa = torch.cat([torch.arange(512, dtype=torch.int32), 0x7FFFFF - torch.arange(512, dtype=torch.int32)])
    bits = ((exponent << 23) | mantissa[None, :]).reshape(-1)
    block = torch.zeros(bits.numel(), 32)
    block[:, 31] = -bits.view(torch.float32)
    block[:, 0] = bits.view(torch.float32) * 0.55
    g = torch.Generator().manual_seed(1)
    rows = torch.randn(4096, 32, generator=g) * torch.exp(20 * torch.randn(4096, 1, generator=g))
    for w in (block, rows):
        got, want = e4b.quantize_mxfp4(w.to(DEV)), Q._quantize_mxfp4_torch(w)
        assert all(torch.equal(a.cpu(), b) for a, b in zip(got, want))
    assert torch.equal(e4b.quantize_mxfp4(block.to(DEV))[1].cpu()[:, 0].int(), ((bits >> 23) - 2).clamp(min=0))
