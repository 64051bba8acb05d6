"""``gemm_mxfp4_grouped(..., act_quant="mxfp4")`` against the product of the same microscaled values in 64 bits.

Tolerance of one output, from the arithmetic: the rounding into the output type, half a step of the
value (``eps / 2``), and the fp32 sums: K products (exact) added in any order, one error of at most 2^-23 of the
running sum's bound per addition (a truncating adder), so K 2^-23 times the sum of the magnitudes."""
import ctypes

import pytest
import torch

import experts4bit_qlora_amd as e4b
from experts4bit_qlora_amd import _native as N
from experts4bit_qlora_amd import ops
from experts4bit_qlora_amd import quant as Q

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _weights(E, n, k, seed):
    g = torch.Generator().manual_seed(seed)
    return Q._quantize_mxfp4_torch(torch.randn(E, n, k, generator=g) * torch.exp(torch.randn(E, n, 1, generator=g)))


def _values(blocks, scales):
    """Microscaled bytes as fp64 values [..., k] (low nibble first; scale byte 255: NaN)."""
    table = torch.tensor(Q.FP4_VALUES, dtype=torch.float64)
    v = table[torch.stack([blocks & 15, blocks >> 4], -1).long()].reshape(*scales.shape, 32)
    power = torch.where(scales == 255, float("nan"), torch.pow(2.0, scales.double() - 127))
    return (v * power.unsqueeze(-1)).reshape(*scales.shape[:-1], -1)


def _check(a, blocks, scales, sizes, ids, out):
    """out [M, n] against the 64-bit product; rows of ids outside [0, E) are zero."""
    E, n, kh = blocks.shape
    ab, asc = Q._quantize_mxfp4_torch(a)
    bad = ~torch.isfinite(a.double()).reshape(a.shape[0], -1, 32).all(-1)
    av, wv = _values(ab, torch.where(bad, 255, asc).to(torch.uint8)), _values(blocks, scales)
    out = out.double().cpu()
    assert out.shape == (a.shape[0], n)
    r = 0
    for s, e in zip(sizes, ids):
        x, got = av[r:r + s], out[r:r + s]
        r += s
        if not 0 <= e < E:
            assert torch.equal(got, torch.zeros_like(got))
            continue
        want = x @ wv[e].T
        bound = torch.finfo(a.dtype).eps / 2 * want.abs() + 2 * kh * 2.0 ** -23 * (x.abs() @ wv[e].abs().T)
        # below the normal range: half a subnormal step of the type, a flushed fp32 subnormal
        bound += torch.finfo(a.dtype).smallest_normal * torch.finfo(a.dtype).eps / 2 + 2.0 ** -126
        assert torch.equal(got.isnan(), want.isnan())
        fine = ~want.isnan()
        err = (got - want).abs()[fine]
        assert (err <= bound[fine]).all(), (err / bound[fine]).max().item()


def _rows(M, k, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(M, k, generator=g) * torch.exp(torch.randn(M, 1, generator=g))).to(dtype)


def _check_both(a, blocks, scales, sizes, ids):
    """The call, and, where a group has more than 32 rows, the same beside a group of zero rows without an expert that
    is large enough (2,700 tiles of 32 x 32) for the 256-row tiles to take them all."""
    _check(a, blocks, scales, sizes, ids, _run(a, blocks, scales, sizes, ids))
    if max(sizes) > 32:
        more = 32 * -(-2700 // -(-blocks.shape[1] // 32))
        out = _run(torch.cat([a, a.new_zeros(more, a.shape[1])]), blocks, scales, [*sizes, more], [*ids, -1])
        assert not out[len(a):].any()
        _check(a, blocks, scales, sizes, ids, out[:len(a)])


def _run(a, blocks, scales, sizes, ids, **kw):
    return e4b.gemm_mxfp4_grouped(a.to(DEV), blocks.to(DEV), scales.to(DEV), sizes, torch.tensor(ids, device=DEV),
                                  act_quant="mxfp4", **kw)


@pytest.mark.parametrize("dtype", (torch.bfloat16, torch.float16))
@pytest.mark.parametrize("k", (32, 64, 96, 224, 256, 288, 704, 1216, 2880))
def test_depths(k, dtype):
    """K below, at and past whole chunks, and with every number of blocks left over."""
    E, n, sizes, ids = 3, 80, [1, 5, 33], [2, 0, 1]
    b, s = _weights(E, n, k, k)
    a = _rows(sum(sizes), k, dtype, k + 1)
    _check_both(a, b, s, sizes, ids)


@pytest.mark.parametrize("n", (1, 3, 31, 32, 33, 127, 130, 256, 257, 516))
def test_widths(n):
    E, k, sizes, ids = 2, 320, [2, 40], [1, 0]
    b, s = _weights(E, n, k, n)
    a = _rows(sum(sizes), k, torch.bfloat16, n)
    _check_both(a, b, s, sizes, ids)


@pytest.mark.parametrize("sizes", ([1], [31], [32], [33], [64], [1, 1, 1, 1], [0, 3, 0], [127, 1, 129], [255], [256],
                                   [257, 300], [513, 30, 290], [3] * 40 + [300], [1] * 40, [7] * 100, [900]))
def test_group_sizes(sizes):
    E, n, k = 5, 272, 544
    ids = [(3 * g + 1) % E for g in range(len(sizes))]
    b, s = _weights(E, n, k, 4)
    a = _rows(sum(sizes), k, torch.bfloat16, len(sizes))
    _check_both(a, b, s, sizes, ids)


def test_512_groups_and_one_more():
    E, n, k = 3, 64, 64
    sizes, ids = [g % 4 for g in range(512)], [g % E for g in range(512)]
    b, s = _weights(E, n, k, 6)
    a = _rows(sum(sizes), k, torch.bfloat16, 6)
    _check_both(a, b, s, sizes, ids)
    with pytest.raises(RuntimeError, match="groups=513"):
        _run(a, b, s, sizes + [0], ids + [0])


@pytest.mark.parametrize("sizes", ([2, 3, 1, 4], [300, 40, 1, 260]))
def test_ids_in_any_order_repeated_and_out_of_range(sizes):
    """Ids are read on the device; groups without an expert give zero rows, the next group is unharmed."""
    E, n, k, ids = 4, 96, 256, [3, -1, 3, 4]
    b, s = _weights(E, n, k, 7)
    a = _rows(sum(sizes), k, torch.bfloat16, 7)
    _check_both(a, b, s, sizes, ids)
    ids = [2, 1 << 40, 0, -(1 << 40)]
    _check_both(a, b, s, sizes, ids)


def test_host_ids_and_no_rows():
    E, n, k = 3, 48, 96
    b, s = _weights(E, n, k, 8)
    a = _rows(6, k, torch.float16, 8)
    w = (b.to(DEV), s.to(DEV))
    out = e4b.gemm_mxfp4_grouped(a.to(DEV), *w, [4, 2], [2, 0], act_quant="mxfp4")
    _check(a, b, s, [4, 2], [2, 0], out)
    assert e4b.gemm_mxfp4_grouped(a[:0].to(DEV), *w, [], [], act_quant="mxfp4").shape == (0, n)
    assert e4b.gemm_mxfp4_grouped(a[:0].to(DEV), *w, [0, 0], [1, 2], act_quant="mxfp4").shape == (0, n)


@pytest.mark.parametrize("rows", (3, 300))
def test_infinities_and_nan_reach_their_rows_only(rows):
    E, n, k = 2, 160, 512
    b, s = _weights(E, n, k, 9)
    a = _rows(rows, k, torch.bfloat16, 9)
    a[0, 17], a[1, 300], a[rows - 1, k - 1] = float("nan"), float("inf"), -float("inf")
    _check_both(a, b, s, [rows], [1])


@pytest.mark.parametrize("rows", (3, 300))
def test_weight_scales_at_the_ends(rows):
    """Scale bytes 0 and 1 (products far below the rest), large ones, and 255 (the column is NaN)."""
    E, n, k = 1, 64, 256
    b, s = _weights(E, n, k, 10)
    s[0, 3], s[0, 4, 2], s[0, 5], s[0, 6, 5] = 0, 1, 200, 255
    a = _rows(rows, k, torch.bfloat16, 10)
    _check_both(a, b, s, [rows], [0])


def test_zero_rows():
    E, n, k = 1, 64, 288
    b, s = _weights(E, n, k, 11)
    a = torch.zeros(5, k, dtype=torch.bfloat16)
    a[3] = _rows(1, k, torch.bfloat16, 11)[0]
    _check_both(a, b, s, [5], [0])


def test_views():
    """Strided activations, a start inside another tensor, transposed ids."""
    E, n, k = 2, 64, 256
    b, s = _weights(E, n, k, 12)
    big = _rows(8, 2 * k + 8, torch.bfloat16, 12)
    dev = big.to(DEV)
    ids = torch.tensor([[1, 0], [0, 1]], device=DEV)[:, 0]
    w = (b.to(DEV), s.to(DEV))
    for lo in (0, 3, 8):
        a = big[::2, lo:lo + k].contiguous()
        out = e4b.gemm_mxfp4_grouped(dev[::2, lo:lo + k], *w, [3, 1], ids, act_quant="mxfp4")
        _check(a, b, s, [3, 1], [1, 0], out)


@pytest.mark.parametrize("sizes", ([1, 2], [300, 20], [300, 17_000]))
def test_captured_and_replayed(sizes):
    """Replays on new inputs in place equal the eager calls bit for bit; two graphs of one pool alternate."""
    E, n, k, ids = 4, 160, 512, torch.tensor([3, 1], device=DEV)
    b, s = (t.to(DEV) for t in _weights(E, n, k, 13))
    M = sum(sizes)
    a = [_rows(M, k, torch.bfloat16, 20 + i).to(DEV) for i in range(2)]

    def call(i):
        return e4b.gemm_mxfp4_grouped(a[i], b, s, sizes, ids, act_quant="mxfp4")

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call(0)
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for i in range(2):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[i], pool=graphs[0].pool() if i else None):
            outs.append(call(i))
    for step in range(4):
        for i in range(2):
            a[i].copy_(_rows(M, k, torch.bfloat16, 30 + 2 * step + i))
            graphs[i].replay()
            got = outs[i].clone()
            assert torch.equal(got, call(i))
            torch.cuda.synchronize()


def test_another_stream_and_no_synchronization():
    E, n, k = 4, 160, 512
    b, s = _weights(E, n, k, 14)
    a = _rows(40, k, torch.bfloat16, 14)
    bd, sd, ad, ids = b.to(DEV), s.to(DEV), a.to(DEV), torch.tensor([3, 1], device=DEV)
    e4b.gemm_mxfp4_grouped(ad, bd, sd, [37, 3], ids, act_quant="mxfp4")
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    torch.cuda.set_sync_debug_mode("error")
    try:
        with torch.cuda.stream(stream):
            out = e4b.gemm_mxfp4_grouped(ad * 2, bd, sd, [37, 3], ids, act_quant="mxfp4")
    finally:
        torch.cuda.set_sync_debug_mode("default")
    stream.synchronize()
    _check(a * 2, b, s, [37, 3], [3, 1], out)


def test_repeats_are_bit_equal():
    E, n, k = 4, 400, 704
    b, s = (t.to(DEV) for t in _weights(E, n, k, 15))
    for sizes in ([2, 1], [700, 90], [700, 6000]):
        a, ids = _rows(sum(sizes), k, torch.bfloat16, 15).to(DEV), torch.tensor([0, 2], device=DEV)
        first = e4b.gemm_mxfp4_grouped(a, b, s, sizes, ids, act_quant="mxfp4")
        assert all(torch.equal(first, e4b.gemm_mxfp4_grouped(a, b, s, sizes, ids, act_quant="mxfp4")) for _ in range(10))


def test_refusals():
    E, n, k = 2, 32, 64
    b, s = (t.to(DEV) for t in _weights(E, n, k, 16))
    a, ids = _rows(3, k, torch.bfloat16, 16).to(DEV), torch.tensor([0, 1], device=DEV)
    call = e4b.gemm_mxfp4_grouped
    with pytest.raises(ValueError, match="act_quant"):
        call(a, b, s, [1, 2], ids, act_quant="fp8")
    with pytest.raises(ValueError, match="sizes sum to"):
        call(a, b, s, [1, 1], ids, act_quant="mxfp4")
    with pytest.raises(ValueError, match="differ in length"):
        call(a, b, s, [3], ids, act_quant="mxfp4")
    with pytest.raises(ValueError, match="columns"):
        call(a[:, :32], b, s, [1, 2], ids, act_quant="mxfp4")
    with pytest.raises(ValueError, match="bad expert ids"):
        call(a, b, s, [1, 2], [0, 2], act_quant="mxfp4")
    with pytest.raises(TypeError):
        call(a.double(), b, s, [1, 2], ids, act_quant="mxfp4")
    with pytest.raises(RuntimeError, match="act_dtype"):
        call(a.float(), b, s, [1, 2], ids, act_quant="mxfp4")
    with pytest.raises(RuntimeError, match="negative size"):
        call(a, b, s, [4, -1], ids, act_quant="mxfp4")
    with pytest.raises(ValueError, match="HIP device"):
        call(a.cpu(), b, s, [1, 2], ids, act_quant="mxfp4")


@pytest.mark.parametrize("dtype", (torch.bfloat16, torch.float16))
@pytest.mark.parametrize("k", (32, 96, 224, 256, 288, 1216, 2880))
@pytest.mark.parametrize("sizes", ([1], [4, 0, 1, 3]))
def test_few_rows(sizes, k, dtype):
    """Groups of at most four rows, whose tiles quantize the rows themselves, and the same rows in a call
    with a larger group: the same bytes."""
    E, n = 3, 72
    b, s = _weights(E, n, k, k)
    ids = [2, 1, 0, 2][:len(sizes)]
    a = _rows(sum(sizes) + 5, k, dtype, k + 7)
    a[0, :32] = 0
    few = a[:sum(sizes)]
    out = _run(few, b, s, sizes, ids)
    _check(few, b, s, sizes, ids, out)
    assert torch.equal(_run(a, b, s, sizes + [5], ids + [1])[:sum(sizes)], out)


def test_refuses_stacks_that_do_not_fit():
    b, s = _weights(2, 16, 64, 1)
    a = _rows(3, 64, torch.bfloat16, 2)
    with pytest.raises(ValueError, match="scales"):
        _run(a, b, s[..., :1].contiguous(), [3], [0])
    with pytest.raises(ValueError, match="bytes"):
        _run(a, b.int(), s, [3], [0])
    with pytest.raises(ValueError, match="columns"):
        _run(a[:, :32].contiguous(), b, s, [3], [0])


def _entry(a, blocks, scales, sizes, ids, out, workspace):
    """e4b_mx_grouped_gemm itself, on the caller's buffers."""
    E, n, kh = blocks.shape
    qw = ops.mxfp4_qweight(blocks, scales, n, 2 * kh)
    return N.lib().e4b_mx_grouped_gemm(a.data_ptr(), ops.dtype_code(a.dtype), (ctypes.c_int64 * len(sizes))(*sizes),
                                       len(sizes), ids.data_ptr(), qw.ref(), workspace.data_ptr(), workspace.numel(),
                                       out.data_ptr(), ops.dtype_code(out.dtype),
                                       torch.cuda.current_stream().cuda_stream)


@pytest.mark.parametrize("out_dtype", (torch.float32, torch.float16, torch.bfloat16))
@pytest.mark.parametrize("n", (72, 267))
@pytest.mark.parametrize("sizes", ([1, 3], [2, 7], [40, 260], [40, 29_000]))
def test_entry_point_output_types_and_what_it_leaves(sizes, n, out_dtype):
    """The entry point's other output types; bytes behind the last row and behind the workspace it asked for stay."""
    E, k, ids, M = 3, 352, [2, 0], sum(sizes)
    b, s = _weights(E, n, k, 40)
    a = _rows(M, k, torch.bfloat16, 41)
    need = N.lib().e4b_mx_gemm_workspace_bytes(M, k)
    ws = torch.full((need + 256,), 0xA5, dtype=torch.uint8, device=DEV)
    out = torch.full((M + 2, n), 77.0, dtype=out_dtype, device=DEV)
    assert _entry(a.to(DEV), b.to(DEV), s.to(DEV), sizes, torch.tensor(ids, device=DEV), out, ws[:need]) == 0
    torch.cuda.synchronize()
    assert (out[M:] == 77).all() and (ws[need:] == 0xA5).all()
    ab, asc = Q._quantize_mxfp4_torch(a)
    av, wv, r = _values(ab, asc), _values(b, s), 0
    for size, e in zip(sizes, ids):
        want = av[r:r + size] @ wv[e].T
        bound = torch.finfo(out_dtype).eps / 2 * want.abs() + k * 2.0 ** -23 * (av[r:r + size].abs() @ wv[e].abs().T)
        bound += torch.finfo(out_dtype).smallest_normal * torch.finfo(out_dtype).eps / 2 + 2.0 ** -126
        top = torch.finfo(out_dtype).max  # a value past fp16's range is infinite
        got = out[r:r + size].double().cpu()
        fine = want.abs() < top
        assert ((got - want).abs()[fine] <= bound[fine]).all() and got[~fine].abs().ge(top / 2).all()
        r += size


@pytest.mark.parametrize("sizes", ([1, 2], [9, 5], [300, 20], [300, 9000]))
def test_two_calls_at_once(sizes):
    """Calls on two streams, each with rows of its own, over the same weights."""
    E, n, k, ids = 4, 320, 704, torch.tensor([3, 1], device=DEV)
    b, s = (t.to(DEV) for t in _weights(E, n, k, 50))
    a = [_rows(sum(sizes), k, torch.bfloat16, 51 + i).to(DEV) for i in range(2)]
    want = [e4b.gemm_mxfp4_grouped(x, b, s, sizes, ids, act_quant="mxfp4") for x in a]
    streams = [torch.cuda.Stream() for _ in a]
    torch.cuda.synchronize()
    for _ in range(10):
        got = []
        for x, stream in zip(a, streams):
            with torch.cuda.stream(stream):
                got.append(e4b.gemm_mxfp4_grouped(x, b, s, sizes, ids, act_quant="mxfp4"))
        torch.cuda.synchronize()
        assert all(torch.equal(g, w) for g, w in zip(got, want))


@pytest.mark.parametrize("n", (1408, 2064))
@pytest.mark.parametrize("most", (4, 8, 16))
def test_many_small_groups(most, n):
    """Groups of up to four, eight and sixteen rows, enough of them (2,064 weight rows: 65 column blocks of 48
    groups) for a workgroup to take several column blocks: the bytes of a call that has a larger group beside them."""
    E, k, G = 4, 320, 48
    b, s = (t.to(DEV) for t in _weights(E, n, k, 60))
    sizes = [most, 0] + [1 + i % most for i in range(G - 2)]
    ids = [i % E for i in range(G)]
    ids[5] = E  # zero rows
    a = _rows(sum(sizes) + 17, k, torch.bfloat16, 61)
    few = a[:sum(sizes)]
    out = _run(few, b, s, sizes, ids)
    _check(few, b.cpu(), s.cpu(), sizes, ids, out)
    assert torch.equal(_run(a, b, s, sizes + [17], ids + [1])[:sum(sizes)], out)


@pytest.mark.parametrize("E", (1, 3))
@pytest.mark.parametrize("n", (1, 2, 7, 40, 300))
@pytest.mark.parametrize("k", (32, 64, 96, 224, 256))
def test_short_rows_in_large_groups(k, n, E):
    """Rows of fewer than eight scale bytes, from the stack's first byte to its last, in 256-row tiles where the stack
    has eight bytes; a byte of 255 makes its own column NaN and no neighbour."""
    b, s = _weights(E, n, k, k + n)
    g = torch.Generator().manual_seed(k * n)
    s[torch.rand(s.shape, generator=g) < 0.1] = 255
    sizes, ids = [300, 45], [E - 1, 0]
    a = _rows(sum(sizes), k, torch.bfloat16, k + n + 1)
    _check_both(a, b, s, sizes, ids)


@pytest.mark.parametrize("dtype", (torch.bfloat16, torch.float16))
@pytest.mark.parametrize("k", (32, 96, 224, 256, 288, 1216, 2880))
@pytest.mark.parametrize("sizes", ([1], [4, 0, 1, 3], [8, 5], [0, 7, 1, 2]))
def test_rows_quantized_inside_the_tiles_and_before_them(sizes, k, dtype):
    """Small groups, whose tiles quantize the rows themselves, and the same rows beside a group of more rows than a tile
    holds, for which all are quantized before the product (test_few_rows adds five rows, which the tiles still
    take): the same bytes."""
    E, n = 3, 72
    b, s = _weights(E, n, k, k)
    ids = [2, 1, 0, 2][:len(sizes)]
    a = _rows(sum(sizes) + 40, k, dtype, k + 9)
    a[0, :32] = 0
    few = a[:sum(sizes)]
    out = _run(few, b, s, sizes, ids)
    _check(few, b, s, sizes, ids, out)
    all_rows = _run(a, b, s, sizes + [40], ids + [1])
    _check(a, b, s, sizes + [40], ids + [1], all_rows)
    assert torch.equal(all_rows[:len(few)], out)
