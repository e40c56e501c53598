"""The 8-bit block quantiser and the product of block-scaled operands, against 64 bits."""
import math

import pytest
import torch

import learn_util as lu
from gpu_util import status_word

pytestmark = pytest.mark.gpu

OUT = [torch.float32, torch.bfloat16, torch.float16]


def _quantize(x, high):
    """Codes (as 64-bit values) and scales by the definition."""
    m, k = x.shape
    v = torch.nn.functional.pad(x.double(), (0, -k % 128, 0, -m % high)).unflatten(1, (-1, 128)).unflatten(0, (-1, high))
    amax = torch.where(torch.isfinite(v), v.abs(), 0.0).amax(dim=(1, 3)).cpu()
    exponent = torch.tensor([[math.frexp(a)[1] + (math.frexp(a)[0] > 0.875) - 9 if a else 0 for a in row] for row in
                             amax.tolist()], dtype=torch.int64).clamp(min=-126)
    scales = (exponent + 1023 << 52).view(torch.float64).to(x.device)
    wide = scales.repeat_interleave(high, 0)[:m].repeat_interleave(128, 1)[:, :k]
    q = x.double() / wide
    e = torch.frexp(q)[1].clamp(min=-5).to(torch.int64) - 1  # 2^e <= |q| < 2^(e + 1); codes below 2^-6 share its step
    step = (e - 3 + 1023 << 52).view(torch.float64)
    return torch.round(q / step) * step, scales


@pytest.mark.parametrize("dtype", OUT)
@pytest.mark.parametrize("high", [1, 128])
@pytest.mark.parametrize("shape", [(1, 1), (3, 128), (5, 129), (128, 256), (130, 1000), (300, 77), (257, 4100)])
def test_quantize(provider, shape, high, dtype):
    gen = torch.Generator().manual_seed(shape[0])
    for pad, offset in ((0, 0), (8, 0), (5, 1)):
        x = torch.randn(shape, generator=gen) * torch.exp(3 * torch.randn((shape[0], 1), generator=gen))
        x = lu.padded(x.double().cuda(), dtype, pad, offset)
        status = provider.new_status()
        codes, scales = provider.block_quantize(x, high, status=status)
        want, want_scales = _quantize(x, high)
        assert torch.equal(scales.double(), want_scales)
        assert torch.equal(codes.double(), want)
        assert status_word(status) == provider.STATUS_OK


def test_quantize_edges(provider):
    """Blocks whose largest value is just at, below and above a step of the scale, zeros, the smallest and
    largest binary32 numbers, ties between codes, values that are not finite."""
    x = torch.zeros((8, 128), device="cuda")
    x[0, 0], x[1, 0] = 448.0, 448.00003
    x[2, 0], x[3, 0] = 447.9, 2.0 ** -149
    x[4, 0] = torch.finfo(torch.float32).max
    x[5, 0], x[5, 1], x[5, 2] = 256.0, 17.0, 19.0  # steps of 2: 17 -> 16, 19 -> 20
    x[5, 3], x[5, 4] = 2.0 ** -10, 3 * 2.0 ** -10  # steps of 2^-9: to 0, to 2^-8
    x[6, :] = -0.0
    x[7, 0], x[7, 1], x[7, 2], x[7, 3] = 1.0, math.nan, math.inf, -math.inf
    status = provider.new_status()
    codes, scales = provider.block_quantize(x, status=status)
    assert scales[:, 0].tolist() == [1.0, 2.0, 1.0, 2.0 ** -126, 2.0 ** 120, 1.0, 1.0, 2.0 ** -8]
    assert codes[5, :5].float().tolist() == [256.0, 16.0, 20.0, 0.0, 2.0 ** -8]
    assert codes[4, 0].float().item() == 256.0 and codes[3, 0].float().item() == 0.0
    assert codes[7, :4].view(torch.uint8).tolist() == [0x78, 0x7f, 0x7f, 0x7f]
    assert provider.decode_status(status_word(status)) == (7 * 128 + 1, 5)


def test_quantize_leaves_the_gaps(provider):
    x = torch.randn((10, 100), device="cuda")
    base = torch.full((10, 112), 0x55, dtype=torch.uint8, device="cuda")
    codes, _ = provider.block_quantize(x, codes=base[:, :100])
    assert bool((base[:, 100:] == 0x55).all())
    assert torch.equal(codes.view(torch.float8_e4m3fn).float(), provider.block_quantize(x)[0].float())


def _operands(rows, inner, columns, seed, room=None):
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn((rows, inner), generator=gen) * torch.exp(torch.randn((rows, 1), generator=gen))
    w = torch.randn((columns, inner), generator=gen)

    def lay(v, high):
        codes, scales = _quantize(v, high)
        stride = (inner + 15) // 16 * 16 if room is None else inner + room
        base = torch.full((v.shape[0], stride), 0x7f, dtype=torch.uint8)  # NaN between the rows
        base[:, :inner] = codes.to(torch.float8_e4m3fn).view(torch.uint8)
        # any powers of two, not only the quantiser's
        scales = (scales * 2.0 ** torch.randint(-3, 4, scales.shape, generator=gen)).float()
        return base.cuda()[:, :inner].view(torch.float8_e4m3fn), scales.cuda()

    return lay(x, 1) + lay(w, 128)


def _exact(a, sa, b, sb):
    wa = sa.double().repeat_interleave(128, 1)[:, :a.shape[1]]
    wb = sb.double().repeat_interleave(128, 0)[:b.shape[0]].repeat_interleave(128, 1)[:, :b.shape[1]]
    x, y = a.double() * wa, b.double() * wb
    return x @ y.t(), x.abs() @ y.abs().t()


def _tolerance(want, size, inner, dtype):
    """Products of codes are exact in binary32, and so is a power of two times them.  The sums are in
    binary32: a group of 32 products in any order (31 u of their magnitudes; the tensor cores align them to
    2^-24 of the largest or finer, which that covers too), the groups one by one."""
    groups = -(-inner // 32)
    return size * (31 + 1 + groups) * lu.u(torch.float32) + lu.u(dtype) * want.abs() * 1.01 + \
        torch.finfo(dtype).smallest_normal


PRODUCTS = [(1, 1, 1), (1, 128, 128), (1, 4096, 520), (3, 1000, 77), (16, 512, 640), (17, 129, 130), (33, 2048, 300),
            (64, 384, 1024), (128, 128, 128), (129, 257, 129), (300, 1111, 1000), (1000, 640, 520), (2049, 256, 1300)]


@pytest.mark.parametrize("dtype", OUT)
@pytest.mark.parametrize("shape", PRODUCTS)
def test_product(provider, shape, dtype):
    rows, inner, columns = shape
    a, sa, b, sb = _operands(rows, inner, columns, rows + inner)
    want, size = _exact(a, sa, b, sb)
    scale = 1.0 if dtype != torch.float16 else 2.0 ** -8
    sa, want, size = sa * scale, want * scale, size * scale
    status = provider.new_status()
    out = provider.block_matmul(a, sa, b, sb, dtype=dtype, status=status)
    lu.within(out, want, _tolerance(want, size, inner, dtype))
    assert status_word(status) == provider.STATUS_OK


@pytest.mark.parametrize("shape", [(1, 200, 130), (5, 129, 33), (140, 300, 150)])
def test_product_of_any_stride(provider, shape):
    """Rows that are not whole 16-byte pieces, and a strided result whose gaps are left alone."""
    rows, inner, columns = shape
    a, sa, b, sb = _operands(rows, inner, columns, 3, room=3)
    want, size = _exact(a, sa, b, sb)
    base = torch.full((rows, columns + 3), 7.0, device="cuda")
    out = provider.block_matmul(a, sa, b, sb, out=base[:, :columns])
    lu.within(out, want, _tolerance(want, size, inner, torch.float32))
    assert bool((base[:, columns:] == 7.0).all())
    a, sa, b, sb = _operands(rows, inner, columns, 3)
    want, size = _exact(a, sa, b, sb)
    out = provider.block_matmul(a, sa, b, sb, out=base[:, :columns])
    lu.within(out, want, _tolerance(want, size, inner, torch.float32))
    assert bool((base[:, columns:] == 7.0).all())


@pytest.mark.parametrize("rows", [2, 40])
def test_offsets_beyond_32_bits(provider, rows):
    """Rows of codes so far apart that the last one begins beyond 2^32 bytes."""
    a, sa, b, sb = _operands(rows, 256, 70, 8)
    want = provider.block_matmul(a, sa, b, sb, dtype=torch.float32)
    stride = ((1 << 32) // (rows - 1) + 16) // 16 * 16
    far = torch.empty(stride * (rows - 1) + 256, dtype=torch.uint8, device="cuda").as_strided((rows, 256), (stride, 1))
    far.copy_(a.view(torch.uint8))
    assert torch.equal(provider.block_matmul(far, sa, b, sb, dtype=torch.float32), want)
    x = torch.randn((rows, 256), device="cuda")
    codes, scales = provider.block_quantize(x)
    out, _ = provider.block_quantize(x, codes=far)
    assert torch.equal(out, codes.view(torch.uint8))


@pytest.mark.parametrize("rows", [1, 9, 200])
def test_cells_are_whole_sums(provider, rows):
    """Integers small enough for every sum to be exact in binary32: the product is exact, whatever the order."""
    gen = torch.Generator().manual_seed(rows)
    a = torch.randint(-8, 9, (rows, 1024), generator=gen).float().cuda().to(torch.float8_e4m3fn)
    b = torch.randint(-8, 9, (400, 1024), generator=gen).float().cuda().to(torch.float8_e4m3fn)
    sa = 2.0 ** torch.randint(-2, 3, (rows, 8), generator=gen).float().cuda()
    sb = 2.0 ** torch.randint(-2, 3, (4, 8), generator=gen).float().cuda()
    want, _ = _exact(a, sa, b, sb)
    out = provider.block_matmul(a, sa, b, sb, dtype=torch.float32)
    assert torch.equal(out.double(), want)


@pytest.mark.parametrize("rows", [1, 20, 300])
def test_faults(provider, rows):
    a, sa, b, sb = _operands(rows, 500, 260, 1)
    at = rows // 2
    a = a.clone()
    a.view(torch.uint8)[at, 300] = 0x7f
    status = provider.new_status()
    out = provider.block_matmul(a, sa, b, sb, status=status)
    assert provider.decode_status(status_word(status)) == (at * 260, 5)
    assert bool(torch.isnan(out[at]).all()) and int(torch.isnan(out).sum()) == 260
    a, sa, b, sb = _operands(rows, 500, 260, 2)
    status = provider.new_status()
    out = provider.block_matmul(a, sa * 2.0 ** 10, b, sb * 2.0 ** 16, dtype=torch.float16, status=status)
    assert provider.decode_status(status_word(status))[1] == 3


@pytest.mark.parametrize("rows,room", [(1, None), (20, None), (300, None), (5, 3)])
def test_a_scale_that_is_no_power_of_two_gives_nan(provider, rows, room):
    for bad in (3.0, 0.0, -1.0, 2.0 ** -127, math.inf, math.nan, 1.0000001):
        a, sa, b, sb = _operands(rows, 500, 260, 3, room)
        sa[rows // 2, 3] = bad
        status = provider.new_status()
        out = provider.block_matmul(a, sa, b, sb, dtype=torch.float32, status=status)
        assert bool(torch.isnan(out[rows // 2]).all()) and int(torch.isnan(out).sum()) == 260
        assert provider.decode_status(status_word(status)) == (rows // 2 * 260, 5)
        a, sa, b, sb = _operands(rows, 500, 260, 3, room)
        sb[1, 2] = bad
        status = provider.new_status()
        out = provider.block_matmul(a, sa, b, sb, dtype=torch.float32, status=status)
        assert bool(torch.isnan(out[:, 128:256]).all()) and int(torch.isnan(out).sum()) == 128 * rows
        assert provider.decode_status(status_word(status)) == (128, 5)


@pytest.mark.parametrize("rows", [1, 20, 300])
def test_large_and_small_scales(provider, rows):
    """Scales far from 1 whose products are not: exact powers of two."""
    a, sa, b, sb = _operands(rows, 300, 200, 5)
    want = provider.block_matmul(a, sa, b, sb, dtype=torch.float32)
    for e in (100, -100):
        got = provider.block_matmul(a, sa * 2.0 ** e, b, sb * 2.0 ** -e, dtype=torch.float32)
        assert torch.equal(got, want)


@pytest.mark.parametrize("rows,room", [(1, None), (20, None), (300, None), (5, 3)])
@pytest.mark.parametrize("left,right,left_code,right_code", [(100, 100, 0.0, 1.0), (-70, -70, 448.0, 448.0),
                                                             (70, 65, 2.0 ** -9, 2.0 ** -9), (-120, 127, 1.0, 448.0)])
def test_scales_whose_product_has_no_exponent(provider, rows, room, left, right, left_code, right_code):
    """2^left by 2^right is beyond binary32 (but for the last), the block's product is not: a power of two times
    a sum of 128 equal products, exact."""
    a, sa, b, sb = _operands(rows, 256, 140, 6, room)
    a.view(torch.uint8)[:] = 0
    a.view(torch.uint8)[:, :128] = torch.tensor(left_code).to(torch.float8_e4m3fn).view(torch.uint8).item()
    b.view(torch.uint8)[:] = torch.tensor(right_code).to(torch.float8_e4m3fn).view(torch.uint8).item()
    sa[:, 0], sb[:, 0], sa[:, 1], sb[:, 1] = 2.0 ** left, 2.0 ** right, 2.0 ** 100, 2.0 ** 100
    status = provider.new_status()
    out = provider.block_matmul(a, sa, b, sb, dtype=torch.float32, status=status)
    want = math.ldexp(128 * left_code * right_code, left + right)
    assert torch.equal(out.double(), torch.full_like(out, want, dtype=torch.float64))
    assert status_word(status) == provider.STATUS_OK


def test_empty(provider):
    f8 = torch.float8_e4m3fn
    z = torch.zeros((4, 0), dtype=torch.uint8, device="cuda").view(f8)
    none = torch.zeros((4, 0), device="cuda")
    out = torch.full((4, 4), 7.0, device="cuda")
    provider.block_matmul(z, none, z, none[:1], out=out)
    assert not out.any()
    a, sa, b, sb = _operands(4, 64, 4, 1)
    assert provider.block_matmul(a[:0], sa[:0], b, sb).shape == (0, 4)
    assert provider.block_matmul(a, sa, b[:0], sb[:0]).shape == (4, 0)
    codes, scales = provider.block_quantize(torch.empty((0, 5), device="cuda"))
    assert codes.shape == (0, 5) and scales.shape == (0, 1)


@pytest.mark.parametrize("rows", [1, 40, 500])
def test_same_bits_on_another_stream_and_in_a_graph(provider, rows):
    gen = torch.Generator().manual_seed(9)
    x = torch.randn((rows, 700), generator=gen).cuda()
    _, _, w, ws = _operands(1, 700, 390, 4)
    codes, scales = provider.block_quantize(x)
    want = provider.block_matmul(codes, scales, w, ws)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    c2, s2 = provider.block_quantize(x, stream=side)
    got = provider.block_matmul(c2, s2, w, ws, stream=side)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(want, got)
    xs = x.clone()
    status = provider.new_status(2)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        c3, s3 = provider.block_quantize(xs, status=status[:1])
        out = provider.block_matmul(c3, s3, w, ws, status=status[1:])
    for factor in (1.0, 3.0, 1.0):
        xs.copy_(x * factor)
        graph.replay()
    assert torch.equal(want, out)
