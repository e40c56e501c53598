"""A call right behind one that wrote its input in place, without a wait between them: tensors whose rows share
16-byte pieces and lines, logits that other blocks of a cluster read before they were overwritten."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _codes(rows, columns):
    """Room for codes whose rows are whole 16-byte pieces."""
    return torch.empty((rows, (columns + 15) // 16 * 16), dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)[:, :columns]


def _same(codes, scales, want):
    return torch.equal(codes.view(torch.uint8), want[0].view(torch.uint8)) and torch.equal(scales, want[1])


@pytest.mark.parametrize("captured", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("shape", [(4, 7, 33, 3), (64, 50, 77, 7), (2, 4095, 321, 3), (300, 1, 999, 3), (3, 9000, 128, 1)])
def test_quantiser_behind_a_norm_in_place(provider, shape, dtype, captured):
    n, s, c, g = shape
    gen = torch.Generator(device="cuda").manual_seed(n)
    given = torch.randn((n, s, c), generator=gen, device="cuda").to(dtype)
    normal = provider.group_norm(given, g, activation="silu")[0]
    torch.cuda.synchronize()
    want = provider.block_quantize(normal.view(n * s, c))
    x, codes, scales = given.clone(), _codes(n * s, c), torch.empty_like(want[1])
    stats, status = torch.empty((n, g, 2), device="cuda"), provider.new_status(2)

    def step():
        provider.group_norm(x, g, activation="silu", out=x, stats=stats, status=status[:1])
        provider.block_quantize(x.view(n * s, c), codes=codes, scales=scales, status=status[1:])

    if captured:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step()
    for _ in range(30):
        x.copy_(given)
        graph.replay() if captured else step()
        torch.cuda.synchronize()
        assert _same(codes, scales, want)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,vocab,k", [(20, 60000, 256), (8, 131071, 1024), (100, 9001, 64)])
def test_quantiser_behind_a_gradient_in_place(provider, rows, vocab, k, dtype):
    gen = torch.Generator(device="cuda").manual_seed(rows)
    given = torch.randn((rows, vocab), generator=gen, device="cuda").to(dtype)
    top, at = given.float().topk(k, dim=1)
    gradient = provider.distill_loss_step(given, at, top)[2]
    torch.cuda.synchronize()
    want = provider.block_quantize(gradient)
    z, codes, scales = given.clone(), _codes(rows, vocab), torch.empty_like(want[1])
    loss, stats, status = torch.empty(rows, device="cuda"), torch.empty((rows, 2), device="cuda"), provider.new_status(2)
    for _ in range(30):
        z.copy_(given)
        provider.distill_loss_step(z, at, top, loss=loss, stats=stats, gradient=z, status=status[:1])
        provider.block_quantize(z, codes=codes, scales=scales, status=status[1:])
        torch.cuda.synchronize()
        assert _same(codes, scales, want)


@pytest.mark.parametrize("rows", [1, 20, 200])
def test_products_over_the_same_buffers(provider, rows):
    """A row form's scales come from a buffer that each step's quantiser writes anew."""
    gen = torch.Generator(device="cuda").manual_seed(rows)
    w = provider.block_quantize(torch.randn((640, 1024), generator=gen, device="cuda"), 128)
    xs = [torch.randn((rows, 1024), generator=gen, device="cuda") * 2.0 ** i for i in range(-6, 7, 2)]
    want = []
    for x in xs:
        want.append(provider.block_matmul(*provider.block_quantize(x), *w, dtype=torch.float32))
        torch.cuda.synchronize()
    codes, scales, status = _codes(rows, 1024), torch.empty((rows, 8), device="cuda"), provider.new_status(2)
    out = [torch.empty_like(v) for v in want]
    for _ in range(20):
        for x, y in zip(xs, out):
            provider.block_quantize(x, codes=codes, scales=scales, status=status[:1])
            provider.block_matmul(codes, scales, *w, out=y, status=status[1:])
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))
