"""Distillation from a teacher's top logits against its definition in 64 bits."""
import math

import pytest
import torch

import learn_util as lu
from gpu_util import status_word

pytestmark = pytest.mark.gpu

# (rows, vocab, k): one entry of everything, fewer logits than a warp, odd sizes, rows split over
# several blocks, more rows than blocks resident, as many entries as there can be
SHAPES = [(1, 1, 1), (3, 2, 2), (2, 31, 5), (5, 1000, 8), (1, 131072, 32), (3, 50003, 17), (700, 1027, 33), (2, 9001, 1024),
          (17, 40000, 300), (1300, 260, 64)]
DTYPES = [torch.float32, torch.bfloat16, torch.float16, torch.float64]


def _data(shape, dtype, seed, pad=0, offset=0, spread=3.0):
    rows, vocab, k = shape
    gen = torch.Generator().manual_seed(seed)
    teacher = spread * torch.randn((rows, vocab), generator=gen)
    top, at = teacher.topk(k, dim=1)
    z = 0.7 * teacher + torch.randn((rows, vocab), generator=gen)
    wide = lu.WIDE[dtype]
    return lu.padded(z.double().cuda(), dtype, pad, offset), at.cuda(), top.to(wide).cuda(), gen


def _tolerances(z, top, t, want, up, w, dtype):
    """An exponent (z - m) c, c = log2(e) / T, is off by 3 u |(z - m) c| (the difference, c and the product
    round), which matters where the term does: A = 24 covers terms above 2^-24 of the largest.  A term is off
    by 2^-22 (the approximation; 2^-50 in 64 bits) + 3 A u, s by that and chain u relative, ln q by s's.  The
    row's other sums are in binary64.  A q below 2^-24 has an exponent of up to E, and 3 E u.
    A p comes from an exponent a = t / T in 64 bits: it is off by (|a| + 8) 2^-53 (the quotient, the
    difference from the maximum, exp, the sum, the division), as the plain form's is by the same, which binary64
    shows; there the plain form's q and sums are off as the kernel's are, which doubles the whole."""
    loss, m, s, gradient, target, q = want
    vocab = z.shape[1]
    wide = lu.WIDE[dtype]
    e = lu.u(wide)
    near = 2.0 ** -22 if wide == torch.float32 else 2.0 ** -50
    rel_s = near + 3 * 24 * e + (lu.chain(vocab) + 8) * e
    weight = (torch.ones_like(loss) if w is None else w.double()).abs()
    t_loss = weight * t * t * (rel_s + 64 * 2.0 ** -50) + 2 * e * loss.abs() + 1e-300
    exponent = ((z.double() - z.double().amax(dim=1, keepdim=True)) / t * math.log2(math.e)).abs()
    exponent = torch.where(torch.isfinite(exponent), exponent, 0.0).clamp(max=200)
    factor = ((1.0 if up is None else up.double()) * weight * t).expand(z.shape[0])[:, None].abs()
    far = torch.where(torch.isfinite(top), top.double(), 0.0).abs().amax() / t if top.numel() else 0.0
    t_p = 3 * e + 2 * (far + 8) * 2.0 ** -53
    t_grad = factor * (q * (rel_s + near + 3 * exponent * e + 4 * e) + t_p * target + 2.0 ** -126)
    if wide == torch.float64:
        t_grad, t_loss, rel_s = 2 * t_grad, 2 * t_loss + weight * t * t * (far + 8) * 2.0 ** -50, 2 * rel_s
    t_grad = t_grad + lu.u(dtype) * gradient.abs() * 1.01 + torch.finfo(dtype).smallest_normal * lu.u(dtype) * 2
    return t_loss, rel_s, t_grad


def _check(provider, z, at, top, t, w, up, dtype):
    want = lu.distill(z, at, top, t, w, up)
    t_loss, rel_s, t_grad = _tolerances(z, top, t, want, up, w, dtype)
    status = provider.new_status()
    loss, stats = provider.distill_loss(z, at, top, temperature=t, row_weights=w, status=status)
    lu.within(loss, want[0], t_loss, "loss")
    assert torch.equal(stats[:, 0].double(), want[1])
    lu.within(stats[:, 1], want[2], rel_s * want[2], "sum")
    gradient = provider.distill_loss_backward(z, at, top, stats, upstream=up, temperature=t, row_weights=w, status=status)
    lu.within(gradient, want[3], t_grad, "gradient")
    loss2, stats2, gradient2 = provider.distill_loss_step(z, at, top, upstream=up, temperature=t, row_weights=w,
                                                          status=status)
    assert torch.equal(loss, loss2) and torch.equal(stats, stats2) and torch.equal(gradient, gradient2)
    assert status_word(status) == provider.STATUS_OK
    return loss, stats, gradient


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_loss_and_gradient(provider, shape, dtype):
    rows, vocab, k = shape
    wide = lu.WIDE[dtype]
    for seed, (pad, offset, t) in enumerate([(0, 0, 1.0), (8, 0, 2.0), (3, 1, 0.7)]):
        z, at, top, gen = _data(shape, dtype, seed, pad, offset)
        w = up = None
        if seed == 1:
            w = (torch.rand(rows, generator=gen) * (torch.rand(rows, generator=gen) > 0.3)).to(wide).cuda()
            up = torch.full((1,), 1.0 / rows, dtype=wide).cuda()
        if seed == 2:
            at = torch.where(torch.rand((rows, k), generator=gen).cuda() < 0.4, -1 - at, at)
            up = torch.randn(rows, generator=gen).to(wide).cuda()
        _check(provider, z, at, top, t, w, up, dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float64])
def test_masks(provider, dtype):
    """Masked vocabulary entries (-infinity and the type's lowest value), whole runs of them, rows whose
    only entry is one finite logit, absent teacher entries by logit and by index, rows without any."""
    z, at, top, gen = _data((12, 3000, 16), dtype, 5)
    keep = torch.zeros((12, 3000), dtype=torch.bool, device="cuda").scatter_(1, at, True)
    z[0] = torch.where(keep[0], z[0], -math.inf)
    z[1] = torch.where(keep[1], z[1], torch.finfo(dtype).min)
    z[2, :2990] = torch.where(keep[2, :2990], z[2, :2990], -math.inf)
    z[3] = -math.inf
    z[3, 17] = 4.0
    at[3] = -1
    at[3, 5] = 17
    top[4, 3:] = -math.inf
    at[5, 1:] = -9
    at[6] = -1
    z[6] = math.nan  # a row without entries is not read
    top[7] = -math.inf
    z[7] = -math.inf
    w = torch.ones(12, dtype=lu.WIDE[dtype], device="cuda")
    w[8] = 0
    z[8] = math.nan
    at[8] = 1 << 40
    zz, a2 = z.clone(), at.clone()
    zz[6], zz[7], zz[8] = 0.0, 0.0, 0.0  # the plain form reads every row
    a2[8] = 0
    want = lu.distill(zz, a2, top, 1.5, w, None)
    t_loss, rel_s, t_grad = _tolerances(zz, top, 1.5, want, None, w, dtype)
    status = provider.new_status()
    loss, stats, gradient = provider.distill_loss_step(z, at, top, temperature=1.5, row_weights=w, status=status)
    lu.within(loss, want[0], t_loss, "loss")
    lu.within(gradient, want[3], t_grad, "gradient")
    lu.within(stats[:, 1], want[2], rel_s * want[2], "sum")
    assert status_word(status) == provider.STATUS_OK
    assert not gradient[6:9].any() and not loss[6:9].any()
    assert torch.equal(stats[6:9].double().cpu(), torch.tensor([[0.0, 1.0]] * 3, dtype=torch.float64))
    # the gradient of a masked entry is 0, also where a whole thread's share is masked
    assert not gradient[0][~keep[0]].any()


def test_repeated_indices_add_up(provider):
    z, at, top, gen = _data((4, 500, 24), torch.float32, 6)
    at[0, :] = at[0, 0]
    at[1, 1] = at[1, 0]
    at[2, 20:] = at[2, 3]
    at[3, ::2] = at[3, 23]
    _check(provider, z, at, top, 1.0, None, None, torch.float32)


def test_gradient_against_differences(provider):
    """Central differences of the loss in binary64, step 1e-5: e^2 / 6 of a third derivative below 10, and
    the rounding of a loss of about 5 divided by e."""
    z, at, top, gen = _data((2, 12, 4), torch.float64, 7)
    up = torch.tensor([0.7, -1.3], dtype=torch.float64, device="cuda")
    at[1, 2] = at[1, 0]
    _, _, gradient = provider.distill_loss_step(z, at, top, upstream=up, temperature=1.7)
    e = 1e-5
    for i in range(2):
        for v in range(12):
            kept = float(z[i, v])
            z[i, v] = kept + e
            a = provider.distill_loss(z, at, top, temperature=1.7)[0]
            z[i, v] = kept - e
            b = provider.distill_loss(z, at, top, temperature=1.7)[0]
            z[i, v] = kept
            assert abs(float(((a - b) * up).sum()) / (2 * e) - float(gradient[i, v])) < 50 * e * e + 1e-13 / e


def test_large_and_far_logits(provider):
    """Logits of magnitude 1e4 in binary32, a low temperature, and a teacher far from the student."""
    z, at, top, gen = _data((5, 700, 9), torch.float32, 8, spread=1.0)
    z = (z * 16).round() / 16 + 10000.0  # exact
    _check(provider, z, at, top * 40, 0.5, None, None, torch.float32)
    _check(provider, z - 20000.0, at.flip(1), top * 1000, 4.0, None, None, torch.float32)


def test_small_and_large_temperatures(provider):
    """A temperature whose reciprocal leaves hardly a term beside the largest, one that makes q uniform, and
    one at which logits divided by it exceed binary32."""
    z, at, top, gen = _data((6, 900, 5), torch.float32, 15)
    for t in (1e-3, 1e6):
        _check(provider, z, at, top, t, None, None, torch.float32)
    t = 1e-37
    z[:, 0] = z.amax(dim=1) + 1
    at[:, 0], at[:, 1:] = 0, -1
    loss, stats, gradient = provider.distill_loss_step(z, at, top, temperature=t)
    # the teacher's only entry is the student's largest logit: nothing else has a share, both are certain
    assert not loss.any() and not gradient.any() and bool((stats[:, 1] == 1).all())


@pytest.mark.parametrize("vocab", [40, 300001])
def test_teacher_beyond_the_range_of_its_exponents(provider, vocab):
    """Teacher logits that a low temperature takes beyond binary64: only their differences count.  Two largest
    ones, equal, and q uniform: the loss is T^2 (ln V - ln 2), the gradient T (1/V - 1/2) there and T/V elsewhere."""
    t = float(torch.tensor(2.0 ** -120))
    z = torch.zeros((1, vocab), dtype=torch.float64, device="cuda")
    at = torch.tensor([[3, 17, 5, -1]], device="cuda")
    top = torch.tensor([[1e290, 1e290, -1e290, 0.0]], dtype=torch.float64, device="cuda")
    status = provider.new_status()
    loss, _, gradient = provider.distill_loss_step(z, at, top, temperature=t, status=status)
    want = torch.full_like(z, t / vocab)
    want[0, 3] = want[0, 17] = t * (1 / vocab - 0.5)
    eps = torch.finfo(torch.float64).eps
    lu.within(loss, torch.full_like(loss, t * t * math.log(vocab / 2)), t * t * math.log(vocab) * 16 * eps)
    lu.within(gradient, want, want.abs() * (16 + lu.chain(vocab)) * eps)
    assert status_word(status) == provider.STATUS_OK


@pytest.mark.parametrize("dtype,vocab", [(torch.float32, 600001), (torch.float64, 300000), (torch.bfloat16, 1000003)])
def test_rows_longer_than_a_cluster_holds(provider, dtype, vocab):
    z, at, top, gen = _data((3, vocab, 20), dtype, 16)
    at[1, 4:] = at[1, 3]
    w = torch.tensor([1.0, 0.5, 0.0], device="cuda").to(lu.WIDE[dtype])
    loss, stats, gradient = _check(provider, z, at, top, 1.3, w, None, dtype)
    a = z.clone()
    provider.distill_loss_step(a, at, top, temperature=1.3, row_weights=w, gradient=a)
    assert torch.equal(a, gradient)
    z[0, vocab - 1] = math.nan
    status = provider.new_status()
    provider.distill_loss_step(z, at, top, temperature=1.3, row_weights=w, status=status)
    assert provider.decode_status(status_word(status)) == (0, 5)


def test_row_offsets_beyond_32_bits(provider):
    """Two rows 2^31 elements apart."""
    z, at, top, _ = _data((2, 500, 8), torch.float16, 17)
    want = provider.distill_loss_step(z, at, top)
    base = torch.empty((1 << 31) + 500, dtype=torch.float16, device="cuda")
    far = base.as_strided((2, 500), (1 << 31, 1))
    far.copy_(z)
    got = provider.distill_loss_step(far, at, top, gradient=far)
    assert all(torch.equal(a, b) for a, b in zip(want, got))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", [(3, 131072, 16), (400, 777, 16), (2, 40, 4)])
def test_gradient_in_place(provider, shape, dtype):
    z, at, top, _ = _data(shape, dtype, 9, pad=5)
    loss, stats, gradient = provider.distill_loss_step(z, at, top)
    a = lu.padded(z, dtype, 5)
    loss2, _, got = provider.distill_loss_step(a, at, top, gradient=a)
    assert got is a and torch.equal(a, gradient) and torch.equal(loss, loss2)
    a = lu.padded(z, dtype, 5)
    provider.distill_loss_backward(a, at, top, stats, gradient=a)
    assert torch.equal(a, gradient)


def test_rows_behind_the_call_are_left(provider):
    z, at, top, _ = _data((4, 300, 8), torch.float32, 10)
    base = torch.full((6, 320), 7.0, device="cuda")
    provider.distill_loss_step(z, at, top, gradient=base[1:5, :300])
    base[1:5, :300] = 7.0
    assert bool((base == 7.0).all())


@pytest.mark.parametrize("vocab", [200, 70000])
def test_faults(provider, vocab):
    def fault(row, change, weights=None, upstream=None):
        z, at, top, _ = _data((6, vocab, 8), torch.float32, 11)
        change(z, at, top)
        status = provider.new_status()
        loss, stats, gradient = provider.distill_loss_step(z, at, top, row_weights=weights, upstream=upstream,
                                                           status=status)
        others = [i for i in range(6) if i != row]
        assert bool(torch.isfinite(loss[others]).all()) and bool(torch.isfinite(gradient[others]).all())
        got = provider.decode_status(status_word(status))
        assert got[0] == row
        return got[1], float(loss[row]), gradient[row]

    def put(t, i, j, v):
        t[i, j] = v

    for v in (math.nan, math.inf):
        kind, loss, g = fault(3, lambda z, at, top: put(z, 3, vocab - 1, v))
        assert kind == 5 and math.isnan(loss) and bool(torch.isnan(g).all())
        kind, loss, g = fault(2, lambda z, at, top: put(top, 2, 7, v))
        assert kind == 5 and math.isnan(loss) and bool(torch.isnan(g).all())
    kind, loss, g = fault(1, lambda z, at, top: z[1].fill_(-math.inf))
    assert kind == 5 and math.isnan(loss) and bool(torch.isnan(g).all())
    for far in (vocab, 1 << 40, (1 << 32) + 1):
        kind, loss, g = fault(5, lambda z, at, top: put(at, 5, 2, far))
        assert kind == 5 and math.isnan(loss) and bool(torch.isnan(g).all())
    # the teacher expects a masked entry: the loss is infinite, the gradient is not
    def masked(z, at, top):
        z[4, at[4, 0]] = -math.inf
    kind, loss, g = fault(4, masked)
    assert kind == 3 and loss == math.inf and bool(torch.isfinite(g).all())
    w = torch.ones(6, device="cuda")
    w[0] = math.nan
    assert fault(0, lambda z, at, top: None, weights=w)[0] == 5
    w[0] = math.inf
    assert fault(0, lambda z, at, top: None, upstream=w)[0] == 5
    # a gradient beyond binary16
    z, at, top, _ = _data((2, vocab, 8), torch.float16, 12)
    status = provider.new_status()
    provider.distill_loss_step(z, at, top, upstream=torch.tensor([1e6], device="cuda"), status=status)
    assert provider.decode_status(status_word(status)) == (0, 3)


def test_backward_reports_bad_statistics(provider):
    z, at, top, _ = _data((4, 100, 4), torch.float32, 13)
    _, stats = provider.distill_loss(z, at, top)
    stats[2, 1] = 0.0
    status = provider.new_status()
    gradient = provider.distill_loss_backward(z, at, top, stats, status=status)
    assert provider.decode_status(status_word(status)) == (2, 5)
    assert bool(torch.isnan(gradient[2]).all()) and bool(torch.isfinite(gradient[[0, 1, 3]]).all())


def test_empty(provider):
    z = torch.empty((0, 10), device="cuda")
    at = torch.empty((0, 3), dtype=torch.int64, device="cuda")
    loss, stats, gradient = provider.distill_loss_step(z, at, torch.empty((0, 3), device="cuda"))
    assert loss.shape == (0,) and gradient.shape == (0, 10)
    z = torch.randn((3, 10), device="cuda")
    at = torch.empty((3, 0), dtype=torch.int64, device="cuda")
    loss, stats, gradient = provider.distill_loss_step(z, at, torch.empty((3, 0), device="cuda"))
    assert not loss.any() and not gradient.any()


@pytest.mark.parametrize("shape", [(3, 100000, 16), (500, 900, 16)])
def test_same_bits_on_another_stream_and_in_a_graph(provider, shape):
    z, at, top, _ = _data(shape, torch.bfloat16, 14)
    want = provider.distill_loss_step(z, at, top)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = provider.distill_loss_step(z, at, top, stream=side)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    zs = z.clone()
    graph = torch.cuda.CUDAGraph()
    status = provider.new_status()
    with torch.cuda.graph(graph):
        loss, stats = provider.distill_loss(zs, at, top, status=status)
        gradient = provider.distill_loss_backward(zs, at, top, stats, status=status)
    for factor in (1.0, 0.5, 1.0):
        zs.copy_(z * factor)
        graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(want, (loss, stats, gradient)))
