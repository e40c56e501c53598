"""Group norm with an activation, forward and backward, against its definition in 64 bits."""
import math

import pytest
import torch

import learn_util as lu
from gpu_util import status_word

pytestmark = pytest.mark.gpu

# (batch, positions, channels, groups): one element a group, narrow and odd widths, one position (an
# MLP's rows), long and short maps, more channels than a warp's vectors, one group over everything
SHAPES = [(1, 1, 4, 4), (1, 1, 1, 1), (3, 1, 8, 2), (2, 7, 33, 3), (5, 1, 4096, 32), (300, 1, 96, 3), (2, 300, 320, 32),
          (1, 1000, 64, 1), (4, 315, 10, 10), (2, 4097, 40, 4), (1, 20001, 16, 2), (3, 2, 5000, 1), (1, 1, 20000, 1),
          (2, 70, 136, 17), (9000, 1, 32, 8)]
DTYPES = [torch.float32, torch.bfloat16, torch.float16, torch.float64]


def _data(shape, dtype, seed, pad=0, offset=0, affine=True, shift=0.0):
    n, s, c, g = shape
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn((n, s, c), generator=gen, dtype=torch.float64) * (torch.rand(c, generator=gen) + 0.5) + shift
    dy = torch.randn((n, s, c), generator=gen, dtype=torch.float64)
    wide = lu.WIDE[dtype]
    w = (1 + 0.3 * torch.randn(c, generator=gen)).to(wide).cuda() if affine else None
    b = (0.3 * torch.randn(c, generator=gen)).to(wide).cuda() if affine else None
    return lu.padded(x.cuda(), dtype, pad, offset), lu.padded(dy.cuda(), dtype, pad, offset), w, b


def _forward_tolerance(x, g, w, b, y, h, dtype):
    """The mean is off by chain(m) u max|x|, the variance's root likewise relative to itself (its terms
    have mean errors of second order); h then by u (chain(m) (max|x| r + |h|) + 3 |h|), z by that times
    |w| and 2 u (|h w| + |b|).  The activations have slopes below 1.13 and add 8 u |z|."""
    n, s, c = x.shape
    e = lu.u(lu.WIDE[dtype])
    m = s * (c // g)
    mean, r = lu.norm_stats(x, g)
    top = x.double().abs().reshape(n, s, g, c // g).amax(dim=(1, 3))
    reach = (top * r)[:, None, :, None].expand(n, s, g, c // g).reshape(n, s, c)
    aw = 1.0 if w is None else w.double().abs()
    ab = 0.0 if b is None else b.double().abs()
    z = e * ((lu.chain(m) + 4) * (reach + h.abs()) * aw + 2 * (h.abs() * aw + ab))
    return 1.13 * z + 8 * e * (h.abs() * aw + ab) + lu.u(dtype) * y.abs() * 1.01 + torch.finfo(dtype).smallest_normal


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_forward(provider, shape, dtype):
    for seed, (name, pad, offset, affine) in enumerate([("none", 0, 0, False), ("relu", 8, 0, True), ("silu", 0, 1, True),
                                                         ("gelu", 3, 0, True)]):
        x, _, w, b = _data(shape, dtype, seed, pad, offset, affine)
        g = shape[3]
        status = provider.new_status()
        out, stats = provider.group_norm(x, g, w, b, activation=name, status=status)
        y, _, h = lu.norm_forward(x, g, w, b, name)
        lu.within(out, y, _forward_tolerance(x, g, w, b, y, h, dtype), name)
        mean, r = lu.norm_stats(x, g)
        e = lu.u(lu.WIDE[dtype]) * (lu.chain(shape[1] * shape[2] // g) + 4)
        top = x.double().abs().reshape(shape[0], shape[1], g, -1).amax(dim=(1, 3))
        lu.within(stats[..., 0], mean, e * top, "mean")
        lu.within(stats[..., 1], r, 2 * e * r * (1 + (top * r * e) ** 2), "r")
        assert status_word(status) == provider.STATUS_OK


def _backward_tolerances(x, dy, g, stats, w, b, name, dtype, want):
    """z is off by 4 u (|h w| + |b|) and h by 3 u |h|; the slopes of silu and gelu change by at most
    1.2 per unit of z and are off by 8 u (1 + |z|) themselves; ReLU's is exact.  So dz is off by
    d = |dy| (4.8 (|h w| + |b|) + 8 (1 + |z|)) u (0 for relu and none, whose slopes are exact), k = dz w by
    d |w| + u |k|.  c1 and c2 are off by the mean of that and chain(m) u of their terms' mean."""
    dx, dw, db, dz, h, k = want
    n, s, c = x.shape
    e = lu.u(lu.WIDE[dtype])
    d = c // g
    m = s * d
    r = stats[..., 1].double()[:, None, :, None]
    aw = torch.ones(c, dtype=torch.float64, device=x.device) if w is None else w.double().abs()
    ab = torch.zeros(c, dtype=torch.float64, device=x.device) if b is None else b.double().abs()
    z = h.abs() * aw + ab
    bend = 0.0 if name in ("none", "relu") else 1.0
    eh = 3 * e * h.abs()
    edz = bend * dy.double().abs() * (1.2 * (eh * aw + 2 * e * z) + 8 * e * (1 + z)) + e * dz.abs()
    ek = edz * aw + e * k.abs()

    def mean(v):
        return v.reshape(n, s, g, d).mean(dim=(1, 3), keepdim=True).expand(n, s, g, d).reshape(n, s, c)

    terms = k.abs() * h.abs()
    c1, c2 = mean(k).abs(), mean(k * h).abs()
    e1 = mean(ek) + lu.chain(m) * e * mean(k.abs())
    e2 = mean(ek * h.abs() + k.abs() * eh) + lu.chain(m) * e * mean(terms)
    off = ek + e1 + h.abs() * e2 + c2 * eh + 4 * e * (k.abs() + c1 + h.abs() * c2)
    t_dx = r.expand(n, s, g, d).reshape(n, s, c) * off + lu.u(dtype) * dx.abs() * 1.01 + torch.finfo(dtype).smallest_normal
    rows = n * s
    t_dw = (edz * h.abs() + dz.abs() * eh).sum(dim=(0, 1)) + (lu.chain(rows) + 2) * e * (dz * h).abs().sum(dim=(0, 1))
    t_db = edz.sum(dim=(0, 1)) + (lu.chain(rows) + 2) * e * dz.abs().sum(dim=(0, 1))
    return t_dx, t_dw + 1e-300, t_db + 1e-300


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_backward(provider, shape, dtype):
    for seed, (name, pad, offset, affine) in enumerate([("none", 0, 1, False), ("relu", 0, 0, True), ("silu", 8, 0, True),
                                                         ("gelu", 3, 0, True)]):
        x, dy, w, b = _data(shape, dtype, 10 + seed, pad, offset, affine)
        g = shape[3]
        wide = lu.WIDE[dtype]
        mean, r = lu.norm_stats(x, g)
        stats = torch.stack([mean, r], dim=2).to(wide)
        status = provider.new_status()
        dx, dw, db = provider.group_norm_backward(x, dy, g, stats, w, b, activation=name, status=status)
        want = lu.norm_backward(x, dy, g, stats, w, b, name)
        t_dx, t_dw, t_db = _backward_tolerances(x, dy, g, stats, w, b, name, dtype, want)
        lu.within(dx, want[0], t_dx, "dx " + name)
        if affine:
            lu.within(dw, want[1], t_dw, "dw " + name)
            lu.within(db, want[2], t_db, "db " + name)
        else:
            assert dw is None and db is None
        assert status_word(status) == provider.STATUS_OK


@pytest.mark.parametrize("name", ["none", "silu", "gelu"])
def test_backward_against_differences(provider, name):
    """Central differences of the forward call in binary64: step e, error e^2 |third derivative| / 6
    (bounded by 10 here) plus the rounding of two sums of 200 terms divided by e."""
    gen = torch.Generator().manual_seed(5)
    x = torch.randn((2, 4, 6), generator=gen, dtype=torch.float64).cuda()
    w, b = (1 + 0.3 * torch.randn(6, generator=gen, dtype=torch.float64)).cuda(), torch.randn(6, generator=gen, dtype=torch.float64).cuda()
    dy = torch.randn((2, 4, 6), generator=gen, dtype=torch.float64).cuda()

    def value(x, w, b):
        return float((provider.group_norm(x, 2, w, b, activation=name)[0] * dy).sum())

    _, stats = provider.group_norm(x, 2, w, b, activation=name)
    got = provider.group_norm_backward(x, dy, 2, stats, w, b, activation=name)
    e = 1e-5
    for which, t in enumerate((x, w, b)):
        flat = t.view(-1)
        for i in range(flat.numel()):
            kept = float(flat[i])
            flat[i] = kept + e
            up = value(x, w, b)
            flat[i] = kept - e
            down = value(x, w, b)
            flat[i] = kept
            assert abs((up - down) / (2 * e) - float(got[which].view(-1)[i])) < 50 * e * e + 1e-14 * 200 / e


def test_far_mean_keeps_the_variance(provider):
    """Values far from 0 beside their spread: the variance is about the mean, so r keeps its digits.
    The data are exact in binary32 (1000 + k / 64); the mean is off by chain u 1002, and the variance by
    the square of that, 1e-6 here, beside u chain relative."""
    gen = torch.Generator().manual_seed(2)
    x = (1000 + torch.randint(-128, 129, (2, 500, 64), generator=gen) / 64.0).float().cuda()
    _, stats = provider.group_norm(x, 4)
    mean, r = lu.norm_stats(x, 4)
    e = lu.u(torch.float32) * (lu.chain(500 * 16) + 4)
    lu.within(stats[..., 0], mean, e * 1002)
    lu.within(stats[..., 1], r, r * (e + (e * 1002) ** 2 * r * r))


def test_one_far_element_keeps_the_variance(provider):
    """An outlier as a group's first element does not become the point that the variance is taken about."""
    gen = torch.Generator().manual_seed(3)
    x = torch.randn((1, 6000, 32), generator=gen).cuda()
    x[0, 0, :] = 4096.0
    _, stats = provider.group_norm(x, 2)
    mean, r = lu.norm_stats(x, 2)
    e = lu.u(torch.float32) * (lu.chain(6000 * 16) + 4)
    lu.within(stats[..., 1], r, r * (e + (e * 4096) ** 2 * r * r))


def test_relu_side_is_decided_in_binary64(provider):
    """z within binary32's rounding of 0: the bias is the negated product h w, rounded, so the sign of z
    is that rounding's."""
    gen = torch.Generator().manual_seed(7)
    x = torch.randn((64, 3, 64), generator=gen).cuda()
    dy = torch.ones_like(x)
    w = (1 + torch.rand(64, generator=gen)).cuda()
    mean, r = lu.norm_stats(x, 4)
    stats = torch.stack([mean, r], dim=2).float()
    h = lu.norm_forward(x, 4, None, None, "none", (stats[..., 0].double(), stats[..., 1].double()))[2]
    b = -(h[10, 1] * w.double()).float()
    want = lu.norm_backward(x, dy, 4, stats, w, b, "relu")
    dx, dw, db = provider.group_norm_backward(x, dy, 4, stats, w, b, activation="relu")
    t_dx, t_dw, t_db = _backward_tolerances(x, dy, 4, stats, w, b, "relu", torch.float32, want)
    lu.within(dx, want[0], t_dx)
    lu.within(db, want[2], t_db)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", [(6, 1, 256, 8), (2, 600, 96, 3), (1, 30001, 16, 2), (2, 5, 7, 7)])
def test_in_place(provider, shape, dtype):
    x, dy, w, b = _data(shape, dtype, 3)
    g = shape[3]
    want, stats = provider.group_norm(x, g, w, b, activation="silu")
    y = x.clone()
    provider.group_norm(y, g, w, b, activation="silu", out=y)
    assert torch.equal(y, want)
    grads = provider.group_norm_backward(x, dy, g, stats, w, b, activation="silu")
    for which in (0, 1):
        a, d = x.clone(), dy.clone()
        again = provider.group_norm_backward(a, d, g, stats, w, b, activation="silu", dx=(a, d)[which])
        assert all(torch.equal(p, q) for p, q in zip(grads, again))


def test_offsets_beyond_32_bits(provider):
    """Positions, and samples, 2^31 elements apart: the rows' offsets need 64 bits in every form."""
    x, dy, w, b = _data((2, 2, 64, 4), torch.bfloat16, 9)
    want = provider.group_norm(x, 4, w, b, activation="silu")
    grads = provider.group_norm_backward(x, dy, 4, want[1], w, b, activation="silu")
    base = torch.empty((1 << 31) * 3 + 64, dtype=torch.bfloat16, device="cuda")
    for strides in ((1 << 31, 64, 1), (64, 1 << 31, 1), (1 << 32, 1 << 31, 1)):
        far = base.as_strided((2, 2, 64), strides)
        far.copy_(x)
        out, stats = provider.group_norm(far, 4, w, b, activation="silu")
        e = lu.u(torch.float32) * 64
        lu.within(stats, want[1].double(), e * (1 + want[1].double().abs()))
        y, _, h = lu.norm_forward(x, 4, w, b, "silu")
        lu.within(out, y, _forward_tolerance(x, 4, w, b, y, h, torch.bfloat16))
        got = provider.group_norm_backward(far, dy, 4, want[1], w, b, activation="silu")
        target = lu.norm_backward(x, dy, 4, want[1], w, b, "silu")
        for g, t, tol in zip(got, target, _backward_tolerances(x, dy, 4, want[1], w, b, "silu", torch.bfloat16, target)):
            lu.within(g, t, tol)


@pytest.mark.parametrize("shape", [(6, 5, 64, 4), (3, 500, 48, 4), (2, 20000, 16, 2)])
def test_positions_first(provider, shape):
    """[positions, batch, channels] in memory, passed as [batch, positions, channels]: the same bits."""
    x, dy, w, b = _data(shape, torch.float32, 13)
    g = shape[3]
    want, stats = provider.group_norm(x, g, w, b, activation="silu")
    grads = provider.group_norm_backward(x, dy, g, stats, w, b, activation="silu")
    xt, yt = (t.transpose(0, 1).contiguous().transpose(0, 1) for t in (x, dy))
    out, stats2 = provider.group_norm(xt, g, w, b, activation="silu")
    assert torch.equal(out, want) and torch.equal(stats, stats2)
    assert all(torch.equal(p, q) for p, q in zip(grads, provider.group_norm_backward(xt, yt, g, stats, w, b, activation="silu")))


def test_constant_groups(provider):
    """No spread at all: the variance is 0, never less, and r is 1 / sqrt(eps)."""
    for shape, g in (((3, 1, 64), 4), ((2, 500, 64), 4), ((1, 40000, 8), 1), ((2, 300, 30), 3)):
        x = torch.full(shape, 1234.567, device="cuda")
        out, stats = provider.group_norm(x, g, eps=0.25)
        lu.within(stats[..., 1], torch.full_like(stats[..., 1], 2.0).double(), 8 * lu.u(torch.float32) + (1234.567 * lu.u(torch.float32) * 700) ** 2 * 8)
        assert float(out.abs().max()) <= 2 * 1234.567 * lu.u(torch.float32) * 1400


def test_masked_upstream_does_not_leak(provider):
    """An infinite or NaN upstream where ReLU is off counts for nothing."""
    for shape in ((4, 1, 64, 4), (2, 300, 64, 4), (1, 20000, 16, 2)):
        x, dy, w, b = _data(shape, torch.float32, 12)
        g = shape[3]
        y, stats = provider.group_norm(x, g, w, b, activation="relu")
        clean = torch.where(y > 0, dy, 0.0)
        dirty = torch.where(y > 0, dy, torch.where(torch.rand_like(dy) < 0.5, math.nan, math.inf))
        a = provider.group_norm_backward(x, clean, g, stats, w, b, activation="relu")
        d = provider.group_norm_backward(x, dirty, g, stats, w, b, activation="relu")
        # y is rounded, z decided in binary64: none lies between here, so the masks agree
        assert all(torch.equal(p, q) for p, q in zip(a, d))


def test_strided_output_leaves_the_gaps(provider):
    x, _, w, b = _data((3, 50, 24, 4), torch.float32, 1)
    base = torch.full((3, 51, 40), 7.0, device="cuda")
    out = base[:, :50, :24]
    provider.group_norm(x, 4, w, b, out=out)
    assert torch.equal(out, provider.group_norm(x, 4, w, b)[0])
    out.fill_(7.0)
    assert bool((base == 7.0).all())


@pytest.mark.parametrize("shape", [(3, 1, 64, 4), (2, 40, 32, 4), (1, 9000, 16, 2)])
def test_faults(provider, shape):
    n, s, c, g = shape
    d = c // g
    x, dy, w, b = _data(shape, torch.float32, 4)
    for bad in (math.nan, math.inf, -math.inf):
        y = x.clone()
        y[n - 1, s - 1, c - 1] = bad
        status = provider.new_status()
        out, stats = provider.group_norm(y, g, w, b, activation="relu", status=status)
        hit = torch.zeros((n, s, c), dtype=torch.bool, device="cuda")
        hit[n - 1, :, c - d:] = True
        assert bool(torch.isnan(out[hit]).all()) and bool(torch.isfinite(out[~hit]).all())
        assert provider.decode_status(status_word(status)) == (((n - 1) * s) * c + c - d, 5)
    # an infinite upstream: NaN throughout its group (c1 is infinite), first at the group's first element
    up = dy.clone()
    up[0, 0, 0] = math.inf
    _, stats = provider.group_norm(x, g)
    status = provider.new_status()
    dx, _, _ = provider.group_norm_backward(x, up, g, stats, status=status)
    event, kind = provider.decode_status(status_word(status))
    assert event == 0 and kind in (3, 5)
    assert not bool(torch.isfinite(dx[0, :, :d]).any()) and bool(torch.isfinite(dx[0, :, d:]).all())
    # a weight that is not finite shows in its channel, and in the parameters' gradients
    w2 = w.clone()
    w2[1] = math.nan
    status = provider.new_status()
    out, _ = provider.group_norm(x, g, w2, b, status=status)
    assert provider.decode_status(status_word(status)) == (1, 5)
    # a result beyond its type
    status = provider.new_status()
    provider.group_norm(x.half(), g, torch.full_like(w, 1e6), b, status=status)
    assert provider.decode_status(status_word(status))[1] == 3
    # a variance beyond binary32
    status = provider.new_status()
    provider.group_norm(x * 1e30, g, status=status)
    assert provider.decode_status(status_word(status)) == (0, 5)


def test_parameter_faults_come_after_the_elements(provider):
    x, dy, w, b = _data((2, 3, 8, 2), torch.float32, 4)
    _, stats = provider.group_norm(x, 2, w, b)
    big = torch.zeros_like(dy)
    big[:, :, 5] = 3e38  # each element's own gradient is finite (w = 0), the sum over the rows is not
    w0 = torch.zeros_like(w)
    status = provider.new_status()
    dx, dw, db = provider.group_norm_backward(x, big, 2, stats, w0, b, status=status)
    event, kind = provider.decode_status(status_word(status))
    assert bool(torch.isfinite(dx).all()) and math.isinf(float(db[5]))
    assert event in (48 + 5, 48 + 8 + 5) and kind in (3, 5)
    assert event == (48 + 5 if not math.isfinite(float(dw[5])) else 48 + 8 + 5)


def test_empty(provider):
    for shape in [(0, 3, 8), (3, 0, 8), (2, 3, 0)]:
        x = torch.empty(shape, device="cuda")
        c = shape[2]
        w, b = torch.ones(c, device="cuda"), torch.ones(c, device="cuda")
        out, stats = provider.group_norm(x, 2, w, b)
        assert out.shape == x.shape and stats.shape == (shape[0], 2, 2)
        stats = torch.ones_like(stats)
        dw, db = torch.full_like(w, 9), torch.full_like(b, 9)
        provider.group_norm_backward(x, x, 2, stats, w, b, dweight=dw, dbias=db)
        assert not dw.any() and not db.any()
    x = torch.empty((3, 0, 8), device="cuda")
    _, stats = provider.group_norm(x, 2, eps=0.25)
    assert torch.equal(stats, torch.tensor([0.0, 2.0], device="cuda").expand(3, 2, 2))


@pytest.mark.parametrize("shape", [(40, 1, 512, 8), (2, 700, 80, 8), (1, 30000, 32, 2)])
def test_same_bits_on_another_stream_and_in_a_graph(provider, shape):
    g = shape[3]
    x, dy, w, b = _data(shape, torch.bfloat16, 6)
    out, stats = provider.group_norm(x, g, w, b, activation="silu")
    grads = provider.group_norm_backward(x, dy, g, stats, w, b, activation="silu")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    o2, s2 = provider.group_norm(x, g, w, b, activation="silu", stream=side)
    g2 = provider.group_norm_backward(x, dy, g, s2, w, b, activation="silu", stream=side)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(out, o2) and torch.equal(stats, s2) and all(torch.equal(p, q) for p, q in zip(grads, g2))
    xs = x.clone()
    status = provider.new_status()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o3, s3 = provider.group_norm(xs, g, w, b, activation="silu", status=status)
        g3 = provider.group_norm_backward(xs, dy, g, s3, w, b, activation="silu", status=status)
    for factor in (1.0, 2.0, 1.0):
        xs.copy_(x * factor)
        graph.replay()
    assert torch.equal(out, o3) and torch.equal(stats, s3) and all(torch.equal(p, q) for p, q in zip(grads, g3))


def test_parameter_gradients_alone_and_none(provider):
    x, dy, w, b = _data((4, 30, 24, 3), torch.float32, 8)
    _, stats = provider.group_norm(x, 3, w, b, activation="gelu")
    dx, dw, db = provider.group_norm_backward(x, dy, 3, stats, w, b, activation="gelu")
    lib = provider.library()
    import ctypes

    def raw(dwp, dbp):
        out = torch.empty_like(x)
        need = lib.pcu_b200_group_norm_backward_workspace_size(0, 4, 30, 24, 3)
        ws = torch.empty(max(need, 1), dtype=torch.uint8, device="cuda")
        status = provider.new_status()
        vp = ctypes.c_void_p
        rc = lib.pcu_b200_group_norm_backward(
            0, 3, vp(x.data_ptr()), vp(dy.data_ptr()), vp(w.data_ptr()), vp(b.data_ptr()), vp(stats.data_ptr()),
            vp(out.data_ptr()), vp(dwp.data_ptr()) if dwp is not None else None,
            vp(dbp.data_ptr()) if dbp is not None else None, 4, 30, 24, 3, 720, 24, 720, 24, 720, 24,
            vp(ws.data_ptr()), need, vp(status.data_ptr()), vp(torch.cuda.current_stream().cuda_stream))
        assert rc == 0
        return out

    assert torch.equal(raw(None, None), dx)
    one = torch.empty_like(w)
    assert torch.equal(raw(one, None), dx) and torch.equal(one, dw)
    assert torch.equal(raw(None, one), dx) and torch.equal(one, db)
    # a gradient for a weight of ones that is not stored
    ones, zeros = torch.ones_like(w), torch.zeros_like(w)
    want = provider.group_norm_backward(x, dy, 3, stats, ones, zeros)
    got = provider.group_norm_backward(x, dy, 3, stats, dweight=torch.empty_like(w), dbias=torch.empty_like(b))
    assert all(torch.equal(p, q) for p, q in zip(got, want))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(2, 90, 2664, 8), (1, 300, 1332, 4), (1, 200, 1022, 2), (3, 64, 4072, 8), (2, 50, 2280, 8)])
def test_wide_blocks_of_odd_groups(provider, shape, dtype):
    """Groups that end inside an access, in blocks of more channels than a CTA has threads."""
    test_forward(provider, shape, dtype)
    test_backward(provider, shape, dtype)
