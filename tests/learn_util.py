"""Plain 64-bit forms of the learning operators, and the error that their kernels may make.

u is half a step of a type relative to the value (finfo.eps / 2).  A sum of n terms in any order is
off by at most (n - 1) u sum|terms|; the kernels never add more than a 32nd of a long sum in one
chain (each thread takes its share, the shares are joined in trees), which `chain` counts."""
import math

import torch

WIDE = {torch.float32: torch.float32, torch.float64: torch.float64, torch.float16: torch.float32,
        torch.bfloat16: torch.float32}


def u(dtype):
    return torch.finfo(dtype).eps / 2


def chain(n):
    return min(n, n / 32 + 40)


def act(z, name):
    if name == "relu":
        return z.clamp(min=0)
    if name == "silu":
        return z * torch.sigmoid(z)
    if name == "gelu":
        return z * 0.5 * torch.erfc(-z / math.sqrt(2))
    return z


def act_slope(z, name):
    if name == "relu":
        return (z > 0).double()
    if name == "silu":
        q = torch.sigmoid(z)
        return q + z * q * (1 - q)
    if name == "gelu":
        return 0.5 * torch.erfc(-z / math.sqrt(2)) + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    return torch.ones_like(z)


def _per_group(v, groups):  # [n, s, c] -> [n, g, s * d]
    n, s, c = v.shape
    return v.reshape(n, s, groups, c // groups).transpose(1, 2).reshape(n, groups, -1)


def norm_stats(x, groups, eps=1e-5):
    """(mean, r) of [n, s, c], in 64 bits."""
    v = _per_group(x.double(), groups)
    mean = v.mean(dim=2)
    var = ((v - mean[..., None]) ** 2).mean(dim=2)
    return mean, 1 / torch.sqrt(var + float(torch.tensor(eps, dtype=torch.float32)))


def norm_forward(x, groups, weight, bias, name, stats=None, eps=1e-5):
    """(y, z, h) in 64 bits; stats: (mean, r) to use instead of x's own."""
    n, s, c = x.shape
    mean, r = norm_stats(x, groups, eps) if stats is None else stats
    v = x.double().reshape(n, s, groups, c // groups)
    h = ((v - mean[:, None, :, None]) * r[:, None, :, None]).reshape(n, s, c)
    z = h * (1.0 if weight is None else weight.double()) + (0.0 if bias is None else bias.double())
    return act(z, name), z, h


def norm_backward(x, dy, groups, stats, weight, bias, name):
    """(dx, dw, db, dz, h, k) in 64 bits for stats [n, g, 2] as given."""
    n, s, c = x.shape
    mean, r = stats[..., 0].double(), stats[..., 1].double()
    _, z, h = norm_forward(x, groups, weight, bias, name, (mean, r))
    dz = dy.double() * act_slope(z, name)
    k = dz * (1.0 if weight is None else weight.double())
    kg, hg = _per_group(k, groups), _per_group(h, groups)
    c1, c2 = kg.mean(dim=2), (kg * hg).mean(dim=2)
    shape = (n, s, groups, c // groups)
    dx = r[:, None, :, None] * (k.reshape(shape) - c1[:, None, :, None] - h.reshape(shape) * c2[:, None, :, None])
    return dx.reshape(n, s, c), (dz * h).sum(dim=(0, 1)), dz.sum(dim=(0, 1)), dz, h, k


def distill(logits, indices, top, temperature, weights, upstream):
    """(loss, m, s, gradient, p, q) in 64 bits, row by row over the vocabulary."""
    rows, vocab = logits.shape
    t = float(torch.tensor(temperature, dtype=torch.float32))
    z = logits.double()
    there = (indices >= 0) & (top != -math.inf)
    some = there.any(dim=1)
    w = torch.ones(rows, dtype=torch.float64, device=z.device) if weights is None else weights.double()
    use = some & (w != 0)
    m = z.amax(dim=1)
    s = torch.exp((z - m[:, None]) / t).sum(dim=1)
    ln_q = (z - m[:, None]) / t - torch.log(s)[:, None]
    a = torch.where(there, top.double() / t, -math.inf)
    a = torch.where(some[:, None], a, 0.0)
    ln_p = torch.log_softmax(a, dim=1)
    p = torch.where(there, ln_p.exp(), 0.0)
    at = torch.where(there, indices, 0)
    terms = torch.where(p > 0, p * (torch.where(p > 0, ln_p, 0.0) - ln_q.gather(1, at)), 0.0)
    loss = torch.where(use, w * t * t * terms.sum(dim=1), 0.0)
    q = ln_q.exp()
    target = torch.zeros_like(q).scatter_add_(1, at, p)
    up = torch.ones(1, dtype=torch.float64, device=z.device) if upstream is None else upstream.double()
    gradient = torch.where(use[:, None], (up * w * t).expand(rows)[:, None] * (q - target), 0.0)
    m, s = torch.where(use, m, 0.0), torch.where(use, s, 1.0)
    return loss, m, s, gradient, target, q


def within(got, want, tolerance, what=""):
    """Every element of `got` is within `tolerance` (a tensor or a number) of `want`; NaN and
    infinities are in the same places."""
    got, want = got.double(), want.double()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), what
    fine = torch.isfinite(want)
    assert torch.equal(fine, torch.isfinite(got)), what
    assert torch.equal(got[~fine].nan_to_num(0), want[~fine].nan_to_num(0)), what
    off = torch.where(fine, (got - want).abs(), 0.0)
    limit = tolerance if isinstance(tolerance, torch.Tensor) else torch.full_like(off, tolerance)
    over = off > limit
    if over.any():
        i = int((off / limit.clamp(min=1e-300)).argmax())
        raise AssertionError(f"{what}: {int(over.sum())} of {over.numel()} off, worst at {i}: got "
                             f"{got.reshape(-1)[i]:.9g}, want {want.reshape(-1)[i]:.9g}, "
                             f"tolerance {limit.expand_as(off).reshape(-1)[i]:.3g}")


def padded(values, dtype, pad, offset=0):
    """`values` as a view with rows `pad` elements longer, starting `offset` elements into its storage;
    what lies between the rows is NaN (it must not be read into a result)."""
    shape = values.shape[:-1] + (values.shape[-1] + pad,)
    count = math.prod(shape)
    base = torch.full((count + offset,), math.nan, dtype=torch.float64).to(dtype).to(values.device)
    view = base[offset:].view(shape)[..., :values.shape[-1]]
    view.copy_(values)
    return view
