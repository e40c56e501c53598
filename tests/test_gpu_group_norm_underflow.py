"""Activations of group norm at the end of binary32: 1 / (1 + exp(-z)) and the normal density are 0 below 2^-126, what
is made of them underflows gradually."""
import math

import pytest
import torch

import learn_util as lu

pytestmark = pytest.mark.gpu

NORMAL, SMALLEST = 2.0 ** -126, 2.0 ** -149


def _at(z):
    """Arguments that make z the input of the activation: weight 0, bias z."""
    c = z.numel()
    x = torch.randn((1, 1, c), generator=torch.Generator().manual_seed(1)).cuda()
    return x, torch.zeros(c, device="cuda"), z.float().cuda()


def _values(name):
    low = -110.0 if name == "silu" else -15.0
    return torch.cat([torch.linspace(low, 4.0, 1021), torch.tensor([-89.0, -88.7, -88.0, -87.5, -87.3, -80.0, -13.3, -13.1,
                                                                    -1e4, -1e30, 1e4, 0.0, 200.0])])


@pytest.mark.parametrize("channels", [1032, 1033])
@pytest.mark.parametrize("name", ["silu", "gelu"])
def test_forward(provider, name, channels):
    """exp(-z) and erfc round their argument (|z| u and z^2 u relative to the result, twice that here) and add a few
    units.  A quotient that is 0 below 2^-126 is off by that, times |z|; erfc is not: steps of 2^-149, times |z|."""
    z = _values(name)[:channels].float().double().cuda()
    x, w, b = _at(z)
    out, _ = provider.group_norm(x, 1, w, b, activation=name)
    want = lu.act(z, name)
    u = 2.0 ** -24
    size = z.abs() if name == "silu" else 2 * z * z
    lost = NORMAL if name == "silu" else SMALLEST
    lu.within(out.reshape(-1), want, want.abs() * u * (2 * size.clamp(max=250) + 16) + lost * (2 + z.abs().clamp(max=110)), name)


@pytest.mark.parametrize("name", ["silu", "gelu"])
def test_slope(provider, name):
    """dbias of one position with an upstream of 2^40 is the slope times it, which takes it away from binary32's end.
    SiLU's q (1 + z (1 - q)) and GELU's Phi(z) + z phi(z) lose a q or phi below 2^-126, times 1 + |z|."""
    z = _values(name).float().double().cuda()
    x, w, b = _at(z)
    up = 2.0 ** 40
    dy = torch.full_like(x, up)
    _, stats = provider.group_norm(x, 1, w, b, activation=name)
    _, _, dbias = provider.group_norm_backward(x, dy, 1, stats, w, b, activation=name)
    want = lu.act_slope(z, name)
    u = 2.0 ** -24
    if name == "silu":
        size = torch.sigmoid(z) * (1 + z.abs())
        off = 2 * z.abs().clamp(max=250) + 16
    else:
        size = 0.5 * torch.erfc(-z / math.sqrt(2)) + z.abs() * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
        off = 4 * (z * z).clamp(max=500) + 16
    lu.within(dbias, want * up, up * (size * u * off + NORMAL * (2 + z.abs().clamp(max=110))), name)


def test_binary64_is_gradual_down_to_its_exponents_end(provider):
    """exp(-z) overflows from z = -709.8 on; before that z / (1 + exp(-z)) is right, subnormal results among them."""
    z = torch.linspace(-709.7, 5.0, 400, dtype=torch.float64).cuda()
    x = torch.randn((1, 1, 400), generator=torch.Generator().manual_seed(2), dtype=torch.float64).cuda()
    out, _ = provider.group_norm(x, 1, torch.zeros(400, dtype=torch.float64, device="cuda"), z, activation="silu")
    want = z / (1 + torch.exp(-z))
    lu.within(out.reshape(-1), want, want.abs() * 2.0 ** -50 + 2.0 ** -1074 * (2 + z.abs()))
