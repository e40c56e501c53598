"""Distillation where logits divided by the temperature are large: masks of finite values, far maxima, low
temperatures."""
import math

import pytest
import torch

import learn_util as lu
from gpu_util import status_word
from test_gpu_distill import _data, _tolerances

pytestmark = pytest.mark.gpu


def _check(provider, z, at, top, t, dtype):
    """Loss, backward and step against the 64-bit form.  In binary64 a loss of large terms needs more than the other
    tests' tolerance: each p_j is off by (|a| + 8) 2^-53 relative, a = top / T, in the kernel and in the plain form, and
    so is its term p_j (ln p_j - ln q_j); a sum of k such terms adds (k - 1) 2^-53 of their magnitudes on either side,
    a term's own two differences, quotient and product 4 2^-53."""
    want = lu.distill(z, at, top, t, None, None)
    t_loss, rel_s, t_grad = _tolerances(z, top, t, want, None, None, dtype)
    if dtype == torch.float64:
        p = torch.softmax(top / t, dim=1)
        ln_q = ((z - want[1][:, None]) / t).gather(1, at) - torch.log(want[2])[:, None]
        terms = t * t * (p * (torch.log(p.clamp(min=1e-300)) - ln_q).abs()).sum(dim=1)
        t_loss = t_loss + terms * 2 * (float(top.abs().amax()) / t + 8 + at.shape[1] + 4) * 2.0 ** -53
    status = provider.new_status()
    loss, stats = provider.distill_loss(z, at, top, temperature=t, status=status)
    lu.within(loss, want[0], t_loss, "loss")
    assert torch.equal(stats[:, 0].double(), want[1])
    lu.within(stats[:, 1], want[2], rel_s * want[2], "sum")
    gradient = provider.distill_loss_backward(z, at, top, stats, temperature=t, status=status)
    lu.within(gradient, want[3], t_grad, "gradient")
    loss2, stats2, gradient2 = provider.distill_loss_step(z, at, top, temperature=t, status=status)
    assert torch.equal(loss, loss2) and torch.equal(stats, stats2) and torch.equal(gradient, gradient2)
    assert status_word(status) == provider.STATUS_OK


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float64])
@pytest.mark.parametrize("vocab", [1000, 9000, 70001])
@pytest.mark.parametrize("mask", [-1e9, -1e10, -1e12, -1e15, -1e20, -1e25, -1e30])
def test_rows_masked_with_a_finite_value(provider, mask, vocab, dtype):
    """Masked but for what the teacher names; but for the last, the first, a middle run of ten (masked pieces before
    real ones, threads and CTAs that meet nothing else); every other piece of 64."""
    z, at, top, gen = _data((5, vocab, 12), dtype, 21)
    real = torch.zeros((5, vocab), dtype=torch.bool, device="cuda")
    real[0, at[0]] = True
    real[1, vocab - 10:] = True
    real[2, :10] = True
    real[3, vocab // 2:vocab // 2 + 10] = True
    real[4] = torch.arange(vocab, device="cuda") // 64 % 2 == 1
    z = torch.where(real, z, mask)
    at[1] = vocab - 1 - torch.arange(12, device="cuda") % 10  # entries that are there, some of them twice
    at[2] = torch.arange(12, device="cuda") % 10
    at[3] = vocab // 2 + torch.arange(12, device="cuda") % 10
    _check(provider, z, at, top, 1.0, dtype)
    if dtype != torch.float64:
        _check(provider, z, at, top, 1e-3, dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("vocab", [1000, 70001])
@pytest.mark.parametrize("far", [1e8, 1e10, 1e13, 1e20])
def test_a_far_maximum(provider, far, vocab, dtype):
    """One logit far above all others, named by the teacher or not; the loss of the others is its distance."""
    z, at, top, gen = _data((4, vocab, 12), dtype, 22)
    z[0, at[0, 3]] = far
    z[1, (at[1].max() + 1) % vocab] = far
    z[2, vocab - 1] = far
    z[3, 0] = far
    _check(provider, z, at, top, 1.0, dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("vocab", [1000, 70001])
@pytest.mark.parametrize("t", [1e-6, 1e-8, 1e-9, 1e-10, 1e-12, 1e-20])
def test_low_temperatures(provider, t, vocab, dtype):
    z, at, top, gen = _data((6, vocab, 5), dtype, 23)
    _check(provider, z, at, top, t, dtype)


@pytest.mark.parametrize("step", [2.0 ** 20, 2.0 ** 22, 2.0 ** 24, 2.0 ** 25])
def test_maxima_on_both_sides_of_the_cut_over(provider, step):
    """A thread's running maximum rises past the place where differences are taken first, by less than the
    terms' range: log2 of the terms, logit / T / ln 2, goes up through `step`, and from below -step to above."""
    vocab, t = 40000, 0.5
    gen = torch.Generator().manual_seed(24)
    rise = torch.arange(vocab) / vocab * 8 - 4 + torch.rand(vocab, generator=gen)
    z = torch.stack([step * t * math.log(2) + rise, -step * t * math.log(2) + rise, rise.flip(0) + step * t * math.log(2),
                     rise.flip(0) - step * t * math.log(2)]).float().cuda()
    top, at = z.topk(9, dim=1)
    _check(provider, z, at, top * 0.5, t, torch.float32)
