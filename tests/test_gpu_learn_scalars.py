"""Scalar arguments of the learning operators' calls are taken anew at each call."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_a_temperature_that_is_changed_in_place(provider):
    gen = torch.Generator().manual_seed(1)
    z = torch.randn((5, 300), generator=gen).cuda()
    top, at = torch.randn((5, 300), generator=gen).cuda().topk(7, dim=1)
    tau = torch.tensor(2.0)
    for value in (2.0, 1.0, 0.5):
        tau.fill_(value)
        loss, stats, gradient = provider.distill_loss_step(z, at, top, temperature=value)
        got, got_stats = provider.distill_loss(z, at, top, temperature=tau)
        assert torch.equal(got, loss)
        assert torch.equal(provider.distill_loss_backward(z, at, top, got_stats, temperature=tau), gradient)
        assert torch.equal(provider.distill_loss_step(z, at, top, temperature=tau)[0], loss)


def test_an_eps_that_is_changed_in_place(provider):
    x = torch.randn((3, 20, 16), generator=torch.Generator().manual_seed(2)).cuda()
    eps = torch.tensor(0.0)
    for value in (0.5, 1e-5, 2.0):
        eps.fill_(value)
        assert torch.equal(provider.group_norm(x, 4, eps=eps)[0], provider.group_norm(x, 4, eps=value)[0])


def test_an_eps_of_zero_after_a_refused_negative_zero(provider):
    x = torch.randn((3, 20, 16), generator=torch.Generator().manual_seed(3)).cuda()
    with pytest.raises(provider.ProviderFailure):
        provider.group_norm(x, 4, eps=-0.0)
    provider.group_norm(x, 4, eps=0.0)
