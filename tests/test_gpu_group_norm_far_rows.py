"""Group norm's statistics where a map begins with rows far from the others, and many rows follow."""
import pytest
import torch

import learn_util as lu

pytestmark = pytest.mark.gpu


def _far_first(n, s, c, dtype, pad, seed):
    """Unit normal values behind a first row of 64 to 4096, as a border or a first token has them."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    base = torch.randn((n, s, c + pad), generator=gen, device="cuda").to(dtype)
    x = base[..., :c]
    far = 2.0 ** torch.randint(6, 13, (n, c), generator=gen, device="cuda")
    x[:, 0] = far.to(dtype)
    return x


def _check(provider, x, groups, first, steps):
    """Rows are summed in blocks about a running mean, the `first` B ones about the far row itself: B - 1 squares D^2
    one by one, B^2 / 2 u D^2 off, less s^2 / B = (B - 1)^2 / B D^2, where s, a sum of B - 1 terms D one by one, is off
    by B / 2 u and its square, the quotient and the product by (B + 3) u; the whole is at least (B - 1) / B D^2.
    Every later block's squares are about a mean that the far row moves by D / B and less, which adds under a tenth.
    The rest (a thread's blocks or rows, threads, channels, chunks, one by one) is `steps` roundings.  r takes half of
    the variance's; the mean is off by steps u of the largest value."""
    _, stats = provider.group_norm(x, groups)
    mean, r = lu.norm_stats(x, groups)
    n, s, c = x.shape
    e = lu.u(torch.float32) * steps
    top = x.abs().amax(dim=1).double().reshape(n, groups, -1).amax(dim=2)
    lu.within(stats[..., 0], mean, e * top, "mean")
    far = first / (first - 1) * (first ** 2 / 2 + (first - 1) ** 2 / first * (first + 3)) * lu.u(torch.float32)
    lu.within(stats[..., 1], r, r * (0.5 * 1.1 * far + e + (e * top * r) ** 2), "r")


@pytest.mark.parametrize("pad", [0, 1])
def test_maps_that_are_read_twice(provider, pad):
    """A group of 2 MB, longer than a cluster's shared memory, and so many maps that a thread takes 512 rows (2048 with
    rows that are not on 16 bytes).  2048 / 16 blocks, at most 4 threads a channel, at most 8 terms a thread and 14
    steps of a tree over 256 channels, ten more for the quotients."""
    _check(provider, _far_first(300, 2048, 256, torch.float32, pad, 1), 1, 16, 128 + 4 + 8 + 14 + 10)


@pytest.mark.parametrize("dtype,channels,pad", [(torch.bfloat16, 64, 1), (torch.bfloat16, 64, 0), (torch.float32, 32, 1)])
@pytest.mark.parametrize("batch", [1, 3])
def test_maps_in_shared_memory(provider, batch, dtype, channels, pad):
    """As long as a cluster holds, a group for each channel: hundreds of rows a thread.  At most 375 rows a thread,
    at most 32 threads a channel in two levels, eight CTAs, ten more for the quotients; half of it for r."""
    _check(provider, _far_first(batch, 12000, channels, dtype, pad, 2), channels, 32, (375 + 32 + 8 + 10) / 2)
