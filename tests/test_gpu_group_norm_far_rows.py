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


def _check(provider, x, groups, steps):
    """Rows are summed in blocks of 16 about a running mean.  The first block's squares, about the far row, are up to
    15 D^2 (120 u D^2 off, as sums of 15 terms one by one) less s^2 / 16 = 14.1 D^2 (15 u relative, s being such a sum,
    211 u D^2), where the whole is at least 15/16 D^2: 353 u.  Every later block's are about a mean that the far row
    moves by D / 16 and less, which adds under a tenth.  The rest (a thread's blocks, threads, channels, chunks, one by
    one) is `steps` roundings.  r takes half of the variance's; the mean is off by steps u of the largest value."""
    _, stats = provider.group_norm(x, groups)
    mean, r = lu.norm_stats(x, groups)
    n, s, c = x.shape
    e = lu.u(torch.float32) * steps
    top = x.abs().amax(dim=1).double().reshape(n, groups, -1).amax(dim=2)
    lu.within(stats[..., 0], mean, e * top, "mean")
    lu.within(stats[..., 1], r, r * (0.5 * 1.1 * 353 * lu.u(torch.float32) + e + (e * top * r) ** 2), "r")


@pytest.mark.parametrize("pad", [0, 1])
def test_maps_that_are_read_twice(provider, pad):
    """A group of 2 MB, longer than a cluster's shared memory, and so many maps that a thread takes 512 rows (2048 with
    rows that are not on 16 bytes).  2048 / 16 blocks, at most 4 threads a channel, at most 8 terms a thread and 14
    steps of a tree over 256 channels, ten more for the quotients."""
    _check(provider, _far_first(300, 2048, 256, torch.float32, pad, 1), 1, 128 + 4 + 8 + 14 + 10)
