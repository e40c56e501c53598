"""The loss of rows whose logits share a large offset: only differences from the maximum count."""
import math

import pytest
import torch

import learn_util as lu
from gpu_util import status_word
from test_gpu_distill import _data
from test_gpu_distill_range import _check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("vocab,k", [(900, 16), (3000, 300), (70001, 40)])
@pytest.mark.parametrize("offset", [1e6, -1e10, 1e13])
def test_a_large_offset_in_binary64(provider, offset, vocab, k):
    z, at, top, gen = _data((5, vocab, k), torch.float64, 31)
    z = (z * 64).round() / 64 + offset
    _check(provider, z, at, top, 1.0, torch.float64)
    _check(provider, z, at.flip(1), top, 2.5, torch.float64)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("vocab,k", [(900, 16), (70001, 300)])
@pytest.mark.parametrize("value", [-1e10, 1e12, -1e15, -1e20, 1e30, -1e30])
def test_rows_of_one_far_value(provider, value, vocab, k, dtype):
    """Every logit alike (a row that is masked as a whole): q is uniform."""
    z, at, top, gen = _data((3, vocab, k), dtype, 32)
    z[:] = value
    _check(provider, z, at, top, 1.0, dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float64])
@pytest.mark.parametrize("named", [1, 32, 256, 300])
def test_named_entries_that_are_masked(provider, named, dtype):
    """The first `named` entries of the teacher, whole warps' shares among them, are masked in the student: the loss
    is infinite, and the only fault is that."""
    z, at, top, gen = _data((3, 5000, 300), dtype, 33)
    z[1, at[1, :named]] = -math.inf
    status = provider.new_status()
    loss, stats, gradient = provider.distill_loss_step(z, at, top, status=status)
    assert provider.decode_status(status_word(status)) == (1, 3)
    assert float(loss[1]) == math.inf and bool(torch.isfinite(loss[[0, 2]]).all()) and bool(torch.isfinite(gradient).all())
    want = lu.distill(z, at, top, 1.0, None, None)
    # each loss is a sum of 300 terms in binary64, rounded once, and ln s (see the other file's tolerances)
    e = lu.u(dtype)
    near = 2.0 ** -22 if dtype == torch.float32 else 2.0 ** -50
    limit = near + (72 + lu.chain(5000) + 8) * e + 64 * 2.0 ** -50 + 4 * e * want[0][[0, 2]].abs()
    lu.within(loss[[0, 2]], want[0][[0, 2]], limit)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float64])
@pytest.mark.parametrize("k", [255, 257, 1023, 1024])
@pytest.mark.parametrize("vocab", [1500, 131071])
def test_loss_of_many_entries_with_the_gradient_in_place(provider, vocab, k, dtype):
    """Named logits lie in other blocks' slices, which the gradient overwrites: the same bits as apart."""
    z, at, top, gen = _data((6, vocab, k), dtype, 34)
    want = provider.distill_loss_step(z, at, top, temperature=1.5)
    _check(provider, z, at, top, 1.5, dtype)
    for _ in range(5):
        a = z.clone()
        got = provider.distill_loss_step(a, at, top, temperature=1.5, gradient=a)
        assert all(torch.equal(x, y) for x, y in zip(got, want))
