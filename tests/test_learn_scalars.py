"""The binary32 patterns of the learning operators' scalar arguments (temperature, eps), on the host."""
import importlib

import numpy as np
import pytest
import torch

learn = importlib.import_module("fusion-pcu_b200.learn")


def test_a_tensor_changed_between_calls():
    tau = torch.tensor(2.0)
    assert learn._bits(tau) == 0x40000000
    tau.mul_(0.5)
    assert learn._bits(tau) == 0x3F800000


@pytest.mark.parametrize("first,second", [(0.0, -0.0), (-0.0, 0.0)])
def test_zeros_of_both_signs(first, second):
    assert [learn._bits(first), learn._bits(second)] == [0x80000000 if str(v)[0] == "-" else 0 for v in (first, second)]


def test_every_kind_of_number():
    for value in (1e-5, 0.1, 2, True, 1e-45, 3.5e38, -1e300, float("nan"), float("inf"), np.float32(0.3), np.float64(0.3),
                  np.array(0.3), torch.tensor(0.3), torch.tensor(0.3, dtype=torch.float64)):
        want = int(np.array([float(value)]).astype(np.float32).view(np.uint32)[0])
        assert learn._bits(value) == want
