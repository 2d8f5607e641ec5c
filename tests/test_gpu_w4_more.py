"""proj_w4 in the forms and at the values that tests/test_gpu_w4.py does not reach, against the formula
in float64 with its bounds."""

import pytest
import torch

from tests.test_gpu_w4 import BF16
from wkvm_amd import W4Weight, proj_w4

pytestmark = pytest.mark.gpu


def test_a_new_weight_is_zero(dev):
    weight = W4Weight(70, 96, 32, dev)
    bias = torch.randn(70, device=dev).to(BF16)
    assert not weight.dequantize().any()
    for m in (1, 20, 200):
        y, = proj_w4([(torch.randn(m, 96, device=dev).to(BF16), weight, bias)])
        assert torch.equal(y, bias.expand(m, 70))
