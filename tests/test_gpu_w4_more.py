"""proj_w4 in the forms and at the values that tests/test_gpu_w4.py does not reach, against the formula
in float64 with its bounds."""

import pytest
import torch

from tests.test_gpu_w4 import BF16, _check, _weight, _x
from wkvm_amd import W4Weight, proj_w4

pytestmark = pytest.mark.gpu


def _on(dev, parts, group):
    return W4Weight.from_codes(*(None if t is None else t.to(dev) for t in parts), group=group)


@pytest.mark.parametrize("group", [64, 128])
@pytest.mark.parametrize("m", [33, 64])
def test_some_tens_of_rows_in_tiles_of_64_columns_at_most_one_a_unit(dev, m, group):
    """Three products whose tiles of 32 columns are more than the units and of 64 are not."""
    gen = torch.Generator().manual_seed(m + group)
    n, k, units = 2001, 416, torch.cuda.get_device_properties(dev).multi_processor_count
    rows = -(-m // 32)
    assert 3 * rows * -(-n // 32) > units >= 3 * rows * -(-n // 64)
    x = _x(gen, m, k)
    parts = [_weight(gen, n, k, group, zero=True) for _ in range(3)]
    bias = torch.randn(n, generator=gen).to(BF16)
    ys = proj_w4([(x.to(dev), _on(dev, p, group), bias.to(dev), "tanh") for p in parts])
    for y, p in zip(ys, parts):
        _check(y, x, p, group, bias, "tanh")


def test_a_new_weight_is_zero(dev):
    weight = W4Weight(70, 96, 32, dev)
    bias = torch.randn(70, device=dev).to(BF16)
    assert not weight.dequantize().any()
    for m in (1, 20, 200):
        y, = proj_w4([(torch.randn(m, 96, device=dev).to(BF16), weight, bias)])
        assert torch.equal(y, bias.expand(m, 70))
