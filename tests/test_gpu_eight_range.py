"""Rows in 8 bits at the ends of their scales' range, back in float32 and bf16."""

import pytest
import torch

from test_gpu_eight import BF16, F32, round8, same

pytestmark = pytest.mark.gpu


def test_the_least_and_the_largest_scale(m3, dev):
    """Every e4m3 value under the scale 2^-126, down to 2^-135, which float32 holds and bf16 rounds below 2^-133;
    and blocks up to float32's last values, of which 256 2^120 is 2^128."""
    vals = torch.arange(0, 127, dtype=torch.uint8).view(torch.float8_e4m3fn).double()
    x = torch.zeros(2, 128, dtype=torch.float64)
    x[0, :127] = vals * 2.0 ** -126
    x[1, ::32], x[1, 1:32] = 2.0 ** 127, -(2.0 ** 127) * vals[-31:] / 448     # blocks of scale 2^119
    x[1, 33] = 3.4e38                                                         # and one of 2^120
    x[0, 127] = -448 * 2.0 ** -126
    q = m3.quantize8(x.float().to(dev))
    want = round8(x.float().double())
    assert torch.equal(want[0], x[0])
    same(q.dequantize(F32), want, "float32")
    same(q.dequantize(), want, "bf16")
    low = q.dequantize().double().cpu()[0]
    assert not torch.equal(low, want[0]) and torch.equal(low[want[0].abs() >= 2.0 ** -129], want[0][want[0].abs() >= 2.0 ** -129])
    assert bool(torch.isinf(q.dequantize()[1, 33]))
