"""The activations of the products in 8 bits, to a bf16 rounding at any argument."""

import math

import pytest
import torch

from test_gpu_eight import BF16, HALF16

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows", [1, 40, 300, 4200])
@pytest.mark.parametrize("n", [64, 65])
@pytest.mark.parametrize("name", ["gelu", "silu"])
def test_far_from_zero(m3, dev, rows, n, name):
    """Sums are the bias alone (rows of zeros), so that arguments are known exactly: from -12 to 12, where
    gelu's 1 + erf has nothing left of its 24 bits beyond -5, and the result is still far above bf16's smallest."""
    T = m3.eightbit
    bias = torch.linspace(-12, 12, n)
    w8 = T.pack8(torch.ones(32, n, device=dev))
    got = T.matmul8(torch.zeros(rows, 32, device=dev, dtype=BF16), w8, bias=bias.to(dev), activation=name).double().cpu()
    v = bias.double()
    want = 0.5 * v * torch.erfc(-v / math.sqrt(2)) if name == "gelu" else v * torch.sigmoid(v)
    # float32 behind the sum: the argument's own rounding is off by 2^-24 relative, by which erfc moves 2 z^2 times as
    # far (z^2 = v^2 / 2 at most 72), and the exponential as |v| of silu; a few ulp of the functions and products
    err = want.abs() * (HALF16 * 1.01 + (v * v + v.abs() + 32) * 2.0 ** -23)
    over = ((got - want).abs() - err)
    assert float(over.max()) <= 0, (float(over.max()), v[over.argmax() % n])
