"""Every form of the products in 8 bits, by the sizes that reach it; bounds as in ``test_gpu_eight.py``."""

import pytest
import torch

from test_gpu_eight import BF16, F32, HALF16, acts, bounded, large_bound, round8, rounded_weight, weight

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def T(dev):
    import mamba3_siso_tpu_amd

    return mamba3_siso_tpu_amd.eightbit


@pytest.mark.parametrize("steps", [1, 2, 3, 4, 5, 6, 7])
def test_inner_dimensions_of_a_few_steps(T, steps):
    """The tiled products' last steps wait for everything: each remainder of the ring of three stages, and
    no turn of the loop at all."""
    k = 128 * steps - 5
    gen = torch.Generator().manual_seed(steps)
    x, w = acts(gen, 1500, k, BF16).cuda(), weight(gen, k, 1100).cuda()
    xr, wr = round8(x.double()), rounded_weight(w)
    want = xr @ wr
    bounded(T.matmul8(x, T.pack8(w)), want.cpu(), (large_bound(xr, wr) + want.abs() * HALF16 * 1.01).cpu(), "product")
