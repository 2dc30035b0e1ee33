"""Every form of the products in 8 bits, by the sizes that reach it; bounds as in ``test_gpu_eight.py``."""

import pytest
import torch

from test_gpu_eight import (BF16, F32, HALF8, HALF16, act_of, acts, bounded, large_bound, round8, rounded_weight,
                            scales_of, unpacked, weight)

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


# The forms (``csrc/m3s_tiles8.h``; ``test_tiles8_cpu.py`` holds these sizes to theirs) with whole pieces of 16
# bytes and with odd widths, partial last tiles both ways.
FORMS = {
    "few16": [(16, 515, 1027), (40, 260, 264)],
    "few32": [(300, 515, 1027), (511, 1040, 840)],
    "tiles64": [(256, 1024, 4480), (130, 260, 8200), (300, 300, 4311)],
    "tiles64wide": [(768, 260, 4480), (600, 300, 5803)],
    "tiles128": [(2500, 130, 1544), (1100, 515, 4487)],
}
GATED_FORMS = {   # (rows, k, outputs)
    "few16": [(16, 515, 501), (40, 260, 320)],
    "few32": [(300, 300, 520), (100, 515, 1155)],
    "tiles64": [(300, 300, 2048), (450, 260, 1155)],
    "tiles64wide": [(450, 260, 2816), (900, 515, 1153)],
    "tiles128": [(2500, 130, 776), (3000, 300, 1153)],
}


def float32_bound(xr, wr):
    return (xr.abs() @ wr.abs()) * (xr.shape[1] / 8 + 16) * 2.0 ** -24


def each(forms):
    return [(name, *size) for name, sizes in forms.items() for size in sizes]


@pytest.mark.parametrize("short", [False, True])
@pytest.mark.parametrize("form,rows,k,n", each(FORMS))
def test_epilogues_of_every_form(T, form, rows, k, n, short):
    gen = torch.Generator().manual_seed(rows + k + n)
    x, w = acts(gen, rows, k, BF16).cuda(), weight(gen, k, n).cuda()
    w8, q = T.pack8(w, short_sums=short), T.quantize8(x)
    xr, wr = round8(x.double()), rounded_weight(w)
    want, err = xr @ wr, (large_bound if short else float32_bound)(xr, wr)
    bias, res = torch.randn(n, generator=gen).cuda(), acts(gen, rows, n, BF16).cuda()
    for b, act, r in ((None, None, None), (bias, None, None), (None, None, res), (bias, None, res), (bias, "gelu", res),
                      (None, "silu", None), (bias, "relu", None)):
        full = act_of(act)(want + (0 if b is None else b.double())) + (0 if r is None else r.double())
        # float32 after the sum: an exponential to 2^-20 and a few roundings; an activation stretches by 1.13
        e = 1.13 * err + 2.0 ** -19 * (want.abs() + bias.double().abs() + res.double().abs()) + full.abs() * HALF16 * 1.01
        bounded(T.matmul8(q, w8, bias=b, activation=act, residual=r), full.cpu(), e.cpu(), f"{b is None} {act} {r is None}")


@pytest.mark.parametrize("short", [False, True])
@pytest.mark.parametrize("biased", [False, True])
@pytest.mark.parametrize("form,rows,k,n", each(GATED_FORMS))
def test_gates_of_every_form(T, form, rows, k, n, biased, short):
    gen = torch.Generator().manual_seed(rows + k + n)
    x, w = acts(gen, rows, k, BF16).cuda(), weight(gen, k, 2 * n).cuda()
    bias = torch.randn(2 * n, generator=gen).cuda() if biased else None
    got = T.swiglu8(T.quantize8(x), T.pack8(w, gated=True, short_sums=short), bias)
    assert not bool(unpacked(got)[0].view(torch.uint8)[:, n:].any())
    xr, wr = round8(x.double()), rounded_weight(w)
    h, e = xr @ wr, (large_bound if short else float32_bound)(xr, wr)
    if biased:
        h = h + bias.double()
    v, g = h[:, :n], h[:, n:]
    silu = g * torch.sigmoid(g)
    want = v * silu
    err = e[:, :n] * (silu.abs() + 1.1 * e[:, n:]) + 1.1 * v.abs() * e[:, n:] + 2.0 ** -19 * v.abs() * (silu.abs() + g.abs())
    top = torch.nn.functional.pad(want.abs() + err, (0, -n % 32)).unflatten(-1, (-1, 32)).amax(-1)
    half = torch.maximum((want.abs() + err) * HALF8, scales_of(top.repeat_interleave(32, -1))[:, :n] * 2.0 ** -10)
    bounded(got.dequantize(F32), want.cpu(), (half + err * 1.01 + 1e-30).cpu(), "gate")


@pytest.mark.parametrize("short", [False, True])
def test_outputs_past_the_caches(T, short):
    """Over 32 MB of output, which goes by the L2s: every row, without a residual and with one."""
    rows, k, n = 16400, 128, 1096
    assert rows * n * 2 > 32 << 20
    gen = torch.Generator().manual_seed(7)
    x, w = acts(gen, rows, k, BF16).cuda(), weight(gen, k, n).cuda()
    w8, q = T.pack8(w, short_sums=short), T.quantize8(x)
    xr, wr = round8(x.double()), rounded_weight(w)
    want, err = xr @ wr, (large_bound if short else float32_bound)(xr, wr)
    bias, res = torch.randn(n, generator=gen).cuda(), acts(gen, rows, n, BF16).cuda()
    for b, r in ((None, None), (bias, None), (None, res), (bias, res)):
        full = want + (0 if b is None else b.double()) + (0 if r is None else r.double())
        e = err + 2.0 ** -22 * (bias.double().abs() + res.double().abs()) + full.abs() * HALF16 * 1.01
        bounded(T.matmul8(q, w8, bias=b, residual=r), full.cpu(), e.cpu(), f"{b is None} {r is None}")
