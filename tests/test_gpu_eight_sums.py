"""The sums of the products in 8 bits, bit by bit: float32's unless a weight asks for short ones.

Whole numbers say it exactly. Rows and weights hold a pair of 128s in each 32 of the inner dimension, whose
products of 2^14 cancel, and whole numbers of at most 3 elsewhere, which 8 bits hold beside a 128 (the block's
scale is 2^-1, and e4m3 holds whole numbers up to 16). All sums of magnitudes stay below 2^24, so float32 sums
are exact in any order and a product rounds once, to bf16. Cut at 2^-13 of the largest of 8 neighbours, the
other products keep nothing below 2.
"""

import pytest
import torch

from test_gpu_eight import (BF16, F32, HALF8, HALF16, acts, bounded, half_step, large_bound, round8, rounded_weight,
                            same, scales_of, unpacked, weight)

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def T(dev):
    import mamba3_siso_tpu_amd

    return mamba3_siso_tpu_amd.eightbit


def whole_numbers(rows, k, n):
    """(rows, k) and (k, n) as above, float64."""
    gen = torch.Generator().manual_seed(rows + 31 * k + n)
    x = torch.randint(-3, 4, (rows, k), generator=gen).double()
    w = torch.randint(-3, 4, (k, n), generator=gen).double()
    at = torch.arange(0, k - 1, 32)
    pair = at + torch.randint(0, 4, (len(at),), generator=gen) * 8 % (k - 1 - at).clamp(max=32)
    x[:, pair], x[:, pair + 1], w[pair], w[pair + 1] = 128.0, 128.0, 128.0, -128.0
    assert float((x.abs() @ w.abs()).max()) < 2 ** 24
    assert torch.equal(round8(x), x) and torch.equal(rounded_weight(w), w)
    return x, w


# one row to many: 16 and 32 rows to a workgroup, then tiles of 128 x 64, 256 x 64 and 256 x 128 outputs x
# rows, each with whole pieces of 16 bytes and with an odd width
SIZES = [(1, 1024, 4480), (5, 515, 31), (16, 200, 17000), (40, 1024, 264), (100, 777, 333), (300, 515, 1027),
         (256, 1024, 4480), (130, 260, 8200), (600, 300, 1803), (450, 515, 2311), (1100, 520, 2000), (900, 260, 4487),
         (2500, 130, 1544), (4200, 1024, 1031)]


@pytest.mark.parametrize("rows,k,n", SIZES)
def test_products_sum_in_float32(T, rows, k, n):
    x, w = whole_numbers(rows, k, n)
    want = (x @ w).to(BF16).double()
    w8 = T.pack8(w.float().cuda())
    same(T.matmul8(x.to(BF16).cuda(), w8), want, "floats")
    same(T.matmul8(T.quantize8(x.float().cuda()), w8), want, "Rows8")
    res = torch.randint(-100, 101, (rows, n), generator=torch.Generator().manual_seed(n)).to(BF16)
    bias = torch.arange(n, dtype=F32) % 7
    full = torch.relu(x @ w + bias.double()) + res.double()
    same(T.matmul8(x.to(BF16).cuda(), w8, bias.cuda(), "relu", res.cuda()), full.to(BF16).double(), "epilogue")
    same(T.matmul8(x.to(BF16).cuda(), w8, bias.cuda(), None, res.cuda()), (x @ w + bias.double() + res.double()).to(BF16).double(), "plain")


@pytest.mark.parametrize("rows,k,n", [(3, 333, 130), (40, 333, 130), (700, 333, 1100)])
@pytest.mark.parametrize("e,f", [(-118, 118), (118, -118), (-130, 118)])
def test_float32_sums_over_the_scales(T, rows, k, n, e, f):
    """Rows near either end of float32 beside weights near the other one: bf16 holds both, below its normal
    values (from 2^-126) too."""
    x, w = whole_numbers(rows, k, n)
    got = T.matmul8((x * 2.0 ** e).float().cuda(), T.pack8((w * 2.0 ** f).float().cuda()))
    same(got, (x @ w).to(BF16).double() * 2.0 ** (e + f))


GATES = [(1, 2048, 5632), (7, 515, 330), (40, 1000, 320), (300, 300, 2048), (450, 260, 1155), (1100, 520, 1000),
         (2500, 130, 772), (3000, 1500, 1153)]


@pytest.mark.parametrize("rows,k,n", GATES)
def test_gates_of_any_number_of_rows_sum_in_float32(T, rows, k, n):
    """Hardly a value falls to its neighbour: those that lie further than float32's error from a border are
    the definition's, and the others one of the two beside it."""
    gen = torch.Generator().manual_seed(rows + k + n)
    x, w = acts(gen, rows, k, F32).cuda(), weight(gen, k, 2 * n, F32).cuda()
    got = T.swiglu8(T.quantize8(x), T.pack8(w, gated=True)).dequantize(F32).double()
    xr, wr = round8(x.double()), rounded_weight(w)
    h, e = xr @ wr, xr.abs() @ wr.abs() * (k / 8 + 16) * 2.0 ** -24
    v, g = h[:, :n], h[:, n:]
    silu = g * torch.sigmoid(g)
    want = v * silu
    # silu and the product in float32: the exponential's argument is off by |g| 2^-24, five roundings more
    err = 1.01 * (e[:, :n] * (silu.abs() + 1.1 * e[:, n:]) + 1.1 * v.abs() * e[:, n:] + want.abs() * (g.abs() + 8) * 2.0 ** -23) + 1e-30
    lo, hi = round8(want - err), round8(want + err)
    sure = (lo == hi) & (scales_of(want.abs() + err) == scales_of((want.abs() - err).clamp(min=0.0)))
    assert float(sure.double().mean()) > 0.8     # at K = 2048 e is twice that of 1024 rows and borders are as far apart
    same(got[sure], lo[sure].cpu(), "far from a border")
    assert bool(((got - want).abs() <= half_step(want, 0.0) * 2 + err).all())


@pytest.mark.parametrize("rows,n", [(5, 640), (300, 2048), (1100, 1000), (2500, 768)])
def test_a_gate_is_no_function_of_its_batch(T, rows, n):
    """Sums that are exact in any order: a row's 8 bits are the same alone and among others."""
    x, w = whole_numbers(rows, 512, 2 * n)
    x, w = x * 2.0 ** -4, w * 2.0 ** -4     # values around the gate's bend
    w8 = T.pack8(w.float().cuda(), gated=True)
    many, one = T.swiglu8(x.to(BF16).cuda(), w8), T.swiglu8(x[-1:].to(BF16).cuda(), w8)
    same(many.dequantize(F32)[-1:], one.dequantize(F32).double().cpu())


@pytest.mark.parametrize("rows,k,n", SIZES)
def test_short_sums_are_asked_for(T, rows, k, n):
    """A weight of short sums: within the cuts' bound, from the call in C++ and the one in Python alike, and
    not what float32 sums give."""
    gen = torch.Generator().manual_seed(rows + k + n)
    x, w = acts(gen, rows, k, BF16).cuda(), weight(gen, k, n).cuda()
    w8 = T.pack8(w, short_sums=True)
    assert w8.short_sums and not T.pack8(w).short_sums
    xr, wr = round8(x.double()), rounded_weight(w)
    bias, res = torch.randn(n, generator=gen).to(BF16).cuda(), acts(gen, rows, n, BF16).cuda()
    full = xr @ wr + bias.double() + res.double()
    err = large_bound(xr, wr) + 2.0 ** -22 * (bias.double().abs() + res.double().abs()) + full.abs() * HALF16 * 1.01
    got = T.matmul8(x, w8, bias.float(), residual=res)
    bounded(got, full.cpu(), err.cpu(), "short")
    same(T.matmul8(x, w8, bias, residual=res), got.double().cpu(), "a bias of bf16 takes the call in Python")
    x, w = whole_numbers(rows, k, n)
    cut = T.matmul8(x.to(BF16).cuda(), T.pack8(w.float().cuda(), short_sums=True)).double().cpu()
    assert not torch.equal(cut, (x @ w).to(BF16).double())


@pytest.mark.parametrize("rows,k,n", GATES)
def test_gates_of_short_sums(T, rows, k, n):
    gen = torch.Generator().manual_seed(rows + k + n)
    x, w = acts(gen, rows, k, BF16).cuda(), weight(gen, k, 2 * n).cuda()
    got = T.swiglu8(x, T.pack8(w, gated=True, short_sums=True))
    assert not bool(unpacked(got)[0].view(torch.uint8)[:, n:].any())
    xr, wr = round8(x.double()), rounded_weight(w)
    h, cuts = xr @ wr, large_bound(xr, wr)
    v, g = h[:, :n], h[:, n:]
    silu = g * torch.sigmoid(g)
    want = v * silu
    err = cuts[:, :n] * (silu.abs() + 1.1 * cuts[:, n:]) + 1.1 * v.abs() * cuts[:, n:] + 2.0 ** -19 * v.abs() * (silu.abs() + g.abs())
    top = torch.nn.functional.pad(want.abs() + err, (0, -n % 32)).unflatten(-1, (-1, 32)).amax(-1)
    half = torch.maximum((want.abs() + err) * HALF8, scales_of(top.repeat_interleave(32, -1))[:, :n] * 2.0 ** -10)
    bounded(got.dequantize(F32), want.cpu(), (half + err * 1.01 + 1e-30).cpu(), "gate")


def test_a_model_of_short_sums(m3, dev):
    """The choice reaches every projection, and the logits stay those of the same weights in bf16."""
    from test_gpu_eight_model import LOGITS_REL, lm, rel, rounded_params

    cfg, params = lm(m3, BF16)
    p8 = m3.model.eight_bit_params(params, cfg, short_sums=True)
    for b in p8.blocks:
        assert all(w.short_sums for w in (b.siso.in_proj, b.siso.out_proj, b.mlp.fc1, b.mlp.fc2))
    assert not m3.model.eight_bit_params(params, cfg).blocks[0].mlp.fc1.short_sums
    xs = torch.randint(0, 61, (2, 192), generator=torch.Generator().manual_seed(1)).cuda()
    with torch.no_grad():
        assert rel(m3.model.lm_forward(p8, xs, cfg), m3.model.lm_forward(rounded_params(m3, params), xs, cfg)) < LOGITS_REL
        st = m3.model.zero_states(cfg, 2, device=dev)
        for i in range(3):
            y, st = m3.model.lm_decode_step(p8, xs[:, i], st, cfg)
        assert bool(torch.isfinite(y).all())
