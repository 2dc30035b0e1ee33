"""The operators in 8 bits without a GPU: what the C entry points refuse, the packed order of a weight,
and that nothing computes on the CPU."""

import ctypes

import pytest
import torch


@pytest.fixture(scope="module")
def lib():
    from mamba3_siso_tpu_amd import _lib

    return _lib


@pytest.fixture(scope="module")
def T(m3):
    return m3.eightbit


def refused(lib, fn, a, text):
    assert fn(ctypes.byref(a), None) == lib.ERR_INVALID
    assert text in lib.load().m3s_last_error(), lib.load().m3s_last_error()


def test_rows8_arguments_are_checked_without_a_launch(lib):
    h = lib.load()
    assert h.m3s_rows8(None, None) == lib.ERR_INVALID
    a = lib.Rows8Args()
    a.struct_size = 8
    refused(lib, h.m3s_rows8, a, b"struct_size")
    a.struct_size = ctypes.sizeof(lib.Rows8Args)
    a.x_dtype, a.width, a.rows, a.ldx = 2, 64, 4, 64
    refused(lib, h.m3s_rows8, a, b"x_dtype")
    a.x_dtype = lib.DTYPE_BF16
    for rows, width in ((-1, 64), (lib.ROWS8_MAX + 1, 64), (4, 0), (4, lib.ROWS8_WIDTH_MAX + 1)):
        a.rows, a.width = rows, width
        refused(lib, h.m3s_rows8, a, b"out of range")
    a.rows, a.width, a.gain = 4, lib.ROWS8_NORM_MAX + 1, 0x1000
    refused(lib, h.m3s_rows8, a, b"norm")
    a.width, a.gain = 64, None
    refused(lib, h.m3s_rows8, a, b"NULL")
    a.x, a.values, a.scales = 0x1000, 0x2000, 0x3000
    a.add, a.ldadd = 0x4000, 64
    refused(lib, h.m3s_rows8, a, b"both add and sum")
    a.sum = 0x5000
    refused(lib, h.m3s_rows8, a, b"with a gain")
    a.gain, a.ldadd = 0x6000, 63
    refused(lib, h.m3s_rows8, a, b"stride")
    a.ldadd, a.ldx = 64, 63
    refused(lib, h.m3s_rows8, a, b"stride")
    a.ldx, a.values = 64, 0x2008
    refused(lib, h.m3s_rows8, a, b"aligned")
    a.rows = 0
    assert h.m3s_rows8(ctypes.byref(a), None) == lib.OK


def test_rows8_values_arguments_are_checked_without_a_launch(lib):
    h = lib.load()
    a = lib.Rows8ValuesArgs()
    refused(lib, h.m3s_rows8_values, a, b"struct_size")
    a.struct_size = ctypes.sizeof(lib.Rows8ValuesArgs)
    a.y_dtype, a.width, a.rows = 3, 64, 4
    refused(lib, h.m3s_rows8_values, a, b"y_dtype")
    a.y_dtype, a.width = lib.DTYPE_F32, 0
    refused(lib, h.m3s_rows8_values, a, b"out of range")
    a.width = 64
    refused(lib, h.m3s_rows8_values, a, b"NULL")
    a.values, a.scales, a.y = 0x1001, 0x2000, 0x3000
    refused(lib, h.m3s_rows8_values, a, b"aligned")
    a.rows = 0
    assert h.m3s_rows8_values(ctypes.byref(a), None) == lib.OK


def test_matmul8_arguments_are_checked_without_a_launch(lib):
    h = lib.load()
    assert h.m3s_matmul8(None, None) == lib.ERR_INVALID
    a = lib.Matmul8Args()
    refused(lib, h.m3s_matmul8, a, b"struct_size")
    a.struct_size = ctypes.sizeof(lib.Matmul8Args)
    a.x_dtype, a.k, a.n, a.rows = 3, 64, 48, 4
    refused(lib, h.m3s_matmul8, a, b"x_dtype")
    a.x_dtype, a.activation = lib.DTYPE_ROWS8, 4
    refused(lib, h.m3s_matmul8, a, b"activation")
    a.activation = 0
    for rows, k, n in ((-1, 64, 48), (lib.ROWS8_MAX + 1, 64, 48), (4, 0, 48), (4, 64, 0), (4, lib.ROWS8_WIDTH_MAX + 1, 1)):
        a.rows, a.k, a.n = rows, k, n
        refused(lib, h.m3s_matmul8, a, b"out of range")
    a.rows, a.k, a.n, a.x_dtype = lib.MATMUL8_FLOAT_ROWS + 1, 64, 48, lib.DTYPE_BF16
    refused(lib, h.m3s_matmul8, a, b"floating point")
    a.x_dtype = lib.DTYPE_ROWS8
    refused(lib, h.m3s_matmul8, a, b"NULL")
    a.x, a.x_scales, a.w, a.w_scales = 0x1000, 0x2000, 0x3000, 0x4000
    refused(lib, h.m3s_matmul8, a, b"another y")
    a.gated, a.y_values, a.y_scales, a.residual = 1, 0x5000, 0x6000, 0x7000
    refused(lib, h.m3s_matmul8, a, b"gated")
    a.residual, a.activation = None, 1
    refused(lib, h.m3s_matmul8, a, b"gated")
    a.activation, a.w = 0, 0x3008
    refused(lib, h.m3s_matmul8, a, b"aligned")
    a.w, a.gated, a.y_values, a.y_scales, a.y = 0x3000, 0, None, None, 0x5000
    a.residual, a.ldres = 0x7000, 47
    refused(lib, h.m3s_matmul8, a, b"ldres")
    a.residual, a.ldy = None, 47
    refused(lib, h.m3s_matmul8, a, b"ldy")
    a.ldy, a.x_dtype, a.ldx = 48, lib.DTYPE_F32, 63
    a.rows = 4
    refused(lib, h.m3s_matmul8, a, b"ldx")
    # steps x rows x 4 bytes of scales behind 32-bit offsets
    a.x_dtype, a.rows, a.k = lib.DTYPE_ROWS8, lib.ROWS8_MAX, 1 << 13
    refused(lib, h.m3s_matmul8, a, b"2 GiB")
    a.rows = 0
    assert h.m3s_matmul8(ctypes.byref(a), None) == lib.OK


@pytest.mark.parametrize("n,gated", [(1, False), (64, False), (65, False), (200, False), (1, True), (32, True),
                                     (128, True), (129, True)])
def test_packed_rows_hold_every_column_once(T, n, gated):
    col = T._packed_rows(n, gated)
    assert len(col) == (-(-n // 128) * 256 if gated else -(-n // 64) * 64)
    assert sorted(col[col >= 0].tolist()) == list(range(2 * n if gated else n))
    # lane group g's four rows in tiles t and t + 1 are 8 neighbouring outputs
    c = col.view(-1, 4, 4, 4)
    for t in (0, 2):
        eight = torch.cat([c[0, t], c[0, t + 1]], -1)
        for g in range(4):
            own = eight[g][eight[g] >= 0]
            assert len(own) < 2 or bool((own[1:] - own[:-1] == 1).all())


def test_nothing_runs_on_the_cpu(T):
    x = torch.randn(3, 64)
    for call in (lambda: T.quantize8(x), lambda: T.rms_norm8(x, torch.ones(64), 1e-5), lambda: T.pack8(x)):
        with pytest.raises(ValueError, match="ROCm device"):
            call()
    for bad, what in ((x.half(), "float32 or bf16"), (torch.tensor(1.0), "an axis")):
        with pytest.raises(ValueError, match=what):
            T.quantize8(bad)
    with pytest.raises(ValueError, match="the weight must be"):
        T.pack8(torch.randn(4, 4, 4))


def test_operands_that_are_not_what_they_say(T):
    """Rows and weights put together or cut by hand are refused by their shapes, before a launch could
    read past them."""
    f8, e8 = torch.float8_e4m3fn, torch.float8_e8m0fnu
    x = torch.randn(3, 200)
    w = T.Weight8(torch.zeros(4, 2, 2, 64, 16, dtype=f8), torch.zeros(2, 1, 64, 4, dtype=torch.uint8).view(e8), 200, 64, False)
    g = T.Weight8(torch.zeros(16, 2, 2, 64, 16, dtype=f8), torch.zeros(2, 4, 64, 4, dtype=torch.uint8).view(e8), 200, 128, True)
    r = T.Rows8(torch.zeros(1, 2, 2, 64, 16, dtype=f8), torch.zeros(8, 128, dtype=torch.uint8).view(e8), 200, (3,))
    for good, call in ((w, T.matmul8), (g, T.swiglu8)):
        with pytest.raises(ValueError, match="ROCm device"):
            call(x, good)
        for bad in (good._replace(n=good.n + 65), good._replace(n=1 << 70), good._replace(values=good.values[:, :1]), good._replace(gated=not good.gated),
                    good._replace(scales=good.scales[:1]), good._replace(values=good.values.view(torch.uint8)),
                    good._replace(values=good.values.transpose(0, 1).contiguous().transpose(0, 1)),
                    good._replace(scales=good.scales.view(torch.uint8))):
            with pytest.raises(ValueError, match="dense Weight8"):
                call(x, bad)
        with pytest.raises(ValueError, match="rows of 200"):
            call(x, good._replace(k=300))
        with pytest.raises(ValueError, match="ROCm device"):
            call(r, good)
    with pytest.raises(ValueError, match="ROCm device"):
        r.dequantize()
    for bad in (r._replace(lead=(17,)), r._replace(width=257), r._replace(scales=r.scales[:4]), r._replace(values=r.values.view(torch.uint8))):
        with pytest.raises(ValueError, match="dense Rows8"):
            bad.dequantize()


def test_exports(m3):
    for name in ("Rows8", "Weight8", "quantize8", "rms_norm8", "pack8", "matmul8", "swiglu8"):
        assert getattr(m3, name) is getattr(m3.eightbit, name)


def test_raw_mode_is_not_for_sub_heads(m3):
    """A head width without a scan kernel of its own runs as sub-heads, which have no raw mode."""
    for chunk, n, p in ((64, 64, 128), (128, 128, 128)):
        assert m3.layout.kernel_headdim("bf16", chunk, n, p) == 64
        assert not m3.kernels.raw_forward_ok("bf16", chunk, n, p, n // 4, 128, 2)
