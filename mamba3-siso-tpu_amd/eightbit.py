"""The language model's rows, weights and products in 8 bits, for serving.

Rows and weights are e4m3 values in blocks of 32 along the axis that a product sums over, each block
with a power of two as its scale: the smallest one (from 2^-126 on) by which the block's largest
magnitude is at most 448, e4m3's largest value (`Rows8`). A weight takes half the memory of bf16 and half
the traffic. Products sum in float32; a weight packed with ``short_sums`` is multiplied by the matrix cores'
own 8-bit form, at twice the rate of bf16 and with sums of fewer bits (`pack8`).

* `quantize8`  -- rows to 8 bits;
* `rms_norm8`  -- the residual's addition and the block norm, its rows in 8 bits;
* `pack8`      -- a projection's weight, rounded and laid out once;
* `matmul8`    -- rows times a packed weight, with bias, activation and residual;
* `swiglu8`    -- the gated MLP's first product and its gate, the rows out in 8 bits.

Each is one launch of ``csrc/m3s_rows8.hip`` or ``csrc/m3s_matmul8.hip`` (`matmul8` and `swiglu8` of
more than a few float rows two), called from C++ (``csrc/m3s_nodes.cpp``) for dense operands of the kernels'
types and from here for others. They take no gradient and refuse operands that need one.
`model.eight_bit_params` makes a model of them.
"""

from __future__ import annotations

import ctypes
from typing import NamedTuple, Optional

import torch

from . import _lib
from . import kernels as K

Tensor = torch.Tensor

#: The width that rows are padded to.
STEP = 128
ACTIVATIONS = {None: 0, "silu": 1, "gelu": 2, "relu": 3}
_FLOATS = (torch.float32, torch.bfloat16)


class Rows8(NamedTuple):
    """Rows in 8 bits, as the products read them: ``values`` (tiles, steps, 2, 64, 16) float8_e4m3fn, a tile
    for 16 rows and a step for 128 of the ``width`` (zeros behind it), whose lane 16 g + r holds 16 values
    of row r; ``scales`` (4 steps, mp) float8_e8m0fnu, the blocks' scales of each row, mp the rows rounded
    up to 128 (``csrc/m3s_eight.h`` has the order of both; rows behind the last may hold anything);
    ``lead``, the shape of the leading axes, whose product is the number of rows."""

    values: Tensor
    scales: Tensor
    width: int
    lead: tuple

    @property
    def shape(self) -> tuple:
        return (*self.lead, self.width)

    def dequantize(self, dtype: torch.dtype = torch.bfloat16) -> Tensor:
        """The values that the 8 bits stand for, (..., width) in float32 or bf16. Both hold them exactly, but for
        float32's last values, which 8 bits hold as 2^128 (an infinity in either), and, in bf16, values of
        a block of the least scale below 2^-130, which it may round (its steps are 2^-133)."""
        if dtype in _FLOATS:
            y = _lib.nodes().rows8_values(self, dtype is torch.bfloat16, K.POISON_OUTPUTS)
            if y is not None:
                return y
        rows = _check_rows8(self, "dequantize")
        K._device_of(self.values, self.scales)
        K.refuse_gradient("dequantize", self.values, self.scales)
        y = K.empty(*self.lead, self.width, device=self.values.device, dtype=dtype)
        a = _lib.Rows8ValuesArgs(ctypes.sizeof(_lib.Rows8ValuesArgs), _lib.dtype_code(dtype), self.width,
                                 rows, self.values.data_ptr(), self.scales.data_ptr(), y.data_ptr())
        _lib.launch(_lib.load().m3s_rows8_values, a, self.values.device, "m3s_rows8_values")
        return y


class Weight8(NamedTuple):
    """A projection's weight (k, n) packed for the products (`pack8`): ``values``
    (tiles, steps, 2, 64, 16) float8_e4m3fn, as of `Rows8` with the outputs for rows, and ``scales`` (steps, tiles / 4, 64, 4) float8_e8m0fnu.
    ``gated``: its columns are value | gate, n of each. ``short_sums``: how its products sum."""

    values: Tensor
    scales: Tensor
    k: int
    n: int
    gated: bool
    short_sums: bool = False

    @property
    def shape(self) -> tuple:
        return (self.k, 2 * self.n if self.gated else self.n)

    @property
    def device(self) -> torch.device:
        return self.values.device


def _padded(n: int, to: int) -> int:
    return (n + to - 1) // to * to


def _check_rows8(x: Rows8, what: str) -> int:
    rows = _count(x.lead)
    if (tuple(x.values.shape), tuple(x.scales.shape)) != _shapes(rows, x.width) or (
            x.values.dtype != torch.float8_e4m3fn or x.scales.dtype != torch.float8_e8m0fnu
            or not x.values.is_contiguous() or not x.scales.is_contiguous()):
        raise ValueError(f"{what}: rows must be dense Rows8 of {rows} x {x.width}")
    return rows


def _check_weight8(w: Weight8, what: str) -> None:
    tiles = _padded(w.n, 128) // 8 if w.gated else _padded(w.n, 64) // 16
    steps = _padded(w.k, STEP) // STEP
    if (tuple(w.values.shape) != (tiles, steps, 2, 64, 16) or tuple(w.scales.shape) != (steps, tiles // 4, 64, 4)
            or w.values.dtype != torch.float8_e4m3fn or w.scales.dtype != torch.float8_e8m0fnu
            or not w.values.is_contiguous() or not w.scales.is_contiguous()):
        raise ValueError(f"{what}: the weight must be a dense Weight8 of {w.shape} (pack8)")


def _shapes(rows: int, width: int) -> tuple:
    steps = _padded(width, STEP) // STEP
    return (_padded(rows, 16) // 16, steps, 2, 64, 16), (4 * steps, _padded(rows, 128))


def _new_rows8(lead: tuple, rows: int, width: int, dev) -> Rows8:
    values, scales = _shapes(rows, width)
    return Rows8(K.empty(*values, device=dev, dtype=torch.float8_e4m3fn),
                 K.empty(*scales, device=dev, dtype=torch.float8_e8m0fnu), width, lead)


def _row_view(x: Tensor) -> Tensor:
    """``x`` (..., width) as (rows, width) with any row stride and unit column stride; a copy where the
    leading axes do not run as one."""
    if x.dim() != 2:
        x = x.reshape(-1, x.shape[-1]) if x.numel() else x.new_empty(_count(x.shape[:-1]), x.shape[-1])
    if (x.shape[1] > 1 and x.stride(1) != 1) or (x.shape[0] > 1 and x.stride(0) < x.shape[1]):
        x = x.contiguous()
    return x


def _count(shape) -> int:
    n = 1
    for s in shape:
        n *= s
    return n


def _row_stride(x: Tensor) -> int:
    return x.stride(0) if x.shape[0] > 1 else x.shape[1]


def _check_sizes(what: str, rows: int, width: int, most: int = _lib.ROWS8_WIDTH_MAX) -> None:
    if not 1 <= width <= most or rows > _lib.ROWS8_MAX:
        raise ValueError(f"{what}: {rows} rows of {width} (at most {_lib.ROWS8_MAX} of 1 to {most})")


def _check_float_rows(x: Tensor, what: str) -> None:
    if x.dtype not in _FLOATS:
        raise ValueError(f"{what}: rows must be float32 or bf16, got {x.dtype}")
    if x.dim() < 1:
        raise ValueError(f"{what}: rows must have an axis, got a scalar")


def quantize8(x: Tensor) -> Rows8:
    """``x`` (..., width) float32 or bf16 as `Rows8`: each value rounded to the nearest e4m3 of its
    block's scale, ties to even. An entry that is not finite becomes NaN and leaves the scale of its
    block to the others. Rows may have any stride between them."""
    done = _lib.nodes().rows8(x, None, 0.0, None, K.POISON_OUTPUTS)
    if done is not None:
        return Rows8._make(done[0])
    _check_float_rows(x, "quantize8")
    dev = K._device_of(x)
    K.refuse_gradient("quantize8", x)
    lead, width = tuple(x.shape[:-1]), x.shape[-1]
    rows = _count(lead)
    _check_sizes("quantize8", rows, width)
    x = _row_view(x)
    out = _new_rows8(lead, rows, width, dev)
    a = _lib.Rows8Args(ctypes.sizeof(_lib.Rows8Args), _lib.dtype_code(x.dtype), width, 0.0, rows,
                       x.data_ptr(), _row_stride(x), None, 0, None, None, out.values.data_ptr(),
                       out.scales.data_ptr())
    _lib.launch(_lib.load().m3s_rows8, a, dev, "m3s_rows8")
    return out


def rms_norm8(x: Tensor, gain: Tensor, eps: float, add: Optional[Tensor] = None):
    """``(s, rows)``: ``s = x + add``, the residual stream ``x`` (..., width) float32 or bf16 after a
    block whose bf16 output is ``add`` (``x`` itself without one), and ``s / sqrt(mean(s^2) + eps) *
    gain`` in 8 bits, with float32 statistics and no rounding before the one to 8 bits. ``s`` is in the
    stream's type. The width is at most 16384."""
    done = _lib.nodes().rows8(x, gain, eps, add, K.POISON_OUTPUTS)
    if done is not None:
        return x if add is None else done[1], Rows8._make(done[0])
    _check_float_rows(x, "rms_norm8")
    lead, width = tuple(x.shape[:-1]), x.shape[-1]
    rows = _count(lead)
    _check_sizes("rms_norm8", rows, width, _lib.ROWS8_NORM_MAX)
    if tuple(gain.shape) != (width,):
        raise ValueError(f"rms_norm8: gain must be ({width},), got {tuple(gain.shape)}")
    if add is not None and (add.dtype != torch.bfloat16 or add.shape != x.shape):
        raise ValueError(f"rms_norm8: add must be bf16 {tuple(x.shape)}, got {add.dtype} {tuple(add.shape)}")
    dev = K._device_of(x, gain, add)
    K.refuse_gradient("rms_norm8", x, gain, add)
    gain = gain.detach()
    if gain.dtype != torch.float32 or not gain.is_contiguous():
        gain = gain.float().contiguous()
    if gain.data_ptr() % 16:
        gain = gain.clone()
    xr = _row_view(x)
    out = _new_rows8(lead, rows, width, dev)
    a = _lib.Rows8Args(ctypes.sizeof(_lib.Rows8Args), _lib.dtype_code(x.dtype), width, eps, rows,
                       xr.data_ptr(), _row_stride(xr), None, 0, gain.data_ptr(), None,
                       out.values.data_ptr(), out.scales.data_ptr())
    s = x
    if add is not None:
        add = _row_view(add)
        s = K.empty(x.shape, device=dev, dtype=x.dtype)
        a.add, a.ldadd, a.sum = add.data_ptr(), _row_stride(add), s.data_ptr()
    _lib.launch(_lib.load().m3s_rows8, a, dev, "m3s_rows8")
    return s, out


def _packed_rows(n: int, gated: bool) -> Tensor:
    """Which column of the weight each packed row holds, -1 behind the last. Four 16-row tiles t are a
    group: row 4 g + i of tile t is output 64 q + 32 (t >> 1) + 8 g + 4 (t & 1) + i of group q, so that
    a lane of the products has 8 neighbouring outputs; gated, the first two tiles are value's
    outputs 32 q + ... and the others gate's."""
    groups = _padded(n, 128) // 32 if gated else _padded(n, 64) // 64
    q, t, g, i = torch.meshgrid(torch.arange(groups), torch.arange(4), torch.arange(4), torch.arange(4),
                                indexing="ij")
    j = 8 * g + 4 * (t & 1) + i
    if gated:
        out = 32 * q + j
        col = torch.where(out < n, out + n * (t >> 1), -1)
    else:
        out = 64 * q + 32 * (t >> 1) + j
        col = torch.where(out < n, out, -1)
    return col.reshape(-1)


def pack8(w: Tensor, gated: bool = False, short_sums: bool = False) -> Weight8:
    """The weight ``w`` (k, n) float32 or bf16 of a projection ``x @ w``, rounded to 8 bits in blocks
    along k (as `quantize8` rounds its columns) and laid out for `matmul8`; with ``gated`` its columns
    are value | gate and it goes to `swiglu8`. Done once, when a model is loaded.

    Products with it sum in float32 (the operands widened to bf16, which holds them). With ``short_sums``
    the matrix cores multiply the 8 bits themselves, at twice that rate, and cut each of 8 neighbouring
    products at 2^-13 of the power of two of the largest of them: 1.3e-5 of a sum over normal values, and
    more of one whose large products cancel."""
    if w.dim() != 2 or w.dtype not in _FLOATS:
        raise ValueError(f"pack8: the weight must be (k, n) float32 or bf16, got {w.dtype} {tuple(w.shape)}")
    k, n = w.shape
    if gated and n % 2:
        raise ValueError(f"pack8: a gated weight has value and gate columns, got {n}")
    n = n // 2 if gated else n
    for size in (k, n):
        if not 1 <= size <= _lib.ROWS8_WIDTH_MAX:
            raise ValueError(f"pack8: a weight of {tuple(w.shape)} (each axis 1 to {_lib.ROWS8_WIDTH_MAX})")
    K._device_of(w)
    w = w.detach()
    col = _packed_rows(n, gated).to(w.device)
    rows = w.t().index_select(0, col.clamp(min=0)).masked_fill_((col < 0).unsqueeze(1), 0.0)
    q = quantize8(rows)
    steps, at = q.values.shape[1], torch.arange(len(col), device=w.device)
    c = q.scales.view(torch.uint8).index_select(1, (at & ~127) + 4 * (at & 31) + (at >> 5 & 3))
    # (step, lane group, group of tiles, tile, row) -> (step, group of tiles, lane, tile)
    c = c.view(steps, 4, -1, 4, 16).permute(0, 2, 1, 4, 3).contiguous()
    return Weight8(q.values, c.view(steps, -1, 64, 4).view(torch.float8_e8m0fnu), k, n, bool(gated),
                   bool(short_sums))


def _operands(x, w: Weight8, bias: Optional[Tensor], what: str):
    """The args struct of a product with its rows, weight and bias filled in, and what it keeps alive."""
    if not isinstance(w, Weight8):
        raise ValueError(f"{what}: the weight must be a Weight8 (pack8)")
    is8 = isinstance(x, Rows8)
    if not is8:
        _check_float_rows(x, what)
    lead, width = tuple(x.shape[:-1]), x.shape[-1]
    if width != w.k:
        raise ValueError(f"{what}: rows of {width} for a weight of {w.shape}")
    _check_weight8(w, what)
    dev = K._device_of(*((x.values, x.scales) if is8 else (x,)), w.values, w.scales, bias)
    K.refuse_gradient(what, None if is8 else x, bias)
    columns = w.shape[1]
    if bias is not None:
        if tuple(bias.shape) != (columns,):
            raise ValueError(f"{what}: bias must be ({columns},), got {tuple(bias.shape)}")
        bias = bias.detach()
        if bias.dtype != torch.float32 or not bias.is_contiguous():
            bias = bias.float().contiguous()
    rows = _count(lead)
    _check_sizes(what, rows, width)
    if not is8 and not _lib.load().m3s_matmul8_takes_floats(rows, w.k, w.n, int(w.gated), _lib.dtype_code(x.dtype)):
        x, is8 = quantize8(x), True
    a = _lib.Matmul8Args()
    a.struct_size = ctypes.sizeof(_lib.Matmul8Args)
    a.k, a.n, a.gated, a.short_sums, a.rows = w.k, w.n, int(w.gated), int(w.short_sums), rows
    if is8:
        _check_rows8(x, what)
        a.x_dtype, a.x, a.x_scales = _lib.DTYPE_ROWS8, x.values.data_ptr(), x.scales.data_ptr()
    else:
        x = _row_view(x)
        a.x_dtype, a.x, a.ldx = _lib.dtype_code(x.dtype), x.data_ptr(), _row_stride(x)
    a.w, a.w_scales, a.bias = w.values.data_ptr(), w.scales.data_ptr(), _lib.ptr(bias)
    return a, dev, lead, rows, (x, bias)


def matmul8(x, w: Weight8, bias: Optional[Tensor] = None, activation: Optional[str] = None,
            residual: Optional[Tensor] = None) -> Tensor:
    """``act(x @ w + bias) + residual`` in bf16, (..., n): ``x`` (..., k) is `Rows8`, or float32 or bf16
    rows, which are rounded to 8 bits first (`quantize8`; a few rows in the same launch); ``bias``
    (n,) float32 or bf16; ``activation`` None, "silu", "gelu" (with erf) or "relu"; ``residual``
    (..., n) bf16, such as a bf16 model's stream. All but the operands in 8 bits is float32 up to the
    one rounding of the result, but for the sums of a weight packed with ``short_sums``. A row with a NaN or
    an infinity comes out NaN, and one with a value that 8 bits hold as 2^128 may come out infinite or NaN."""
    if activation not in ACTIVATIONS:
        raise ValueError(f"matmul8: activation must be one of {list(ACTIVATIONS)}, got {activation!r}")
    y = _lib.nodes().matmul8(x, w, False, ACTIVATIONS[activation], bias, residual, K.POISON_OUTPUTS)
    if y is not None:
        return y
    a, dev, lead, rows, keep = _operands(x, w, bias, "matmul8")
    if w.gated:
        raise ValueError("matmul8: a gated weight goes to swiglu8")
    a.activation = ACTIVATIONS[activation]
    if residual is not None:
        if residual.dtype != torch.bfloat16 or tuple(residual.shape) != (*lead, w.n):
            raise ValueError(f"matmul8: residual must be bf16 {(*lead, w.n)}, got {residual.dtype} "
                             f"{tuple(residual.shape)}")
        K._device_of(w.values, residual)
        K.refuse_gradient("matmul8", residual)
        residual = _row_view(residual)
        a.residual, a.ldres = residual.data_ptr(), _row_stride(residual)
    y = K.empty(*lead, w.n, device=dev, dtype=torch.bfloat16)
    a.y, a.ldy = y.data_ptr(), w.n
    _lib.launch(_lib.load().m3s_matmul8, a, dev, "m3s_matmul8")
    return y


def matmul8_into(x, w: Weight8, stride: int) -> Tensor:
    """`matmul8` without an epilogue into rows of ``stride`` (at least n) elements: a dense
    (rows, stride) buffer whose first n columns are the product and whose others nothing writes."""
    a, dev, _, rows, keep = _operands(x, w, None, "matmul8")
    if w.gated or stride < w.n:
        raise ValueError(f"matmul8: rows of {stride} for a product of {w.shape}")
    y = K.empty(rows, stride, device=dev, dtype=torch.bfloat16)
    a.y, a.ldy = y.data_ptr(), stride
    _lib.launch(_lib.load().m3s_matmul8, a, dev, "m3s_matmul8")
    return y


def swiglu8(x, w: Weight8, bias: Optional[Tensor] = None) -> Rows8:
    """``value * silu(gate)`` of ``value | gate = x @ w + bias`` in 8 bits (..., n), in float32 up to that
    rounding (but for the sums of a weight packed with ``short_sums``): the gated MLP's first product on a
    weight packed with ``gated=True``. ``x`` and ``bias`` (2 n,) as in `matmul8`."""
    done = _lib.nodes().matmul8(x, w, True, 0, bias, None, K.POISON_OUTPUTS)
    if done is not None:
        return Rows8._make(done)
    a, dev, lead, rows, keep = _operands(x, w, bias, "swiglu8")
    if not w.gated:
        raise ValueError("swiglu8: the weight must be packed with gated=True")
    out = _new_rows8(lead, rows, w.n, dev)
    a.y_values, a.y_scales = out.values.data_ptr(), out.scales.data_ptr()
    _lib.launch(_lib.load().m3s_matmul8, a, dev, "m3s_matmul8")
    return out
