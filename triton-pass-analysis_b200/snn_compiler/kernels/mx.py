"""Microscaled 4- and 8-bit operators (no counterpart in the reference): quantisation, the product
with 4-bit weights, and the RMS norm that feeds it.

A microscaled tensor holds blocks of 32 values along its last axis, each with one power-of-two
scale: ``"mxfp4"`` has E2M1 elements (magnitudes 0, .5, 1, 1.5, 2, 3, 4, 6), ``"mxfp8"`` E4M3.
Spikes {0, 1} are exact in either.

  mx_quantize(x, fmt) -> MXTensor                        a value to its nearest code
  mx_dequantize(t, dtype) -> tensor                      the values that the codes stand for
  mx_linear(a, w, bias, dtype=...) -> tensor             a w^T + bias, float32 sums, w in mxfp4
  rms_norm_mx(x, weight, residual, ...) -> MXTensor, h   norm of h = x + residual, quantised

Each call is one launch of libsnnb200.so on the current stream of its input's device.
"""
from __future__ import annotations

import math

import torch

from .. import _lib

FORMATS = {"mxfp4": 0, "mxfp8": 1}
_ROW_BLOCK_BYTES = {"mxfp4": 16, "mxfp8": 32}


def _blocks(K: int) -> int:
    return (K + 31) // 32


def mx_scales_shape(rows: int, K: int) -> tuple:
    """Shape of the scale bytes of a tensor [rows, K]: the byte of row 128 i + 32 c + l, block
    4 j + b is scales[i, j, l, c, b]."""
    return ((rows + 127) // 128, (_blocks(K) + 3) // 4, 32, 4, 4)


class MXTensor:
    """Codes and scales of a tensor of `shape` (any leading axes, flattened to rows):
    data uint8 [rows, 16 ceil(K/32)] (mxfp4, the even element in the low four bits) or
    [rows, 32 ceil(K/32)] (mxfp8), scales uint8 of mx_scales_shape(rows, K).  Elements past K and
    scale bytes that no block owns are zero."""

    __slots__ = ("data", "scales", "shape", "fmt", "rows")

    def __init__(self, data: torch.Tensor, scales: torch.Tensor, shape, fmt: str):
        if fmt not in FORMATS:
            raise ValueError(f"unknown microscaled format {fmt!r} (one of {sorted(FORMATS)})")
        shape = tuple(shape)
        K = shape[-1]
        rows = math.prod(shape[:-1])
        nb = _blocks(K)
        assert K >= 1, shape
        assert data.dtype == torch.uint8 and data.is_contiguous() and \
            data.numel() == rows * nb * _ROW_BLOCK_BYTES[fmt], (tuple(data.shape), shape, fmt)
        assert scales.dtype == torch.uint8 and scales.is_contiguous() and \
            scales.numel() == (rows + 127) // 128 * ((nb + 3) // 4) * 512, \
            (tuple(scales.shape), shape)
        assert data.device == scales.device
        self.data, self.scales, self.shape, self.fmt, self.rows = data, scales, shape, fmt, rows

    @property
    def device(self):
        return self.data.device

    @classmethod
    def from_rows(cls, data: torch.Tensor, row_scales: torch.Tensor, K: int, fmt: str):
        """From codes [rows, ...] and row-major scale bytes [rows, ceil(K/32)] (uint8), the form
        in which checkpoints hold them; the scales are laid out once."""
        rows, nb = row_scales.shape
        assert row_scales.dtype == torch.uint8 and nb == _blocks(K), (tuple(row_scales.shape), K)
        tr, tb = mx_scales_shape(rows, K)[:2]
        full = torch.zeros(tr * 128, tb * 4, dtype=torch.uint8, device=row_scales.device)
        full[:rows, :nb] = row_scales
        tiled = full.view(tr, 4, 32, tb, 4).permute(0, 3, 2, 1, 4).contiguous()
        return cls(data.contiguous(), tiled, (rows, K), fmt)

    def row_scales(self) -> torch.Tensor:
        """The scale bytes row-major, [rows, ceil(K/32)]."""
        nb = _blocks(self.shape[-1])
        tr, tb = mx_scales_shape(self.rows, self.shape[-1])[:2]
        s = self.scales.view(tr, tb, 32, 4, 4).permute(0, 3, 2, 1, 4)
        return s.reshape(tr * 128, tb * 4)[:self.rows, :nb].contiguous()

    def to(self, device) -> "MXTensor":
        return MXTensor(self.data.to(device), self.scales.to(device), self.shape, self.fmt)

    def dequantize(self, dtype=torch.bfloat16) -> torch.Tensor:
        return mx_dequantize(self, dtype)


def _rows_of(x: torch.Tensor):
    """(x as [rows, K] with unit column stride, its row stride): a view where x has one."""
    if x.dim() != 2:
        x = x.reshape(-1, x.shape[-1])
    if x.stride(1) != 1 and x.shape[1] > 1:
        x = x.contiguous()
    return x, x.stride(0)


def _empty(rows: int, K: int, fmt: str, device):
    nb = _blocks(K)
    data = torch.empty(rows, nb * _ROW_BLOCK_BYTES[fmt], dtype=torch.uint8, device=device)
    scales = torch.empty(mx_scales_shape(rows, K), dtype=torch.uint8, device=device)
    return data, scales


def _on_device(fn):
    """Runs fn on the device of its first argument, as its launches go to the current device."""
    def call(x, *args, **kw):
        dev = x.device
        assert dev.type == "cuda", f"a CUDA tensor is needed, got {dev}"
        if dev.index == torch.cuda.current_device():
            return fn(x, *args, **kw)
        with torch.cuda.device(dev):
            return fn(x, *args, **kw)
    call.__name__, call.__doc__, call.__wrapped__ = fn.__name__, fn.__doc__, fn
    return call


def _fmt(fmt):
    if fmt not in FORMATS:
        raise ValueError(f"unknown microscaled format {fmt!r} (one of {sorted(FORMATS)})")
    return FORMATS[fmt]


@_on_device
def mx_quantize(x: torch.Tensor, fmt: str = "mxfp4") -> MXTensor:
    """x [..., K] float32 / float16 / bfloat16 -> MXTensor.  A block's scale is
    2^(floor(log2(largest magnitude)) - 2) (- 8 for mxfp8), its elements are rounded to the
    nearest, ties to even, and clamped to the largest element; a block that holds an infinity or
    a NaN becomes NaN.  Rows may be strided (a slice of a wider tensor) without a copy."""
    code = _fmt(fmt)
    assert x.dim() >= 1 and x.dtype in (torch.float32, torch.float16, torch.bfloat16), x.dtype
    shape = x.shape
    if shape[-1] < 1:
        raise ValueError("mx_quantize: the last axis is empty")
    K = shape[-1]
    x2, ld = _rows_of(x)
    rows = x2.shape[0]
    data, scales = _empty(rows, K, fmt, x.device)
    st = _lib.lib().snnb_mx_quantize(x2.data_ptr(), _lib.dtype_code(x.dtype), rows, K, ld, code,
                                     data.data_ptr(), scales.data_ptr(), _lib.stream_of(x))
    _lib.check(st, "snnb_mx_quantize")
    return MXTensor(data, scales, shape, fmt)


@_on_device
def mx_dequantize(t: MXTensor, dtype=torch.bfloat16) -> torch.Tensor:
    """The values that t's codes stand for, rounded once to dtype (bfloat16 holds them all)."""
    K = t.shape[-1]
    out = torch.empty(t.shape, dtype=dtype, device=t.device)
    st = _lib.lib().snnb_mx_dequantize(t.data.data_ptr(), t.scales.data_ptr(), FORMATS[t.fmt],
                                       t.rows, K, out.data_ptr(), _lib.dtype_code(dtype),
                                       _lib.stream_of(t.data))
    _lib.check(st, "snnb_mx_dequantize")
    return out


@_on_device
def mx_linear(a: MXTensor, w: MXTensor, bias: torch.Tensor | None = None, *,
              dtype=torch.bfloat16, out: torch.Tensor | None = None) -> torch.Tensor:
    """a [..., K] (mxfp4 or mxfp8) times w [N, K]^T (mxfp4) + bias [N] (float32) -> [..., N] of
    dtype (or of `out`): products and sums in float32, rounded once."""
    if w.fmt != "mxfp4":
        raise ValueError(f"mx_linear: the weights are held in mxfp4, got {w.fmt}")
    assert len(w.shape) == 2 and a.shape[-1] == w.shape[1], (a.shape, w.shape)
    assert w.device == a.device
    N, K = w.shape
    if N < 1:
        raise ValueError("mx_linear: no output features")
    if bias is not None:
        assert bias.dtype == torch.float32 and bias.is_contiguous() and \
            bias.numel() == N and bias.device == a.device, tuple(bias.shape)
    shape = (*a.shape[:-1], N)
    if out is None:
        out = torch.empty(shape, dtype=dtype, device=a.device)
    else:
        assert out.device == a.device and out.is_contiguous() and tuple(out.shape) == shape
        dtype = out.dtype
    if dtype == torch.uint8:
        raise AssertionError("mx_linear: out is float32, float16 or bfloat16")
    st = _lib.lib().snnb_mx_linear(a.data.data_ptr(), a.scales.data_ptr(), FORMATS[a.fmt], a.rows,
                                   K, w.data.data_ptr(), w.scales.data_ptr(), N,
                                   None if bias is None else bias.data_ptr(), out.data_ptr(),
                                   _lib.dtype_code(dtype), _lib.stream_of(a.data))
    _lib.check(st, "snnb_mx_linear")
    return out


@_on_device
def rms_norm_mx(x: torch.Tensor, weight: torch.Tensor, residual: torch.Tensor | None = None, *,
                eps: float = 1e-6, fmt: str = "mxfp8"):
    """h = x + residual; (h / sqrt(mean(h^2) + eps)) * weight over the last axis, quantised to
    `fmt` -> (MXTensor, h).  The sum and the norm are float32; the returned h, the next residual,
    is rounded to x's dtype (x itself without a residual).  weight [K] of x's dtype or float32."""
    code = _fmt(fmt)
    assert x.dim() >= 1 and x.dtype in (torch.float32, torch.float16, torch.bfloat16), x.dtype
    shape = x.shape
    K = shape[-1]
    if K < 1:
        raise ValueError("rms_norm_mx: the last axis is empty")
    assert weight.dtype in (x.dtype, torch.float32) and weight.is_contiguous() and \
        weight.numel() == K and weight.device == x.device, (tuple(weight.shape), weight.dtype)
    x2, ldx = _rows_of(x)
    rows = x2.shape[0]
    r2, ldr, h = None, 0, x
    if residual is not None:
        assert residual.shape == shape and residual.dtype == x.dtype and \
            residual.device == x.device, (tuple(residual.shape), residual.dtype)
        r2, ldr = _rows_of(residual)
        h = torch.empty(shape, dtype=x.dtype, device=x.device)
    data, scales = _empty(rows, K, fmt, x.device)
    st = _lib.lib().snnb_rms_norm_mx(
        x2.data_ptr(), ldx, None if r2 is None else r2.data_ptr(), ldr, _lib.dtype_code(x.dtype),
        weight.data_ptr(), _lib.dtype_code(weight.dtype), float(eps), rows, K, code,
        data.data_ptr(), scales.data_ptr(), None if r2 is None else h.data_ptr(),
        _lib.stream_of(x))
    _lib.check(st, "snnb_rms_norm_mx")
    return MXTensor(data, scales, shape, fmt), h
