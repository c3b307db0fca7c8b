"""Microscaled 4- and 8-bit operators (no counterpart in the reference): quantisation, the product
with 4-bit weights, and the RMS norm that feeds it.

A microscaled tensor holds blocks of 32 values along its last axis, each with one power-of-two
scale: ``"mxfp4"`` has E2M1 elements (magnitudes 0, .5, 1, 1.5, 2, 3, 4, 6), ``"mxfp8"`` E4M3.
Spikes {0, 1} are exact in either.

  mx_quantize(x, fmt) -> MXTensor                        a value to its nearest code
  mx_dequantize(t, dtype) -> tensor                      the values that the codes stand for
  mx_linear(a, w, bias, dtype=...) -> tensor             a w^T + bias, float32 sums, w in mxfp4
  rms_norm_mx(x, weight, residual, ...) -> MXTensor, h   norm of h = x + residual, quantised

Each call is one launch of libsnnb200.so on the current stream of its input's device.  Waits inside
mx_linear and rms_norm_mx are bounded: one that gives up leaves the output unspecified and is
reported by the device status word (kernels.conv.raise_on_device_status), not by the call.
"""
from __future__ import annotations

import math

import torch

from .. import _lib

FORMATS = {"mxfp4": 0, "mxfp8": 1}
_BLOCK_BYTES = (16, 32)
_DTYPES = {torch.float32: _lib.F32, torch.float16: _lib.F16, torch.bfloat16: _lib.BF16}


def _fmt(fmt: str) -> int:
    code = FORMATS.get(fmt)
    if code is None:
        raise ValueError(f"unknown microscaled format {fmt!r} (one of {sorted(FORMATS)})")
    return code


def _dtype(dtype) -> int:
    code = _DTYPES.get(dtype)
    assert code is not None, f"float32, float16 or bfloat16 is needed, got {dtype}"
    return code


def mx_scales_shape(rows: int, K: int) -> tuple:
    """Shape of the scale bytes of a tensor [rows, K]: the byte of row 128 i + 32 c + l, block
    4 j + b is scales[i, j, l, c, b]."""
    return ((rows + 127) // 128, ((K + 31) // 32 + 3) // 4, 32, 4, 4)


class MXTensor:
    """Codes and scales of a tensor of `shape` (any leading axes, flattened to rows):
    data uint8 [rows, 16 ceil(K/32)] (mxfp4, the even element in the low four bits) or
    [rows, 32 ceil(K/32)] (mxfp8), scales uint8 of mx_scales_shape(rows, K).  Elements past K and
    scale bytes that no block owns are zero."""

    # _data holds the codes, or codes and scales in one allocation (_size: where the scales start,
    # -1 where they lie apart); _parts the two as tensors, once they are known
    __slots__ = ("shape", "fmt", "rows", "_code", "_data", "_size", "_parts")

    def __init__(self, data: torch.Tensor, scales: torch.Tensor, shape, fmt: str):
        code = _fmt(fmt)
        K = shape[-1]
        rows = shape[0] if len(shape) == 2 else math.prod(shape[:-1])
        nb = (K + 31) // 32
        assert K >= 1, shape
        assert data.dtype == scales.dtype == torch.uint8
        assert data.get_device() == scales.get_device()
        assert data.is_contiguous() and data.numel() == rows * nb * _BLOCK_BYTES[code], \
            (tuple(data.shape), tuple(shape), fmt)
        assert scales.is_contiguous() and \
            scales.numel() == (rows + 127) // 128 * ((nb + 3) // 4) * 512, \
            (tuple(scales.shape), tuple(shape))
        self.shape, self.fmt, self.rows = tuple(shape), fmt, rows
        self._code, self._data, self._size, self._parts = code, data, -1, (data, scales)

    @classmethod
    def _new(cls, like: torch.Tensor, rows: int, shape, fmt: str, code: int):
        """Uninitialised, on like's device: codes and scales in one allocation."""
        self = cls.__new__(cls)
        nb = (shape[-1] + 31) // 32
        size = rows * nb * _BLOCK_BYTES[code]
        buf = like.new_empty(size + (rows + 127) // 128 * ((nb + 3) // 4) * 512,
                             dtype=torch.uint8)
        self.shape, self.fmt, self.rows = shape, fmt, rows
        self._code, self._data, self._size, self._parts = code, buf, size, None
        return self

    def _pointers(self):
        """Addresses of the codes and the scales."""
        p = self._data.data_ptr()
        return p, p + self._size if self._size >= 0 else self._parts[1].data_ptr()

    def _split(self):
        """Codes and scales as two tensors.  Set together: other threads see both or neither."""
        parts = self._parts
        if parts is None:
            buf, size, K = self._data, self._size, self.shape[-1]
            scales = buf[size:].view(mx_scales_shape(self.rows, K))
            data = buf[:size].view(self.rows, (K + 31) // 32 * _BLOCK_BYTES[self._code])
            parts = self._parts = (data, scales)
        return parts

    @property
    def device(self) -> torch.device:
        return self._data.device

    @property
    def data(self) -> torch.Tensor:
        return self._split()[0]

    @property
    def scales(self) -> torch.Tensor:
        return self._split()[1]

    @classmethod
    def from_rows(cls, data: torch.Tensor, row_scales: torch.Tensor, K: int, fmt: str):
        """From codes [rows, ...] and row-major scale bytes [rows, ceil(K/32)] (uint8), the form
        in which checkpoints hold them; the scales are laid out once.  Codes past K become zero."""
        _fmt(fmt)
        rows, nb = row_scales.shape
        assert row_scales.dtype == torch.uint8 and nb == (K + 31) // 32, \
            (tuple(row_scales.shape), K)
        tr, tb = mx_scales_shape(rows, K)[:2]
        full = torch.zeros(tr * 128, tb * 4, dtype=torch.uint8, device=row_scales.device)
        full[:rows, :nb] = row_scales
        tiled = full.view(tr, 4, 32, tb, 4).permute(0, 3, 2, 1, 4).contiguous()
        data = data.contiguous()
        if K % 32:
            per_byte = 2 if fmt == "mxfp4" else 1
            used = -(-K // per_byte)                              # bytes of a row that hold codes
            data = data.reshape(rows, nb * 32 // per_byte).clone()
            data[:, used:] = 0
            if K % per_byte:
                data[:, used - 1] &= 15
        return cls(data, tiled, (rows, K), fmt)

    def row_scales(self) -> torch.Tensor:
        """The scale bytes row-major, [rows, ceil(K/32)]."""
        K = self.shape[-1]
        tr, tb = mx_scales_shape(self.rows, K)[:2]
        s = self.scales.view(tr, tb, 32, 4, 4).permute(0, 3, 2, 1, 4)
        return s.reshape(tr * 128, tb * 4)[:self.rows, :(K + 31) // 32].contiguous()

    def to(self, device) -> "MXTensor":
        return MXTensor(self.data.to(device), self.scales.to(device), self.shape, self.fmt)

    def dequantize(self, dtype=torch.bfloat16) -> torch.Tensor:
        return mx_dequantize(self, dtype)


def _rows_of(x: torch.Tensor):
    """(x as [rows, K] with unit column stride, its row stride): a view where x has one."""
    if x.dim() != 2:
        x = x.reshape(-1, x.shape[-1])
    ld, unit = x.stride()
    if unit != 1 and x.shape[1] > 1:
        x = x.contiguous()
        ld = x.stride(0)
    return x, ld


_entries = {}


def _launch(name: str, index: int, *args) -> None:
    """One library call on the current stream of CUDA device `index`, which becomes the current
    device for it (launches go to the current device)."""
    fn = _entries.get(name)
    if fn is None:
        fn = _entries[name] = getattr(_lib.lib(), name)
    if index == torch.cuda.current_device():
        st = fn(*args, _lib.raw_stream(index))
    else:
        with torch.cuda.device(index):
            st = fn(*args, _lib.raw_stream(index))
    if st:
        _lib.check(st, name)


def _index(t: torch.Tensor) -> int:
    index = t.get_device()
    assert index >= 0, f"a CUDA tensor is needed, got {t.device}"
    return index


def mx_quantize(x: torch.Tensor, fmt: str = "mxfp4") -> MXTensor:
    """x [..., K] float32 / float16 / bfloat16 -> MXTensor.  A block's scale is
    2^(floor(log2(largest magnitude)) - 2) (- 8 for mxfp8), its elements are rounded to the
    nearest, ties to even, and clamped to the largest element; a block that holds an infinity or
    a NaN becomes NaN.  Rows may be strided (a slice of a wider tensor) without a copy."""
    code, dt, shape = _fmt(fmt), _dtype(x.dtype), x.shape
    assert len(shape) >= 1, "mx_quantize: x has no axis"
    K = shape[-1]
    if K < 1:
        raise ValueError("mx_quantize: the last axis is empty")
    index = _index(x)
    x2, ld = _rows_of(x)
    rows = x2.shape[0]
    t = MXTensor._new(x, rows, tuple(shape), fmt, code)
    _launch("snnb_mx_quantize", index, x2.data_ptr(), dt, rows, K, ld, code, *t._pointers())
    return t


def mx_dequantize(t: MXTensor, dtype=torch.bfloat16) -> torch.Tensor:
    """The values that t's codes stand for, rounded once to dtype (bfloat16 holds them all but some
    of E4M3's under the scale bytes 0 to 2, which lie below its smallest)."""
    dt = _dtype(dtype)
    index = _index(t._data)
    out = t._data.new_empty(t.shape, dtype=dtype)
    _launch("snnb_mx_dequantize", index, *t._pointers(), t._code, t.rows, t.shape[-1],
            out.data_ptr(), dt)
    return out


def mx_linear(a: MXTensor, w: MXTensor, bias: torch.Tensor | None = None, *,
              dtype=torch.bfloat16, out: torch.Tensor | None = None) -> torch.Tensor:
    """a [..., K] (mxfp4 or mxfp8) times w [N, K]^T (mxfp4) + bias [N] (float32) -> [..., N] of
    dtype (or of `out`): products and sums in float32, rounded once."""
    if w._code != 0:
        raise ValueError(f"mx_linear: the weights are held in mxfp4, got {w.fmt}")
    assert len(w.shape) == 2 and a.shape[-1] == w.shape[1], (a.shape, w.shape)
    N, K = w.shape
    index = _index(a._data)
    assert w._data.get_device() == index, (w.device, a.device)
    if N < 1:
        raise ValueError("mx_linear: no output features")
    if bias is not None:
        assert bias.dtype == torch.float32 and bias.is_contiguous() and \
            bias.numel() == N and bias.get_device() == index, (tuple(bias.shape), bias.dtype)
    shape = a.shape[:-1] + (N,)
    if out is None:
        dt = _dtype(dtype)
        out = a._data.new_empty(shape, dtype=dtype)
    else:
        dt = _dtype(out.dtype)
        assert out.get_device() == index and out.is_contiguous() and tuple(out.shape) == shape
    _launch("snnb_mx_linear", index, *a._pointers(), a._code, a.rows, K, *w._pointers(), N,
            None if bias is None else bias.data_ptr(), out.data_ptr(), dt)
    return out


def rms_norm_mx(x: torch.Tensor, weight: torch.Tensor, residual: torch.Tensor | None = None, *,
                eps: float = 1e-6, fmt: str = "mxfp8"):
    """h = x + residual; (h / sqrt(mean(h^2) + eps)) * weight over the last axis, quantised to
    `fmt` -> (MXTensor, h).  The sum and the norm are held in float32 or more; the returned h, the
    next residual, is rounded to x's dtype (x itself without a residual).  weight [K] of x's dtype or
    float32."""
    code, dt, shape = _fmt(fmt), _dtype(x.dtype), x.shape
    assert len(shape) >= 1, "rms_norm_mx: x has no axis"
    K = shape[-1]
    if K < 1:
        raise ValueError("rms_norm_mx: the last axis is empty")
    if not eps >= 0.0:
        raise ValueError(f"rms_norm_mx: eps is {eps}")
    index, wd = _index(x), weight.dtype
    assert (wd == x.dtype or wd == torch.float32) and weight.is_contiguous() and \
        weight.numel() == K and weight.get_device() == index, (tuple(weight.shape), wd)
    x2, ldx = _rows_of(x)
    rows = x2.shape[0]
    r2, ldr, h, hp = None, 0, x, None
    if residual is not None:
        assert residual.shape == shape and residual.dtype == x.dtype and \
            residual.get_device() == index, (tuple(residual.shape), residual.dtype)
        r2, ldr = _rows_of(residual)
        h = x.new_empty(shape)
        hp = h.data_ptr()
    t = MXTensor._new(x, rows, tuple(shape), fmt, code)
    _launch("snnb_rms_norm_mx", index, x2.data_ptr(), ldx,
            None if r2 is None else r2.data_ptr(), ldr, dt, weight.data_ptr(), _DTYPES[wd], eps,
            rows, K, code, *t._pointers(), hp)
    return t, h
