"""The microscaled kernels' forms that only large tensors reach, and the bytes around their outputs.

Large: a few rows, checked against the float64 oracle, repeated in an order that puts each of them
everywhere; every repetition has the same bits (none of the kernels' results depends on where a
row lies).  Bytes around: the C entries write into buffers whose other bytes are known."""
import numpy as np
import pytest
import torch

import test_mx_gpu as M
from oracle import mx as OM

pytestmark = pytest.mark.gpu
DEV = "cuda"
BASE = 61


def _spread(rows, base=BASE):
    """Which of the `base` rows stands at each place: neighbours, and places a stride apart, differ."""
    i = torch.arange(rows)
    return (i * 37 + i // base * 11) % base


def _firsts(idx, base=BASE):
    return torch.tensor([int((idx == b).nonzero()[0]) for b in range(base)])


def _rows_apart(x, gap):
    """x's values with `gap` NaN columns between its rows (a slice of a wider tensor)."""
    rows, K = x.shape
    wide = torch.full((rows, K + gap), float("nan"), dtype=x.dtype, device=x.device)
    wide[:, :K] = x
    return wide[:, :K]


def _same_rows(t, idx, at):
    """Each row of t has the codes and scale bytes of the row at[idx]."""
    data, scales = t.data, t.row_scales()
    src = at[idx].to(DEV)
    assert torch.equal(data, data[src]) and torch.equal(scales, scales[src])


def _pick(t, at):
    """The rows `at` of t alone."""
    mx = M._mx()
    return mx.MXTensor.from_rows(t.data[at.to(DEV)], t.row_scales()[at.to(DEV)], t.shape[-1], t.fmt)


# ---- quantise and back ---------------------------------------------------------------------

# rows x K that give a thread several blocks of 32 (aligned) or several pieces (not): contiguous
# whole groups of 128; others; and pieces of 8, 16 and 32 lanes
LARGE = [(40009, 128, 0), (40009, 104, 0), (40009, 96, 16), (80021, 34, 0), (40009, 113, 0),
         (80021, 61, 3), (20011, 300, 1), (8209, 1003, 0), (2503, 2501, 3)]


@pytest.mark.parametrize("fmt", ["mxfp4", "mxfp8"])
@pytest.mark.parametrize("dtype", M.DTYPES)
@pytest.mark.parametrize("rows,K,gap", LARGE)
def test_quantise_large(rows, K, gap, dtype, fmt):
    mx = M._mx()
    base = M._data(BASE, K, dtype, K, spread=1.0)
    idx = _spread(rows)
    at = _firsts(idx)
    x = base.to(DEV)[idx.to(DEV)]
    t = mx.mx_quantize(_rows_apart(x, gap) if gap else x, fmt)
    M._check_quantised(_pick(t, at), base.double().numpy(), fmt)
    _same_rows(t, idx, at)
    # bytes that no block owns are zero
    full = mx.MXTensor.from_rows(t.data, t.row_scales(), K, fmt)
    assert torch.equal(full.scales, t.scales) and torch.equal(full.data, t.data)
    codes, scales = OM.quantize(base.double().numpy(), fmt)
    want = torch.from_numpy(OM.values(codes, scales, fmt)[:, :K]).float()
    for out in M.DTYPES:
        v = mx.mx_dequantize(t, out)
        assert torch.equal(v, want.to(out).to(DEV)[idx.to(DEV)])


# ---- norm ----------------------------------------------------------------------------------

# Teams of 64, 128, 256 and 512 threads that walk more rows than two turns of the longest ring, at
# lengths that fill a team and at others; with and without residual, both kinds of weights
RING = [(20011, 2048, "bf16", True, False), (20011, 1536, "bf16", True, False),
        (20011, 1032, "f16", False, True), (20011, 2048, "f32", True, False),
        (9001, 4096, "bf16", True, True), (9001, 2256, "bf16", True, False),
        (9001, 4096, "f16", False, False), (9001, 3256, "f32", False, False),
        (5003, 8192, "bf16", True, False), (5003, 4104, "bf16", True, True),
        (5003, 8184, "f16", True, False), (5003, 8192, "f32", False, False),
        (5003, 5000, "f32", True, False), (3001, 16384, "bf16", True, False),
        (3001, 8200, "bf16", False, True), (3001, 12000, "f16", True, False),
        (3001, 12800, "f32", True, False), (3001, 16384, "f32", False, False)]
NAMES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def _norm_everywhere(rows, K, dtype, residual, wide_weights, fmt, gap=0):
    mx = M._mx()
    g = M._gen(rows + K)
    base = (torch.randn(BASE, K, generator=g) * 3).to(dtype)
    other = torch.randn(BASE, K, generator=g).to(dtype) if residual else None
    w = (torch.rand(K, generator=g) + 0.5).to(torch.float32 if wide_weights else dtype)
    idx = _spread(rows)
    at = _firsts(idx)
    x = base.to(DEV)[idx.to(DEV)]
    r = other.to(DEV)[idx.to(DEV)] if residual else None
    if gap:
        x, r = _rows_apart(x, gap), _rows_apart(r, gap) if residual else None
    q, h = mx.rms_norm_mx(x, w.to(DEV), r, eps=1e-5, fmt=fmt)
    M._check_norm(_pick(q, at), h[at.to(DEV)], base, w, other, 1e-5, fmt)
    _same_rows(q, idx, at)
    if residual:
        assert torch.equal(h, h[at[idx].to(DEV)])
    full = mx.MXTensor.from_rows(q.data, q.row_scales(), K, fmt)
    assert torch.equal(full.scales, q.scales) and torch.equal(full.data, q.data)


@pytest.mark.parametrize("rows,K,dtype,residual,wide_weights", RING)
def test_norm_ring_turns(rows, K, dtype, residual, wide_weights):
    _norm_everywhere(rows, K, NAMES[dtype], residual, wide_weights, "mxfp8" if K % 3 else "mxfp4")


@pytest.mark.parametrize("rows,K,gap", [(3, 8193, 0), (301, 8200, 3), (150, 16001, 0), (5, 16383, 2),
                                        (2, 16385, 0), (170, 17001, 5), (1, 40001, 0)])
@pytest.mark.parametrize("dtype,residual", [("bf16", True), ("f16", False), ("f32", True)])
def test_norm_of_long_unaligned_rows(rows, K, gap, dtype, residual):
    g = M._gen(K)
    mx, dt = M._mx(), NAMES[dtype]
    x = (torch.randn(rows, K, generator=g) * 3).to(dt)
    r = torch.randn(rows, K, generator=g).to(dt) if residual else None
    w = (torch.rand(K, generator=g) + 0.5).to(dt)
    put = lambda t: None if t is None else _rows_apart(t.to(DEV), gap)
    for fmt in ("mxfp8", "mxfp4"):
        q, h = mx.rms_norm_mx(put(x), w.to(DEV), put(r), eps=1e-5, fmt=fmt)
        M._check_norm(q, h, x, w, r, 1e-5, fmt)


@pytest.mark.parametrize("rows,K,gap", [(70001, 34, 0), (30011, 404, 1), (30011, 96, 0), (12553, 384, 0),
                                        (9001, 1000, 0), (9001, 2047, 0), (4001, 4099, 5)])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_norm_of_many_rows(rows, K, gap, dtype):
    _norm_everywhere(rows, K, NAMES[dtype], True, False, "mxfp8", gap)


# ---- bytes around the outputs --------------------------------------------------------------

GUARD = 512


class _Guarded:
    """`size` bytes, `shift` of them past a 16-byte boundary, inside bytes of 0xA5."""

    def __init__(self, size, shift=0):
        self.buf = torch.full((size + 2 * GUARD + 16,), 0xA5, dtype=torch.uint8, device=DEV)
        self.at, self.size = GUARD + shift, size
        assert self.buf.data_ptr() % 16 == 0

    def ptr(self):
        return self.buf.data_ptr() + self.at

    def value(self):
        return self.buf[self.at: self.at + self.size]

    def untouched(self):
        around = torch.cat([self.buf[: self.at], self.buf[self.at + self.size:]])
        return bool((around == 0xA5).all())


WIDTHS = [1, 7, 8, 9, 31, 33, 64, 65, 100, 128, 129, 250, 257, 500, 513, 1003, 1024, 2051, 4100, 8200]


@pytest.mark.parametrize("K", WIDTHS)
@pytest.mark.parametrize("rows", [1, 5, 130, 303])
def test_nothing_is_written_around_the_outputs(rows, K):
    """Codes, scales, values and the next residual, at every alignment of the last two."""
    from snn_compiler import _lib
    mx = M._mx()
    L, stream = _lib.lib(), torch.cuda.current_stream().cuda_stream
    g = M._gen(rows + K)
    for code, (fmt, block) in enumerate((("mxfp4", 16), ("mxfp8", 32))):
        for dtype in (torch.bfloat16, torch.float32):
            es = dtype.itemsize
            dt = _lib.dtype_code(dtype)
            x = torch.randn(rows, K, generator=g).to(dtype).to(DEV)
            r = torch.randn(rows, K, generator=g).to(dtype).to(DEV)
            w = torch.ones(K, dtype=dtype, device=DEV)
            nb = -(-K // 32)
            size, scales = rows * nb * block, int(np.prod(mx.mx_scales_shape(rows, K)))
            d, s = _Guarded(size), _Guarded(scales)
            _lib.check(L.snnb_mx_quantize(x.data_ptr(), dt, rows, K, K, code, d.ptr(), s.ptr(),
                                          stream), "quantise")
            t = mx.mx_quantize(x, fmt)
            assert d.untouched() and s.untouched()
            assert torch.equal(d.value(), t.data.flatten())
            assert torch.equal(s.value(), t.scales.flatten())
            q, h = mx.rms_norm_mx(x, w, r, fmt=fmt)
            back = t.dequantize(dtype)
            for shift in range(0, 16, es * (1 if rows < 100 else 3)):
                v = _Guarded(rows * K * es, shift)
                _lib.check(L.snnb_mx_dequantize(*t._pointers(), code, rows, K, v.ptr(), dt, stream),
                           "dequantise")
                assert v.untouched()
                assert torch.equal(v.value(), back.flatten().view(torch.uint8))
                d, s, v = _Guarded(size), _Guarded(scales), _Guarded(rows * K * es, shift)
                _lib.check(L.snnb_rms_norm_mx(x.data_ptr(), K, r.data_ptr(), K, dt, w.data_ptr(), dt,
                                              1e-6, rows, K, code, d.ptr(), s.ptr(), v.ptr(), stream),
                           "norm")
                assert d.untouched() and s.untouched() and v.untouched()
                assert torch.equal(d.value(), q.data.flatten())
                assert torch.equal(s.value(), q.scales.flatten())
                assert torch.equal(v.value(), h.flatten().view(torch.uint8))
