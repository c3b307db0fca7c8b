"""Microscaled operators on the GPU against the float64 oracle (oracle/mx.py).

Tolerances, derived:
  quantise / dequantise   none: codes, scale bytes and values are equal bit for bit.
  linear                  products of the element values are exact in float32; a sum is rounded
                          (or cut) to 24 bits at most once inside an MMA's K (32 or 64), once per
                          MMA onto the accumulator, and once per joined split, each relative to at
                          most sum |a w|: (2 K / 32 + 16) * 2^-23 * sum |a w|; the bias adds 2^-24
                          of the result, and the output rounds by half an ulp of its type.
  norm                    codes and scales are equal: y is decided at code boundaries in float64,
                          good to ~2^-40, so only values within 2^-36 of a boundary may differ;
                          h is x + residual in float32, rounded once to x's type (equal).
"""
import numpy as np
import pytest
import torch

from oracle import mx as OM

pytestmark = pytest.mark.gpu
DEV = "cuda"
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def _mx():
    from snn_compiler.kernels import mx
    return mx


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _held(t):
    """(codes [rows, nb, 32], scale bytes [rows, nb]) of an MXTensor."""
    nb = -(-t.shape[-1] // 32)
    return (OM.split_codes(t.data.cpu().numpy(), t.fmt),
            OM.row_scales(t.scales.cpu().numpy(), t.rows, nb))


def _unowned_zero(t):
    """Elements past K and scale bytes that no block owns are zero."""
    K, rows = t.shape[-1], t.rows
    nb = -(-K // 32)
    codes = OM.split_codes(t.data.cpu().numpy(), t.fmt).reshape(rows, -1)
    assert not codes[:, K:].any()
    s = t.scales.cpu().numpy().copy()
    r, j = np.arange(rows)[:, None], np.arange(nb)[None]
    s[r // 128, j // 4, r % 32, r % 128 // 32, j % 4] = 0
    assert not s.any()


def _check_quantised(t, x, fmt):
    codes, scales = _held(t)
    ref_codes, ref_scales = OM.quantize(x, fmt)
    assert np.array_equal(scales, ref_scales)
    # the sign of a zero is not a value
    sign = 8 if fmt == "mxfp4" else 128
    for c in (codes, ref_codes):
        c[c == sign] = 0
    assert np.array_equal(codes, ref_codes)
    _unowned_zero(t)


def _data(rows, K, dtype, seed, spread=3.0):
    g = _gen(seed)
    x = torch.randn(rows, K, generator=g) * torch.exp(spread * torch.randn(rows, 1, generator=g))
    return x.to(dtype)


SHAPES = [(1, 1), (1, 32), (3, 31), (2, 33), (5, 127), (127, 128), (128, 129), (129, 256),
          (1, 4096), (70, 1000), (40, 1003), (1030, 96), (3, 5000)]


@pytest.mark.parametrize("fmt", ["mxfp4", "mxfp8"])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,K", SHAPES)
def test_quantise_against_oracle(rows, K, dtype, fmt):
    x = _data(rows, K, dtype, rows + K, spread=2.0 if dtype == torch.float16 else 5.0)
    t = _mx().mx_quantize(x.to(DEV), fmt)
    assert t.shape == (rows, K) and t.fmt == fmt
    _check_quantised(t, x.double().numpy(), fmt)
    for out in DTYPES:
        v = _mx().mx_dequantize(t, out)
        codes, scales = _held(t)
        ref = torch.from_numpy(OM.values(codes, scales, fmt)[:, :K])
        assert v.dtype == out and torch.equal(v.cpu(), ref.float().to(out))


@pytest.mark.parametrize("fmt", ["mxfp4", "mxfp8"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,K,cols,at", [(9, 64, 96, 0), (9, 64, 96, 32), (70, 100, 103, 0),
                                            (70, 100, 103, 3), (33, 257, 300, 1), (5, 40, 41, 1),
                                            (300, 24, 27, 2), (6, 1024, 1031, 5)])
def test_quantise_slices_of_a_wider_tensor(rows, K, cols, at, dtype, fmt):
    """Row strides and base addresses of every alignment, without a copy; nothing outside the
    slice counts (it is NaN here)."""
    x = _data(rows, K, dtype, cols)
    wide = torch.full((rows, cols), float("nan"), dtype=dtype, device=DEV)
    wide[:, at: at + K] = x.to(DEV)
    t = _mx().mx_quantize(wide[:, at: at + K], fmt)
    _check_quantised(t, x.double().numpy(), fmt)


def test_quantise_any_axes_and_orders():
    mx = _mx()
    x = torch.randn(3, 4, 50, generator=_gen(1))
    ref = mx.mx_quantize(x.to(DEV).reshape(12, 50), "mxfp8")
    for y in (x.to(DEV), x.to(DEV).transpose(0, 1).contiguous().transpose(0, 1),
              x.to(DEV).transpose(1, 2).contiguous().transpose(1, 2)):
        t = mx.mx_quantize(y, "mxfp8")
        assert t.shape == (3, 4, 50)
        assert torch.equal(t.data, ref.data) and torch.equal(t.scales, ref.scales)
    one = mx.mx_quantize(x[0, 0].to(DEV), "mxfp8")            # [K]: one row
    assert one.shape == (50,) and torch.equal(one.data, ref.data[:1])
    assert one.dequantize().shape == (50,)
    e = x[0, :1].to(DEV).expand(6, 50)                        # row stride 0
    t = mx.mx_quantize(e)
    _check_quantised(t, x[0, :1].expand(6, 50).double().numpy(), "mxfp4")


def test_empty_tensors():
    mx = _mx()
    t = mx.mx_quantize(torch.empty(0, 64, device=DEV, dtype=torch.bfloat16))
    assert t.rows == 0 and t.dequantize().shape == (0, 64)
    w = mx.mx_quantize(torch.randn(16, 64, device=DEV))
    assert mx.mx_linear(t, w).shape == (0, 16)
    q, h = mx.rms_norm_mx(torch.empty(2, 0, 64, device=DEV), torch.ones(64, device=DEV),
                          torch.empty(2, 0, 64, device=DEV))
    assert q.shape == (2, 0, 64) and h.shape == (2, 0, 64)
    with pytest.raises(ValueError):
        mx.mx_quantize(torch.empty(4, 0, device=DEV))
    with pytest.raises(ValueError):
        mx.rms_norm_mx(torch.empty(4, 0, device=DEV), torch.empty(0, device=DEV))


@pytest.mark.parametrize("fmt", ["mxfp4", "mxfp8"])
@pytest.mark.parametrize("dtype", DTYPES)
def test_quantise_extremes(dtype, fmt):
    """Blocks of zeros, of the type's smallest and largest values, subnormals, exact ties, and
    blocks with an infinity or a NaN (those become NaN, their neighbours do not)."""
    fi = torch.finfo(dtype)
    g = _gen(3)
    rows = [torch.zeros(64), torch.full((64,), fi.max), torch.full((64,), fi.tiny),
            torch.full((64,), fi.smallest_normal) * torch.rand(64, generator=g),
            torch.randn(64, generator=g) * fi.tiny, -torch.full((64,), fi.max)]
    mids = (OM.grid(fmt)[1:] + OM.grid(fmt)[:-1]) / 2         # ties, with the top value in place
    for k in (1.0, 2.0 ** -3, 2.0 ** 4):
        m = torch.tensor(np.resize(mids, 64))
        m[0] = m[32] = OM.grid(fmt)[-1]
        rows.append(m * k)
    r = torch.randn(64, generator=g)
    for bad in (float("inf"), -float("inf"), float("nan")):
        b = r.clone()
        b[5] = bad
        rows.append(b)
    x = torch.stack([v.double() for v in rows]).to(dtype)
    t = _mx().mx_quantize(x.to(DEV), fmt)
    _check_quantised(t, x.double().numpy(), fmt)
    v = t.dequantize(torch.float32).cpu()
    assert torch.isnan(v[-3:, :32]).all() and torch.isfinite(v[-3:, 32:]).all()
    assert torch.isfinite(v[:-3]).all()


def test_spikes_are_exact():
    x = (torch.rand(50, 300, generator=_gen(0)) < 0.2).to(torch.bfloat16).to(DEV)
    for fmt in ("mxfp4", "mxfp8"):
        assert torch.equal(_mx().mx_quantize(x, fmt).dequantize(), x)


def test_dequantise_every_code_and_scale():
    """All 16 / 256 codes under every scale byte, and outputs rounded once (to 16 bits too)."""
    mx = _mx()
    for fmt in ("mxfp4", "mxfp8"):
        n = 16 if fmt == "mxfp4" else 256
        codes = np.resize(np.arange(n, dtype=np.uint8), (256, max(n, 32)))
        K = codes.shape[1]
        data = codes if fmt == "mxfp8" else codes[:, 0::2] | (codes[:, 1::2] << 4)
        s = np.repeat(np.arange(256, dtype=np.uint8)[:, None], K // 32, 1)
        t = mx.MXTensor.from_rows(torch.from_numpy(data.copy()).to(DEV), torch.from_numpy(s).to(DEV),
                                  K, fmt)
        ref = torch.from_numpy(OM.values(codes.reshape(256, -1, 32), s, fmt))
        for dtype in DTYPES:
            v = t.dequantize(dtype).cpu()
            want = ref.float().to(dtype)                       # exact in float32, or infinite
            assert torch.equal(torch.isnan(v), torch.isnan(want))
            assert torch.equal(v.nan_to_num(7.0), want.nan_to_num(7.0)), (fmt, dtype)


# ---- product -------------------------------------------------------------------------------


def _linear_case(rows, N, K, afmt, seed, bias):
    mx = _mx()
    g = _gen(seed)
    a = torch.randn(rows, K, generator=g) * torch.exp(torch.randn(rows, 1, generator=g))
    a[:, ::17] *= 20
    w = torch.randn(N, K, generator=g) * torch.exp(0.5 * torch.randn(N, 1, generator=g))
    ta, tw = mx.mx_quantize(a.to(DEV), afmt), mx.mx_quantize(w.to(DEV), "mxfp4")
    b = torch.randn(N, generator=g) if bias else None
    va = torch.from_numpy(OM.values(*_held(ta), afmt)[:, :K])
    vw = torch.from_numpy(OM.values(*_held(tw), "mxfp4")[:, :K])
    ref = va @ vw.t()
    span = va.abs() @ vw.abs().t()
    if bias:
        ref, span = ref + b.double(), span + b.abs().double()
    return ta, tw, None if b is None else b.to(DEV), ref, span


def _tolerance(ref, span, K, dtype):
    half_ulp = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
    tiny = {torch.float32: 0.0, torch.float16: 2.0 ** -25, torch.bfloat16: 0.0}[dtype]
    acc = (2 * K / 32 + 16) * 2.0 ** -23 * span
    return acc + (ref.abs() + acc) * half_ulp[dtype] + tiny


# every form: 16, 32, 64, 128 tokens with K split over 1 .. 8 CTAs, pairs of 128 and 256 tokens
# with one and several rounds of tiles; odd sizes in every axis
LINEAR = [(1, 1, 1), (1, 7, 31), (1, 128, 32), (1, 4096, 4096), (2, 129, 33), (16, 130, 1000),
          (17, 256, 257), (32, 1001, 512), (33, 200, 2048), (64, 384, 640), (65, 100, 100),
          (128, 257, 4100), (129, 130, 96), (200, 1001, 1000), (300, 256, 2500), (333, 77, 129),
          (513, 2050, 300), (1000, 4097, 416), (2300, 2304, 1100), (2500, 4000, 256)]


@pytest.mark.parametrize("afmt", ["mxfp4", "mxfp8"])
@pytest.mark.parametrize("rows,N,K", LINEAR)
def test_linear_against_oracle(rows, N, K, afmt):
    dtype = DTYPES[(rows + N + K) % 3]
    ta, tw, b, ref, span = _linear_case(rows, N, K, afmt, rows * 3 + N + K, (rows + K) % 2 == 0)
    y = _mx().mx_linear(ta, tw, b, dtype=dtype)
    assert y.dtype == dtype and y.shape == (rows, N)
    if dtype == torch.float16:
        ref = ref.clamp(-65504, 65504)
        y = y.clamp(-65504, 65504)
    err = (y.double().cpu() - ref).abs()
    tol = _tolerance(ref, span, K, dtype)
    assert (err <= tol).all(), ((err / tol).max().item(), (err > tol).sum().item())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("afmt", ["mxfp4", "mxfp8"])
@pytest.mark.parametrize("rows,N,K", [(3, 50, 96), (40, 33, 200), (150, 258, 130), (700, 4100, 512)])
def test_linear_types_and_bias(rows, N, K, afmt, dtype):
    for bias in (False, True):
        ta, tw, b, ref, span = _linear_case(rows, N, K, afmt, N + K, bias)
        y = _mx().mx_linear(ta, tw, b, dtype=dtype).double().cpu()
        ref16 = ref.clamp(-65504, 65504) if dtype == torch.float16 else ref
        tol = _tolerance(ref16, span, K, dtype)
        assert ((y.clamp(ref16.min(), ref16.max()) - ref16).abs() <= tol).all()


@pytest.mark.parametrize("rows", [1, 20, 100, 200, 1500])
@pytest.mark.parametrize("afmt", ["mxfp4", "mxfp8"])
def test_linear_of_small_whole_numbers_is_exact(rows, afmt):
    """Whole numbers whose sums stay below 2^24 leave nothing to round: equality with the
    integer product, so every code, scale and position counts."""
    mx = _mx()
    g = _gen(rows)
    K, N = 1056, 515
    a = torch.randint(-4, 5, (rows, K), generator=g).float()
    w = torch.randint(-4, 5, (N, K), generator=g).float()
    a[:, ::32] = 4                                 # the block's scale keeps the grid of halves
    w[:, ::32] = 4
    ta, tw = mx.mx_quantize(a.to(DEV), afmt), mx.mx_quantize(w.to(DEV))
    assert torch.equal(ta.dequantize(torch.float32).cpu(), a)
    y = mx.mx_linear(ta, tw, dtype=torch.float32)
    assert torch.equal(y.cpu().double(), a.double() @ w.double().t())


@pytest.mark.parametrize("rows", [4, 300])
@pytest.mark.parametrize("afmt", ["mxfp4", "mxfp8"])
def test_linear_nan_stays_in_its_row_and_column(rows, afmt):
    mx = _mx()
    a = torch.randn(rows, 300, generator=_gen(0))
    w = torch.randn(140, 300, generator=_gen(1))
    clean = mx.mx_linear(mx.mx_quantize(a.to(DEV), afmt), mx.mx_quantize(w.to(DEV)),
                         dtype=torch.float32)
    a[2, 299] = float("nan")
    w[131, 0] = float("inf")
    y = mx.mx_linear(mx.mx_quantize(a.to(DEV), afmt), mx.mx_quantize(w.to(DEV)),
                     dtype=torch.float32)
    bad = torch.zeros(rows, 140, dtype=torch.bool)
    bad[2], bad[:, 131] = True, True
    assert torch.isnan(y.cpu()[bad]).all()
    assert torch.equal(y.cpu()[~bad], clean.cpu()[~bad])


def test_linear_repeats_bit_for_bit():
    """Split sums are joined in a fixed order: no run differs from another."""
    for rows, N, K, afmt in ((1, 512, 8192, "mxfp8"), (5, 640, 4096, "mxfp4"),
                             (128, 256, 4096, "mxfp8"), (600, 1000, 2048, "mxfp8")):
        ta, tw, b, _, _ = _linear_case(rows, N, K, afmt, 1, True)
        first = _mx().mx_linear(ta, tw, b, dtype=torch.float32)
        for _ in range(20):
            assert torch.equal(_mx().mx_linear(ta, tw, b, dtype=torch.float32), first)


def test_linear_out_argument_leading_axes_and_unaligned_out():
    mx = _mx()
    a = torch.randn(2, 3, 96, generator=_gen(0)).to(DEV)
    w = mx.mx_quantize(torch.randn(34, 96, generator=_gen(1)).to(DEV))
    t = mx.mx_quantize(a, "mxfp8")
    y = mx.mx_linear(t, w)
    assert y.shape == (2, 3, 34)
    flat = torch.zeros(6 * 34 + 1, device=DEV, dtype=torch.bfloat16)
    odd = flat[1:].view(2, 3, 34)                             # 2-byte aligned only
    assert mx.mx_linear(t, w, out=odd) is odd
    assert torch.equal(odd, y) and flat[0] == 0
    with pytest.raises(AssertionError):
        mx.mx_linear(t, w, out=torch.empty(6, 34, device=DEV))
    one = mx.mx_quantize(a[0, 0], "mxfp8")
    assert torch.equal(mx.mx_linear(one, w), y[0, 0])


def test_offsets_past_32_bits():
    """More than 2^31 values in, and out: the last rows are those of a call on them alone."""
    mx = _mx()
    rows, K = 70000, 32768                                    # 2.29e9 values, 4.6 GB
    x = torch.empty(rows, K, device=DEV, dtype=torch.bfloat16)
    tail = torch.randn(300, K, generator=_gen(0)).to(torch.bfloat16).to(DEV)
    x.zero_()
    x[-300:] = tail
    t = mx.mx_quantize(x)
    ref = mx.mx_quantize(tail)
    assert torch.equal(t.data[-300:], ref.data)
    v = mx.mx_dequantize(t)
    assert torch.equal(v[-300:], ref.dequantize()) and not v[:256].any()
    del x, v
    # the product's output: 70000 x 32768 in bfloat16
    w = mx.mx_quantize(torch.randn(K, 64, generator=_gen(1)).to(DEV))
    a = torch.randn(rows, 64, generator=_gen(2)).to(DEV)
    y = mx.mx_linear(mx.mx_quantize(a, "mxfp8"), w)
    assert torch.equal(y[-300:], mx.mx_linear(mx.mx_quantize(a[-300:], "mxfp8"), w))


# ---- norm ----------------------------------------------------------------------------------


def _check_norm(q, h, x, w, r, eps, fmt):
    y, href = OM.rms_norm(x.float().numpy(), w.double().numpy(),
                          None if r is None else r.float().numpy(), eps)
    codes, scales = _held(q)
    ref_codes, ref_scales = OM.quantize(y, fmt)
    sign = 8 if fmt == "mxfp4" else 128
    for c in (codes, ref_codes):
        c[c == sign] = 0
    K = x.shape[-1]
    rows, nb = ref_scales.shape
    differ = (codes != ref_codes) | (scales != ref_scales)[..., None]
    if differ.any():
        # only values that a relative change of 2^-36 takes across a boundary
        lo, hi = OM.quantize(y * (1 - 2.0 ** -36), fmt), OM.quantize(y * (1 + 2.0 ** -36), fmt)
        same = (lo[0] == hi[0]) & (lo[1] == hi[1])[..., None]
        assert not (differ & same).any()
    _unowned_zero(q)
    if r is not None:
        want = (x.float() + r.float()).to(x.dtype)
        assert torch.equal(h.cpu(), want)


@pytest.mark.parametrize("fmt", ["mxfp8", "mxfp4"])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,K", [(1, 1), (1, 4096), (2, 8192), (1, 9000), (1, 40000), (3, 31), (5, 200),
                                    (129, 96), (150, 33), (160, 250), (300, 384), (200, 1000),
                                    (170, 1003), (200, 1536), (149, 4096), (160, 4100),
                                    (150, 8192), (150, 16384), (150, 17000)])
def test_norm_against_oracle(rows, K, dtype, fmt):
    g = _gen(rows + K)
    x = (torch.randn(rows, K, generator=g) * 3).to(dtype)
    w = (torch.rand(K, generator=g) + 0.5).to(dtype)
    r = torch.randn(rows, K, generator=g).to(dtype) if (rows + K) % 3 else None
    d = x.to(DEV)
    q, h = _mx().rms_norm_mx(d, w.to(DEV), None if r is None else r.to(DEV), eps=1e-5, fmt=fmt)
    if r is None:
        assert h is d
    assert torch.equal(d.cpu(), x)                            # the inputs are left alone
    _check_norm(q, h, x, w, r, 1e-5, fmt)


@pytest.mark.parametrize("rows,K", [(7, 64), (200, 64), (200, 2048), (3, 700)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_norm_float32_weights(rows, K, dtype):
    g = _gen(K)
    x, r = torch.randn(rows, K, generator=g).to(dtype), torch.randn(rows, K, generator=g).to(dtype)
    w = torch.rand(K, generator=g) + 0.5
    q, h = _mx().rms_norm_mx(x.to(DEV), w.to(DEV), r.to(DEV))
    _check_norm(q, h, x, w, r, 1e-6, "mxfp8")


@pytest.mark.parametrize("rows,K,cols,at", [(5, 64, 72, 8), (5, 64, 67, 1), (200, 512, 520, 0),
                                            (200, 512, 515, 2), (160, 1003, 1010, 3)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_norm_slices_of_wider_tensors(rows, K, cols, at, dtype):
    g = _gen(cols)
    wide = torch.full((2, rows, cols), float("nan"), dtype=dtype)
    wide[:, :, at: at + K] = torch.randn(2, rows, K, generator=g).to(dtype)
    w = (torch.rand(K, generator=g) + 0.5).to(dtype)
    d = wide.to(DEV)
    x, r = wide[0, :, at: at + K], wide[1, :, at: at + K]
    q, h = _mx().rms_norm_mx(d[0, :, at: at + K], w.to(DEV), d[1, :, at: at + K], fmt="mxfp4")
    assert h.is_contiguous()
    _check_norm(q, h, x, w, r, 1e-6, "mxfp4")


@pytest.mark.parametrize("K", [1, 7, 9, 34, 100, 128, 129, 189, 250, 257, 404, 500, 777, 3001])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_norm_of_unaligned_rows_between_nans(K, dtype):
    """Rows inside a wider tensor whose other columns are NaN: loads may cover them, results do
    not.  The first row starts the storage, the last ends it."""
    mx = _mx()
    g = _gen(K)
    rows = 37
    for fmt, ld, at in (("mxfp4", K + 3, 0), ("mxfp8", K + 3, 3), ("mxfp8", K + 17, 5)):
        hold = [torch.full((rows, ld), float("nan"), dtype=dtype) for _ in range(2)]
        x, r = (t[:, at:at + K] for t in hold)
        x.copy_(torch.randn(rows, K, generator=g))
        r.copy_(torch.randn(rows, K, generator=g))
        w = torch.rand(K, generator=g).to(dtype) + 0.5
        xd, rd = (t.to(DEV)[:, at:at + K] for t in hold)
        q, h = mx.rms_norm_mx(xd, w.to(DEV), rd, eps=1e-6, fmt=fmt)
        _check_norm(q, h, x, w, r, 1e-6, fmt)


@pytest.mark.parametrize("K", [1, 8, 31, 34, 48, 63, 64, 65, 120, 127, 129, 260, 300, 511, 513])
@pytest.mark.parametrize("rows", [1, 9, 301])
def test_short_rows(K, rows):
    """Quantise, back and norm at every team width of short rows, aligned or not, the gap between
    rows NaN."""
    mx = _mx()
    g = _gen(rows * 1000 + K)
    for gap, at, dtype, fmt in ((0, 0, torch.float32, "mxfp4"), (16, 8, torch.bfloat16, "mxfp8"),
                                (3, 1, torch.float16, "mxfp4"), (5, 2, torch.float32, "mxfp8")):
        hold = torch.full((rows, K + gap), float("nan"), dtype=dtype)
        x = hold[:, at:at + K]
        x.copy_(torch.randn(rows, K, generator=g))
        d = hold.to(DEV)[:, at:at + K]
        t = mx.mx_quantize(d, fmt)
        _check_quantised(t, x.double().numpy(), fmt)
        back = mx.mx_dequantize(t, torch.float32).cpu()
        codes, scales = OM.quantize(x.double().numpy(), fmt)
        want = OM.values(codes, scales, fmt).reshape(rows, -1)[:, :K]
        assert np.array_equal(back.double().numpy(), want)
        w = (torch.rand(K, generator=g) + 0.5).to(dtype)
        q, h = mx.rms_norm_mx(d, w.to(DEV), None, eps=1e-6, fmt=fmt)
        _check_norm(q, h, x, w, None, 1e-6, fmt)


@pytest.mark.parametrize("K", [5, 100, 189, 500, 1003])
def test_norm_of_one_row_for_all(K):
    """Row stride 0."""
    mx = _mx()
    g = _gen(K)
    x, w = torch.randn(1, K, generator=g), torch.rand(K, generator=g) + 0.5
    r = torch.randn(40, K, generator=g)
    q, h = mx.rms_norm_mx(x.to(DEV).expand(40, K), w.to(DEV), r.to(DEV), eps=1e-6, fmt="mxfp8")
    _check_norm(q, h, x.expand(40, K), w, r, 1e-6, "mxfp8")


def test_norm_rows_of_extremes():
    """Zero rows (eps alone), values whose squares leave float32, and NaN or infinite rows, which
    stay NaN (or zero around an infinity) and leave their neighbours alone."""
    K = 96
    g = _gen(0)
    for rows in (12, 400):
        x = torch.randn(rows, K, generator=g)
        x[0] = 0
        x[1] *= 1e30
        x[2] *= 1e-30
        x[3, 5] = float("nan")
        x[4, 40] = float("inf")
        w = torch.rand(K, generator=g) + 0.5
        q, _ = _mx().rms_norm_mx(x.to(DEV), w.to(DEV))
        v = q.dequantize(torch.float32).cpu()
        assert not v[0].any()
        assert torch.isnan(v[3]).all()
        assert torch.isnan(v[4, 32:64]).all() and not v[4, :32].any() and not v[4, 64:].any()
        keep = [0, 1, 2] + list(range(5, rows))
        y, _ = OM.rms_norm(x[keep].numpy(), w.double().numpy(), None, 1e-6)
        ref = torch.from_numpy(OM.values(*OM.quantize(y, "mxfp8"), "mxfp8")).float()
        assert torch.equal(v[keep], ref)


def test_norm_exact_ties():
    """Rows of +-1 with eps 0 leave y = weight exactly: ties go to the even code."""
    mids = (OM.grid("mxfp8")[1:] + OM.grid("mxfp8")[:-1]) / 2
    K = 256
    w = torch.tensor(np.resize(mids, K), dtype=torch.float32)
    w[::32] = 448.0
    x = torch.where(torch.rand(300, K, generator=_gen(0)) < 0.5, -1.0, 1.0)
    q, h = _mx().rms_norm_mx(x.to(DEV), w.to(DEV), eps=0.0)
    _check_norm(q, h, x, w, None, 0.0, "mxfp8")


# ---- streams, graphs, modules --------------------------------------------------------------


def test_other_streams_and_graph_capture():
    """Launches go to the current stream and can be captured; a replay follows its inputs."""
    mx = _mx()
    x = torch.randn(40, 512, generator=_gen(0)).to(DEV)
    w = torch.rand(512, generator=_gen(1)).to(DEV)
    wt = mx.mx_quantize(torch.randn(300, 512, generator=_gen(2)).to(DEV))

    def step(v):
        q, h = mx.rms_norm_mx(v, w, v)
        return mx.mx_linear(q, wt, dtype=torch.float32), h
    ref = step(x)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        torch.cuda._sleep(20_000_000)                # the default stream is far ahead
        y = x * 2
        got = step(y)
    s.synchronize()
    want = step(x * 2)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert not torch.equal(want[1], ref[1])
    static = x.clone()
    with torch.cuda.stream(s):
        step(static)
        s.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            out = step(static)
    for k in (1.0, 3.0):
        static.copy_(x * k)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, step(x * k)))


def test_status_word_stays_clear():
    from snn_compiler.kernels import conv as KC
    assert KC.device_status() == 0


@pytest.mark.parametrize("rows,N,K", [(6523, 4000, 32), (2000, 4000, 96), (2000, 3000, 1000)])
def test_linear_of_packed_weights_repeated(rows, N, K):
    """Rows of K that are no whole groups of 128 beside 8-bit tokens: weights pass through a ring of
    their own, whose copies may land in any order.  Every repetition gives the first one's bits,
    and those are the oracle's within the bound."""
    mx = _mx()
    g = _gen(K)
    a = mx.mx_quantize(torch.randn(rows, K, generator=g).to(DEV), "mxfp8")
    ws = [mx.mx_quantize(torch.randn(N, K, generator=g).to(DEV)) for _ in range(3)]
    first = [mx.mx_linear(a, w, dtype=torch.float32) for w in ws]
    va = torch.from_numpy(OM.values(*_held(a), "mxfp8")[:, :K]).to(DEV)
    for w, out in zip(ws, first):
        vw = torch.from_numpy(OM.values(*_held(w), "mxfp4")[:, :K]).to(DEV)
        tol = (2 * K / 32 + 16) * 2.0 ** -23 * (va.abs() @ vw.abs().t()) + 2.0 ** -24 * (va @ vw.t()).abs()
        assert ((out.double() - va @ vw.t()).abs() <= tol).all()
    for _ in range(300):
        for w, out in zip(ws, first):
            assert torch.equal(mx.mx_linear(a, w, dtype=torch.float32), out)


@pytest.mark.parametrize("stages", list(range(1, 27)))
@pytest.mark.parametrize("fmt", ["mxfp4", "mxfp8"])
def test_linear_every_number_of_stages(stages, fmt):
    """Few tiles and a K of 1 to 26 ring stages (256 of K in mxfp4, 128 in mxfp8), whole or ragged:
    K is split over as many thread blocks as pay, and each has work."""
    from snn_compiler.kernels import conv as KC
    mx = _mx()
    step = 256 if fmt == "mxfp4" else 128
    for rows, N, K in ((2, 16, stages * step), (2, 16, stages * step - step // 2 - 32),
                       (40, 200, stages * step - 7), (140, 100, stages * step - 32)):
        if K < 1:
            continue
        g = _gen(K)
        a = mx.mx_quantize(torch.randn(rows, K, generator=g).to(DEV), fmt)
        w = mx.mx_quantize(torch.randn(N, K, generator=g).to(DEV))
        out = mx.mx_linear(a, w, dtype=torch.float32).double().cpu()
        va = torch.from_numpy(OM.values(*_held(a), fmt)[:, :K])
        vw = torch.from_numpy(OM.values(*_held(w), "mxfp4")[:, :K])
        tol = (2 * K / 32 + 16) * 2.0 ** -23 * (va.abs() @ vw.abs().t()) + 2.0 ** -24 * (va @ vw.t()).abs()
        assert ((out - va @ vw.t()).abs() <= tol).all(), (rows, N, K)
    assert KC.device_status() == 0


@pytest.mark.parametrize("rows,N,K", [(1, 1, 32), (2, 3, 32), (15, 31, 40), (17, 33, 64), (64, 129, 96),
                                      (101, 255, 33), (301, 257, 64), (1001, 1023, 40),
                                      (1300, 2051, 160)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("fmt", ["mxfp4", "mxfp8"])
def test_linear_odd_features_in_16_bits(rows, N, K, dtype, fmt):
    """An odd number of features: words of two that begin at even or odd features by the row, at
    either alignment of `out`.  The same product in float32, rounded once, is the same bits."""
    mx = _mx()
    g = _gen(rows + N)
    a = mx.mx_quantize(torch.randn(rows, K, generator=g).to(DEV), fmt)
    w = mx.mx_quantize(torch.randn(N, K, generator=g).to(DEV))
    bias = torch.randn(N, generator=g).to(DEV)
    want = mx.mx_linear(a, w, bias, dtype=torch.float32).to(dtype)
    for at in (0, 1, 2):
        hold = torch.full((rows * N + 4,), 7.0, dtype=dtype, device=DEV)
        mx.mx_linear(a, w, bias, out=hold[at: at + rows * N].view(rows, N))
        assert torch.equal(hold[at: at + rows * N].view(rows, N), want)
        assert (hold[:at] == 7).all() and (hold[at + rows * N:] == 7).all()


def test_mx_linear_module():
    from snn_compiler.nn import MXLinear
    mx = _mx()
    torch.manual_seed(0)
    lin = torch.nn.Linear(200, 96).to(DEV)
    m = MXLinear.from_linear(lin, dtype=torch.float32)
    x = torch.randn(2, 7, 200, device=DEV)
    want = mx.mx_linear(mx.mx_quantize(x, "mxfp8"), mx.mx_quantize(lin.weight.detach()),
                        lin.bias.detach(), dtype=torch.float32)
    assert torch.equal(m(x), want) and not m(x).requires_grad
    other = MXLinear.from_linear(torch.nn.Linear(200, 96).to(DEV), dtype=torch.float32)
    assert not torch.equal(other(x), want)
    other.load_state_dict(m.state_dict())
    assert torch.equal(other(x), want)
    # near the float layer: 4-bit weights round by 2^-2 relative at most, 8-bit values by 2^-4
    y = lin(x).detach()
    assert ((m(x) - y).norm() / y.norm()).item() < 0.25


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_linear_module_whose_bias_was_cast(dtype):
    """model.to(dtype) casts the bias buffer; the product takes it at that value."""
    from snn_compiler.nn import MXLinear
    torch.manual_seed(4)
    m = MXLinear.from_linear(torch.nn.Linear(200, 96).to(DEV), dtype=torch.float32)
    x = torch.randn(5, 200, device=DEV)
    without = MXLinear(m.weight, None, dtype=torch.float32)(x)
    m = m.to(dtype)
    assert m.bias.dtype == dtype
    assert torch.equal(m(x), without + m.bias.float())


def test_spiking_mlp_block():
    """norm -> fc1 -> LIF -> fc2 over [T, B, N, D]: each stage against the oracle on the stage's
    own input, and two chained blocks through the residual."""
    from oracle import neurons as ON
    from snn_compiler.nn import SpikingMLP
    mx = _mx()
    torch.manual_seed(1)
    T, B, N, D, H = 4, 2, 49, 384, 1536
    block = SpikingMLP.from_linears(torch.nn.Linear(D, H).to(DEV), torch.nn.Linear(H, D).to(DEV),
                                    norm_weight=torch.rand(D).to(DEV) + 0.5, v_threshold=0.5)
    x = torch.randn(T, B, N, D, device=DEV).to(torch.bfloat16)
    y, h = block(x)
    assert y.shape == (T, B, N, D) and h.data_ptr() == x.data_ptr()
    q, _ = block.norm(x)
    _check_norm(q, x, x.cpu().reshape(-1, D), block.norm.weight.cpu(), None, 1e-6, "mxfp8")
    u = block.fc1(q)
    s = block.neuron(u)
    o = ON.lif_multistep(u.float().cpu().numpy().reshape(T, -1), df=np.float32(0.5),
                         sc=np.float32(0.5), thr=0.5)
    assert np.array_equal(s.float().cpu().numpy().reshape(T, -1), o["spikes"])
    assert 0 < s.float().mean().item() < 1
    ts = mx.mx_quantize(s, "mxfp4")
    assert torch.equal(ts.dequantize(), s)
    vw = torch.from_numpy(OM.values(*_held(block.fc2.weight), "mxfp4")[:, :H])
    vs = s.double().cpu().reshape(-1, H)
    ref = vs @ vw.t() + block.fc2.bias.double().cpu()
    span = vs @ vw.abs().t() + block.fc2.bias.abs().double().cpu()
    err = (y.double().cpu().reshape(-1, D) - ref).abs()
    assert (err <= _tolerance(ref, span, H, torch.bfloat16)).all()
    y2, h2 = block(y, h)
    assert torch.equal(h2, (x.float() + y.float()).to(torch.bfloat16))
    assert torch.isfinite(y2.float()).all()


# every form of the packed ring: one tile of 16, 32, 64 and 128 tokens with K split, pairs of 128
# tokens (few tiles; short K) and of 256
@pytest.mark.parametrize("rows,N,K", [(1, 512, 8100), (20, 640, 4000), (60, 1001, 4050),
                                      (128, 256, 4016), (300, 1000, 1100),
                                      (2000, 4000, 416), (2000, 3000, 1100), (1300, 4097, 2500),
                                      (256, 2304, 4000)])
def test_linear_forms_of_the_packed_ring_repeated(rows, N, K):
    """Weights placed by warps, of which one CTA of a pair reads the other's: every repetition
    gives the first one's bits, and those are the oracle's within the bound."""
    mx = _mx()
    assert -(-K // 32) % 4, "rows of whole groups of 128 are unpacked by the copies instead"
    g = _gen(K + rows)
    a = mx.mx_quantize(torch.randn(rows, K, generator=g).to(DEV), "mxfp8")
    ws = [mx.mx_quantize(torch.randn(N, K, generator=g).to(DEV)) for _ in range(3)]
    first = [mx.mx_linear(a, w, dtype=torch.float32) for w in ws]
    va = torch.from_numpy(OM.values(*_held(a), "mxfp8")[:, :K]).to(DEV)
    for w, out in zip(ws, first):
        vw = torch.from_numpy(OM.values(*_held(w), "mxfp4")[:, :K]).to(DEV)
        tol = (2 * K / 32 + 16) * 2.0 ** -23 * (va.abs() @ vw.abs().t()) + 2.0 ** -24 * (va @ vw.t()).abs()
        assert ((out.double() - va @ vw.t()).abs() <= tol).all()
    for _ in range(200):
        for w, out in zip(ws, first):
            assert torch.equal(mx.mx_linear(a, w, dtype=torch.float32), out)
