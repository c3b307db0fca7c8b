"""Microscaled operators without a GPU: the layout helpers, the oracle's own formats, argument
checks of the Python layer and of the C entries (rejected before any device work)."""
import ctypes

import numpy as np
import pytest
import torch

from oracle import mx as OM


def _mx():
    from snn_compiler.kernels import mx
    return mx


@pytest.mark.parametrize("rows,K", [(1, 1), (1, 32), (127, 33), (128, 128), (129, 4096), (300, 1000)])
def test_scale_layout_round_trip(rows, K):
    mx = _mx()
    nb = -(-K // 32)
    g = torch.Generator().manual_seed(rows * 7 + K)
    s = torch.randint(0, 256, (rows, nb), generator=g, dtype=torch.uint8)
    data = torch.randint(0, 256, (rows, nb * 16), generator=g, dtype=torch.uint8)
    t = mx.MXTensor.from_rows(data, s, K, "mxfp4")
    assert tuple(t.scales.shape) == mx.mx_scales_shape(rows, K)
    assert torch.equal(t.row_scales(), s)
    # byte by byte, the order that the C header states
    flat = t.scales.flatten().numpy()
    groups = -(-nb // 4)
    r, j = np.arange(rows)[:, None], np.arange(nb)[None]
    at = ((r // 128) * groups + j // 4) * 512 + (r % 32) * 16 + (r % 128 // 32) * 4 + j % 4
    assert np.array_equal(flat[at], s.numpy())
    owned = np.zeros(flat.size, bool)
    owned[at] = True
    assert not flat[~owned].any()
    assert np.array_equal(OM.row_scales(t.scales.numpy(), rows, nb), s.numpy())


@pytest.mark.parametrize("K", [1, 31, 32, 33, 40, 96, 127])
@pytest.mark.parametrize("fmt", ["mxfp4", "mxfp8"])
def test_from_rows_clears_codes_past_the_last_column(K, fmt):
    mx = _mx()
    nb, size = -(-K // 32), 16 if fmt == "mxfp4" else 32
    data = torch.full((3, nb, size), 0x77, dtype=torch.uint8)
    t = mx.MXTensor.from_rows(data, torch.full((3, nb), 127, dtype=torch.uint8), K, fmt)
    flat = t.data.reshape(3, -1)
    codes = torch.stack([flat & 15, flat >> 4], -1).flatten(1) if fmt == "mxfp4" else flat
    assert (codes[:, :K] != 0).all() and not codes[:, K:].any()
    assert (data == 0x77).all()                               # the caller's bytes stay


@pytest.mark.parametrize("fmt", ["mxfp4", "mxfp8"])
def test_oracle_formats(fmt):
    """Every value of the format is a fixed point of the oracle's rounding, midpoints go to the
    even code, and spikes {0, 1} are exact."""
    g = OM.grid(fmt)
    assert np.array_equal(OM.nearest(g, fmt), np.arange(g.size))
    mid = (g[1:] + g[:-1]) / 2
    assert not (OM.nearest(mid, fmt) & 1).any()
    assert OM.nearest(np.array([g[-1] * 1.3]), fmt)[0] == g.size - 1
    if fmt == "mxfp8":
        t = torch.tensor(np.arange(127), dtype=torch.uint8).view(torch.float8_e4m3fn)
        assert np.array_equal(t.double().numpy(), g)
    x = (np.random.default_rng(0).random((5, 70)) < 0.3).astype(np.float64)
    c, s = OM.quantize(x, fmt)
    assert np.array_equal(OM.values(c, s, fmt)[:, :70], x)


def test_mxtensor_checks():
    mx = _mx()
    data = torch.zeros(4, 32, dtype=torch.uint8)
    scales = torch.zeros(mx.mx_scales_shape(4, 64), dtype=torch.uint8)
    t = mx.MXTensor(data, scales, (2, 2, 64), "mxfp4")
    assert t.rows == 4 and t.shape == (2, 2, 64) and t.data is data and t.scales is scales
    with pytest.raises(ValueError):
        mx.MXTensor(data, scales, (4, 64), "fp4")
    with pytest.raises(AssertionError):
        mx.MXTensor(data, scales, (4, 65), "mxfp4")          # 3 blocks a row, not 2
    with pytest.raises(AssertionError):
        mx.MXTensor(data, scales, (4, 64), "mxfp8")
    with pytest.raises(AssertionError):
        mx.MXTensor(data, scales[:, :, :16].contiguous(), (4, 64), "mxfp4")
    with pytest.raises(AssertionError):
        mx.MXTensor(data.float(), scales, (4, 64), "mxfp4")


def test_python_refusals_without_a_device():
    """CPU tensors, unknown formats and mismatched shapes raise before the library is called."""
    mx = _mx()
    x = torch.randn(4, 64)
    with pytest.raises(AssertionError):
        mx.mx_quantize(x)
    with pytest.raises(ValueError):
        mx.mx_quantize(x, "int4")
    with pytest.raises(ValueError):
        mx.mx_quantize(x[:, :0])
    with pytest.raises(AssertionError):
        mx.mx_quantize(x.double())
    with pytest.raises(AssertionError):
        mx.mx_quantize(x.to(torch.uint8))
    t4 = mx.MXTensor(torch.zeros(4, 32, dtype=torch.uint8),
                     torch.zeros(mx.mx_scales_shape(4, 64), dtype=torch.uint8), (4, 64), "mxfp4")
    t8 = mx.MXTensor(torch.zeros(4, 64, dtype=torch.uint8),
                     torch.zeros(mx.mx_scales_shape(4, 64), dtype=torch.uint8), (4, 64), "mxfp8")
    with pytest.raises(AssertionError):
        mx.mx_dequantize(t4)
    with pytest.raises(AssertionError):
        mx.mx_dequantize(t4, torch.int32)
    with pytest.raises(ValueError):
        mx.mx_linear(t4, t8)                                 # 8-bit weights
    with pytest.raises(AssertionError):
        mx.mx_linear(t8, mx.MXTensor(torch.zeros(4, 16, dtype=torch.uint8),
                                     torch.zeros(mx.mx_scales_shape(4, 32), dtype=torch.uint8),
                                     (4, 32), "mxfp4"))      # another K
    with pytest.raises(AssertionError):
        mx.mx_linear(t8, t4, torch.zeros(5))                 # bias of another length
    with pytest.raises(AssertionError):
        mx.mx_linear(t8, t4, torch.zeros(4, dtype=torch.float16))
    with pytest.raises(AssertionError):
        mx.mx_linear(t8, t4, dtype=torch.uint8)
    with pytest.raises(AssertionError):
        mx.mx_linear(t8, t4)                                 # no CUDA tensors
    w = torch.ones(64)
    with pytest.raises(AssertionError):
        mx.rms_norm_mx(x, w)
    with pytest.raises(AssertionError):
        mx.rms_norm_mx(x, w[:63])
    with pytest.raises(AssertionError):
        mx.rms_norm_mx(x, w.half())
    with pytest.raises(AssertionError):
        mx.rms_norm_mx(x, w, x[:3])
    with pytest.raises(ValueError):
        mx.rms_norm_mx(x, w, eps=-1.0)
    with pytest.raises(ValueError):
        mx.rms_norm_mx(x, w, fmt="fp8")


def test_module_refusals():
    from snn_compiler.nn import MXLinear
    mx = _mx()
    t8 = mx.MXTensor(torch.zeros(4, 64, dtype=torch.uint8),
                     torch.zeros(mx.mx_scales_shape(4, 64), dtype=torch.uint8), (4, 64), "mxfp8")
    with pytest.raises(ValueError):
        MXLinear(t8)
    t4 = mx.MXTensor(torch.zeros(4, 32, dtype=torch.uint8),
                     torch.zeros(mx.mx_scales_shape(4, 64), dtype=torch.uint8), (4, 64), "mxfp4")
    with pytest.raises(ValueError):
        MXLinear(t4, act="bf16")
    m = MXLinear(t4, torch.zeros(4))
    assert m.weight is m.weight and m.weight.data is m.weight_data
    assert set(m.state_dict()) == {"weight_data", "weight_scales", "bias"}


def test_c_entries_reject_bad_arguments_without_a_device():
    from snn_compiler import _lib
    L = _lib.lib()
    p = ctypes.c_void_p(1 << 20)             # aligned stand-ins: rejected before any access
    odd = ctypes.c_void_p((1 << 20) + 1)
    by8 = ctypes.c_void_p((1 << 20) + 8)

    def q(**kw):
        a = dict(x=p, dt=2, rows=4, K=64, ld=64, fmt=0, data=p, scales=p, st=None)
        a.update(kw)
        return L.snnb_mx_quantize(*a.values())
    assert q(rows=0) == 0
    for bad in (dict(dt=3), dict(dt=-1), dict(fmt=2), dict(fmt=-1), dict(rows=-1), dict(K=0),
                dict(K=-4), dict(ld=-1), dict(x=None), dict(data=None), dict(scales=None),
                dict(x=odd), dict(data=by8), dict(scales=by8), dict(rows=1 << 31),
                dict(rows=1 << 24, K=1 << 20), dict(K=1 << 31), dict(ld=1 << 40)):
        assert q(**bad) == -1, bad

    def d(**kw):
        a = dict(data=p, scales=p, fmt=1, rows=4, K=64, out=p, dt=2, st=None)
        a.update(kw)
        return L.snnb_mx_dequantize(*a.values())
    assert d(rows=0) == 0
    for bad in (dict(dt=3), dict(fmt=7), dict(rows=-1), dict(K=0), dict(out=None), dict(data=None),
                dict(scales=None), dict(out=odd), dict(data=by8), dict(rows=1 << 31)):
        assert d(**bad) == -1, bad

    def lin(**kw):
        a = dict(a=p, asc=p, fmt=0, rows=4, K=64, w=p, ws=p, N=8, bias=None, out=p, dt=2, st=None)
        a.update(kw)
        return L.snnb_mx_linear(*a.values())
    assert lin(rows=0) == 0
    for bad in (dict(fmt=2), dict(dt=3), dict(rows=-1), dict(K=0), dict(N=0), dict(N=-1),
                dict(a=None), dict(asc=None), dict(w=None), dict(ws=None), dict(out=None),
                dict(a=by8), dict(w=by8), dict(asc=by8), dict(ws=by8), dict(out=odd),
                dict(bias=odd), dict(rows=1 << 31), dict(N=1 << 31), dict(K=1 << 31)):
        assert lin(**bad) == -1, bad

    def n(**kw):
        a = dict(x=p, ldx=64, r=None, ldr=0, dt=2, w=p, wd=2, eps=1e-6, rows=4, K=64, fmt=1,
                 data=p, scales=p, h=None, st=None)
        a.update(kw)
        return L.snnb_rms_norm_mx(*a.values())
    assert n(rows=0) == 0
    for bad in (dict(dt=3), dict(wd=1), dict(wd=5), dict(fmt=2), dict(rows=-1), dict(K=0),
                dict(eps=-1.0), dict(eps=float("nan")), dict(x=None), dict(w=None),
                dict(data=None), dict(scales=None), dict(x=odd), dict(r=odd), dict(h=odd),
                dict(w=odd), dict(data=by8), dict(ldx=-1), dict(ldr=-1), dict(rows=1 << 31)):
        assert n(**bad) == -1, bad


@pytest.mark.parametrize("step", [0, 1])
def test_another_thread_reads_a_tensor_while_it_is_split(monkeypatch, step):
    """Codes and scales of one allocation become two tensors at their first use.  Whichever step of
    that another thread's read falls on, it sees whole codes and whole scales."""
    import threading
    mx = _mx()
    rows, K = 130, 200
    sizes, scales_shape = mx._BLOCK_BYTES, mx.mx_scales_shape(rows, K)
    t = mx.MXTensor._new(torch.empty(0), rows, (rows, K), "mxfp4", 0)
    main, steps, seen = threading.current_thread(), [], []

    def read():
        try:
            seen.append((tuple(t.data.shape), tuple(t.scales.shape)))
        except Exception as e:                     # reported by the main thread
            seen.append(repr(e))

    def pause():
        if threading.current_thread() is main:
            steps.append(1)
            if len(steps) == step + 1:
                other = threading.Thread(target=read)
                other.start()
                other.join()

    class Sizes:
        def __getitem__(self, i):
            pause()
            return sizes[i]
    monkeypatch.setattr(mx, "_BLOCK_BYTES", Sizes())
    monkeypatch.setattr(mx, "mx_scales_shape", lambda *a: (pause(), scales_shape)[1])
    whole = ((rows, 7 * 16), scales_shape)
    assert (tuple(t.data.shape), tuple(t.scales.shape)) == whole
    assert seen == [whole]
