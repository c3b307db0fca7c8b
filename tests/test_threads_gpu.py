"""Kernels whose shared memory depends on the sizes, called from several host threads at once.  How
much a kernel may use is a setting of the kernel, not of the launch: no thread's call may take it
from another's, so every call launches and gives the results of a call alone.

The threads call the C entries, which leave them little to do between two launches."""
import threading

import pytest
import torch

from snn_compiler import _lib

pytestmark = pytest.mark.gpu
DEV = "cuda"


class _Case:
    """One call of the C entry `name`; `args` without the stream, `outs` its output tensors."""

    def __init__(self, name, args, outs):
        self.fn, self.args, self.outs = getattr(_lib.lib(), name), args, outs
        _lib.check(self.fn(*args, torch.cuda.current_stream().cuda_stream), name)
        torch.cuda.synchronize()
        self.want = [o.clone() for o in outs]
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()


def _together(cases, calls=20000):
    """One thread for each case, on a stream of its own."""
    failed = []

    def work(case):
        stream = torch.cuda.Stream()
        at = stream.cuda_stream
        for i in range(calls):
            status = case.fn(*case.args, at)
            if status:
                failed.append((case.args, status, i))
                break
        stream.synchronize()
    threads = [threading.Thread(target=work, args=(c,)) for c in cases]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed, failed
    for c in cases:
        assert all(torch.equal(a, b) for a, b in zip(c.outs, c.want))


def test_norms_of_several_lengths():
    """Rows of 2256 and 3256 values share a kernel (128 threads a row), of 4104 and 8184 another."""
    from snn_compiler.kernels import mx
    g = torch.Generator().manual_seed(9)

    def case(K):
        rows = 200
        x, r = (torch.randn(rows, K, generator=g).to(torch.bfloat16).to(DEV) for _ in range(2))
        w = (torch.rand(K, generator=g) + 0.5).to(torch.bfloat16).to(DEV)
        data = torch.empty(rows, (K + 31) // 32 * 32, dtype=torch.uint8, device=DEV)
        scales = torch.empty(mx.mx_scales_shape(rows, K), dtype=torch.uint8, device=DEV)
        h = torch.empty_like(x)
        c = _Case("snnb_rms_norm_mx",
                  (x.data_ptr(), K, r.data_ptr(), K, _lib.BF16, w.data_ptr(), _lib.BF16, 1e-6, rows,
                   K, 1, data.data_ptr(), scales.data_ptr(), h.data_ptr()), (data, scales, h))
        c.inputs = x, r, w
        return c
    _together([case(K) for K in (2256, 3256, 8184, 4104)])


@pytest.mark.parametrize("op", ["conv", "linear"])
def test_first_cuda_call_of_a_thread(op):
    """A host thread whose first CUDA call is one of the entries that describe tensors to the
    copy engine: it has no context of its own yet."""
    from snn_compiler.kernels import conv as C, mx
    g = torch.Generator().manual_seed(14)
    if op == "linear":
        a = mx.mx_quantize(torch.randn(8, 256, generator=g).to(DEV), "mxfp8")
        w = mx.mx_quantize(torch.randn(64, 256, generator=g).to(DEV))
        call = lambda: mx.mx_linear(a, w)
    else:
        x = (torch.rand(4, 2, 8, 8, 64, generator=g) < 0.2).to(torch.bfloat16).to(DEV)
        w = (torch.randn(64, 3, 3, 64, generator=g) * 0.06).to(torch.bfloat16).to(DEV)
        b = (torch.rand(64, generator=g) * 0.9).to(DEV)
        call = lambda: C.conv3x3_lif(x, w, b, tau=2.0, v_threshold=1.0)
    want = call()
    torch.cuda.synchronize()
    got = []

    def work():
        try:
            got.append(call())
        except Exception as e:                     # reported by the main thread
            got.append(repr(e))
    t = threading.Thread(target=work)
    t.start()
    t.join()
    assert isinstance(got[0], torch.Tensor), got
    torch.cuda.synchronize()
    assert torch.equal(got[0], want)


def _first_conv(g, cin, cout, size, pool=False):
    T, B = 4, 2
    x = torch.rand(1, B, cin, size, size, generator=g).to(DEV)
    w = (torch.randn(cout, cin, 3, 3, generator=g) * 0.2).to(DEV)
    b = (torch.rand(cout, generator=g) * 0.6).to(DEV)
    side = size // 2 if pool else size
    out = torch.empty(T, B, side, side, cout, device=DEV, dtype=torch.bfloat16)
    c = _Case("snnb_first_conv_lif",
              (x.data_ptr(), 1, T, B, cin, size, size, w.data_ptr(), b.data_ptr(), cout, 0.5, 0.5,
               1.0, 0.0, 1, int(pool), out.data_ptr()), (out,))
    c.inputs = x, w, b
    return c


def test_first_convs_of_several_sizes():
    """The image layer over quads of pixels, whose shared memory goes by channels and width."""
    g = torch.Generator().manual_seed(10)
    _together([_first_conv(g, 3, 64, 32), _first_conv(g, 1, 16, 16), _first_conv(g, 2, 64, 32),
               _first_conv(g, 1, 32, 32)])


def test_first_convs_of_bands_of_several_sizes():
    """Over bands of rows, with weights that a quad's shared memory does not hold."""
    g = torch.Generator().manual_seed(12)
    _together([_first_conv(g, 16, 128, 32), _first_conv(g, 14, 128, 8), _first_conv(g, 16, 128, 64),
               _first_conv(g, 15, 128, 16)])


def test_pooled_first_convs_of_several_sizes():
    g = torch.Generator().manual_seed(13)
    _together([_first_conv(g, 3, 64, 32, True), _first_conv(g, 1, 16, 16, True),
               _first_conv(g, 8, 64, 16, True), _first_conv(g, 2, 32, 16, True)])


def test_band_convs_of_several_sizes():
    """Row-band convolutions of 64 and 128 input channels over rows of 8 and 32 pixels."""
    g = torch.Generator().manual_seed(11)

    def case(cin, W, variant):
        T, B = 4, 2
        x = (torch.rand(T, B, W, W, cin, generator=g) < 0.2).to(torch.bfloat16).to(DEV)
        w = (torch.randn(64, 3, 3, cin, generator=g) * 0.06).to(torch.bfloat16).to(DEV)
        b = (torch.rand(64, generator=g) * 0.9).to(DEV)
        out = torch.empty(T, B, W, W, 64, device=DEV, dtype=torch.bfloat16)
        c = _Case("snnb_conv3x3_lif",
                  (x.data_ptr(), T, B, W, W, cin, w.data_ptr(), b.data_ptr(), 64, 0.5, 0.5, 1.0,
                   0.0, 1, 0, variant, 32, 1, None, 0, out.data_ptr()), (out,))
        c.inputs = x, w, b
        return c
    _together([case(64, 8, 3), case(128, 32, 3), case(64, 8, 7), case(128, 32, 7)])
