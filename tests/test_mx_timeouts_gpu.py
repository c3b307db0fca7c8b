"""Waits that run out in the microscaled kernels: with a wait limit far below a product's time, or
with a copy that is withheld, launches give up with copies in flight, let those land and return.
The device status word reads the time-out once, and the next launch with the usual limit is right.

A launch holds the GPU for the limit and at most one wait of the fixed limit that outlasts any copy
(4e9 cycles, 2.1 s at 1.9 GHz), in the pairs for stages that are never handed on."""
import time

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
TIMEOUT = -4


def _gives_up_and_recovers(call, stall=False):
    from snn_compiler import _lib
    from snn_compiler.kernels import conv as KC
    L = _lib.lib()
    want = call()
    flush = torch.empty(1 << 28, dtype=torch.uint8, device=DEV)
    flush.zero_()                                  # the inputs come from memory
    assert KC.device_status() == 0
    try:
        _lib.check(L.snnb_set_wait_limit(1000), "snnb_set_wait_limit")        # ~0.5 us
        if stall:
            _lib.check(L.snnb_debug_inject_stall(1), "snnb_debug_inject_stall")
        t0 = time.time()
        call()
        torch.cuda.synchronize()
        took = time.time() - t0
    finally:
        L.snnb_debug_inject_stall(0)
        L.snnb_set_wait_limit(0)
    assert KC.device_status() == TIMEOUT           # cleared by the read
    assert KC.device_status() == 0
    assert took < 8.0
    got = call()
    assert KC.device_status() == 0
    assert all(torch.equal(a, b) for a, b in zip(got, want))


# one tile with K split (unpacked by the copies, and from a packed ring), pairs of 256 and 128
# tokens, in both formats
@pytest.mark.parametrize("rows,N,K,fmt", [(1, 4096, 8192, "mxfp8"), (1, 4096, 8100, "mxfp8"),
                                          (16, 4096, 8192, "mxfp4"), (2000, 4000, 8192, "mxfp4"),
                                          (2000, 4000, 4096, "mxfp8"), (2000, 4000, 4000, "mxfp8"),
                                          (300, 1000, 1100, "mxfp8")])
def test_linear(rows, N, K, fmt):
    from snn_compiler.kernels import mx
    g = torch.Generator().manual_seed(K)
    a = mx.mx_quantize(torch.randn(rows, K, generator=g).to(DEV), fmt)
    w = mx.mx_quantize(torch.randn(N, K, generator=g).to(DEV))
    _gives_up_and_recovers(lambda: (mx.mx_linear(a, w, dtype=torch.float32),))


# teams of 64, 128, 256 and 512 threads, several turns of the ring
@pytest.mark.parametrize("rows,K", [(16384, 2048), (8192, 4000), (8192, 8192), (4096, 16384)])
def test_norm_ring(rows, K):
    from snn_compiler.kernels import mx
    g = torch.Generator(device=DEV).manual_seed(K)
    x, r = (torch.randn(rows, K, generator=g, device=DEV).to(torch.bfloat16) for _ in range(2))
    w = torch.ones(K, device=DEV)

    def call():
        q, h = mx.rms_norm_mx(x, w, r)
        return q.data, q.scales, h
    _gives_up_and_recovers(call, stall=True)
