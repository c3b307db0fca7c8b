"""Sizes that the decay attention's C entries refuse, without a device."""
import ctypes

import pytest


def _call(N, dtype, H=1, d=1):
    from snn_compiler import _lib
    p, zero = ctypes.c_void_p(1 << 20), (ctypes.c_int64 * 3)(0, 0, 0)
    return _lib.lib().snnb_decay_attention(p, zero, p, zero, p, zero, dtype, 1, N, H, H, d, d, p, 1.0, None, None, 0,
                                           p, None, p, 1 << 50, None)


@pytest.mark.parametrize("dtype", [0, 1, 2])
@pytest.mark.parametrize("N", [(1 << 31) - 255, (1 << 31) - 1, 1 << 31, 1 << 35, (1 << 40) - 1])
def test_more_tokens_than_32_bits_count(N, dtype):
    """Chunks, their powers of the decay and tensor maps count tokens in 32 bits.  At 2^35 tokens of one
    head (keys and values may be one token, expanded) a segment has 2^31 tokens, and the loop that forms the
    power of the decay over it would not have ended."""
    from snn_compiler import _lib
    assert _call(N, dtype) == -1
    assert _lib.lib().snnb_decay_attention_workspace_bytes(dtype, 1, N, 1, 1, 1) < 0
