"""Decay attention of 16-bit inputs is a float32 sum, rounded once, at every length, number of heads and
alignment, against the float64 oracle.

Tolerances, derived: on the tensor cores P and the state are held as two terms of at least 8 bits (2^-16
each of what they hold), sums as in test_sequence_gpu.py, (dk + N / 8 + 64) 2^-23 of the magnitude; the
output's one rounding is half a step of its type.  The state's operands have 22 bits or more: 2^-22
(float16's two terms of 11) and the sums.
"""
import pytest
import torch

from oracle import sequence as OS
from test_sequence_gpu import BF16, DEV, DTYPES, F16, F32, _gen, _k, _lam, _near, _tiny, _tokens, _u
from test_sequence_ranges_gpu import _views

pytestmark = pytest.mark.gpu


def _check(q, k, v, lam, scale=1.0, state=None, lengths=None, pad=0, in_place=False):
    old = None if state is None else state.to(DEV)
    o, S = _k().decay_attention(*_views((q, k, v), pad), lam.to(DEV), scale=scale, state=old,
                                lengths=None if lengths is None else lengths.to(DEV),
                                state_out=old if in_place else None)
    ro, rS, oa, A = OS.decay(q, k, v, lam, scale, state, lengths)
    sums = (q.shape[-1] + q.shape[1] / 8 + 64) * 2.0 ** -23
    terms = 0.0 if q.dtype == F32 else 2.0 ** -15
    _near(o, ro, (terms + sums) * oa + _u(q.dtype) * ro.abs() + _tiny(q.dtype) + 1e-37)
    _near(S, rS, (2.0 ** -22 + sums) * A + 1e-37)
    return o, S, ro


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("pad", [0, 1])
@pytest.mark.parametrize("B,N,H,d", [(1, 2, 1, 64), (1, 8, 2, 64), (1, 9, 1, 128), (2, 33, 1, 48), (1, 64, 1, 64),
                                     (1, 64, 2, 64), (1, 65, 1, 64), (2, 64, 4, 128), (1, 128, 1, 64), (1, 200, 2, 128)])
def test_outputs_are_rounded_once(B, N, H, d, pad, dtype):
    """Of every size alike: no output is off by more than its own rounding and float32's sums, and all
    together by no more than a tenth above the rounding's."""
    q, k, v = _tokens(B, N, H, H, d, d, dtype, 50 + N)
    state = torch.randn(B, H, d, d, generator=_gen(7))
    lam = 1 - torch.exp2(-5.0 - torch.arange(H))
    o, _, ro = _check(q, k, v, lam, d ** -0.5, state, None, pad)
    if dtype != F32 and B * N * H * d >= 512:                 # enough values for a mean
        assert (o.cpu().double() - ro).norm() <= 1.1 * (ro.to(dtype).double() - ro).norm()


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("N,H,d", [(2, 1, 64), (8, 8, 32), (9, 2, 64), (40, 1, 128), (64, 2, 64)])
def test_a_sequence_alone_is_the_one_in_a_batch(N, H, d, dtype):
    """One form takes the same sequence, however many stand beside it: the same bits."""
    q, k, v = (x.to(DEV) for x in _tokens(200, N, H, H, d, d, dtype, 51))
    lam = _lam(H).to(DEV)
    o, S = _k().decay_attention(q, k, v, lam)
    for b in (1, 3):
        a, s = _k().decay_attention(q[:b], k[:b], v[:b], lam)
        assert torch.equal(a, o[:b]) and torch.equal(s, S[:b])


# 9 to 19 chunks of 128 tokens (18 to 38 of 64 on the CUDA cores) of few heads: 3 to 7 segments (9 to 13), each of
# which starts from what those before it leave
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("pad", [0, 1])
@pytest.mark.parametrize("H,Hk,dk,dv,N", [(2, 1, 64, 64, 2390), (1, 1, 128, 128, 1100), (2, 2, 40, 72, 1500)])
def test_long_sequences_in_segments(H, Hk, dk, dv, N, pad, dtype):
    """Lengths that end in the first, a middle and the last segment, at a chunk's border, at none; from no
    state, from one, and in place."""
    B = 6
    q, k, v = _tokens(B, N, H, Hk, dk, dv, dtype, 52)
    lam = torch.tensor([0.999, 0.9])[:H]
    state = torch.randn(B, H, dk, dv, generator=_gen(8)) * 4
    lengths = torch.tensor([0, 1, N // 2, 1024, N - 1, N], dtype=torch.int64)
    o, S, _ = _check(q, k, v, lam, dk ** -0.5, state, lengths, pad)
    for b, n in enumerate(lengths.tolist()):
        assert not o[b, n:].any()
    assert torch.equal(S[0].cpu(), state[0])
    o2, S2, _ = _check(q, k, v, lam, dk ** -0.5, state, lengths, pad, in_place=True)
    assert torch.equal(o2, o) and torch.equal(S2, S)
    _check(q[:1], k[:1], v[:1], lam, dk ** -0.5, None, None, pad)
    o3, S3, _ = _check(q[-1:], k[-1:], v[-1:], lam, dk ** -0.5, state[-1:], None, pad)
    assert torch.equal(o3, o[-1:]) and torch.equal(S3, S[-1:])       # in as many segments
