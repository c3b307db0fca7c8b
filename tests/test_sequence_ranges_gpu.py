"""Decay attention on the GPU where values of one sequence lie orders of magnitude apart, against the
float64 oracle (oracle/sequence.py) at the bounds of test_sequence_gpu.py.

float16 holds 2^-24 to 2^16, scores, states and sums far more: what one token or one column holds may not
cost the others their bits, whatever form (tensor cores, or CUDA cores for rows that are not aligned) runs.
"""
import pytest
import torch

from oracle import sequence as OS
from test_sequence_gpu import BF16, DEV, DTYPES, F16, F32, _decay_tol, _gen, _k, _lam, _near, _tokens

pytestmark = pytest.mark.gpu


def _views(xs, pad):
    """On the GPU, in rows of odd strides where pad is odd."""
    out = []
    for x in xs:
        row = torch.zeros(*x.shape[:2], x.shape[2] * x.shape[3] + pad, dtype=x.dtype, device=DEV)
        view = row[..., pad:].unflatten(-1, x.shape[2:])
        view.copy_(x.to(DEV))
        out.append(view)
    return out


def _check(q, k, v, lam, scale=1.0, state=None, lengths=None, pad=0):
    o, S = _k().decay_attention(*_views((q, k, v), pad), lam.to(DEV), scale=scale,
                                state=None if state is None else state.to(DEV),
                                lengths=None if lengths is None else lengths.to(DEV))
    ro, rS, oa, A = OS.decay(q, k, v, lam, scale, state, lengths)
    to, tS = _decay_tol(ro, oa, rS, A, q.dtype, q.shape[-1], q.shape[1])
    assert ro.abs().max() < torch.finfo(q.dtype).max
    _near(o, ro, to)
    _near(S, rS, tS)
    return o, S


LAM = torch.tensor([0.97, 1.0, 0.5, 0.999])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("pad", [0, 1])
@pytest.mark.parametrize("d", [64, 128, 48])
@pytest.mark.parametrize("small,large", [(1.0, 100.0), (0.1, 1000.0), (1.0, 10000.0), (0.01, 100.0), (0.01, 1000.0)])
def test_rows_beside_large_ones(small, large, d, pad, dtype):
    """Rows of q and k 10^2 to 10^5 apart in one chunk; rows before the large ones are the same with them
    as without them."""
    q, k, v = _tokens(1, 150, 4, 4, d, d, dtype, 40)
    q, k = (q.float() * small).to(dtype), (k.float() * small * d ** 0.5).to(dtype)
    scale = {100.0: 1.0, 1000.0: 0.08, 10000.0: 1e-3}[large]  # outputs stay in float16's range
    before, _ = _check(q, k, v, LAM, scale, pad=pad)
    q2, k2 = q.clone(), k.clone()
    q2[:, 110] = torch.randn(4, d, generator=_gen(1)) * large
    k2[:, 100] = torch.randn(4, d, generator=_gen(2)) * large / 8
    after, _ = _check(q2, k2, v, LAM, scale * 0.125, pad=pad)
    again, _ = _check(q, k, v, LAM, scale * 0.125, pad=pad)
    assert torch.equal(after[:, :100], again[:, :100])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("pad", [0, 1])
@pytest.mark.parametrize("dk,dv", [(64, 64), (128, 96), (40, 72)])
def test_columns_beside_large_ones(dk, dv, pad, dtype):
    """Columns of v and of the state 10^-4 to 10^5 apart."""
    q, k, v = _tokens(2, 300, 4, 2, dk, dv, dtype, 41)
    size = 10.0 ** (torch.arange(dv) % 8 - 4.0)
    state = torch.randn(2, 4, dk, dv, generator=_gen(3)) * size.flip(0)
    v = (v.float().clamp(-3, 3) * 0.2 * size).to(dtype)
    q = q * 0.05
    _check(q.to(dtype), k, v, LAM, 0.05, state, torch.tensor([300, 131], dtype=torch.int32), pad)
    # one large value in a column of small ones, not the last token
    v[:, 40, :, 5] = 5e4
    q[:, :, :, :] *= 0.01
    _check(q.to(dtype), k, v, LAM, 0.05, state, None, pad)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("pad", [0, 1])
def test_smallest_and_largest_values(pad, dtype):
    """Subnormals of float16 beside its largest values, zeros, states far outside its range."""
    B, N, H, d = 1, 260, 4, 64
    q, k, v = _tokens(B, N, H, H, d, d, dtype, 42)
    rows = 2.0 ** (torch.arange(N) * 7 % 29 - 14.0)[None, :, None, None]
    q, k = (q.float().clamp(-3, 3) * rows).to(dtype), (k.float() * rows.flip(1)).to(dtype)
    q[:, 7], k[:, 9], k[:, 128:150] = 0, 0, 0
    _check(q, k, v, LAM, 2.0 ** -16, pad=pad)
    _check(q, (k.float() * 2.0 ** -10).to(dtype), v, LAM, 2.0 ** -8, pad=pad)
    for size in (1e-30, 1e-12, 1e12):
        state = torch.randn(B, H, d, d, generator=_gen(4)) * size
        q1, k1, v1 = _tokens(B, N, H, H, d, d, dtype, 43)
        _check(q1, k1, v1, LAM, min(1.0, 1.0 / size), state, pad=pad)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("pad", [0, 1])
@pytest.mark.parametrize("N,d", [(64, 64), (120, 128), (48, 48)])
def test_a_state_of_single_tokens(N, d, pad, dtype):
    """Keys that are unit vectors, one token each: a row of the state is decay^(N-1-j) v_j, rounded when
    the power is made, in their product and where terms are put together: three halves of 2^-23, and
    float16's two terms of 11 bits leave 2^-23 of a value.  Nothing but that token is in its row, so a
    decayed one stands beside nothing there, while on the tensor cores float16 holds it beside the
    largest |v| of the chunk, m: brought to [2^14, 2^15), the first term of a value is off by 2^-25 at
    most however small it is, what that leaves is multiplied by 2^11 and again off by 2^-25, so
    2^-36 remain of 2^14: 2^-50 m."""
    _, _, v = _tokens(2, N, 4, 4, d, d, dtype, 44)
    k = torch.zeros(2, N, 4, d, dtype=dtype)
    k[:, torch.arange(N), :, torch.arange(N) % d] = 1
    q = k.roll(3, 1)
    _, S = _k().decay_attention(*_views((q, k, v), pad), LAM.to(DEV))
    _, rS, _, _ = OS.decay(q, k, v, LAM)
    largest = v.double().abs().amax((1, 3))[:, :, None, None]
    _near(S, rS, 2.0 ** -21 * rS.abs() + (2.0 ** -50 * largest if dtype == F16 else 0.0) + 1e-37)


@pytest.mark.parametrize("pad", [0, 1])
def test_float16_values_that_are_not_finite(pad):
    """An infinity or a NaN in q, k, v or the state spoils what it reaches, and nothing else loses bits."""
    lam = torch.tensor([0.9, 1.0])
    q, k, v = _tokens(1, 300, 2, 2, 64, 64, F16, 45)
    state = torch.randn(1, 2, 64, 64, generator=_gen(5))
    ref, rS = _k().decay_attention(*_views((q, k, v), pad), lam.to(DEV), state=state.to(DEV))
    for bad in (float("inf"), float("-inf"), float("nan")):
        x = q.clone()
        x[0, 150, 0, 5] = bad
        o, S = _k().decay_attention(*_views((x, k, v), pad), lam.to(DEV), state=state.to(DEV))
        assert not o[0, 150, 0].isfinite().any() and torch.equal(S, rS)
        keep = torch.arange(300) != 150
        assert torch.equal(o[:, keep], ref[:, keep])
        x = state.clone()
        x[0, 1, 3, 7] = bad
        o, S = _k().decay_attention(*_views((q, k, v), pad), lam.to(DEV), state=x.to(DEV))
        assert not o[0, :, 1, 7].isfinite().any() and not S[0, 1, 3, 7].isfinite()
        others = [c for c in range(64) if c != 7]
        assert torch.equal(o[..., others], ref[..., others]) and torch.equal(o[:, :, 0], ref[:, :, 0])
        assert torch.equal(S[..., others], rS[..., others])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("pad", [0, 1])
@pytest.mark.parametrize("size", [1e-30, 1e30])
def test_scale_that_undoes_the_state(size, pad, dtype):
    """A scale of 1e-30 beside a state of 1e30: what a decayed state leaves is a number of ordinary size
    or far below it, never one that the scale pushed out of float32's range on the way."""
    q, k, v = _tokens(1, 260, 4, 4, 64, 64, dtype, 46)
    state = torch.randn(1, 4, 64, 64, generator=_gen(6)) * size
    _check(q, k, v, LAM, min(1.0, 1.0 / size), state, pad=pad)
