"""Rotary positions of more than 32 bits, and negative ones, on the GPU against angles that are reduced
exactly (in 80 digits).

The kernel's angle is position * (frequency / 2 pi) in float64 turns: the power is good to 2^-52 of
itself, 2 pi, the quotient and the product round by 2^-53 each, in all at most 2^-50 of the angle; what
stands in test_sequence_gpu.py for the rest, 2^-21 of the pair and half a step of the output.
"""
import decimal
import math

import pytest
import torch

from test_sequence_gpu import DEV, DTYPES, _gen, _k, _near, _tiny, _u

pytestmark = pytest.mark.gpu
PI = decimal.Decimal("3.14159265358979323846264338327950288419716939937510582097494459230781640628620899863")


def _angles(positions, pairs, base):
    """positions [N] whole -> (cos, sin [N, pairs], |angle|) of position * base^(-i / pairs)."""
    with decimal.localcontext() as c:
        c.prec = 80
        f = [decimal.Decimal(base) ** (-decimal.Decimal(i) / pairs) for i in range(pairs)]
        full = [[n * x for x in f] for n in positions]
        left = [[float(t - 2 * PI * (t / (2 * PI)).to_integral_value()) for t in row] for row in full]
        size = [[abs(float(t)) for t in row] for row in full]
    t = torch.tensor(left, dtype=torch.float64)
    return torch.cos(t), torch.sin(t), torch.tensor(size, dtype=torch.float64)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("base", [1.0, 10000.0])
def test_positions_past_32_bits(base, interleaved, dtype):
    far = [0, 1, -1, -5000, 2 ** 31 - 1, 2 ** 31, -2 ** 31, 2 ** 32 + 3, -2 ** 32 - 3, 3 * 2 ** 33 + 1, -2 ** 36 + 77,
           2 ** 38 + 12345]
    pairs, d = 8, 20
    x = torch.randn(1, len(far), 3, d, generator=_gen(60)).to(dtype)
    pos = torch.tensor(far, dtype=torch.int64)[:, None]
    y = _k().rotary_axes(x.to(DEV), None, pos.to(DEV), sections=(pairs,), base=base, interleaved=interleaved)[0]
    cos, sin, size = _angles(far, pairs, base)
    cos, sin, size = (t[None, :, None] for t in (cos, sin, size))
    xd, ref = x.double(), x.double().clone()
    one, two = (slice(0, 2 * pairs, 2), slice(1, 2 * pairs, 2)) if interleaved else \
        (slice(0, pairs), slice(pairs, 2 * pairs))
    a, b = xd[..., one], xd[..., two]
    ref[..., one], ref[..., two] = a * cos - b * sin, a * sin + b * cos
    tol = torch.zeros_like(ref)
    both = (2.0 ** -21 + 2.0 ** -50 * size) * (a.abs() + b.abs())
    tol[..., one], tol[..., two] = both, both
    _near(y, ref, tol + _u(dtype) * ref.abs() + _tiny(dtype))
    # what the low 32 bits alone would give is something else
    low, _, _ = _angles([((n + 2 ** 31) % 2 ** 32) - 2 ** 31 for n in far], pairs, base)
    assert (low[7:] - cos[0, 7:, 0]).abs().max() > 0.1 and math.isclose(cos[0, 0, 0, 0].item(), 1.0)


def test_back_and_forth_at_far_positions():
    x = torch.randn(2, 50, 2, 64, generator=_gen(61)).to(DEV)
    pos = torch.randint(-2 ** 45, 2 ** 45, (2, 50, 2), generator=_gen(62)).to(DEV)
    kw = dict(sections=(16, 16))
    back = _k().rotary_axes(_k().rotary_axes(x, None, pos, **kw)[0], None, pos, inverse=True, **kw)[0]
    # the same sines and cosines both ways: each turn rounds by 2^-21 of a pair at most
    assert ((back - x).abs() <= 2.0 ** -20 * 2 * x.abs().amax(-1, keepdim=True) * 2).all()
