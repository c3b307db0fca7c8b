"""Group norm's statistics on the GPU, of every form: a part of the values that is left out, counted twice or
weighed wrongly has to show, so the last rows and the last channels of each group lie far from the others, and
the tolerances follow the sums as they are made.

A thread sums `rows` rows one after another, and then at most 96 partial sums follow one another (of its block's
threads, a group's channels, a sample's blocks): (rows + 96) 2^-24 of the mean magnitude for the mean; as much
of the variance for its squares, which are taken around the thread's first row and are twice the variance's on
the average; 1.2 (SiLU's slope is below 1.1) times that of the oracle's magnitude d plus |y|; and u |y|.
That each mistake would show is asserted too, on the oracle.
"""
import pytest
import torch

from oracle import sequence as OS
from test_sequence_gpu import DEV, DTYPES, F32, _k, _tiny, _u

pytestmark = pytest.mark.gpu

# (shape, groups, padding of the rows, rows that a thread sums at most)
ONE_PASS = [((1, 70000, 64), 1, 0, 547), ((5, 300, 6, 512), 4, 0, 29), ((64, 28, 28, 256), 32, 0, 13),
            ((3, 700, 90), 5, 6, 700)]
TWO_PASSES = [((1, 140000, 256), 32, 0, 60), ((3, 17000, 700), 7, 0, 87), ((5, 2300, 4096), 1, 0, 80),
              ((2, 13000, 1305), 1, 0, 407), ((70, 56, 56, 256), 32, 3, 392), ((600, 100, 600), 3, 0, 100)]


def _oracle(x, groups, of, w, b, eps):
    """The norm of x with the statistics of `of`, in float64, and its magnitude d."""
    B, S, C = x.shape
    if of is x:
        return OS.group_norm(x, groups, w, b, eps, "silu")
    g = of.double().reshape(B, of.shape[1], groups, -1)
    mean, var = g.mean((1, 3)), g.var((1, 3), unbiased=False)
    mean, var = (t.repeat_interleave(C // groups, 1)[:, None] for t in (mean, var))
    y = (x.double() - mean) / torch.sqrt(var + eps) * w.double() + b.double()
    return y * torch.sigmoid(y), None


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape,groups,pad,rows", ONE_PASS + TWO_PASSES)
def test_every_value_counts_once(shape, groups, pad, rows, dtype):
    from snn_compiler import _lib
    K, C = _k(), shape[-1]
    cg, size = C // groups, 4 if dtype == F32 else 2
    g = torch.Generator(device=DEV).manual_seed(sum(shape))
    x = torch.randn(*shape[:-1], C + pad, generator=g, device=DEV) * 2
    x += torch.randn(C + pad, generator=g, device=DEV) * 3
    S = x[0, ..., 0].numel()
    late = max(1, S // 20)
    x.view(shape[0], S, C + pad)[:, S - late:] += 20                     # the last rows
    last = max(1, cg // 9)
    at = torch.arange(C + pad, device=DEV) % cg >= cg - last             # and channels of each group
    x[..., at] -= 15
    x = x.to(dtype)
    view = x[..., :C]
    w, b = (torch.randn(C, generator=g, device=DEV).to(dtype) for _ in range(2))
    x3 = view.reshape(shape[0], S, C)
    dt = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}[dtype]
    need = _lib.lib().snnb_group_norm_act_workspace_bytes(dt, shape[0], S, C, groups)
    assert (need > 0) == (x3.numel() * size >= 64 << 20)                 # the two passes' workspace
    y = K.group_norm_act(view, groups, w, b, eps=1e-3, act="silu").reshape(shape[0], S, C).double()
    ref, d = _oracle(x3, groups, x3, w, b, 1e-3)
    tol = 1.2 * (rows + 96) * 2.0 ** -24 * (d + ref.abs()) + _u(dtype) * ref.abs() + _tiny(dtype)
    bad = ~((y - ref).abs() <= tol)
    assert not bad.any(), (int(bad.sum()), ((y - ref).abs() / tol).max().item())
    fewer = torch.arange(C, device=DEV) % cg < cg - last
    for of in (x3[:, :S - late], torch.cat([x3, x3[:, S - late:]], 1), x3[..., fewer]):
        wrong, _ = _oracle(x3, groups, of, w, b, 1e-3)
        assert ((wrong - ref).abs() > tol).double().mean() > 0.5
