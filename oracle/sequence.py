"""Float64 oracle of the linear-attention block's operators, from their definitions: rotary positions
with several axes, linear attention with a decay per head (token by token), group norm.  Each also
gives the magnitudes that rounding errors are relative to."""
import math

import torch


def rotary(x, positions, sections, base=10000.0, ladder="shared", interleaved=False,
           inverse=False):
    """x [B, N, heads, d], positions [B, N, axes] -> (y, |a| + |b| of each value's pair)."""
    x = x.double()
    y, mag = x.clone(), x.abs()
    total, i = sum(sections), 0
    for a, count in enumerate(sections):
        for j in range(count):
            f = base ** -((i / total) if ladder == "shared" else (j / count))
            t = positions[..., a].double() * f * (-1.0 if inverse else 1.0)
            c, s = torch.cos(t)[..., None], torch.sin(t)[..., None]
            p, r = (2 * i, 2 * i + 1) if interleaved else (i, i + total)
            y[..., p] = x[..., p] * c - x[..., r] * s
            y[..., r] = x[..., p] * s + x[..., r] * c
            both = x[..., p].abs() + x[..., r].abs()
            mag[..., p] = both
            mag[..., r] = both
            i += 1
    return y, mag


def _expand(x, H):
    return x.double().repeat_interleave(H // x.shape[-2], dim=-2)


def decay(q, k, v, lam, scale=1.0, state=None, lengths=None):
    """The recurrence over q [B, N, H, dk], k, v [B, N, Hkv, d] -> (o, S, |o|, |S|): the outputs, and
    the same with every factor's magnitude."""
    B, N, H, dk = q.shape
    q, k, v = q.double(), _expand(k, H), _expand(v, H)
    lam = lam.double()[:, None, None]
    dv = v.shape[-1]
    S = torch.zeros(B, H, dk, dv, dtype=torch.float64) if state is None else state.double().clone()
    A = S.abs()
    o = torch.zeros(B, N, H, dv, dtype=torch.float64)
    oa = torch.zeros_like(o)
    for b in range(B):
        n = N if lengths is None else min(max(int(lengths[b]), 0), N)
        for t in range(n):
            S[b] = lam * S[b] + k[b, t, :, :, None] * v[b, t, :, None, :]
            A[b] = lam * A[b] + (k[b, t, :, :, None] * v[b, t, :, None, :]).abs()
            o[b, t] = (q[b, t, :, :, None] * S[b]).sum(-2) * scale
            oa[b, t] = (q[b, t, :, :, None].abs() * A[b]).sum(-2) * abs(scale)
    return o, S, oa, A


def group_norm(x, groups, weight=None, bias=None, eps=1e-5, act="none"):
    """x [B, S, C] -> (y, d): the output, and the magnitude of what a relative error of the mean, the
    variance and the products moves y by."""
    B, S, C = x.shape
    x = x.double()
    g = x.reshape(B, S, groups, C // groups)
    mean = g.mean((1, 3), keepdim=True)
    var = ((g - mean) ** 2).mean((1, 3), keepdim=True)
    r = 1.0 / torch.sqrt(var + eps)
    y = (g - mean) * r
    d = y.abs() + (g.abs() + g.abs().mean((1, 3), keepdim=True)) * r
    y, d = y.reshape(B, S, C), d.reshape(B, S, C)
    if weight is not None:
        y, d = y * weight.double(), d * weight.double().abs()
    if bias is not None:
        y, d = y + bias.double(), d + bias.double().abs()
    if act == "silu":
        y = y * torch.sigmoid(y)
    elif act == "relu":
        y = torch.where(y < 0, 0.0, y)
    elif act == "gelu":
        y = 0.5 * y * (1 + torch.erf(y / math.sqrt(2.0)))
    return y, d
