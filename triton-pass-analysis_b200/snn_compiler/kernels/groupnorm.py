"""Group norm with an activation on channels-last tensors (no counterpart in the reference): NHWC
images beside the convolutions, and each token's heads behind an attention.

  group_norm_act(x, groups, weight, bias, ...) -> act((x - mean) / sqrt(var + eps) * weight + bias)

Inference only: outputs carry no gradient.
"""
from __future__ import annotations

import functools

import torch

from .. import _lib
from .mx import _DTYPES, _dtype, _index, _launch

MAX_CHANNELS = 16384
ACTIVATIONS = {"none": 0, "silu": 1, "relu": 2, "gelu": 3}


@functools.lru_cache(maxsize=4096)
def _workspace(dt, B, S, C, groups):
    return _lib.lib().snnb_group_norm_act_workspace_bytes(dt, B, S, C, groups)


def group_norm_act(x: torch.Tensor, groups: int, weight: torch.Tensor | None = None,
                   bias: torch.Tensor | None = None, *, eps: float = 1e-5, act: str = "none",
                   out: torch.Tensor | None = None) -> torch.Tensor:
    """x [B, ..., C] (float32, float16 or bfloat16), its C channels in `groups` groups; the mean and
    the biased variance of a group are over its channels and all axes between the first and the
    last, in float32.  weight and bias [C], of x's type or float32 (the same for both); act "none",
    "silu", "relu" or "gelu" (the exact form).  Rows may be strided (a slice of a wider tensor)
    without a copy; the output is contiguous, of x's type; `out` may be x where that is contiguous, and
    otherwise does not overlap it."""
    dt, shape = _dtype(x.dtype), x.shape
    code = ACTIVATIONS.get(act)
    if code is None:
        raise ValueError(f"group_norm_act: unknown activation {act!r} (one of {sorted(ACTIVATIONS)})")
    if not eps >= 0.0:
        raise ValueError(f"group_norm_act: eps is {eps}")
    assert len(shape) >= 2, f"group_norm_act: x is [B, ..., C], got {tuple(shape)}"
    B, C = shape[0], shape[-1]
    if groups < 1 or C < 1 or C % groups or C > MAX_CHANNELS:
        raise ValueError(f"group_norm_act: {C} channels in {groups} groups (up to {MAX_CHANNELS})")
    index = _index(x)
    wd = None
    for name, t in (("weight", weight), ("bias", bias)):
        if t is None:
            continue
        assert t.dtype in (x.dtype, torch.float32) and t.is_contiguous() and t.numel() == C and \
            t.get_device() == index and wd in (None, t.dtype), \
            f"group_norm_act: {name} {tuple(t.shape)} {t.dtype} beside x {tuple(shape)} {x.dtype}"
        wd = t.dtype
    if out is None:
        out = x.new_empty(shape)
    else:
        assert out.shape == shape and out.dtype == x.dtype and out.is_contiguous() and \
            out.get_device() == index, (tuple(out.shape), out.dtype)
    if x.numel() == 0:
        return out
    # [B, S, C] with unit column stride: a view where x has one
    x3 = x.view(B, 1, C) if x.dim() == 2 else x.flatten(1, -2)
    if x3.stride(2) != 1 and C > 1:
        x3 = x3.contiguous()
    need = _workspace(dt, B, x3.shape[1], C, groups)
    work = x.new_empty(need, dtype=torch.uint8) if need > 0 else None
    _launch("snnb_group_norm_act", index, x3.data_ptr(), x3.stride(0), x3.stride(1), dt, B,
            x3.shape[1], C, groups, None if weight is None else weight.data_ptr(),
            None if bias is None else bias.data_ptr(), _DTYPES[wd or torch.float32], eps, code,
            out.data_ptr(), None if work is None else work.data_ptr(), max(need, 0))
    return out
