"""Rotary positions with several axes (no counterpart in the reference): queries and keys of an
attention turned by where their tokens stand in time, height and width.

  rotary_axes(q, k, positions, sections=...) -> q', k'      one launch of snnb_rotary_axes
  grid_positions(T, H, W) -> [T H W, 3]                     the positions of a grid in raster order

The pairs of a head's columns are divided among the axes by `sections`; pair i of axis a turns by
positions[..., a] * frequency(i).  Inference only: outputs carry no gradient (the gradient of a
turned tensor is that tensor's, turned back: inverse=True).
"""
from __future__ import annotations

import ctypes
import functools
import math

import torch

from .. import _lib
from .mx import _dtype, _index, _launch

MAX_PAIRS = 256
_POSITIONS = {torch.int32: 0, torch.int64: 1, torch.float32: 2}


@functools.lru_cache(maxsize=64)
def _ladder(sections: tuple, base: float, ladder: str):
    """(frequency / 2 pi, axis) of every pair, as host arrays."""
    total, turns, axis = sum(sections), [], []
    for a, count in enumerate(sections):
        for j in range(count):
            power = len(turns) / total if ladder == "shared" else j / count
            turns.append(base ** -power / (2.0 * math.pi))
            axis.append(a)
    return (ctypes.c_double * total)(*turns), (ctypes.c_uint8 * total)(*axis)


def _unit_columns(x: torch.Tensor) -> torch.Tensor:
    return x if x.stride(-1) == 1 or x.shape[-1] <= 1 else x.contiguous()


@functools.lru_cache(maxsize=4096)
def _host_array(*values):
    return (ctypes.c_int64 * len(values))(*values)


def _strides(*tensors):
    """The strides of all axes but the last, of one tensor after the other, as a host array."""
    values = ()
    for t in tensors:
        values += t.stride()[:-1]
    return _host_array(*values)


def _output(out, x, what):
    if out is None:
        return x.new_empty(x.shape)
    assert out.shape == x.shape and out.dtype == x.dtype and out.device == x.device and \
        (out.stride(-1) == 1 or out.shape[-1] <= 1), \
        f"rotary_axes: {what} {tuple(out.shape)} {out.dtype} does not fit {tuple(x.shape)} {x.dtype}"
    return out


def rotary_axes(q: torch.Tensor, k: torch.Tensor | None, positions: torch.Tensor, *, sections,
                base: float = 10000.0, ladder: str = "shared", interleaved: bool = False,
                inverse: bool = False, q_out: torch.Tensor | None = None,
                k_out: torch.Tensor | None = None):
    """q [B, N, heads, d] and k [B, N, heads of its own, d] (or None) -> (q', k'), contiguous or in
    q_out and k_out, which may be q and k themselves and otherwise overlap neither.  Rows may be
    strided (slices of a fused projection) without a copy.

    positions [N, axes] or [B, N, axes], int32, int64 or float32; sections: pairs of columns for each
    axis, sum(sections) = R <= d / 2 (and <= 256); columns from 2 R on are copied.  Pair i is
    columns (i, i + R), or (2i, 2i + 1) when interleaved.  Its frequency is base^(-i / R)
    (ladder="shared"), or base^(-j / sections[a]) for the j-th pair of axis a (ladder="axis").
    Angles lose nothing at far positions: they are held in float64 turns."""
    sections = tuple(sections)
    if ladder not in ("shared", "axis"):
        raise ValueError(f"rotary_axes: unknown ladder {ladder!r} (shared or axis)")
    if not 0.0 < base < math.inf:
        raise ValueError(f"rotary_axes: base is {base}")
    dt, shape = _dtype(q.dtype), q.shape
    assert len(shape) == 4, tuple(shape)
    B, N, H, d = shape
    axes, pairs = len(sections), sum(sections)
    if not sections or min(sections) < 0 or pairs < 1 or 2 * pairs > d or pairs > MAX_PAIRS:
        raise ValueError(f"rotary_axes: sections {sections} do not fit a head of {d} columns")
    index = _index(q)
    ptype, place = _POSITIONS.get(positions.dtype), positions.stride()
    assert ptype is not None, f"positions are int32, int64 or float32, got {positions.dtype}"
    if len(place) == 2:
        place = (0,) + place
        assert positions.shape == (N, axes), (tuple(positions.shape), (N, axes))
    else:
        assert positions.shape == (B, N, axes), (tuple(positions.shape), (B, N, axes))
    assert positions.get_device() == index, (positions.device, q.device)
    turns, axis = _ladder(sections, float(base), ladder)
    q = _unit_columns(q)
    qo = _output(q_out, q, "q_out")
    ko, k_args = None, (None, None, 0, None)
    if k is not None:
        ks = k.shape
        assert len(ks) == 4 and ks[0] == B and ks[1] == N and ks[3] == d and \
            k.dtype == q.dtype and k.get_device() == index, (tuple(ks), k.dtype)
        k = _unit_columns(k)
        ko = _output(k_out, k, "k_out")
        k_args = (k.data_ptr(), ko.data_ptr(), ks[2], _strides(k, ko))
    _launch("snnb_rotary_axes", index, q.data_ptr(), qo.data_ptr(), H, _strides(q, qo), *k_args, dt,
            B, N, d, positions.data_ptr(), ptype, _host_array(*place), turns, axis, pairs,
            int(interleaved), int(inverse))
    return qo, ko


def grid_positions(T: int, H: int, W: int, *, start=(0, 0, 0), device="cuda") -> torch.Tensor:
    """[T H W, 3] int32: (time, height, width) of each cell of a T x H x W grid in raster order."""
    axes = [torch.arange(s, s + n, dtype=torch.int32, device=device)
            for s, n in zip(start, (T, H, W))]
    return torch.stack(torch.meshgrid(*axes, indexing="ij"), -1).reshape(-1, 3)
