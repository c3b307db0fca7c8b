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
    """Addresses of (frequency / 2 pi, axis) of every pair, and the arrays, which a caller holds on
    to while it uses the addresses."""
    total, turns, axis = sum(sections), [], []
    for a, count in enumerate(sections):
        for j in range(count):
            power = len(turns) / total if ladder == "shared" else j / count
            turns.append(base ** -power / (2.0 * math.pi))
            axis.append(a)
    turns, axis = (ctypes.c_double * total)(*turns), (ctypes.c_uint8 * total)(*axis)
    return ctypes.addressof(turns), ctypes.addressof(axis), (turns, axis)


@functools.lru_cache(maxsize=4096)
def _host_array(values: tuple):
    """(address, array) of 64-bit integers; a caller holds the array while it uses the address."""
    array = (ctypes.c_int64 * len(values))(*values)
    return ctypes.addressof(array), array


def _rows(x: torch.Tensor):
    """(x with unit column stride: itself where it has one, the strides of its other axes)."""
    strides = x.stride()
    if strides[-1] != 1 and x.shape[-1] > 1:
        x = x.contiguous()
        strides = x.stride()
    return x, strides[:-1]


def _output(out, x, shape, what):
    """(out or a new tensor for it, the strides of all its axes but the last)."""
    if out is None:
        out = x.new_empty(shape)
        return out, out.stride()[:-1]
    strides = out.stride()
    assert out.shape == shape and out.dtype == x.dtype and out.get_device() == x.get_device() and \
        (strides[-1] == 1 or shape[-1] <= 1), \
        f"rotary_axes: {what} {tuple(out.shape)} {out.dtype} does not fit {tuple(shape)} {x.dtype}"
    return out, strides[:-1]


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
    Angles are formed in float64 turns: good to 2^-50 of themselves, however far the position (whole
    positions are exact up to 2^53)."""
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
    turns, axis, _held = _ladder(sections, float(base), ladder)
    q, strides = _rows(q)
    qo, out_strides = _output(q_out, q, shape, "q_out")
    q_strides, _held_q = _host_array(strides + out_strides)
    ko, kp, kop, Hk, k_strides = None, None, None, 0, None
    if k is not None:
        ks = k.shape
        assert len(ks) == 4 and ks[0] == B and ks[1] == N and ks[3] == d and \
            k.dtype == q.dtype and k.get_device() == index, (tuple(ks), k.dtype)
        k, strides = _rows(k)
        ko, out_strides = _output(k_out, k, ks, "k_out")
        kp, kop, Hk = k.data_ptr(), ko.data_ptr(), ks[2]
        k_strides, _held_k = _host_array(strides + out_strides)
    place, _held_p = _host_array(place)
    _launch("snnb_rotary_axes", index, q.data_ptr(), qo.data_ptr(), H, q_strides, kp, kop, Hk,
            k_strides, dt, B, N, d, positions.data_ptr(), ptype, place, turns, axis, pairs,
            1 if interleaved else 0, 1 if inverse else 0)
    return qo, ko


def grid_positions(T: int, H: int, W: int, *, start=(0, 0, 0), device="cuda") -> torch.Tensor:
    """[T H W, 3] int32: (time, height, width) of each cell of a T x H x W grid in raster order."""
    axes = [torch.arange(s, s + n, dtype=torch.int32, device=device)
            for s, n in zip(start, (T, H, W))]
    return torch.stack(torch.meshgrid(*axes, indexing="ij"), -1).reshape(-1, 3)
