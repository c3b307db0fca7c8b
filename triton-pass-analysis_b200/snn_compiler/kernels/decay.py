"""Linear attention with a decay for each head (no counterpart in the reference, whose spiking
attention sums over all tokens alike): causal, with a state that carries over.

  S_t = decay S_{t-1} + k_t v_t^T,   o_t = scale q_t S_t

  decay_attention(q, k, v, decay, ...) -> o, S         whole sequences, in chunks
  decay_attention_step(q, k, v, decay, S, ...) -> o, S  one token of each sequence

Tokens are [B, N, heads, d], as a projection leaves them; the state is [B, heads, dk, dv] float32.
Key and value heads may be fewer than query heads: query head h reads head h // (H // Hkv).
Inference only: outputs carry no gradient.
"""
from __future__ import annotations


import functools

import torch

from .. import _lib
from .mx import _dtype, _index, _launch
from .rotary import _host_array, _rows

MAX_DIM = 256


def _check(q, k, v, decay, lead, what):
    """Argument checks shared by the two forms -> (dtype code, device index, H, Hkv, dk, dv)."""
    dt, n, qs, ks, vs = _dtype(q.dtype), len(lead), q.shape, k.shape, v.shape
    assert len(qs) == len(ks) == len(vs) == n + 2, (tuple(qs), tuple(ks), tuple(vs))
    H, dk, Hkv, dv = qs[n], qs[n + 1], vs[n], vs[n + 1]
    assert ks[:n] == vs[:n] == lead and ks[n] == Hkv and ks[n + 1] == dk, \
        (tuple(qs), tuple(ks), tuple(vs))
    assert k.dtype == v.dtype == q.dtype, (q.dtype, k.dtype, v.dtype)
    if H < 1 or Hkv < 1 or H % Hkv:
        raise ValueError(f"{what}: {H} query heads do not share {Hkv} key heads")
    if not 1 <= dk <= MAX_DIM or not 1 <= dv <= MAX_DIM:
        raise ValueError(f"{what}: heads of {dk} and {dv} columns (1 to {MAX_DIM})")
    index = _index(q)
    assert k.get_device() == v.get_device() == decay.get_device() == index, \
        (q.device, k.device, v.device, decay.device)
    assert decay.dtype == torch.float32 and decay.shape == (H,) and \
        decay.is_contiguous(), (tuple(decay.shape), decay.dtype)
    return dt, index, H, Hkv, dk, dv


def _state(state, shape, index, what):
    assert state.dtype == torch.float32 and state.shape == shape and \
        state.is_contiguous() and state.get_device() == index, \
        f"{what}: a contiguous float32 {shape} is needed, got {tuple(state.shape)} {state.dtype}"
    return state


def _out(out, shape, q, what):
    if out is None:
        return q.new_empty(shape)
    assert out.shape == shape and out.dtype == q.dtype and out.is_contiguous() and \
        out.get_device() == q.get_device(), f"{what}: out {tuple(out.shape)} {out.dtype}"
    return out


@functools.lru_cache(maxsize=4096)
def _workspace(dt, B, N, H, dk, dv, index):
    """Bytes of workspace; they follow from the sizes and, on the tensor cores, the device's number of SMs."""
    with torch.cuda.device(index):
        return _lib.lib().snnb_decay_attention_workspace_bytes(dt, B, N, H, dk, dv)


def decay_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, decay: torch.Tensor, *,
                    scale: float = 1.0, state: torch.Tensor | None = None,
                    lengths: torch.Tensor | None = None, out: torch.Tensor | None = None,
                    state_out: torch.Tensor | None = None):
    """q [B, N, H, dk], k [B, N, Hkv, dk], v [B, N, Hkv, dv] (float32, float16 or bfloat16; rows may
    be strided) and decay [H] float32 in [0, 1] -> (o [B, N, H, dv] of q's type, the state after each
    sequence's last token [B, H, dk, dv] float32).

    state: the state before the first token (zero without one); state_out receives the state
    behind the last and may be `state` itself.  lengths [B] int32 or int64: tokens of each sequence,
    clamped to [0, N]; what lies behind them is not used, o is zero there, and the state is that
    after the last token (`state` for a length of zero).  dk, dv: 1 to 256, N below 2^31 - 255.  Powers, sums and the
    state are held in float32.  16-bit operands of the tensor cores are held to 2^-16 of themselves or better: an
    output is off by half a step of its type and about 2^-15 of the sum of its terms' magnitudes, and a state by a
    float32 sum's error and 2^-22 of that sum.  float16 has less range than that: beside it, scores are held there
    to 2^-49 of 128 |q_i| times the largest |k_j| so far, values to 2^-50 of their chunk's largest and the state
    that q reads to 2^-50 of its largest (64 columns of v at a time).  out and state_out overlap no other argument (but for state_out, state
    as a whole).  A token that is not finite shows in itself and those behind it only."""
    assert q.dim() == 4, tuple(q.shape)
    B, N = q.shape[:2]
    dt, index, H, Hkv, dk, dv = _check(q, k, v, decay, q.shape[:2], "decay_attention")
    sshape = (B, H, dk, dv)
    if state is not None:
        _state(state, sshape, index, "decay_attention: state")
    if state_out is None:
        state_out = decay.new_empty(sshape)
    else:
        _state(state_out, sshape, index, "decay_attention: state_out")
    ltype = 0
    if lengths is not None:
        assert lengths.dtype in (torch.int32, torch.int64) and tuple(lengths.shape) == (B,) and \
            lengths.is_contiguous() and lengths.get_device() == index, \
            (tuple(lengths.shape), lengths.dtype)
        ltype = 1 if lengths.dtype == torch.int64 else 0
    out = _out(out, (B, N, H, dv), q, "decay_attention")
    need = _workspace(dt, B, N, H, dk, dv, index)
    work = torch.empty(need, dtype=torch.uint8, device=q.device) if need > 0 else None
    (q, qs), (k, ks), (v, vs) = _rows(q), _rows(k), _rows(v)
    (qs, _held_q), (ks, _held_k), (vs, _held_v) = _host_array(qs), _host_array(ks), _host_array(vs)
    _launch("snnb_decay_attention", index, q.data_ptr(), qs, k.data_ptr(), ks, v.data_ptr(), vs, dt, B, N, H, Hkv, dk, dv, decay.data_ptr(), scale,
            None if state is None else state.data_ptr(),
            None if lengths is None else lengths.data_ptr(), ltype, out.data_ptr(),
            state_out.data_ptr(), None if work is None else work.data_ptr(), max(need, 0))
    return out, state_out


def decay_attention_step(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, decay: torch.Tensor,
                         state: torch.Tensor, *, scale: float = 1.0,
                         out: torch.Tensor | None = None, state_out: torch.Tensor | None = None):
    """One token of each sequence: q [B, H, dk], k [B, Hkv, dk], v [B, Hkv, dv], state [B, H, dk, dv]
    float32 -> (o [B, H, dv], the new state), the state updated in place unless state_out is
    given.  out and state_out overlap no other argument (but for state_out, state as a whole)."""
    assert q.dim() == 3, tuple(q.shape)
    B = q.shape[0]
    dt, index, H, Hkv, dk, dv = _check(q, k, v, decay, q.shape[:1], "decay_attention_step")
    sshape = (B, H, dk, dv)
    _state(state, sshape, index, "decay_attention_step: state")
    state_out = state if state_out is None else \
        _state(state_out, sshape, index, "decay_attention_step: state_out")
    out = _out(out, (B, H, dv), q, "decay_attention_step")
    (q, qs), (k, ks), (v, vs) = _rows(q), _rows(k), _rows(v)
    (qs, _held_q), (ks, _held_k), (vs, _held_v) = _host_array(qs), _host_array(ks), _host_array(vs)
    _launch("snnb_decay_attention_step", index, q.data_ptr(), qs, k.data_ptr(), ks, v.data_ptr(), vs, dt, B, H, Hkv, dk, dv, decay.data_ptr(), scale,
            state.data_ptr(), out.data_ptr(), state_out.data_ptr())
    return out, state_out
