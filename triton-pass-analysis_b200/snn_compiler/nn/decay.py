"""Causal linear-attention block on the low-bit operators (no counterpart in the reference, whose
attention blocks sum over all tokens alike).

``DecayAttention`` runs, pre-norm, with the microscaled norm and products around the attention:

  h = x + residual;  [q k v] = qkv(norm(h))         8-bit activations x 4-bit weights
  q, k turned by the tokens' positions              rotary_axes, in place
  S_t = decay S_{t-1} + k_t v_t^T, o_t = q_t S_t    decay_attention, a state that carries over
  u = act(group norm of o's heads), or neuron(it)   group_norm_act
  y = out(u)

``step`` does the same for one token of each sequence.  Inference only, as the rest of the package:
weights are buffers, outputs carry no gradient.
"""
from __future__ import annotations

import torch
import torch.nn as nn

from ..kernels.decay import decay_attention, decay_attention_step
from ..kernels.groupnorm import ACTIVATIONS, group_norm_act
from ..kernels.rotary import rotary_axes
from .mx import MXLinear, RMSNormMX


class GroupNormAct(nn.Module):
    """act(group norm) of channels-last tensors [B, ..., C]."""

    def __init__(self, groups: int, channels: int, *, eps: float = 1e-5, act: str = "none",
                 weight=None, bias=None, device=None, dtype=torch.float32):
        super().__init__()
        if act not in ACTIVATIONS:
            raise ValueError(f"GroupNormAct: unknown activation {act!r}")
        if groups < 1 or channels % groups:
            raise ValueError(f"GroupNormAct: {channels} channels in {groups} groups")
        self.groups, self.eps, self.act = groups, eps, act
        w = torch.ones(channels, device=device, dtype=dtype) if weight is None else weight.detach()
        b = torch.zeros_like(w) if bias is None else bias.detach()
        self.register_buffer("weight", w.contiguous())
        self.register_buffer("bias", b.contiguous())

    @classmethod
    def from_norm(cls, norm: nn.GroupNorm, *, act: str = "none") -> "GroupNormAct":
        """The same norm, of channels-last tensors."""
        return cls(norm.num_groups, norm.num_channels, eps=norm.eps, act=act, weight=norm.weight,
                   bias=norm.bias)

    def forward(self, x, out=None):
        w, b = self.weight, self.bias
        if w.dtype != b.dtype or w.dtype not in (x.dtype, torch.float32):
            w, b = w.to(x.dtype), b.to(x.dtype)
        return group_norm_act(x, self.groups, w, b, eps=self.eps, act=self.act, out=out)

    def extra_repr(self):
        return f"{self.groups}, {self.weight.numel()}, eps={self.eps}, act={self.act}"


class DecayAttention(nn.Module):
    """The block of the module text.  decay: [heads] in [0, 1]; sections, base, ladder as for
    rotary_axes (sections=None: no positions); neuron: a multi-step module in the activation's place
    (x is then [T, ..., N, D]: the neurons run over T, the attention over N)."""

    def __init__(self, norm: RMSNormMX, qkv: MXLinear, out: MXLinear, decay: torch.Tensor, *,
                 heads: int, kv_heads: int | None = None, dk: int, dv: int, sections=None,
                 base: float = 10000.0, ladder: str = "shared", head_norm: GroupNormAct | None = None,
                 neuron: nn.Module | None = None):
        super().__init__()
        kv_heads = heads if kv_heads is None else kv_heads
        if heads < 1 or kv_heads < 1 or heads % kv_heads:
            raise ValueError(f"DecayAttention: {heads} heads do not share {kv_heads} key heads")
        if qkv.out_features != heads * dk + kv_heads * (dk + dv) or out.in_features != heads * dv:
            raise ValueError(f"DecayAttention: projections of {qkv.out_features} and "
                             f"{out.in_features} features for {heads} and {kv_heads} heads of {dk}, {dv}")
        if decay.numel() != heads:
            raise ValueError(f"DecayAttention: {decay.numel()} decays for {heads} heads")
        self.heads, self.kv_heads, self.dk, self.dv = heads, kv_heads, dk, dv
        self.sections = None if sections is None else tuple(sections)
        self.base, self.ladder, self.scale = base, ladder, dk ** -0.5
        self.norm, self.qkv, self.out, self.neuron = norm, qkv, out, neuron
        device = qkv.weight_data.device
        self.head_norm = head_norm if head_norm is not None else \
            GroupNormAct(heads, heads * dv, act="none" if neuron is not None else "silu", device=device)
        self.register_buffer("decay", decay.detach().float().reshape(-1).contiguous().to(device))

    @classmethod
    def from_linears(cls, q: nn.Linear, k: nn.Linear, v: nn.Linear, out: nn.Linear, decay, *, heads: int,
                     kv_heads: int | None = None, norm_weight=None, eps: float = 1e-6,
                     dtype=torch.bfloat16, neuron: nn.Module | None = None, **kw):
        """Quantises four float layers; the head dimensions follow from their sizes."""
        kv_heads = heads if kv_heads is None else kv_heads
        if heads < 1 or kv_heads < 1 or q.out_features % heads or v.out_features % kv_heads or \
                k.out_features * heads != q.out_features * kv_heads:
            raise ValueError(f"DecayAttention: layers of {q.out_features}, {k.out_features} and {v.out_features} "
                             f"features do not divide into {heads} and {kv_heads} heads")
        dk, dv = q.out_features // heads, v.out_features // kv_heads
        parts = (q, k, v)
        joint = nn.Linear(q.in_features, sum(m.out_features for m in parts),
                          bias=any(m.bias is not None for m in parts), device=q.weight.device,
                          dtype=q.weight.dtype)
        with torch.no_grad():
            joint.weight.copy_(torch.cat([m.weight for m in parts]))
            if joint.bias is not None:             # zeros for those without one
                joint.bias.copy_(torch.cat([m.weight.new_zeros(m.out_features) if m.bias is None
                                            else m.bias for m in parts]))
        return cls(RMSNormMX(q.in_features, eps=eps, weight=norm_weight, device=q.weight.device),
                   MXLinear.from_linear(joint, act="mxfp8", dtype=dtype),
                   MXLinear.from_linear(out, act="mxfp8" if neuron is None else "mxfp4", dtype=dtype),
                   torch.as_tensor(decay), heads=heads, kv_heads=kv_heads, dk=dk, dv=dv, neuron=neuron,
                   **kw)

    def _apply(self, fn, recurse=True):
        decay = self.decay
        super()._apply(fn, recurse)
        if self.decay.dtype != torch.float32:      # .half() and the like: 0.999 in bfloat16 is one
            self.decay = decay.to(self.decay.device)
        return self

    def _turn(self, q, k, positions):
        if self.sections is None:
            return
        if positions is None:
            raise ValueError(f"DecayAttention: sections {self.sections} need positions")
        rotary_axes(q, k, positions, sections=self.sections, base=self.base, ladder=self.ladder,
                    q_out=q, k_out=k)

    def _heads(self, row, lead):
        H, Hk, dk, dv = self.heads, self.kv_heads, self.dk, self.dv
        q, k, v = row.view(*lead, -1).split([H * dk, Hk * dk, Hk * dv], -1)
        return (q.unflatten(-1, (H, dk)), k.unflatten(-1, (Hk, dk)), v.unflatten(-1, (Hk, dv)))

    def _finish(self, o, shape):
        u = o.view(-1, self.heads * self.dv)
        u = self.head_norm(u, out=u)
        if self.neuron is not None:
            u = self.neuron(u.view(*shape[:-1], -1))
        return self.out(u).view(*shape[:-1], -1)

    def forward(self, x, positions=None, residual=None, *, state=None, lengths=None):
        """x [..., N, D] (leading axes are sequences), positions [N, axes] or [sequences, N, axes],
        state [sequences, heads, dk, dv] -> (y [..., N, D], h = x + residual, the state behind each
        sequence's last token)."""
        codes, h = self.norm(x, residual)
        N = x.shape[-2]
        q, k, v = self._heads(self.qkv(codes), (x.shape[:-2].numel(), N))
        self._turn(q, k, positions)
        o, state = decay_attention(q, k, v, self.decay, scale=self.scale, state=state, lengths=lengths)
        return self._finish(o, x.shape), h, state

    def step(self, x, state, positions=None, residual=None):
        """x [..., D], one token of each sequence, positions [axes] or [sequences, axes] ->
        (y [..., D], h, state), the state updated in place."""
        codes, h = self.norm(x, residual)
        q, k, v = self._heads(self.qkv(codes), (x.shape[:-1].numel(),))
        if positions is not None:
            positions = positions[None] if positions.dim() == 1 else positions[:, None]
        self._turn(q[:, None], k[:, None], positions)
        o, state = decay_attention_step(q, k, v, self.decay, state, scale=self.scale)
        return self._finish(o, x.shape), h, state
