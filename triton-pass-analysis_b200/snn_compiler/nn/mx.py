"""Low-bit layers on the microscaled operators (no counterpart in the reference).

``MXLinear`` holds a linear layer's weights in 4 bits, ``RMSNormMX`` is the norm in front of it,
and ``SpikingMLP`` runs the two with the multi-step neurons as a pre-norm block:

  h = x + residual;  u = fc1(norm(h))     8-bit activations x 4-bit weights
  s = LIF(u)                              multi-step, [T, ...] spikes
  y = fc2(s)                              spikes are exact in 4 bits: 4-bit x 4-bit

Inference only, as the rest of the package: weights are buffers, outputs carry no gradient.
"""
from __future__ import annotations

import torch
import torch.nn as nn

from ..kernels.mx import MXTensor, mx_linear, mx_quantize, rms_norm_mx
from .modules import LIFNode


class MXLinear(nn.Module):
    """y = x w^T + b with w [out_features, in_features] held in mxfp4 (laid out once).  x is an
    MXTensor, or a tensor that is quantised to `act` ("mxfp8" or "mxfp4") first."""

    def __init__(self, weight: MXTensor, bias: torch.Tensor | None = None, *, act: str = "mxfp8",
                 dtype=torch.bfloat16):
        super().__init__()
        if weight.fmt != "mxfp4":
            raise ValueError(f"MXLinear: the weights are held in mxfp4, got {weight.fmt}")
        if act not in ("mxfp4", "mxfp8"):
            raise ValueError(f"MXLinear: unknown activation format {act!r}")
        self.out_features, self.in_features = weight.shape
        self.act, self.dtype = act, dtype
        self.register_buffer("weight_data", weight.data)
        self.register_buffer("weight_scales", weight.scales)
        self.register_buffer("bias", None if bias is None else bias.detach().float().contiguous())
        self._weight = None

    @classmethod
    def from_linear(cls, linear: nn.Linear, **kw) -> "MXLinear":
        """Quantises linear's weights (on its CUDA device)."""
        return cls(mx_quantize(linear.weight.detach(), "mxfp4"), linear.bias, **kw)

    @property
    def weight(self) -> MXTensor:
        w = self._weight
        # the buffers may have moved (.to(device), load_state_dict into them keeps the storage)
        if w is None or w.data is not self.weight_data or w.scales is not self.weight_scales:
            w = self._weight = MXTensor(self.weight_data, self.weight_scales,
                                        (self.out_features, self.in_features), "mxfp4")
        return w

    def forward(self, x):
        if not isinstance(x, MXTensor):
            x = mx_quantize(x, self.act)
        bias = self.bias
        if bias is not None and bias.dtype != torch.float32:      # after .half() or .to(bfloat16)
            bias = bias.float()
        return mx_linear(x, self.weight, bias, dtype=self.dtype)

    def extra_repr(self):
        return (f"{self.in_features}, {self.out_features}, bias={self.bias is not None}, "
                f"act={self.act}")


class RMSNormMX(nn.Module):
    """(x, residual) -> (the norm of x + residual as an MXTensor of `fmt`, x + residual)."""

    def __init__(self, dim: int, *, eps: float = 1e-6, fmt: str = "mxfp8", weight=None,
                 device=None, dtype=torch.float32):
        super().__init__()
        self.eps, self.fmt = eps, fmt
        w = torch.ones(dim, device=device, dtype=dtype) if weight is None else weight.detach()
        self.register_buffer("weight", w.contiguous())

    def forward(self, x, residual=None):
        w = self.weight
        if w.dtype not in (x.dtype, torch.float32):
            w = w.to(x.dtype)
        return rms_norm_mx(x, w, residual, eps=self.eps, fmt=self.fmt)


class SpikingMLP(nn.Module):
    """The pre-norm spiking MLP block of the module text.  forward(x [T, ..., D], residual) ->
    (y [T, ..., D], h): pass both on to the next block, whose norm adds them."""

    def __init__(self, norm: RMSNormMX, fc1: MXLinear, neuron: nn.Module, fc2: MXLinear):
        super().__init__()
        self.norm, self.fc1, self.neuron, self.fc2 = norm, fc1, neuron, fc2

    @classmethod
    def from_linears(cls, fc1: nn.Linear, fc2: nn.Linear, *, norm_weight=None, eps: float = 1e-6,
                     tau: float = 2.0, v_threshold: float = 1.0, dtype=torch.bfloat16):
        """Quantises two float layers [hidden, D] and [D, hidden]."""
        return cls(RMSNormMX(fc1.in_features, eps=eps, weight=norm_weight,
                             device=fc1.weight.device),
                   MXLinear.from_linear(fc1, act="mxfp8", dtype=dtype),
                   LIFNode(tau=tau, v_threshold=v_threshold),
                   MXLinear.from_linear(fc2, act="mxfp4", dtype=dtype))

    def forward(self, x, residual=None):
        q, h = self.norm(x, residual)
        spikes = self.neuron(self.fc1(q))
        return self.fc2(spikes), h
