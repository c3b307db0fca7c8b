"""nn.DecayAttention built from float layers, and its single tokens, on the GPU."""
import pytest
import torch
import torch.nn as nn

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _linears(biases, D=96, H=6, Hk=3, d=32):
    torch.manual_seed(4)
    sizes = ((D, H * d), (D, Hk * d), (D, Hk * d), (H * d, D))
    return [nn.Linear(i, o, bias=b).to(DEV, torch.bfloat16) for (i, o), b in zip(sizes, biases)]


@pytest.mark.parametrize("biases", [(True, False, True), (False, False, True), (False, True, False),
                                    (True, False, False), (False, False, False), (True, True, True)])
def test_biases_of_some_projections(biases):
    """The joint projection gives what each layer by itself gives, whichever of them have a bias."""
    from snn_compiler import kernels as K
    from snn_compiler.nn import DecayAttention, MXLinear
    layers = _linears(biases + (True,))
    m = DecayAttention.from_linears(*layers, torch.full((6,), 0.9), heads=6, kv_heads=3)
    x = torch.randn(7, 96, generator=torch.Generator().manual_seed(5)).to(torch.bfloat16).to(DEV)
    codes = K.mx_quantize(x, "mxfp8")
    want = torch.cat([MXLinear.from_linear(p)(codes) for p in layers[:3]], -1)
    got = m.qkv(codes)
    # the same products and sums, at most in another order: float32 sums of 96 terms, rounded once
    assert ((got - want).float().abs() <= 2.0 ** -7 * want.float().abs() + 2.0 ** -14).all()
    assert (m.qkv.bias is not None) == any(biases)
