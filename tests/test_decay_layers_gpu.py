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


def _block(D=96, H=6, Hk=3, d=32):
    from snn_compiler.nn import DecayAttention
    return DecayAttention.from_linears(*_linears((True,) * 4, D, H, Hk, d), 1 - torch.exp2(-1.0 - torch.arange(H)),
                                       heads=H, kv_heads=Hk, sections=(4, 6, 6))


def _inputs(*shape):
    g = torch.Generator().manual_seed(6)
    return [torch.randn(*shape, generator=g).to(torch.bfloat16).to(DEV) for _ in range(2)]


def _near(got, ref, tol):
    off = (got.cpu().double() - ref).abs()
    assert (off <= tol).all(), (off / tol).max().item()


def _linear(codes, m):
    """A product of microscaled operands in float64 and the bound of its float32 sums, rounded once."""
    a, w = (t.dequantize(torch.float32).cpu().double() for t in (codes, m.weight))
    y = a @ w.t() + m.bias.cpu().double()
    return y, 2.0 ** -18 * (a.abs() @ w.abs().t() + m.bias.cpu().double().abs()) + 2.0 ** -8 * y.abs() + 1e-30


def test_step_is_its_operators_in_a_row_and_near_the_oracle():
    """A step's output and state are those of its operators, bit for bit, and each of those is near its
    definition in float64 on what the one before it gave (the norm's codes: its own tests)."""
    from oracle import sequence as OS
    from snn_compiler import kernels as K
    m = _block()
    x, r = _inputs(5, 96)
    pos = torch.randint(0, 5000, (5, 3), generator=torch.Generator().manual_seed(7), dtype=torch.int32).to(DEV)
    old = torch.randn(5, 6, 32, 32, generator=torch.Generator().manual_seed(8)).to(DEV)
    state = old.clone()
    y, h, S = m.step(x, state, pos, r)
    assert S is state
    codes, h2 = K.rms_norm_mx(x, m.norm.weight, r)
    assert torch.equal(h, h2) and torch.equal(h, x + r)
    row = m.qkv(codes)
    _near(row, *_linear(codes, m.qkv))
    q, k, v = (t.unflatten(-1, (-1, 32)) for t in row.split([192, 96, 96], -1))
    q2, k2 = K.rotary_axes(q[:, None], k[:, None], pos[:, None], sections=(4, 6, 6))
    for a, b in ((q, q2), (k, k2)):
        ref, mag = OS.rotary(a[:, None].cpu(), pos[:, None].cpu(), (4, 6, 6))
        _near(b, ref, 2.0 ** -21 * mag + 2.0 ** -8 * ref.abs() + 1e-30)
    o, S2 = K.decay_attention_step(q2[:, 0], k2[:, 0], v, m.decay, old.clone(), scale=32 ** -0.5)
    assert torch.equal(S, S2)
    ro, rS, oa, A = OS.decay(q2.cpu(), k2.cpu(), v[:, None].cpu(), m.decay.cpu(), 32 ** -0.5, old.cpu())
    _near(o[:, None], ro, (32 + 16) * 2.0 ** -23 * oa + 2.0 ** -8 * ro.abs() + 1e-30)
    _near(S, rS, 2.0 ** -22 * A + 1e-30)
    u = K.group_norm_act(o.view(5, 192), 6, m.head_norm.weight, m.head_norm.bias, act="silu")
    ru, d = OS.group_norm(o.view(5, 1, 192).cpu(), 6, m.head_norm.weight.cpu(), m.head_norm.bias.cpu(), act="silu")
    _near(u[:, None], ru, 1.2 * 49 * 2.0 ** -24 * (d + ru.abs()) + 2.0 ** -8 * ru.abs() + 1e-30)
    codes = K.mx_quantize(u, "mxfp8")
    assert torch.equal(y, m.out(codes))
    _near(y, *_linear(codes, m.out))


def test_sequence_is_near_the_oracle():
    """The same of a sequence's projections, norm of heads and output."""
    from oracle import sequence as OS
    from snn_compiler import kernels as K
    m = _block()
    x, r = _inputs(2, 150, 96)
    pos = K.grid_positions(6, 5, 5)
    y, h, S = m(x, pos, r)
    codes, _ = K.rms_norm_mx(x, m.norm.weight, r)
    row = m.qkv(codes)
    ref, tol = _linear(codes, m.qkv)
    _near(row, ref.view(row.shape), tol.view(row.shape))
    q, k, v = (t.unflatten(-1, (-1, 32)) for t in row.split([192, 96, 96], -1))
    q, k = K.rotary_axes(q, k, pos, sections=(4, 6, 6))
    o, S2 = K.decay_attention(q, k, v, m.decay, scale=32 ** -0.5)
    assert torch.equal(S, S2)
    ro, rS, oa, A = OS.decay(q.cpu(), k.cpu(), v.cpu(), m.decay.cpu(), 32 ** -0.5)
    sums = (32 + 150 / 8 + 64) * 2.0 ** -23
    _near(o, ro, (2.0 ** -15 + sums) * oa + 2.0 ** -8 * ro.abs() + 1e-30)
    _near(S, rS, (2.0 ** -22 + sums) * A + 1e-30)
    u = K.group_norm_act(o.view(300, 192), 6, m.head_norm.weight, m.head_norm.bias, act="silu")
    ru, d = OS.group_norm(o.view(300, 1, 192).cpu(), 6, m.head_norm.weight.cpu(), m.head_norm.bias.cpu(), act="silu")
    _near(u[:, None], ru, 1.2 * 49 * 2.0 ** -24 * (d + ru.abs()) + 2.0 ** -8 * ru.abs() + 1e-30)
    codes = K.mx_quantize(u, "mxfp8")
    ref, tol = _linear(codes, m.out)
    assert torch.equal(y.view(300, 96), m.out(codes))
    _near(y.view(300, 96), ref, tol)
