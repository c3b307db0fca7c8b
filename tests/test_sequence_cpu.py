"""The linear-attention block's operators without a GPU: the oracle against closed forms, argument
checks of the Python layer and of the C entries (rejected before any device work)."""
import ctypes

import pytest
import torch

from oracle import sequence as OS

CPU = "cpu"


def _k():
    from snn_compiler import kernels
    return kernels


def test_oracle_rotary_is_a_rotation_and_its_inverse():
    g = torch.Generator().manual_seed(0)
    x = torch.randn(2, 5, 3, 20, generator=g, dtype=torch.float64)
    pos = torch.randint(0, 1000, (2, 5, 2), generator=g)
    for inter in (False, True):
        y, _ = OS.rotary(x, pos, (3, 5), ladder="axis", interleaved=inter)
        assert torch.allclose((y ** 2).sum(-1), (x ** 2).sum(-1), rtol=1e-12)
        assert torch.equal(y[..., 16:], x[..., 16:])
        back, _ = OS.rotary(y, pos, (3, 5), ladder="axis", interleaved=inter, inverse=True)
        assert torch.allclose(back, x, atol=1e-12)


def test_oracle_rotary_gradient_is_the_inverse():
    """d (w . rotary(x)) / dx = rotary(w, inverse): against differences."""
    g = torch.Generator().manual_seed(1)
    x = torch.randn(1, 3, 1, 8, generator=g, dtype=torch.float64)
    w = torch.randn(1, 3, 1, 8, generator=g, dtype=torch.float64)
    pos = torch.randint(0, 50, (1, 3, 2), generator=g)
    grad, _ = OS.rotary(w, pos, (1, 3), inverse=True)
    for i in range(x.numel()):
        e = torch.zeros_like(x).flatten()
        e[i] = 1e-4
        e = e.view_as(x)
        up, dn = (OS.rotary(x + s * e, pos, (1, 3))[0] for s in (1, -1))
        assert abs(((up - dn) * w).sum() / 2e-4 - grad.flatten()[i]) < 1e-9


def test_oracle_decay_against_the_quadratic_form():
    g = torch.Generator().manual_seed(2)
    q, k = torch.randn(2, 9, 4, 3, generator=g), torch.randn(2, 9, 2, 3, generator=g)
    v, lam = torch.randn(2, 9, 2, 5, generator=g), torch.tensor([1.0, 0.9, 0.3, 0.0])
    o, S, _, _ = OS.decay(q, k, v, lam, scale=0.5)
    i = torch.arange(9)
    gap = (i[:, None] - i[None]).clamp(min=0)
    w = torch.where(i[:, None] >= i[None], lam.double()[:, None, None] ** gap, 0.0)
    kk, vv = (x.double().repeat_interleave(2, 2).transpose(1, 2) for x in (k, v))
    p = (q.double().transpose(1, 2) @ kk.transpose(-1, -2)) * w
    assert torch.allclose(o, 0.5 * (p @ vv).transpose(1, 2), atol=1e-12)
    assert torch.allclose(S, (kk * w[:, -1, :, None]).transpose(-1, -2) @ vv, atol=1e-12)


def test_oracle_group_norm_against_torch():
    g = torch.Generator().manual_seed(3)
    x, w, b = (torch.randn(*s, generator=g, dtype=torch.float64) for s in ((2, 7, 12), (12,), (12,)))
    ref = torch.nn.functional.group_norm(x.transpose(1, 2), 4, w, b, 1e-3).transpose(1, 2)
    y, _ = OS.group_norm(x, 4, w, b, 1e-3)
    assert torch.allclose(y, ref, atol=1e-12)
    s, _ = OS.group_norm(x, 4, w, b, 1e-3, "gelu")
    assert torch.allclose(s, torch.nn.functional.gelu(ref), atol=1e-12)


def test_grid_positions():
    p = _k().grid_positions(2, 3, 4, start=(5, 0, 1), device=CPU)
    assert p.shape == (24, 3) and p.dtype == torch.int32
    assert p[0].tolist() == [5, 0, 1] and p[-1].tolist() == [6, 2, 4] and p[5].tolist() == [5, 1, 2]


def test_rotary_refusals():
    K = _k()
    q, k = torch.zeros(2, 5, 3, 16), torch.zeros(2, 5, 1, 16)
    pos = torch.zeros(5, 2, dtype=torch.int32)
    ok = dict(sections=(4, 4))
    with pytest.raises(AssertionError):
        K.rotary_axes(q, k, pos, **ok)                       # no CUDA tensors
    for sections in ((), (0, 0), (4, 5), (-1, 4)):
        with pytest.raises(ValueError):
            K.rotary_axes(q, k, pos, sections=sections)
    with pytest.raises(ValueError):
        K.rotary_axes(q, k, pos, ladder="each", **ok)
    for base in (0.0, -1.0, float("nan"), float("inf")):
        with pytest.raises(ValueError):
            K.rotary_axes(q, k, pos, base=base, **ok)
    with pytest.raises(AssertionError):
        K.rotary_axes(q.double(), k, pos, **ok)
    with pytest.raises(AssertionError):
        K.rotary_axes(q[0], k, pos, **ok)
    with pytest.raises(ValueError):
        K.rotary_axes(torch.zeros(1, 1, 1, 600), None, pos[:1], sections=(250, 50))


@pytest.mark.parametrize("step", [False, True])
def test_decay_refusals(step):
    K = _k()
    lead = (2,) if step else (2, 5)
    q, k, v = torch.zeros(*lead, 4, 8), torch.zeros(*lead, 2, 8), torch.zeros(*lead, 2, 6)
    lam, S = torch.ones(4), torch.zeros(2, 4, 8, 6)

    def call(q=q, k=k, v=v, lam=lam, S=S, **kw):
        if step:
            return K.decay_attention_step(q, k, v, lam, S, **kw)
        return K.decay_attention(q, k, v, lam, state=S, **kw)
    with pytest.raises(AssertionError):
        call()                                               # no CUDA tensors
    with pytest.raises(ValueError):
        call(k=torch.zeros(*lead, 3, 8), v=torch.zeros(*lead, 3, 6))
    with pytest.raises(ValueError):
        call(v=torch.zeros(*lead, 2, 257))
    with pytest.raises(ValueError):
        call(q=torch.zeros(*lead, 4, 0), k=torch.zeros(*lead, 2, 0))
    with pytest.raises(AssertionError):
        call(k=torch.zeros(*lead, 2, 7))
    with pytest.raises(AssertionError):
        call(k=k.half())
    with pytest.raises(AssertionError):
        call(q=q.double(), k=k.double(), v=v.double())
    with pytest.raises(AssertionError):
        call(q=q[0])


def test_group_norm_refusals():
    K = _k()
    x = torch.zeros(2, 3, 12)
    with pytest.raises(AssertionError):
        K.group_norm_act(x, 4)                               # no CUDA tensor
    for groups in (0, 5, -1, 24):
        with pytest.raises(ValueError):
            K.group_norm_act(x, groups)
    with pytest.raises(ValueError):
        K.group_norm_act(x, 4, act="swish")
    for eps in (-1.0, float("nan")):
        with pytest.raises(ValueError):
            K.group_norm_act(x, 4, eps=eps)
    with pytest.raises(AssertionError):
        K.group_norm_act(x[0, 0], 4)
    with pytest.raises(AssertionError):
        K.group_norm_act(x.double(), 4)


def _array(kind, *v):
    return (kind * len(v))(*v)


def test_c_entries_reject_bad_arguments_without_a_device():
    from snn_compiler import _lib
    L = _lib.lib()
    p = ctypes.c_void_p(1 << 20)            # aligned stand-ins: rejected before any access
    odd = ctypes.c_void_p((1 << 20) + 1)
    s6, s3, s2 = (_array(ctypes.c_int64, *([16] * n)) for n in (6, 3, 2))
    turns, axis = _array(ctypes.c_double, *([0.1] * 4)), _array(ctypes.c_uint8, *([0] * 4))

    def rotary(**kw):
        a = dict(q=p, qo=p, hq=2, qs=s6, k=p, ko=p, hk=1, ks=s6, dt=2, B=1, N=3, d=8, pos=p, pt=0,
                 ps=s3, turns=turns, axis=axis, pairs=4, inter=0, inv=0, st=None)
        a.update(kw)
        return L.snnb_rotary_axes(*a.values())
    for bad in (dict(dt=7), dict(pt=3), dict(B=-1), dict(N=-1), dict(hq=-1), dict(d=7),
                dict(pairs=0), dict(pairs=257, d=1000), dict(q=None), dict(ko=None),
                dict(qs=None), dict(pos=None), dict(ps=None), dict(turns=None), dict(axis=None),
                dict(q=odd), dict(ko=odd), dict(pos=odd), dict(B=1 << 38)):
        assert rotary(**bad) == -1, bad
    assert rotary(B=0) == 0 and rotary(N=0) == 0 and rotary(hq=0, hk=0) == 0

    def attention(**kw):
        a = dict(q=p, qs=s3, k=p, ks=s3, v=p, vs=s3, dt=2, B=1, N=3, H=2, Hk=1, dk=8, dv=8, lam=p,
                 scale=1.0, si=None, ln=None, lt=0, out=p, so=None, ws=None, wsb=0, st=None)
        a.update(kw)
        return L.snnb_decay_attention(*a.values())

    def step(**kw):
        a = dict(q=p, qs=s2, k=p, ks=s2, v=p, vs=s2, dt=2, B=1, H=2, Hk=1, dk=8, dv=8, lam=p,
                 scale=1.0, si=p, out=p, so=p, st=None)
        a.update(kw)
        return L.snnb_decay_attention_step(*a.values())
    for call in (attention, step):
        for bad in (dict(dt=3), dict(B=-1), dict(H=0), dict(Hk=0), dict(H=3, Hk=2), dict(dk=0),
                    dict(dk=257), dict(dv=257), dict(q=None), dict(k=None), dict(v=None),
                    dict(lam=None), dict(out=None), dict(qs=None), dict(vs=None), dict(q=odd),
                    dict(lam=odd), dict(si=odd), dict(so=odd), dict(B=1 << 40)):
            assert call(**bad) == -1, bad
        assert call(B=0) == 0
    assert attention(N=-1) == -1 and attention(ln=p, lt=2) == -1 and attention(ln=odd) == -1
    assert attention(N=1 << 45) == -1
    assert step(si=None) == -1 and step(so=None) == -1
    assert L.snnb_decay_attention_workspace_bytes(2, 1, 100, 2, 0, 8) < 0
    assert L.snnb_decay_attention_workspace_bytes(2, 1, -1, 2, 8, 8) < 0
    assert L.snnb_decay_attention_workspace_bytes(5, 1, 1, 2, 8, 8) < 0
    assert L.snnb_decay_attention_workspace_bytes(2, 1, 100, 2, 8, 8) >= 0

    def norm(**kw):
        a = dict(x=p, xb=96, xs=12, dt=2, B=2, S=8, C=12, G=4, w=p, b=p, wd=0, eps=1e-5, act=0,
                 out=p, ws=None, wsb=0, st=None)
        a.update(kw)
        return L.snnb_group_norm_act(*a.values())
    for bad in (dict(dt=3), dict(wd=1), dict(act=4), dict(act=-1), dict(eps=-1.0),
                dict(eps=float("nan")), dict(G=5), dict(G=0), dict(C=0), dict(B=-1), dict(S=-1),
                dict(x=None), dict(out=None), dict(x=odd), dict(out=odd), dict(w=odd), dict(b=odd),
                dict(B=1 << 31), dict(S=1 << 31), dict(C=1 << 30, G=1)):
        assert norm(**bad) == -1, bad
    assert norm(B=0) == 0 and norm(S=0) == 0
    need = L.snnb_group_norm_act_workspace_bytes(2, 64, 3136, 256, 32)
    assert need > 0 and L.snnb_group_norm_act_workspace_bytes(2, 2, 8, 12, 4) == 0
    assert L.snnb_group_norm_act_workspace_bytes(2, 2, 8, 12, 5) < 0
    large = dict(B=64, S=3136, C=256, G=32, xb=3136 * 256, xs=256)
    assert norm(**large) == -1 and norm(ws=p, wsb=need - 1, **large) == -1
    assert norm(ws=ctypes.c_void_p((1 << 20) + 4), wsb=need, **large) == -1
