"""Rotary positions, decay attention and group norm on the GPU against the float64 oracle
(oracle/sequence.py).

Tolerances, derived (u: half a step of the output's type relative to the value, eps / 2):
  rotary   what is left of the angle is at most half a turn, rounded to float32 (2^-25 of a turn,
           2^-22.3 of a radian) and the sine and cosine are good to 2^-22; the products and the
           sum round three times: 2^-21 (|a| + |b|), and u |y|.
  decay    products of the inputs are exact in float32 or round once, and so do the powers; sums
           of dk terms and of the tokens round (or are cut) at most once per term onto a partial
           sum that sum |q||k||v| bounds, N / 8 + 64 times where chunks sum in between:
           (dk + N / 8 + 64) 2^-23 of that magnitude.  16-bit inputs may go through the tensor
           cores: there scores round once to the inputs' type, by half a step of it (2^-8, 2^-11),
           and the other operands are held as two terms of at least 8 bits (2^-8 of 2^-8 each):
           u and 3 * 2^-16 of the magnitude for the outputs, 2 * 2^-16 for the state.
  norm     sums over n values in at least 32 partial ones: (n / 32 + 32) 2^-24 relative to the
           mean magnitude, and as much of the variance's; about 16 roundings behind that; SiLU
           and GELU have slopes below 1.13: 1.2 (n / 32 + 48) 2^-24 of the oracle's magnitude
           d plus |y|, and u |y|.
"""
import threading

import pytest
import torch

from oracle import sequence as OS

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
DTYPES = [BF16, F16, F32]


def _k():
    from snn_compiler import kernels
    return kernels


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _u(dtype):
    return torch.finfo(dtype).eps / 2


def _tiny(dtype):
    """Half a step of the subnormals."""
    return torch.finfo(dtype).smallest_normal * _u(dtype)


def _near(got, ref, tol):
    got = got.cpu().double()
    assert got.shape == ref.shape
    bad = ~((got - ref).abs() <= tol)
    assert not bad.any(), \
        f"{int(bad.sum())} of {bad.numel()} off, at {bad.nonzero()[0].tolist()}: " \
        f"{got[bad][0].item()} for {ref[bad][0].item()} (tolerance {tol.expand_as(ref)[bad][0].item()})"


# ---- rotary --------------------------------------------------------------------------------


def _rotary_check(q, k, pos, **kw):
    """On CPU tensors; returns what the GPU gave."""
    qo, ko = _k().rotary_axes(q.to(DEV), None if k is None else k.to(DEV), pos.to(DEV), **kw)
    full = pos[None].expand(q.shape[0], *pos.shape) if pos.dim() == 2 else pos
    for x, y in ((q, qo), (k, ko)):
        if x is None:
            assert y is None
            continue
        ref, mag = OS.rotary(x, full, **kw)
        assert y.dtype == x.dtype and y.is_contiguous()
        _near(y, ref, 2.0 ** -21 * mag + _u(x.dtype) * ref.abs() + _tiny(x.dtype))
        rest = 2 * sum(kw["sections"])
        assert torch.equal(y[..., rest:].cpu(), x[..., rest:])
    return qo, ko


ROTARY = [(1, 1, 1, 1, 2, (1,)), (2, 5, 3, 1, 6, (1, 1)), (1, 7, 4, 2, 16, (4, 2, 2)),
          (2, 3, 5, 5, 48, (8, 8, 8)), (1, 33, 8, 2, 128, (16, 24, 24)), (3, 2, 2, 1, 100, (7, 13)),
          (1, 4, 9, 3, 64, (0, 32)), (1, 3, 2, 2, 97, (10, 11, 12, 13)), (1, 2, 1, 1, 512, (256,)),
          (1, 300, 40, 8, 64, (32,)), (2, 9, 33, 7, 40, (12,)), (1, 6, 12, 12, 56, (14, 14))]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("B,N,H,Hk,d,sections", ROTARY)
def test_rotary_against_oracle(B, N, H, Hk, d, sections, interleaved, dtype):
    g = _gen(B * N + d)
    q, k = (torch.randn(B, N, h, d, generator=g).to(dtype) for h in (H, Hk))
    for ladder, shape, inverse in (("shared", (N,), False), ("axis", (B, N), True)):
        pos = torch.randint(0, 5000, (*shape, len(sections)), generator=g, dtype=torch.int32)
        _rotary_check(q, k, pos, sections=sections, ladder=ladder, interleaved=interleaved,
                      inverse=inverse)


@pytest.mark.parametrize("kind", [torch.int32, torch.int64, torch.float32])
def test_rotary_far_negative_and_fractional_positions(kind):
    g = _gen(4)
    q = torch.randn(1, 40, 2, 32, generator=g)
    far = 2 ** 40 if kind == torch.int64 else 2 ** 30
    pos = torch.randint(-far, far, (40, 2), generator=g)
    pos = (pos.double() / 1024).to(kind) if kind == torch.float32 else pos.to(kind)
    # the oracle's own angle is a float64 product: at 2^40 radians it is good to 2^-13 of one, so
    # compare there with frequencies that are powers of two of a turn through float positions
    if kind == torch.int64:
        pos = pos % (2 ** 31)
    _rotary_check(q, None, pos, sections=(8, 8))


def test_rotary_slices_orders_and_in_place():
    K, g = _k(), _gen(5)
    B, N, H, Hk, d = 2, 9, 4, 2, 32
    kw = dict(sections=(4, 6, 6))
    pos = torch.randint(0, 99, (N, 3), generator=g, dtype=torch.int32).to(DEV)
    for dtype in DTYPES:
        for pad in (0, 3, 8):
            row = torch.randn(B, N, (H + Hk) * d + pad, generator=g).to(dtype).to(DEV)
            q = row[..., pad:pad + H * d].unflatten(-1, (H, d))
            k = row[..., pad + H * d:].unflatten(-1, (Hk, d))
            ref = K.rotary_axes(q.contiguous(), k.contiguous(), pos, **kw)
            got = K.rotary_axes(q, k, pos, **kw)
            assert all(torch.equal(a, b) for a, b in zip(got, ref))
            # head-major tensors
            t = q.transpose(1, 2).contiguous().transpose(1, 2)
            assert torch.equal(K.rotary_axes(t, None, pos, **kw)[0], ref[0])
            # columns that are not contiguous
            c = q.transpose(2, 3).contiguous().transpose(2, 3)
            assert torch.equal(K.rotary_axes(c, None, pos, **kw)[0], ref[0])
            before = row.clone()
            a, b = K.rotary_axes(q, k, pos, q_out=q, k_out=k, **kw)
            assert a.data_ptr() == q.data_ptr() and b.data_ptr() == k.data_ptr()
            assert torch.equal(q, ref[0]) and torch.equal(k, ref[1])
            assert torch.equal(row[..., :pad], before[..., :pad])      # what lies beside them
    # positions of any strides
    wide = torch.randint(0, 99, (3, N), dtype=torch.int32, device=DEV)
    a = K.rotary_axes(q, k, wide.t(), **kw)
    b = K.rotary_axes(q, k, wide.t().contiguous(), **kw)
    assert torch.equal(a[0], b[0])


def test_rotary_nothing_to_do_and_non_finite():
    K = _k()
    for shape in ((0, 3, 2, 8), (2, 0, 2, 8)):
        q = torch.zeros(*shape, device=DEV)
        pos = torch.zeros(shape[1], 1, dtype=torch.int32, device=DEV)
        assert K.rotary_axes(q, q[:, :, :0], pos, sections=(4,))[0].shape == shape
    q = torch.ones(1, 3, 1, 8, device=DEV)
    pos = torch.tensor([[0.0], [float("nan")], [1.0]], device=DEV)
    y = K.rotary_axes(q, None, pos, sections=(3,))[0]
    assert y[0, 1, 0, :6].isnan().all() and (y[0, 1, 0, 6:] == 1).all()
    assert torch.equal(y[0, 0], q[0, 0]) and y[0, 2].isfinite().all()
    with pytest.raises(AssertionError):
        K.rotary_axes(q, None, torch.zeros(3, 2, device=DEV), sections=(3,))
    with pytest.raises(AssertionError):
        K.rotary_axes(q, None, torch.zeros(3, 1, device=DEV, dtype=torch.int16), sections=(3,))
    with pytest.raises(AssertionError):
        K.rotary_axes(q, None, torch.zeros(3, 1), sections=(3,))
    with pytest.raises(AssertionError):
        K.rotary_axes(q, None, pos, sections=(3,), q_out=q.half())


def test_rotary_offsets_past_32_bits():
    """Two sequences whose rows lie more than 2^32 bytes apart."""
    K = _k()
    if torch.cuda.mem_get_info()[0] < 24 << 30:
        pytest.skip("needs 24 GB")
    big = torch.empty((1 << 32) + (1 << 20), dtype=BF16, device=DEV)
    q = big.as_strided((2, 4, 2, 16), ((1 << 32), 32, 16, 1))
    x = torch.randn(2, 4, 2, 16, generator=_gen(6)).to(BF16)
    q.copy_(x.to(DEV))
    pos = torch.arange(4, dtype=torch.int32)[:, None]
    ref = K.rotary_axes(x.to(DEV), None, pos.to(DEV), sections=(8,))[0]
    assert torch.equal(K.rotary_axes(q, None, pos.to(DEV), sections=(8,), q_out=q)[0], ref)


# ---- decay attention -----------------------------------------------------------------------


def _lam(H):
    """From no memory at all to no decay."""
    return torch.tensor([1.0, 0.0, 0.5, 0.97, 0.9995, 2.0 ** -20, 0.75, 0.999])[:H] if H <= 8 \
        else 1 - torch.exp2(-1 - 9 * torch.arange(H) / (H - 1))


def _decay_tol(o, oa, S, A, dtype, dk, N):
    sums = (dk + N / 8 + 64) * 2.0 ** -23
    extra = 0.0 if dtype == F32 else _u(dtype) + 3 * 2.0 ** -16
    state = 0.0 if dtype == F32 else 2 * 2.0 ** -16
    return ((extra + sums) * oa + _u(dtype) * o.abs() + _tiny(dtype) + 1e-37,
            (state + sums) * A + 1e-37)


def _tokens(B, N, H, Hk, dk, dv, dtype, seed):
    g = _gen(seed)
    return (torch.randn(B, N, H, dk, generator=g).to(dtype),
            (torch.randn(B, N, Hk, dk, generator=g) * dk ** -0.5).to(dtype),
            torch.randn(B, N, Hk, dv, generator=g).to(dtype))


def _decay_check(q, k, v, lam, scale=1.0, state=None, lengths=None, views=None):
    dev = [x.to(DEV) for x in (q, k, v)] if views is None else views
    o, S = _k().decay_attention(*dev, lam.to(DEV), scale=scale,
                                state=None if state is None else state.to(DEV),
                                lengths=None if lengths is None else lengths.to(DEV))
    ro, rS, oa, A = OS.decay(q, k, v, lam, scale, state, lengths)
    assert o.dtype == q.dtype and S.dtype == F32 and o.is_contiguous() and S.is_contiguous()
    to, tS = _decay_tol(ro, oa, rS, A, q.dtype, q.shape[-1], q.shape[1])
    _near(o, ro, to)
    _near(S, rS, tS)
    return o, S


DECAY = [(1, 1, 1, 1, 1, 1), (2, 2, 2, 1, 3, 5), (1, 31, 3, 3, 8, 8), (2, 33, 2, 2, 16, 40),
         (1, 128, 2, 1, 64, 64), (2, 129, 4, 2, 48, 48), (1, 196, 8, 8, 32, 32),
         (1, 300, 2, 2, 128, 128), (2, 257, 6, 3, 64, 96), (1, 130, 3, 1, 72, 24),
         (1, 70, 2, 2, 200, 136), (1, 40, 1, 1, 256, 256), (1, 65, 2, 2, 97, 33),
         (3, 127, 1, 1, 128, 8), (1, 640, 1, 1, 64, 128), (1, 513, 5, 5, 40, 72)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,N,H,Hk,dk,dv", DECAY)
def test_decay_against_oracle(B, N, H, Hk, dk, dv, dtype):
    q, k, v = _tokens(B, N, H, Hk, dk, dv, dtype, N + dk)
    state = torch.randn(B, H, dk, dv, generator=_gen(9))
    lam = _lam(H)
    _decay_check(q, k, v, lam, scale=dk ** -0.5)
    g = _gen(10)
    lengths = torch.randint(0, N + 1, (B,), generator=g, dtype=torch.int32)
    _decay_check(q, k, v, lam, scale=-0.7, state=state, lengths=lengths)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lengths", [[0, 0], [0, 200], [1, 128], [129, 127], [300, -5], [199, 64]])
def test_decay_lengths_hide_what_lies_behind_them(lengths, dtype):
    """Infinities and NaN behind the lengths count nowhere; rows there are zero; lengths outside
    [0, N] are clamped."""
    B, N, H, dk, dv = 2, 200, 3, 48, 64
    q, k, v = _tokens(B, N, H, H, dk, dv, dtype, 3)
    state = torch.randn(B, H, dk, dv, generator=_gen(2))
    for kind in (torch.int32, torch.int64):
        n = torch.tensor(lengths, dtype=kind)
        for x, bad in ((q, "nan"), (k, "inf"), (v, "nan")):
            for b in range(B):
                x[b, max(0, min(N, lengths[b])):] = float(bad)
        o, S = _decay_check(q, k, v, _lam(H), state=state, lengths=n)
        for b in range(B):
            m = max(0, min(N, lengths[b]))
            assert not o[b, m:].any()
            if m == 0:
                assert torch.equal(S[b].cpu(), state[b])


@pytest.mark.parametrize("dtype", DTYPES)
def test_decay_later_tokens_touch_no_earlier_ones(dtype):
    """A token that is not finite is seen by itself and those behind it only."""
    q, k, v = _tokens(1, 300, 2, 2, 64, 64, dtype, 8)
    lam = torch.tensor([0.9, 1.0])
    ref, _ = _k().decay_attention(q.to(DEV), k.to(DEV), v.to(DEV), lam.to(DEV))
    for which, bad in ((k, float("inf")), (v, float("nan")), (v, float("inf"))):
        keep = which[0, 150, 0, 5].clone()
        which[0, 150, 0, 5] = bad
        o, _ = _k().decay_attention(q.to(DEV), k.to(DEV), v.to(DEV), lam.to(DEV))
        assert torch.equal(o[:, :150], ref[:, :150])
        assert torch.equal(o[:, :, 1], ref[:, :, 1])             # another head
        hit = o[0, 150:, 0] if which is k else o[0, 150:, 0, 5]
        assert not hit.float().isfinite().any()
        if which is v:
            others = [c for c in range(64) if c != 5]
            assert torch.equal(o[..., others], ref[..., others])
        which[0, 150, 0, 5] = keep


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("pad", [0, 8, 3])
def test_decay_slices_orders_and_alignments(pad, dtype):
    B, N, H, Hk, dk, dv = 2, 150, 4, 2, 32, 64
    q, k, v = _tokens(B, N, H, Hk, dk, dv, dtype, 11)
    sizes = [H * dk, Hk * dk, Hk * dv]
    row = torch.full((B, N, sum(sizes) + pad), float("nan"), dtype=dtype, device=DEV)
    parts = row[..., pad:].split(sizes, -1)
    views = [p.unflatten(-1, (x.shape[2], x.shape[3])) for p, x in zip(parts, (q, k, v))]
    for p, x in zip(views, (q, k, v)):
        p.copy_(x.to(DEV))
    _decay_check(q, k, v, _lam(H), views=views)
    major = [x.to(DEV).transpose(1, 2).contiguous().transpose(1, 2) for x in (q, k, v)]
    _decay_check(q, k, v, _lam(H), views=major)
    cols = [x.to(DEV).transpose(2, 3).contiguous().transpose(2, 3) for x in (q, k, v)]
    _decay_check(q, k, v, _lam(H), views=cols)


@pytest.mark.parametrize("dtype", DTYPES)
def test_decay_pieces_and_steps_give_the_whole(dtype):
    """A sequence in pieces through its state, and token by token, against the oracle's whole."""
    K = _k()
    B, N, H, Hk, dk, dv = 2, 150, 4, 2, 64, 48
    q, k, v = _tokens(B, N, H, Hk, dk, dv, dtype, 12)
    lam, g = _lam(H), [x.to(DEV) for x in _tokens(B, N, H, Hk, dk, dv, dtype, 12)]
    ro, rS, oa, A = OS.decay(q, k, v, lam, 0.3)
    to, tS = _decay_tol(ro, oa, rS, A, dtype, dk, N)
    S, outs, at = None, [], 0
    for n in (1, 100, 0, 20):
        o, S = K.decay_attention(*[x[:, at:at + n] for x in g], lam.to(DEV), scale=0.3, state=S,
                                 state_out=S)                     # in place from the second on
        outs.append(o)
        at += n
    for t in range(at, N):
        o, S2 = K.decay_attention_step(*[x[:, t] for x in g], lam.to(DEV), S, scale=0.3)
        assert S2 is S
        outs.append(o[:, None])
    _near(torch.cat(outs, 1), ro, to)
    _near(S, rS, tS)


STEP = [(1, 1, 1, 1, 1), (2, 3, 1, 5, 7), (1, 32, 32, 128, 128), (5, 4, 2, 64, 96), (3, 6, 3, 48, 48),
        (2, 2, 2, 256, 256), (1, 7, 7, 97, 33), (64, 2, 1, 32, 40), (300, 1, 1, 16, 4)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,H,Hk,dk,dv", STEP)
def test_step_against_oracle(B, H, Hk, dk, dv, dtype):
    K = _k()
    q, k, v = (x[:, 0] for x in _tokens(B, 1, H, Hk, dk, dv, dtype, dk))
    state, lam = torch.randn(B, H, dk, dv, generator=_gen(5)), _lam(H)
    ro, rS, oa, A = OS.decay(q[:, None], k[:, None], v[:, None], lam, 0.5, state)
    sums = (dk + 16) * 2.0 ** -23
    old = state.to(DEV)
    new = torch.full_like(old, 7.0)
    o, S = K.decay_attention_step(q.to(DEV), k.to(DEV), v.to(DEV), lam.to(DEV), old, scale=0.5,
                                  state_out=new)
    assert S is new and torch.equal(old.cpu(), state)
    _near(o, ro[:, 0], (sums * oa + _u(dtype) * ro.abs() + _tiny(dtype))[:, 0])
    _near(S, rS, 2.0 ** -22 * A + 1e-37)
    o2, S2 = K.decay_attention_step(q.to(DEV), k.to(DEV), v.to(DEV), lam.to(DEV), old, scale=0.5)
    assert S2 is old and torch.equal(old, new) and torch.equal(o2, o)
    # slices of one projection's row
    row = torch.cat([x.flatten(1) for x in (q, k, v)], 1).to(DEV)
    a, b, c = row.split([H * dk, Hk * dk, Hk * dv], 1)
    o3, _ = K.decay_attention_step(a.unflatten(1, (H, dk)), b.unflatten(1, (Hk, dk)),
                                   c.unflatten(1, (Hk, dv)), lam.to(DEV), state.to(DEV), scale=0.5)
    assert torch.equal(o3, o)


def test_decay_nothing_to_do_and_refusals():
    K = _k()
    q, k, v = (x.to(DEV) for x in _tokens(2, 0, 2, 2, 8, 8, F32, 1))
    lam, state = torch.tensor([0.5, 1.0], device=DEV), torch.randn(2, 2, 8, 8, device=DEV)
    o, S = K.decay_attention(q, k, v, lam, state=state)
    assert o.shape == (2, 0, 2, 8) and torch.equal(S, state)
    o, S = K.decay_attention(q, k, v, lam)
    assert not S.any()
    o, S = K.decay_attention(q[:0], k[:0], v[:0], lam)
    assert S.shape == (0, 2, 8, 8)
    q, k, v = (x.to(DEV) for x in _tokens(2, 5, 2, 2, 8, 8, F32, 1))
    for kw in (dict(state=state.half()), dict(state=state[:1]), dict(state=state.transpose(2, 3)),
               dict(state=state.cpu()), dict(lengths=torch.tensor([1, 2])),
               dict(lengths=torch.tensor([1.0, 2.0], device=DEV)),
               dict(lengths=torch.tensor([1], device=DEV)), dict(out=torch.empty_like(q).half()),
               dict(state_out=state.cpu())):
        with pytest.raises(AssertionError):
            K.decay_attention(q, k, v, lam, **kw)
    with pytest.raises(AssertionError):
        K.decay_attention(q, k, v, lam.double())
    with pytest.raises(AssertionError):
        K.decay_attention(q, k, v, lam.cpu())
    with pytest.raises(AssertionError):
        K.decay_attention_step(q[:, 0], k[:, 0], v[:, 0], lam, state.cpu())


@pytest.mark.parametrize("dtype", DTYPES)
def test_decay_twice_is_the_same(dtype):
    q, k, v = (x.to(DEV) for x in _tokens(2, 700, 3, 3, 64, 64, dtype, 21))
    lam = _lam(3).to(DEV)
    a, b = (_k().decay_attention(q, k, v, lam) for _ in range(2))
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


# ---- group norm ----------------------------------------------------------------------------


def _norm_check(x, groups, weight=None, bias=None, eps=1e-5, act="none", view=None):
    to = lambda t: None if t is None else t.to(DEV)                       # noqa: E731
    y = _k().group_norm_act(to(x) if view is None else view, groups, to(weight), to(bias), eps=eps,
                            act=act)
    assert y.shape == x.shape and y.dtype == x.dtype and y.is_contiguous()
    B, C = x.shape[0], x.shape[-1]
    x3 = x.reshape(B, -1, C)
    ref, d = OS.group_norm(x3, groups, weight, bias, eps, act)
    n = x3.shape[1] * C // groups
    tol = 1.2 * (n / 32 + 48) * 2.0 ** -24 * (d + ref.abs()) + _u(x.dtype) * ref.abs() + \
        _tiny(x.dtype)
    _near(y.reshape(B, -1, C), ref, tol)
    return y


NORM = [((1, 1), 1), ((3, 8), 2), ((2, 5, 12), 4), ((1, 7, 3, 90), 30), ((2, 16, 16, 64), 32),
        ((700, 384), 8), ((1, 33, 31, 96), 6), ((3, 1, 1, 2048), 64), ((2, 1000, 24), 24),
        ((1, 3000, 7), 1), ((5, 14, 14, 320), 32), ((2, 56, 56, 64), 32), ((1, 9, 2050), 2),
        ((9000, 40), 5), ((300, 2048), 1), ((300, 1005), 3), ((257, 1023), 1), ((130, 1500), 1), ((1, 4096, 8), 1), ((2, 50, 1003), 17)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape,groups", NORM)
def test_group_norm_against_oracle(shape, groups, dtype):
    g = _gen(sum(shape))
    C = shape[-1]
    x = (torch.randn(shape, generator=g) * 2 + torch.randn(C, generator=g) * 3).to(dtype)
    w, b = torch.rand(C, generator=g) + 0.5, torch.randn(C, generator=g)
    _norm_check(x, groups, w.to(dtype), b.to(dtype), act="silu")
    _norm_check(x, groups, w, b, act="gelu")
    _norm_check(x, groups, eps=0.1, act="relu")
    _norm_check(x, groups, w, None)
    _norm_check(x, groups, None, b, act="silu")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape,groups,pad", [((9, 37, 41, 330), 33, 0), ((3, 9000, 257), 257, 0),
                                              ((40, 200, 1030), 2, 3), ((2, 20000, 130), 26, 6),
                                              ((33, 4, 40000), 8, 0), ((1, 70000, 64), 1, 0),
                                              ((5, 300, 6, 512), 4, 16), ((1100, 4096), 1, 0)])
def test_group_norm_of_large_tensors(shape, groups, pad, dtype):
    g = _gen(groups)
    C = min(shape[-1], 16384)
    x = torch.randn(*shape[:-1], C + pad, generator=g) * 2
    x = (x + torch.randn(C + pad, generator=g) * 3).to(dtype)
    w, b = (torch.randn(C, generator=g).to(dtype) for _ in range(2))
    view = x.to(DEV)[..., :C]
    _norm_check(x[..., :C].contiguous(), groups, w, b, act="silu", view=view)
    if not pad:                                                 # in place
        y = _k().group_norm_act(view, groups, act="gelu")
        assert torch.equal(_k().group_norm_act(view, groups, act="gelu", out=view), y)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("cols,at,C,groups", [(48, 0, 40, 5), (48, 8, 40, 5), (47, 3, 40, 5), (391, 7, 384, 8),
                                              (90, 1, 66, 22)])
def test_group_norm_slices_of_a_wider_tensor(cols, at, C, groups, dtype):
    g = _gen(cols)
    for lead in ((3, 37), (150,), (2, 500)):
        wide = torch.full((*lead, cols), float("nan"), dtype=dtype)
        wide[..., at:at + C] = torch.randn(*lead, C, generator=g).to(dtype)
        x = wide[..., at:at + C]
        _norm_check(x.contiguous(), groups, act="silu", view=wide.to(DEV)[..., at:at + C])


def test_group_norm_orders_large_means_and_non_finite():
    K, g = _k(), _gen(3)
    x = torch.randn(2, 24, 6, 5, generator=g)                  # an NCHW image, seen channels last
    _norm_check(x.permute(0, 2, 3, 1).contiguous(), 4, view=x.to(DEV).permute(0, 2, 3, 1))
    y = x.to(DEV).permute(0, 2, 3, 1).contiguous()             # rows in another order
    _norm_check(y.transpose(1, 2).contiguous().cpu(), 4, view=y.transpose(1, 2))
    # a mean of a thousand deviations: E[x^2] - mean^2 would leave nothing of the variance
    _norm_check(torch.randn(2, 300, 16, generator=g) + 1000.0, 2)
    # constant groups: the variance is zero, the bias is left
    c = torch.full((2, 9, 8), 3.0, device=DEV)
    b = torch.randn(8, generator=g)
    assert torch.equal(K.group_norm_act(c, 2, None, b.to(DEV)), b.to(DEV).expand(2, 9, 8))
    # a value that is not finite spoils its group of its sample, nothing else
    for bad in (float("nan"), float("inf")):
        x = torch.randn(2, 50, 16, generator=g)
        ref = K.group_norm_act(x.to(DEV), 4, act="silu")
        x[1, 20, 5] = bad
        for act in ("silu", "relu"):
            z = K.group_norm_act(x.to(DEV), 4, act=act)
            assert z[1, :, 4:8].isnan().all()
        z = K.group_norm_act(x.to(DEV), 4, act="silu")
        assert torch.equal(z[0], ref[0]) and torch.equal(z[1, :, 8:], ref[1, :, 8:])
    assert K.group_norm_act(torch.zeros(0, 5, 8, device=DEV), 2).shape == (0, 5, 8)
    assert K.group_norm_act(torch.zeros(3, 0, 8, device=DEV), 2).shape == (3, 0, 8)
    o = torch.full((2, 50, 16), 5.0, device=DEV)
    assert K.group_norm_act(x.to(DEV), 4, out=o) is o and (o != 5.0).any()
    with pytest.raises(AssertionError):
        K.group_norm_act(o, 4, torch.ones(15, device=DEV))
    with pytest.raises(AssertionError):
        K.group_norm_act(o, 4, torch.ones(16, device=DEV, dtype=F16))
    with pytest.raises(AssertionError):
        K.group_norm_act(o, 4, torch.ones(16))
    with pytest.raises(AssertionError):
        K.group_norm_act(o.half(), 4, torch.ones(16, device=DEV).half(), torch.ones(16, device=DEV))
    with pytest.raises(AssertionError):
        K.group_norm_act(o, 4, out=o.half())


def test_group_norm_in_place():
    K = _k()
    for shape in ((700, 384), (2, 56, 56, 64), (2, 50, 90)):
        x = torch.randn(*shape, generator=_gen(1)).to(BF16).to(DEV)
        ref = K.group_norm_act(x, 2, act="silu")
        assert torch.equal(K.group_norm_act(x, 2, act="silu", out=x), ref)


# ---- together ------------------------------------------------------------------------------


def _run(K, q, k, v, pos, lam):
    q, k = K.rotary_axes(q, k, pos, sections=(8, 12, 12))
    o, S = K.decay_attention(q, k, v, lam, scale=0.125)
    return K.group_norm_act(o.flatten(0, 1).flatten(1), o.shape[2], act="silu"), S


def _run_inputs(seed, dtype=BF16, B=2, N=300, H=4, d=64):
    q, k, v = (x.to(DEV) for x in _tokens(B, N, H, H, d, d, dtype, seed))
    return q, k, v, _k().grid_positions(3, 10, 10), _lam(H).to(DEV)


@pytest.mark.parametrize("dtype", DTYPES)
def test_the_three_in_a_row_against_oracle(dtype):
    K = _k()
    q, k, v, pos, lam = _run_inputs(31, dtype)
    y, S = _run(K, q, k, v, pos, lam)
    full = pos.cpu()[None].expand(2, 300, 3)
    # the oracle goes on from what each operator rounded to its output's type
    kq, kk = K.rotary_axes(q, k, pos, sections=(8, 12, 12))
    for x, t in ((q, kq), (k, kk)):
        r, mag = OS.rotary(x.cpu(), full, (8, 12, 12))
        _near(t, r, 2.0 ** -21 * mag + _u(dtype) * r.abs() + _tiny(dtype))
    ro, rS, oa, A = OS.decay(kq.cpu(), kk.cpu(), v.cpu(), lam.cpu(), 0.125)
    to, tS = _decay_tol(ro, oa, rS, A, dtype, 64, 300)
    o, _ = K.decay_attention(kq, kk, v, lam, scale=0.125)
    _near(o, ro, to)
    _near(S, rS, tS)
    o2 = o.cpu().flatten(0, 1).flatten(1)[:, None]
    rn, d = OS.group_norm(o2, 4, act="silu")
    _near(y[:, None], rn, 1.2 * 50 * 2.0 ** -24 * (d + rn.abs()) + _u(dtype) * rn.abs() + _tiny(dtype))


def test_graph_replays_and_streams():
    """Captured once and replayed on other inputs; two graphs live at a time; a side stream."""
    K = _k()
    sets = [_run_inputs(s) for s in (1, 2, 3)]
    refs = [_run(K, *s) for s in sets]
    graphs = []
    for s in sets[:2]:
        buf = [x.clone() for x in s]
        for _ in range(2):
            _run(K, *buf)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = _run(K, *buf)
        graphs.append((graph, buf, out))
    for order in ((0, 1, 2), (2, 0, 1)):
        for (graph, buf, out), i in zip(graphs, order):
            for a, b in zip(buf, sets[i]):
                a.copy_(b)
        for graph, _, _ in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for (_, _, out), i in zip(graphs, order):
            assert all(torch.equal(a, b) for a, b in zip(out, refs[i]))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out = _run(K, *sets[2])
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(out, refs[2]))


def test_two_threads_at_once():
    K = _k()
    sets = [_run_inputs(s) for s in (4, 5)]
    refs = [_run(K, *s) for s in sets]
    torch.cuda.synchronize()
    wrong = []

    def work(i):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            for _ in range(20):
                out = _run(K, *sets[i])
                stream.synchronize()
                if not all(torch.equal(a, b) for a, b in zip(out, refs[i])):
                    wrong.append(i)
    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


def test_another_device_than_the_current_one():
    if torch.cuda.device_count() < 2:
        pytest.skip("needs two GPUs")
    K = _k()
    s = _run_inputs(6)
    ref = _run(K, *s)
    out = _run(K, *[x.to("cuda:1") for x in s])
    assert all(torch.equal(a, b.cpu().to(DEV)) for a, b in zip(ref, out))


def test_injected_status_reaches_the_caller():
    from snn_compiler import _lib
    K = _k()
    s = _run_inputs(7)
    for call in (lambda: K.rotary_axes(s[0], s[1], s[3], sections=(8, 12, 12)),
                 lambda: K.decay_attention(*s[:3], s[4]),
                 lambda: K.decay_attention_step(s[0][:, 0], s[1][:, 0], s[2][:, 0], s[4],
                                                torch.zeros(2, 4, 64, 64, device=DEV)),
                 lambda: K.group_norm_act(s[0], 2)):
        _lib.check(_lib.lib().snnb_debug_inject_status(-2, 1), "inject")
        with pytest.raises(_lib.SnnbError):
            call()
        call()
