"""The linear-attention block (nn.DecayAttention) and the group norm layer on the GPU, the waits of the
tensor-core kernel, and its outputs under the bounds-checking build."""
import os
import subprocess
import sys
import time

import pytest
import torch
import torch.nn as nn

from oracle import sequence as OS

pytestmark = pytest.mark.gpu
DEV = "cuda"
HERE = os.path.dirname(os.path.abspath(__file__))
PKG = os.path.join(os.path.dirname(HERE), "triton-pass-analysis_b200")
TIMEOUT = -4


def _linears(D, H, Hk, d, seed=0, bias=True):
    torch.manual_seed(seed)
    sizes = ((D, H * d), (D, Hk * d), (D, Hk * d), (H * d, D))
    return [nn.Linear(i, o, bias=bias).to(DEV, torch.bfloat16) for i, o in sizes]


def _block(D=96, H=6, Hk=3, d=32, **kw):
    from snn_compiler.nn import DecayAttention
    lam = 1 - torch.exp2(-1.0 - torch.arange(H))
    return DecayAttention.from_linears(*_linears(D, H, Hk, d), lam, heads=H, kv_heads=Hk,
                                       sections=(4, 6, 6), **kw)


def _inputs(shape, seed=1):
    g = torch.Generator().manual_seed(seed)
    return [torch.randn(*shape, generator=g).to(torch.bfloat16).to(DEV) for _ in range(2)]


def test_block_is_its_operators_in_a_row():
    from snn_compiler import kernels as K
    m = _block()
    x, r = _inputs((2, 150, 96))
    pos = K.grid_positions(6, 5, 5)
    lengths = torch.tensor([150, 40], dtype=torch.int32, device=DEV)
    y, h, S = m(x, pos, r, lengths=lengths)
    codes, h2 = K.rms_norm_mx(x, m.norm.weight, r)
    row = m.qkv(codes)
    q, k, v = row.split([192, 96, 96], -1)
    q, k, v = (t.unflatten(-1, (-1, 32)) for t in (q, k, v))
    q, k = K.rotary_axes(q, k, pos, sections=(4, 6, 6))
    o, S2 = K.decay_attention(q, k, v, m.decay, scale=32 ** -0.5, lengths=lengths)
    u = K.group_norm_act(o.view(300, 192), 6, m.head_norm.weight, m.head_norm.bias, act="silu")
    assert torch.equal(h, h2) and torch.equal(S, S2)
    assert torch.equal(y, m.out(u).view(2, 150, 96)) and y.abs().sum() > 0
    ro, rS, oa, A = OS.decay(q.cpu(), k.cpu(), v.cpu(), m.decay.cpu(), 32 ** -0.5, None, lengths.cpu())
    assert ((o.cpu().double() - ro).abs() <= 2.0 ** -8 * (1.02 * oa + ro.abs()) + 1e-30).all()
    assert ((S.cpu().double() - rS).abs() <= 2.0 ** -14 * A + 1e-30).all()


def test_steps_follow_the_sequence():
    """The last tokens one by one from the state of those before.  A projection's sums may differ in
    their order between the two forms, so q, k and v may differ by one rounding, 2^-7: the state by
    twice that of its magnitude."""
    from snn_compiler import kernels as K
    m = _block()
    x, r = _inputs((3, 40, 96), 2)
    pos = K.grid_positions(2, 4, 5)
    y, h, S = m(x, pos, r)
    _, _, s = m(x[:, :30], pos[:30], r[:, :30])
    for t in range(30, 40):
        yt, ht, s2 = m.step(x[:, t], s, pos[t] if t % 2 else pos[t].expand(3, 3), r[:, t])
        assert s2 is s and torch.equal(ht, h[:, t])
        assert yt.shape == (3, 96) and yt.dtype == y.dtype and yt.isfinite().all()
    assert (s - S).norm() <= 2.0 ** -6 * S.norm()
    assert (yt - y[:, -1]).float().norm() <= 0.25 * y[:, -1].float().norm()


def test_spiking_block_runs_over_time_steps():
    from snn_compiler.nn import LIFNode
    m = _block(neuron=LIFNode(v_threshold=0.5))
    x, r = _inputs((4, 2, 50, 96), 3)                          # [T, B, N, D]
    from snn_compiler import kernels as K
    y, h, S = m(x, K.grid_positions(2, 5, 5), r)
    assert y.shape == x.shape and h.shape == x.shape and S.shape == (8, 6, 32, 32)
    assert y.isfinite().all() and y.abs().sum() > 0


def test_group_norm_layer_matches_the_float_one():
    from snn_compiler.nn import GroupNormAct
    g = torch.Generator().manual_seed(5)
    ref = nn.GroupNorm(8, 64).to(DEV)
    with torch.no_grad():
        ref.weight.copy_(torch.rand(64, generator=g) + 0.5)
        ref.bias.copy_(torch.randn(64, generator=g))
    x = torch.randn(3, 9, 11, 64, generator=g).to(DEV)
    m = GroupNormAct.from_norm(ref, act="silu")
    want = nn.functional.silu(ref(x.permute(0, 3, 1, 2))).permute(0, 2, 3, 1)
    assert (m(x) - want).abs().max() < 1e-5
    h = m.half()(x.half())
    assert h.dtype == torch.float16 and (h.float() - want).abs().max() < 0.02
    assert (m(x) - want).abs().max() < 0.02                    # half parameters beside float32 values


def test_module_refusals():
    from snn_compiler.nn import DecayAttention, GroupNormAct
    with pytest.raises(ValueError):
        GroupNormAct(5, 64)
    with pytest.raises(ValueError):
        GroupNormAct(8, 64, act="tanh")
    with pytest.raises(ValueError):
        DecayAttention.from_linears(*_linears(96, 6, 3, 32), torch.ones(5), heads=6, kv_heads=3)
    with pytest.raises(ValueError):
        DecayAttention.from_linears(*_linears(96, 6, 3, 32), torch.ones(6), heads=6, kv_heads=4)


def test_block_after_a_cast():
    from snn_compiler import kernels as K
    m = _block()
    x, r = _inputs((2, 40, 96), 8)
    pos = K.grid_positions(2, 4, 5)
    y, _, S = m(x, pos, r)
    decay = m.decay.clone()
    y2, _, S2 = m.to(torch.bfloat16)(x, pos, r)                # norms rounded, decays as they were
    assert m.decay.dtype == torch.float32 and torch.equal(m.decay, decay)
    with pytest.raises(ValueError, match="positions"):
        m(x)
    with pytest.raises(ValueError, match="positions"):
        m.step(x[:, 0], S)
    assert y2.isfinite().all() and (S2 - S).norm() < 0.1 * S.norm()


def test_two_captured_graphs_hold_their_own_workspaces():
    """Sequences in segments: each captured call has a workspace of its own; replays on two streams at
    once give what the eager calls gave."""
    from snn_compiler import kernels as K
    g = torch.Generator(device=DEV).manual_seed(11)
    lam = torch.tensor([0.9, 0.999], device=DEV)
    sets = [[torch.randn(1, 6000, 2, 64, generator=g, device=DEV).to(torch.bfloat16) for _ in range(3)]
            for _ in range(2)]
    state = torch.randn(1, 2, 64, 64, generator=g, device=DEV)
    want = [K.decay_attention(*s, lam, state=state) for s in sets]
    again = state.clone()                                      # in place, through the segments
    o, S = K.decay_attention(*sets[0], lam, state=again, state_out=again)
    assert S is again and torch.equal(S, want[0][1]) and torch.equal(o, want[0][0])
    graphs = []
    for s in sets:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            graphs.append((graph, K.decay_attention(*s, lam, state=state)))
        graphs[-1] = (graph, graphs[-1][1])
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(5):
        for stream, (graph, _) in zip(streams, graphs):
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    for (_, got), ref in zip(graphs, want):
        assert all(torch.equal(a, b) for a, b in zip(got, ref))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_offsets_past_32_bits(dtype):
    """Sequences, samples and states whose starts lie more than 2^32 bytes apart."""
    from snn_compiler import kernels as K
    if torch.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip("needs 40 GB")
    far = (1 << 32) // (2 if dtype == torch.float32 else 1)
    big = torch.empty(far + (1 << 20), dtype=dtype, device=DEV)
    g = torch.Generator().manual_seed(12)
    x = torch.randn(2, 40, 192, generator=g).to(dtype).to(DEV)
    row = big.as_strided((2, 40, 192), (far, 192, 1))
    row.copy_(x)
    lam = torch.tensor([0.9, 1.0], device=DEV)

    def parts(r):
        return [t.unflatten(-1, (2, 32)) for t in r.split(64, -1)]
    for a, b in zip(K.decay_attention(*parts(row), lam), K.decay_attention(*parts(x), lam)):
        assert torch.equal(a, b)
    old = torch.randn(2, 2, 32, 32, generator=g).to(DEV)
    a = K.decay_attention_step(*[t[:, 3] for t in parts(row)], lam, old.clone())
    b = K.decay_attention_step(*[t[:, 3] for t in parts(x)], lam, old.clone())
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    assert torch.equal(K.group_norm_act(row, 4, act="silu"), K.group_norm_act(x, 4, act="silu"))


def test_captured_block_replays():
    from snn_compiler import kernels as K
    m = _block()
    pos = K.grid_positions(6, 5, 5)
    x, r = _inputs((2, 150, 96), 6)
    other = _inputs((2, 150, 96), 7)
    want = m(other[0], pos, other[1])
    m(x, pos, r)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = m(x, pos, r)
    x.copy_(other[0])
    r.copy_(other[1])
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(out, want))


# many chunks an item, one item and many items a block, both widths of k, both 16-bit types, segments
@pytest.mark.parametrize("B,N,H,d,dtype", [(1, 8192, 2, 64, torch.bfloat16), (1, 8192, 2, 128, torch.float16),
                                           (40, 600, 8, 48, torch.bfloat16), (2, 4096, 40, 128, torch.bfloat16)])
def test_waits_that_run_out(B, N, H, d, dtype):
    """With a wait limit far below the kernel's time a launch gives up, lets what is in flight land and
    returns; the status word reads the time-out once, and the next launch is right."""
    from snn_compiler import _lib
    from snn_compiler import kernels as K
    from snn_compiler.kernels import conv as KC
    L = _lib.lib()
    g = torch.Generator(device=DEV).manual_seed(N)
    q, k, v = (torch.randn(B, N, H, d, generator=g, device=DEV).to(dtype) for _ in range(3))
    lam = torch.full((H,), 0.99, device=DEV)
    want = K.decay_attention(q, k, v, lam)
    flush = torch.empty(1 << 28, dtype=torch.uint8, device=DEV)
    flush.zero_()                                  # the inputs come from memory
    assert KC.device_status() == 0
    try:
        _lib.check(L.snnb_set_wait_limit(1000), "snnb_set_wait_limit")        # ~0.5 us
        t0 = time.time()
        K.decay_attention(q, k, v, lam)
        torch.cuda.synchronize()
        took = time.time() - t0
    finally:
        L.snnb_set_wait_limit(0)
    assert KC.device_status() == TIMEOUT           # cleared by the read
    assert KC.device_status() == 0
    assert took < 8.0
    got = K.decay_attention(q, k, v, lam)
    assert KC.device_status() == 0
    assert all(torch.equal(a, b) for a, b in zip(got, want))


CASES = """
import sys
sys.path.insert(0, sys.argv[2])
import torch
from snn_compiler import kernels as K
from snn_compiler.kernels import conv as KC
out, g = {}, torch.Generator().manual_seed(3)
for B, N, H, dk, dv in ((1, 9, 3, 8, 8), (2, 129, 2, 48, 72), (1, 300, 2, 128, 128), (3, 257, 4, 72, 40),
                        (1, 2000, 1, 64, 64)):
    for dtype in (torch.bfloat16, torch.float16, torch.float32):
        q, k, v = (torch.randn(B, N, H, d, generator=g).to(dtype).cuda() for d in (dk, dk, dv))
        lam = torch.rand(H, generator=g).cuda()
        o, S = K.decay_attention(q, k, v, lam, lengths=torch.full((B,), N - 3, device="cuda"))
        out[f"{B}x{N}x{H}x{dk}x{dv}{dtype}"] = torch.cat([o.flatten().float(), S.flatten()]).cpu()
torch.cuda.synchronize()
out["status"] = torch.tensor(KC.device_status())
torch.save(out, sys.argv[1])
"""


def _run(tmp_path, name, library):
    path = str(tmp_path / f"{name}.pt")
    env = dict(os.environ)
    env.pop("SNNB_LIBRARY", None)
    if library:
        env["SNNB_LIBRARY"] = library
    subprocess.run([sys.executable, "-c", CASES, path, PKG], env=env, check=True, timeout=600)
    return torch.load(path)


def test_tail_shapes_pass_the_bounds_checks(tmp_path):
    check_lib = os.path.join(PKG, "libsnnb200_check.so")
    assert os.path.exists(check_lib), "build it with `make -C triton-pass-analysis_b200 check`"
    rel, chk = _run(tmp_path, "release", None), _run(tmp_path, "check", check_lib)
    assert int(rel["status"]) == 0 and int(chk["status"]) == 0
    assert rel.keys() == chk.keys()
    for k in rel:
        assert torch.equal(rel[k], chk[k]), k
