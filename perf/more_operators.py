"""What is measured of the operators of a linear-attention block: ``snn_compiler.kernels.rotary``,
``.decay`` and ``.groupnorm``.

Four operators, each as a user calls it:

  rotary  queries and keys [B, N, H, d] turned by positions with several axes (time, height, width):
          the pair i of axis a by positions[..., a] * frequency[i]
  decay   linear attention with a decay for each head: S_t = decay S_{t-1} + k_t v_t^T,
          o_t = scale q_t S_t, over whole sequences, from a state and to a state
  step    the same for one token of each sequence
  norm    group norm of channels-last tensors, then an activation

``run`` computes them in a plain form of elementary torch operations, or, with ``own`` set, through
the framework's operators.
"""
import math
import os
import sys

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}


def listed():
    return [
        # one new token in front of the attention: latency alone
        {"name": "rotary one token", "op": "rotary", "b": 1, "n": 1, "h": 32, "hk": 8, "d": 128,
         "sections": "16,24,24", "ladder": "shared", "interleaved": False, "fused": True,
         "far": True, "batched": True, "dtype": "bf16"},
        # 4 steps of 14 x 14 patches in a block of width 384, slices of a fused projection
        {"name": "rotary 16 x 4 x 14 x 14", "op": "rotary", "b": 16, "n": 784, "h": 8, "hk": 8,
         "d": 48, "sections": "8,8,8", "ladder": "axis", "interleaved": False, "fused": True,
         "far": False, "batched": False, "dtype": "bf16"},
        # a long video prompt: memory alone
        {"name": "rotary 32768 tokens", "op": "rotary", "b": 1, "n": 32768, "h": 32, "hk": 8,
         "d": 128, "sections": "16,24,24", "ladder": "shared", "interleaved": False,
         "fused": False, "far": True, "batched": False, "dtype": "bf16"},
        # the tokens of 4 steps x 16 images in a block of width 384
        {"name": "decay 64 x 196 tokens", "op": "decay", "b": 64, "n": 196, "h": 8, "hk": 8,
         "dk": 48, "dv": 48, "state": False, "ragged": False, "fused": True, "dtype": "bf16"},
        # a padded batch that goes on from a state, shared key and value heads, float32
        {"name": "decay 3 x 1003 float32", "op": "decay", "b": 3, "n": 1003, "h": 6, "hk": 2,
         "dk": 64, "dv": 96, "state": True, "ragged": True, "fused": False, "dtype": "f32"},
        # a batch of prompts
        {"name": "decay 8 x 2048 tokens", "op": "decay", "b": 8, "n": 2048, "h": 16, "hk": 16,
         "dk": 64, "dv": 64, "state": False, "ragged": True, "fused": True, "dtype": "f16"},
        # one long prompt: few heads for the machine, many tokens each
        {"name": "decay 16384 tokens", "op": "decay", "b": 1, "n": 16384, "h": 32, "hk": 32,
         "dk": 128, "dv": 128, "state": False, "ragged": False, "fused": True, "dtype": "bf16"},
        # one sequence's next token: latency alone
        {"name": "step one sequence", "op": "step", "b": 1, "h": 32, "hk": 32, "dk": 128,
         "dv": 128, "dtype": "bf16"},
        # a full batch's next tokens: the states' traffic alone
        {"name": "step 64 sequences", "op": "step", "b": 64, "h": 32, "hk": 32, "dk": 128,
         "dv": 128, "dtype": "bf16"},
        # each token's heads behind the attention (4 x 16 x 196 tokens, width 384)
        {"name": "norm 12544 tokens", "op": "norm", "b": 12544, "s": 1, "c": 384, "groups": 8,
         "act": "silu", "affine": True, "pad": 0, "dtype": "bf16"},
        # odd sizes, float32, rows of a wider tensor
        {"name": "norm 5 x 33 x 31 x 90", "op": "norm", "b": 5, "s": 1023, "c": 90, "groups": 30,
         "act": "gelu", "affine": True, "pad": 6, "dtype": "f32"},
        # a batch of images: memory alone
        {"name": "norm 64 x 56 x 56 x 256", "op": "norm", "b": 64, "s": 3136, "c": 256,
         "groups": 32, "act": "silu", "affine": True, "pad": 0, "dtype": "bf16"},
    ]


def _size(rng, low, high, multiple=1):
    """A size spread over the logarithm of its range."""
    n = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
    return max(low, min(high, n // multiple * multiple))


def _draw_rotary(rng):
    d = _size(rng, 16, 256, rng.choice([2, 8, 16]))
    axes = rng.choice([1, 2, 3, 3])
    pairs = d // 2 if rng.random() < 0.7 else rng.randint(axes, d // 2)
    cuts = sorted(rng.sample(range(1, pairs), axes - 1))
    sections = [b - a for a, b in zip([0] + cuts, cuts + [pairs])]
    if rng.random() < 0.6:                         # the even division that configurations use
        sections = [pairs // axes] * axes
    h = _size(rng, 1, 64)
    hk = rng.choice([h, max(1, h // 4), 1])
    b = 1 if rng.random() < 0.3 else _size(rng, 1, 64)
    n = 1 if rng.random() < 0.15 else _size(rng, 1, 32768)
    while b * n * (h + hk) * d > 32768 * 40 * 128:
        b, n = (b // 2, n) if b > 1 else (b, n // 2)
    return {"op": "rotary", "b": b, "n": n, "h": h, "hk": hk, "d": d,
            "sections": ",".join(str(s) for s in sections),
            "ladder": rng.choice(["shared", "axis"]), "interleaved": rng.random() < 0.3,
            "fused": rng.random() < 0.5, "far": rng.random() < 0.5,
            "batched": rng.random() < 0.3, "dtype": rng.choice(["bf16", "bf16", "f16", "f32"])}


def _draw_heads(rng):
    """Heads and their dimensions, as an attention and its step share them."""
    h = _size(rng, 1, 32)
    hk = rng.choice([x for x in range(1, h + 1) if h % x == 0] + [h, h, h])
    multiple = rng.choice([1, 8, 16, 32])
    dk = _size(rng, max(8, multiple), 128, multiple)
    dv = dk if rng.random() < 0.6 else _size(rng, max(8, multiple), 128, multiple)
    return {"h": h, "hk": hk, "dk": dk, "dv": dv,
            "dtype": rng.choice(["bf16", "bf16", "f16", "f32"])}


def draw(rng):
    op = rng.choice(["rotary", "decay", "decay", "step", "norm"])
    if op == "rotary":
        return _draw_rotary(rng)
    if op == "step":
        heads = _draw_heads(rng)
        return {"op": op, "b": _size(rng, 1, 64), **heads}
    if op == "decay":
        heads = _draw_heads(rng)
        b = 1 if rng.random() < 0.3 else _size(rng, 1, 64)
        n = 1 if rng.random() < 0.1 else _size(rng, 1, 16384)
        while b * n * heads["h"] * (heads["dk"] + heads["dv"]) * BYTES[heads["dtype"]] > \
                16384 * 32 * 256 * 2:
            b, n = (b // 2, n) if b > 1 else (b, n // 2)
        return {"op": op, "b": b, "n": n, **heads, "state": rng.random() < 0.5,
                "ragged": rng.random() < 0.4, "fused": rng.random() < 0.6}
    groups = _size(rng, 1, 64)
    c = groups * _size(rng, 1, max(2, 2048 // groups))
    s = 1 if rng.random() < 0.3 else _size(rng, 2, 12544)
    if s == 1 and c == groups:
        c *= 4                                     # a group of one value is its bias alone
    b = _size(rng, 1, 16384 if s == 1 else 64)
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    while b * s * c * BYTES[dtype] > 64 * 3136 * 256 * 2:
        b, s = (b // 2, s) if b > 1 else (b, s // 2)
    return {"op": op, "b": b, "s": s, "c": c, "groups": groups,
            "act": rng.choice(["none", "silu", "silu", "relu", "gelu"]),
            "affine": rng.random() < 0.8, "pad": rng.choice([0, 0, 0, 32, 3]), "dtype": dtype}


# ---- the plain form ------------------------------------------------------------------------


def _frequencies(case_sections, ladder, base):
    """(frequency, axis) of every pair, frequencies in float64."""
    sections = [int(s) for s in case_sections.split(",")]
    total, freq, axis = sum(sections), [], []
    for a, count in enumerate(sections):
        for j in range(count):
            power = len(freq) / total if ladder == "shared" else j / count
            freq.append(base ** -power)
            axis.append(a)
    return freq, axis


def _turned(x, cos, sin, pairs, interleaved):
    """x [B, N, H, d] float32 with its first 2 * pairs columns turned."""
    rot, rest = x[..., :2 * pairs], x[..., 2 * pairs:]
    first, second = (rot[..., 0::2], rot[..., 1::2]) if interleaved else \
        (rot[..., :pairs], rot[..., pairs:])
    a = first * cos - second * sin
    b = first * sin + second * cos
    both = torch.stack([a, b], -1).flatten(-2) if interleaved else torch.cat([a, b], -1)
    return torch.cat([both, rest], -1)


def _plain_rotary(s):
    dev = s["q"].device
    freq = torch.tensor(s["freq"], dtype=torch.float64, device=dev)
    pos = s["positions"].double()[..., s["axis"]]              # [N, pairs] or [B, N, pairs]
    angle = pos * freq                                         # far positions: 64 bits
    cos, sin = angle.cos().float().unsqueeze(-2), angle.sin().float().unsqueeze(-2)
    if cos.dim() == 3:
        cos, sin = cos[None], sin[None]
    pairs = len(s["axis"])
    return [_turned(x.float(), cos, sin, pairs, s["interleaved"]).to(x.dtype)
            for x in (s["q"], s["k"])]


def _powers(decay, count):
    """decay^0 .. decay^(count - 1) [H, count] float32, from 64 bits."""
    return (decay.double()[:, None] ** torch.arange(count, device=decay.device)).float()


def _shared_heads(x, h):
    return x.repeat_interleave(h // x.shape[2], dim=2)


def _plain_decay(s, chunk=256):
    q, k, v = s["q"].float(), _shared_heads(s["k"].float(), s["h"]), \
        _shared_heads(s["v"].float(), s["h"])
    q, k, v = (x.transpose(1, 2) for x in (q, k, v))           # [B, H, N, d]
    bsz, h, n, dk = q.shape
    dev = q.device
    lengths = s["lengths"] if s["lengths"] is not None else \
        torch.full((bsz,), n, device=dev, dtype=torch.int32)
    alive = torch.arange(n, device=dev)[None] < lengths[:, None]           # [B, N]
    k = torch.where(alive[:, None, :, None], k, 0.0)
    v = torch.where(alive[:, None, :, None], v, 0.0)
    pw = _powers(s["decay"], chunk + 1)                                     # [H, chunk + 1]
    i = torch.arange(chunk, device=dev)
    gap = i[:, None] - i[None]
    within = torch.where(gap >= 0, pw[:, gap.clamp(min=0)], 0.0)            # [H, chunk, chunk]
    S = s["state"] if s["state"] is not None else \
        torch.zeros(bsz, h, dk, v.shape[-1], device=dev)
    outs = []
    for c in range(0, n, chunk):
        m = min(chunk, n - c)
        qc, kc, vc = q[:, :, c:c + m], k[:, :, c:c + m], v[:, :, c:c + m]
        p = (qc @ kc.transpose(-1, -2)) * within[:, :m, :m]
        outs.append(p @ vc + pw[:, 1:m + 1, None] * (qc @ S))
        held = (lengths - c).clamp(0, m).long()                             # tokens of this chunk
        left = (held[:, None] - 1 - i[None, :m]).clamp(min=0)               # [B, m]
        w = pw[:, left].transpose(0, 1)                                     # [B, H, m]
        S = pw[:, held].t()[..., None, None] * S + (kc * w[..., None]).transpose(-1, -2) @ vc
    o = torch.cat(outs, 2) * s["scale"]
    o = torch.where(alive[:, None, :, None], o, 0.0)
    return [o.transpose(1, 2).to(s["q"].dtype).contiguous(), S]


def _plain_step(s):
    h = s["h"]
    q = s["q"].float()
    k, v = (x.float().repeat_interleave(h // x.shape[1], dim=1) for x in (s["k"], s["v"]))
    S = s["decay"][None, :, None, None] * s["state"] + k[..., :, None] * v[..., None, :]
    o = (q[..., :, None] * S).sum(-2) * s["scale"]
    return [o.to(s["q"].dtype), S]


def _plain_norm(s):
    x, g = s["x"].float(), s["groups"]
    b, n, c = x.shape
    x = x.reshape(b, n, g, c // g)
    mean = x.mean((1, 3), keepdim=True)
    x = x - mean
    var = (x * x).mean((1, 3), keepdim=True)
    y = (x * torch.rsqrt(var + s["eps"])).reshape(b, n, c)
    if s["weight"] is not None:
        y = y * s["weight"].float() + s["bias"].float()
    if s["act"] == "silu":
        y = y / (1 + torch.exp(-y))
    elif s["act"] == "relu":
        y = y.clamp(min=0)
    elif s["act"] == "gelu":
        y = 0.5 * y * (1 + torch.erf(y * 0.5 ** 0.5))
    return y.to(s["x"].dtype)


_PLAIN = {"rotary": _plain_rotary, "decay": _plain_decay, "step": _plain_step,
          "norm": _plain_norm}


# ---- the framework's operators -------------------------------------------------------------

_kernels = None


def _operators():
    global _kernels
    if _kernels is None:
        root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
        package = os.path.join(root, "triton-pass-analysis_b200")
        if package not in sys.path:
            sys.path.insert(0, package)
        from snn_compiler import kernels
        _kernels = kernels
    return _kernels


def _framework(s):
    K = _operators()
    if s["op"] == "rotary":
        return list(K.rotary_axes(s["q"], s["k"], s["positions"], sections=s["sections"],
                                  base=s["base"], ladder=s["ladder"],
                                  interleaved=s["interleaved"]))
    if s["op"] == "decay":
        return list(K.decay_attention(s["q"], s["k"], s["v"], s["decay"], scale=s["scale"],
                                      state=s["state"], lengths=s["lengths"]))
    if s["op"] == "step":
        return list(K.decay_attention_step(s["q"], s["k"], s["v"], s["decay"], s["state"],
                                           scale=s["scale"], state_out=s["state_out"]))
    return K.group_norm_act(s["x"], s["groups"], s["weight"], s["bias"], eps=s["eps"],
                            act=s["act"])


# ---- inputs --------------------------------------------------------------------------------


def _heads(g, lead, counts, widths, dtype, fused, scales):
    """Tensors [*lead, heads, d]: slices of one projection's rows where `fused`."""
    sizes = [c * w for c, w in zip(counts, widths)]
    if fused:
        row = torch.randn(*lead, sum(sizes), generator=g, device="cuda")
        at = 0
        for size, scale in zip(sizes, scales):
            row[..., at:at + size] *= scale
            at += size
        row = row.to(dtype)
        parts = list(row.split(sizes, dim=-1))
    else:
        parts = [(torch.randn(*lead, size, generator=g, device="cuda") * scale).to(dtype)
                 for size, scale in zip(sizes, scales)]
    return [p.unflatten(-1, (c, w)) for p, c, w in zip(parts, counts, widths)]


def _decays(h):
    """From heads that forget within some tens of tokens to heads that hold thousands."""
    return 1 - torch.exp2(-5 - 7 * torch.arange(h, device="cuda") / max(1, h - 1))


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    op, dtype = case["op"], DTYPES[case["dtype"]]
    if op == "rotary":
        b, n = case["b"], case["n"]
        q, k = _heads(g, (b, n), (case["h"], case["hk"]), (case["d"], case["d"]), dtype,
                      case["fused"], (1.0, 1.0))
        base = 10000.0
        freq, axis = _frequencies(case["sections"], case["ladder"], base)
        axes = max(axis) + 1
        # a grid of patches in raster order, seen from a start that differs from call to call
        t = torch.arange(n, device="cuda")
        grid = torch.stack([t // 196, t % 196 // 14, t % 14][-axes:] if axes > 1 else [t], -1)
        shape = (b, 1, axes) if case["batched"] else (axes,)
        start = torch.randint(0, 2000000 if case["far"] else 64, shape, generator=g,
                              device="cuda")
        return {"op": op, "q": q, "k": k, "positions": (grid + start).to(torch.int32),
                "freq": freq, "axis": axis, "base": base, "ladder": case["ladder"],
                "sections": tuple(int(x) for x in case["sections"].split(",")),
                "interleaved": case["interleaved"]}
    if op == "norm":
        b, n, c = case["b"], case["s"], case["c"]
        x = torch.randn(b, n, c + case["pad"], generator=g, device="cuda")
        # channels of different size and mean, as the streams of trained blocks have
        x = x * (torch.rand(c + case["pad"], generator=g, device="cuda") * 2 + 0.2)
        x = (x + torch.randn(c + case["pad"], generator=g, device="cuda")).to(dtype)[..., :c]
        w = bias = None
        if case["affine"]:
            w = (torch.rand(c, generator=g, device="cuda") + 0.5).to(dtype)
            bias = (torch.randn(c, generator=g, device="cuda") * 0.2).to(dtype)
        return {"op": op, "x": x, "groups": case["groups"], "weight": w, "bias": bias,
                "eps": 1e-5, "act": case["act"]}
    b, h, hk, dk, dv = (case[x] for x in ("b", "h", "hk", "dk", "dv"))
    lead = (b, case["n"]) if op == "decay" else (b,)
    q, k, v = _heads(g, lead, (h, hk, hk), (dk, dk, dv), dtype,
                     case["fused"] if op == "decay" else True, (1.0, dk ** -0.5, 1.0))
    s = {"op": op, "q": q, "k": k, "v": v, "h": h, "decay": _decays(h), "scale": dk ** -0.5}
    state = torch.randn(b, h, dk, dv, generator=g, device="cuda") \
        if op == "step" or case["state"] else None
    s["state"] = state
    if op == "step":
        s["state_out"] = torch.empty_like(state)       # a program that keeps two takes turns
        return s
    s["lengths"] = None
    if case["ragged"]:
        s["lengths"] = torch.randint(max(1, case["n"] // 2), case["n"] + 1, (b,), generator=g,
                                     device="cuda", dtype=torch.int32)
    return s


def run(state):
    return _framework(state) if own else _PLAIN[state["op"]](state)


def work(case):
    op, size = case["op"], BYTES[case["dtype"]]
    if op == "rotary":
        elements = case["b"] * case["n"] * (case["h"] + case["hk"]) * case["d"]
        places = case["n"] * (case["b"] if case["batched"] else 1)
        axes = len(case["sections"].split(","))
        return {"bytes": 2 * elements * size + 4 * axes * places, "flops": 3 * elements}
    if op == "norm":
        elements = case["b"] * case["s"] * case["c"]
        return {"bytes": 2 * elements * size + (2 * case["c"] * size if case["affine"] else 0),
                "flops": 8 * elements}
    b, h, hk, dk, dv = (case[x] for x in ("b", "h", "hk", "dk", "dv"))
    tokens = b * (case["n"] if op == "decay" else 1)
    if op == "decay" and case["ragged"]:               # three quarters of the rows are tokens
        tokens = tokens * 3 // 4
    moved = tokens * (h * (dk + dv) + hk * (dk + dv)) * size
    states = 1 if op == "decay" and not case["state"] else 2
    return {"bytes": moved + states * 4 * b * h * dk * dv + 4 * h,
            "flops": 5 * tokens * h * dk * dv}


# ---- the definition in 64 bits -------------------------------------------------------------


def _exact_rotary(case, s):
    out = []
    pos = s["positions"].double()
    if pos.dim() == 2:
        pos = pos[None]
    sections, base = s["sections"], s["base"]
    total = sum(sections)
    for x in (s["q"], s["k"]):
        y = x.double()
        z = y.clone()
        i = 0
        for a, count in enumerate(sections):
            for j in range(count):
                one = i if case["interleaved"] is False else 2 * i
                two = i + total if case["interleaved"] is False else 2 * i + 1
                f = base ** (-(i / total) if case["ladder"] == "shared" else -(j / count))
                t = (pos[..., a] * f)[..., None]
                z[..., one] = y[..., one] * torch.cos(t) - y[..., two] * torch.sin(t)
                z[..., two] = y[..., two] * torch.cos(t) + y[..., one] * torch.sin(t)
                i += 1
        out.append(z)
    return out


def _exact_decay(case, s):
    """Every pair of tokens by itself: o_i = scale sum_{j <= i} decay^(i - j) (q_i . k_j) v_j."""
    q, k, v = s["q"].double(), s["k"].double(), s["v"].double()
    bsz, n, h, dk = q.shape
    hk, dv = k.shape[2], v.shape[3]
    lam = s["decay"].double().log()
    o = torch.zeros(bsz, n, h, dv, dtype=torch.float64, device=q.device)
    final = torch.zeros(bsz, h, dk, dv, dtype=torch.float64, device=q.device)
    count = [n] * bsz if s["lengths"] is None else [int(x) for x in s["lengths"].tolist()]
    at = torch.arange(n, device=q.device, dtype=torch.float64)
    for b in range(bsz):
        m = count[b]
        group = max(1, min(h, (1 << 25) // max(1, min(m, 2048) * m)))
        for h0 in range(0, h, group):
            hs = torch.arange(h0, min(h, h0 + group), device=q.device)
            ks = hs // (h // hk)
            kk, vv = k[b, :m, ks].transpose(0, 1), v[b, :m, ks].transpose(0, 1)   # [g, m, d]
            L = lam[hs, None, None]
            for r in range(0, m, 2048):
                e = min(m, r + 2048)
                gap = at[r:e, None] - at[None, :e]
                w = torch.where(gap >= 0, torch.exp(L * gap.clamp(min=0)), 0.0)
                qq = q[b, r:e, hs].transpose(0, 1)
                y = ((qq @ kk[:, :e].transpose(1, 2)) * w) @ vv[:, :e]
                if s["state"] is not None:
                    y = y + torch.exp(L * (at[r:e, None] + 1)) * (qq @ s["state"][b, hs].double())
                o[b, r:e, hs] = (y * s["scale"]).transpose(0, 1)
            w = torch.exp(lam[hs, None] * (m - 1 - at[None, :m]))
            final[b, hs] = (kk * w[..., None]).transpose(1, 2) @ vv
            if s["state"] is not None:
                final[b, hs] += torch.exp(L * m) * s["state"][b, hs].double()
    return [o, final]


def _exact_step(case, s):
    b, h, hk = case["b"], case["h"], case["hk"]
    q, k, v, old = (s[x].double() for x in ("q", "k", "v", "state"))
    of = torch.arange(h, device=q.device) // (h // hk)
    new = torch.einsum("h,bhkv->bhkv", s["decay"].double(), old) + \
        torch.einsum("bhk,bhv->bhkv", k[:, of], v[:, of])
    return [torch.einsum("bhk,bhkv->bhv", q, new) * s["scale"], new]


def _exact_norm(case, s):
    x, g = s["x"].double(), s["groups"]
    b, n, c = x.shape
    out = torch.empty_like(x)
    for i in range(g):
        at = slice(i * (c // g), (i + 1) * (c // g))
        part = x[..., at].flatten(1)
        var, mean = torch.var_mean(part, 1, unbiased=False, keepdim=True)
        out[..., at] = ((part - mean) / (var + s["eps"]).sqrt()).reshape(b, n, c // g)
    if s["weight"] is not None:
        out = out * s["weight"].double() + s["bias"].double()
    act = {"none": lambda y: y, "silu": lambda y: y * torch.sigmoid(y),
           "relu": torch.relu, "gelu": lambda y: y * torch.special.ndtr(y)}
    return act[s["act"]](out)


def exact(case, seed):
    s = prepare(case, seed)
    return {"rotary": _exact_rotary, "decay": _exact_decay, "step": _exact_step,
            "norm": _exact_norm}[case["op"]](case, s)
