"""What is measured of the microscaled operators of ``snn_compiler.kernels.mx``.

Three operators of a low-bit transformer block, each as a user calls it:

  quantise  a tensor to a microscaled format (blocks of 32 values along the last axis share one
            power-of-two scale): E2M1 elements of 4 bits ("mxfp4") or E4M3 of 8 ("mxfp8"), and back
            to the values that the codes stand for
  linear    activations in 4 or 8 bits times a 4-bit weight matrix, plus a bias
  norm      root-mean-square norm of x + residual, its output in 4 or 8 bits with scales, and the
            new residual

``run`` computes them in a plain form of elementary torch operations in 32 bits, or, with ``own``
set, through the framework's operators.

Layout of a microscaled tensor [rows, K], nb = ceil(K / 32) blocks a row:
  data    uint8 [rows, 16 nb] (E2M1, the even element in the low four bits) or [rows, 32 nb] (E4M3);
          elements past K are zero
  scales  uint8 [ceil(rows / 128), ceil(nb / 4), 32, 4, 4]: the E8M0 byte of row 128 i + 32 c + l,
          block 4 j + b, is scales[i, j, l, c, b]; bytes outside the tensor are zero
"""
import math
import os
import sys

import torch

own = False

BLOCK = 32
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}
# the largest exponent of an element: 6 = 1.5 * 2^2, 448 = 1.75 * 2^8
EMAX = {"mxfp4": 2, "mxfp8": 8}


def listed():
    return [
        # one token's hidden state in front of a 4-bit product: latency alone
        {"name": "quantise one token", "op": "quantise", "rows": 1, "k": 4096, "dtype": "bf16",
         "fmt": "mxfp4", "values": "normal", "pad": 0},
        # the spikes of 4 steps x 16 images x 196 tokens in the hidden layer of an MLP of width 384
        {"name": "quantise spikes", "op": "quantise", "rows": 12544, "k": 1536, "dtype": "bf16",
         "fmt": "mxfp4", "values": "spikes", "pad": 0},
        # a long batch of tokens: memory alone
        {"name": "quantise 16384 x 8192", "op": "quantise", "rows": 16384, "k": 8192,
         "dtype": "bf16", "fmt": "mxfp4", "values": "normal", "pad": 0},
        # serving one token: the weights are read once, nothing else counts
        {"name": "linear one token", "op": "linear", "rows": 1, "n": 4096, "k": 4096,
         "afmt": "mxfp8", "dtype": "bf16", "bias": False},
        # a small batch of requests through a wide layer
        {"name": "linear 16 tokens", "op": "linear", "rows": 16, "n": 16384, "k": 4096,
         "afmt": "mxfp4", "dtype": "bf16", "bias": True},
        # sizes that no tile divides, float32 out
        {"name": "linear 333 x 1001 x 1000", "op": "linear", "rows": 333, "n": 1001, "k": 1000,
         "afmt": "mxfp8", "dtype": "f32", "bias": True},
        # the first layer of the MLP beside spiking attention (4 x 16 x 196 tokens, width 384)
        {"name": "linear 12544 tokens, 384 wide", "op": "linear", "rows": 12544, "n": 1536,
         "k": 384, "afmt": "mxfp4", "dtype": "bf16", "bias": True},
        # a long prompt, activations in 8 bits
        {"name": "linear 4096 tokens, 8 bits", "op": "linear", "rows": 4096, "n": 8192, "k": 4096,
         "afmt": "mxfp8", "dtype": "bf16", "bias": False},
        # a large batch, activations in 4 bits: the tensor cores alone
        {"name": "linear 8192 x 8192 x 8192", "op": "linear", "rows": 8192, "n": 8192, "k": 8192,
         "afmt": "mxfp4", "dtype": "bf16", "bias": False},
        # serving one token: latency alone
        {"name": "norm one token", "op": "norm", "rows": 1, "k": 4096, "dtype": "bf16",
         "fmt": "mxfp8", "residual": True, "pad": 0},
        # odd rows of a wider tensor, no residual, float32
        {"name": "norm 517 x 1003", "op": "norm", "rows": 517, "k": 1003, "dtype": "f32",
         "fmt": "mxfp4", "residual": False, "pad": 5},
        # a long batch of tokens: memory alone
        {"name": "norm 16384 x 8192", "op": "norm", "rows": 16384, "k": 8192, "dtype": "bf16",
         "fmt": "mxfp8", "residual": True, "pad": 0},
    ]


def _size(rng, low, high, multiple=1):
    """A size spread over the logarithm of its range."""
    n = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
    n = max(low, min(high, n // multiple * multiple))
    return n + multiple if n == 3072 else n


def draw(rng):
    op = rng.choice(["quantise", "linear", "linear", "norm"])
    multiple = rng.choice([1, 1, 8, 32, 64])
    if op == "linear":
        rows = 1 if rng.random() < 0.15 else _size(rng, 1, 8192)
        n = _size(rng, 16, 16384, multiple if multiple <= 16 else 16)
        k = _size(rng, 32, 16384, multiple)
        while rows * n * k > 8192 ** 3:
            rows = max(1, rows // 2)
        return {"op": op, "rows": rows, "n": n, "k": k, "afmt": rng.choice(["mxfp4", "mxfp8"]),
                "dtype": rng.choice(["bf16", "bf16", "f16", "f32"]), "bias": rng.random() < 0.5}
    rows = 1 if rng.random() < 0.15 else _size(rng, 1, 65536)
    k = _size(rng, 16 if multiple == 1 else multiple, 16384, multiple)
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    while rows * k * BYTES[dtype] > 16384 * 8192 * 2:
        rows //= 2
    pad = rng.choice([0, 0, 0, 64, 3])
    if op == "quantise":
        return {"op": op, "rows": rows, "k": k, "dtype": dtype,
                "fmt": rng.choice(["mxfp4", "mxfp8"]),
                "values": rng.choice(["normal", "normal", "spikes"]), "pad": pad}
    return {"op": op, "rows": rows, "k": k, "dtype": dtype, "fmt": rng.choice(["mxfp8", "mxfp4"]),
            "residual": rng.random() < 0.75, "pad": pad}


# ---- the plain form ------------------------------------------------------------------------


def _element_values(fmt, device):
    """The value of every element code, by index: E2M1 (16 codes) or E4M3 (256; two are NaN)."""
    exp_bits, man_bits, bias = (2, 1, 1) if fmt == "mxfp4" else (4, 3, 7)
    codes = torch.arange(1 << (1 + exp_bits + man_bits), device=device)
    man = (codes & ((1 << man_bits) - 1)).float() / (1 << man_bits)
    exp = (codes >> man_bits) & ((1 << exp_bits) - 1)
    mag = torch.where(exp == 0, man * 2.0 ** (1 - bias), (1 + man) * torch.exp2((exp - bias).float()))
    if fmt == "mxfp8":
        mag = torch.where((codes & 127) == 127, float("nan"), mag)
    return torch.where(codes >> (exp_bits + man_bits) == 1, -mag, mag)


def _scale_values(b):
    """2^(b - 127) of E8M0 bytes, NaN for 255, in 32 bits."""
    b = b.to(torch.int32)
    v = torch.where(b == 0, 1 << 22, b << 23).view(torch.float32)
    return torch.where(b == 255, float("nan"), v)


def _round_blocks(x, fmt):
    """x [rows, K] float32 -> (elements [rows, nb, 32] rounded to the format's values, E8M0 bytes
    [rows, nb]): a block's scale is 2^(floor(log2(largest magnitude)) - EMAX), its elements are
    rounded to the nearest value, ties to even, and clamped to the largest."""
    rows, k = x.shape
    nb = -(-k // BLOCK)
    if nb * BLOCK != k:
        x = torch.nn.functional.pad(x, (0, nb * BLOCK - k))
    x = x.view(rows, nb, BLOCK)
    top = x.abs().amax(-1)
    byte = ((top.view(torch.int32) >> 23) - EMAX[fmt]).clamp(min=0)
    y = x * _scale_values(254 - byte)[..., None]
    mag = y.abs()
    if fmt == "mxfp4":
        step = torch.where(mag < 2, 0.5, torch.where(mag < 4, 1.0, 2.0))
        most = 6.0
    else:
        exp = (mag.view(torch.int32) >> 23).clamp(min=127 - 6) - 3
        step = (exp << 23).view(torch.float32)
        most = 448.0
    mag = (torch.round(mag / step) * step).clamp(max=most)
    return torch.where(y < 0, -mag, mag), byte


def _plain_values(x, fmt, dtype):
    """The values that x [rows, K] stands for once it is held in `fmt`."""
    q, byte = _round_blocks(x.float(), fmt)
    return (q * _scale_values(byte)[..., None]).flatten(1)[:, : x.shape[1]].to(dtype)


def _tile_scales(byte):
    rows, nb = byte.shape
    tr, tb = -(-rows // 128), -(-nb // 4)
    full = torch.zeros(tr * 128, tb * 4, dtype=torch.uint8, device=byte.device)
    full[:rows, :nb] = byte
    return full.view(tr, 4, 32, tb, 4).permute(0, 3, 2, 1, 4).contiguous()


def _row_scales(scales, rows, nb):
    tr, tb = scales.shape[:2]
    return scales.permute(0, 3, 2, 1, 4).reshape(tr * 128, tb * 4)[:rows, :nb]


def _pack(x, fmt):
    """x [rows, K] -> (data, scales) in the layout above."""
    q, byte = _round_blocks(x.float(), fmt)
    q = q.flatten(1)
    if fmt == "mxfp4":
        mag = q.abs()
        code = torch.where(mag <= 2, mag * 2, torch.where(mag <= 4, mag + 2, torch.full_like(mag, 7)))
        code = code.to(torch.uint8) | ((q < 0).to(torch.uint8) << 3)
        data = code[:, 0::2] | (code[:, 1::2] << 4)
    else:
        data = q.to(torch.float8_e4m3fn).view(torch.uint8)
    return data.contiguous(), _tile_scales(byte.to(torch.uint8))


def _unpack(data, scales, k, fmt):
    """The float32 values [rows, k] of (data, scales)."""
    rows = data.shape[0]
    codes = torch.stack([data & 15, data >> 4], -1).flatten(1) if fmt == "mxfp4" else data
    nb = -(-k // BLOCK)
    v = _element_values(fmt, data.device)[codes.long()].view(rows, nb, BLOCK)
    return (v * _scale_values(_row_scales(scales, rows, nb))[..., None]).flatten(1)[:, :k]


def _plain(s):
    if s["op"] == "quantise":
        return _plain_values(s["x"], s["fmt"], torch.bfloat16)
    if s["op"] == "linear":
        a = _unpack(s["a_data"], s["a_scales"], s["k"], s["afmt"])
        w = _unpack(s["w_data"], s["w_scales"], s["k"], "mxfp4")
        y = a @ w.t()
        if s["bias"] is not None:
            y = y + s["bias"]
        return y.to(s["dtype"])
    h = s["x"].float()
    if s["residual"] is not None:
        h = h + s["residual"].float()
    y = h * torch.rsqrt((h * h).mean(-1, keepdim=True) + s["eps"]) * s["weight"].float()
    q = _plain_values(y, s["fmt"], torch.bfloat16)
    return [q] if s["residual"] is None else [q, h.to(s["x"].dtype)]


# ---- the framework's operators -------------------------------------------------------------

_mx = None


def _operators():
    global _mx
    if _mx is None:
        root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
        package = os.path.join(root, "triton-pass-analysis_b200")
        if package not in sys.path:
            sys.path.insert(0, package)
        from snn_compiler.kernels import mx
        _mx = mx
    return _mx


def _framework(s):
    mx = _operators()
    if s["op"] == "quantise":
        return mx.mx_dequantize(mx.mx_quantize(s["x"], s["fmt"]), torch.bfloat16)
    if s["op"] == "linear":
        a = mx.MXTensor(s["a_data"], s["a_scales"], (s["rows"], s["k"]), s["afmt"])
        w = mx.MXTensor(s["w_data"], s["w_scales"], (s["n"], s["k"]), "mxfp4")
        return mx.mx_linear(a, w, s["bias"], dtype=s["dtype"])
    q, h = mx.rms_norm_mx(s["x"], s["weight"], s["residual"], eps=s["eps"], fmt=s["fmt"])
    q = mx.mx_dequantize(q, torch.bfloat16)
    return [q] if s["residual"] is None else [q, h]


# ---- inputs --------------------------------------------------------------------------------


def _activations(g, rows, k, dtype, pad=0, kind="normal"):
    """Rows of a wider tensor where pad > 0 (a slice of a fused projection's output)."""
    if kind == "spikes":
        x = (torch.rand(rows, k + pad, generator=g, device="cuda") < 0.15).to(dtype)
    else:
        x = torch.randn(rows, k + pad, generator=g, device="cuda")
        # a few channels of large magnitude, as the streams of trained blocks have
        x = (x * torch.where(torch.rand(k + pad, generator=g, device="cuda") < 0.01, 12.0, 1.0)).to(dtype)
    return x[:, :k]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    op, rows, k = case["op"], case["rows"], case["k"]
    dtype = DTYPES[case["dtype"]]
    if op == "quantise":
        return {"op": op, "fmt": case["fmt"],
                "x": _activations(g, rows, k, dtype, case["pad"], case["values"])}
    if op == "linear":
        n = case["n"]
        a_data, a_scales = _pack(_activations(g, rows, k, torch.float32), case["afmt"])
        w_data, w_scales = _pack(torch.randn(n, k, generator=g, device="cuda") * k ** -0.5, "mxfp4")
        return {"op": op, "rows": rows, "n": n, "k": k, "afmt": case["afmt"], "dtype": dtype,
                "a_data": a_data, "a_scales": a_scales, "w_data": w_data, "w_scales": w_scales,
                "bias": torch.randn(n, generator=g, device="cuda") * 0.1 if case["bias"] else None}
    return {"op": op, "fmt": case["fmt"], "eps": 1e-6,
            "x": _activations(g, rows, k, dtype, case["pad"]),
            "residual": _activations(g, rows, k, dtype) if case["residual"] else None,
            "weight": (torch.rand(k, generator=g, device="cuda") * 0.5 + 0.75).to(dtype)}


def run(state):
    return _framework(state) if own else _plain(state)


def work(case):
    rows, k = case["rows"], case["k"]
    nb = -(-k // BLOCK)

    def held(r, fmt):
        return r * nb * (17 if fmt == "mxfp4" else 33)
    if case["op"] == "linear":
        n = case["n"]
        return {"bytes": held(rows, case["afmt"]) + held(n, "mxfp4") + (4 * n if case["bias"] else 0)
                + rows * n * BYTES[case["dtype"]], "flops": 2 * rows * n * k}
    # x in, the codes and scales out; then the codes in and their values out
    size = rows * k * BYTES[case["dtype"]] + 2 * held(rows, case["fmt"]) + rows * k * 2
    if case["op"] == "quantise":
        return {"bytes": size, "flops": 4 * rows * k}
    size += k * BYTES[case["dtype"]]
    if case["residual"]:                      # the residual in and out
        size += 2 * rows * k * BYTES[case["dtype"]]
    return {"bytes": size, "flops": 9 * rows * k}


# ---- the definition in 64 bits -------------------------------------------------------------


def _grid64(fmt, device):
    """The non-negative finite values of the element format, in ascending order (index = code)."""
    if fmt == "mxfp4":
        v = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]
    else:
        v = [m * 2.0 ** -9 for m in range(8)]
        v += [(8 + m) * 2.0 ** (e - 3) for e in range(-6, 9) for m in range(8)][:-1]
    return torch.tensor(v, dtype=torch.float64, device=device)


def _held64(x, fmt):
    """x [rows, k] float64 -> the float64 values that its microscaled form stands for."""
    rows, k = x.shape
    grid = _grid64(fmt, x.device)
    halfway = (grid[1:] + grid[:-1]) / 2
    out = torch.empty_like(x)
    step = max(1, (1 << 25) // max(1, k))
    for r in range(0, rows, step):
        part = x[r: r + step]
        nb = -(-k // 32)
        b = torch.zeros(part.shape[0], nb * 32, dtype=torch.float64, device=x.device)
        b[:, :k] = part
        b = b.view(part.shape[0], nb, 32)
        largest = b.abs().max(-1).values
        # frexp: largest = m 2^e with 0.5 <= m < 1
        e = torch.frexp(largest).exponent.long() - 1 - EMAX[fmt]
        e = torch.where(largest > 0, e, -127).clamp(-127, 127)
        scale = torch.ldexp(torch.ones_like(largest), e)[..., None]
        v = b / scale
        below = torch.bucketize(v.abs(), halfway)
        upto = torch.bucketize(v.abs(), halfway, right=True)
        code = torch.where(below == upto, below, below + (below & 1))   # a tie: the even code
        out[r: r + step] = (grid[code] * v.sign() * scale).flatten(1)[:, :k]
    return out


def _read64(data, scales, k, fmt):
    """The float64 values of codes and scales in the layout above."""
    rows, dev = data.shape[0], data.device
    nb = -(-k // 32)
    grid = _grid64(fmt, dev)
    if fmt == "mxfp4":
        c = torch.empty(rows, nb * 32, dtype=torch.int64, device=dev)
        c[:, 0::2] = (data % 16).long()
        c[:, 1::2] = (data // 16).long()
        sign, code = c // 8, c % 8
    else:
        sign, code = (data // 128).long(), (data % 128).long()
    v = grid[code] * (1 - 2 * sign)
    r = torch.arange(rows, device=dev)[:, None]
    j = torch.arange(nb, device=dev)[None]
    byte = scales[r // 128, j // 4, r % 32, r % 128 // 32, j % 4].double()
    return (v.view(rows, nb, 32) * torch.exp2(byte - 127)[..., None]).flatten(1)[:, :k]


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "quantise":
        return _held64(s["x"].double(), case["fmt"])
    if case["op"] == "linear":
        y = _read64(s["a_data"], s["a_scales"], s["k"], s["afmt"]) @ \
            _read64(s["w_data"], s["w_scales"], s["k"], "mxfp4").t()
        return y if s["bias"] is None else y + s["bias"].double()
    h = s["x"].double()
    if s["residual"] is not None:
        h = h + s["residual"].double()
    root = ((h ** 2).sum(-1, keepdim=True) / case["k"] + s["eps"]).sqrt()
    q = _held64(h / root * s["weight"].double(), case["fmt"])
    return [q] if s["residual"] is None else [q, h]
