"""Workloads of the block-scaled operators (centernet_amd.mx): quantisation to 8- and 4-bit floating point with one power-of-two
scale per 32 channels, the product of 4-bit activations and 4-bit weights (a 1x1 convolution / linear layer), and the two backward passes that read 8-bit
activation checkpoints (weight gradient; batch norm + ReLU + residual).

Every case is rows x channels: an NHWC activation [B, H, W, C] has B * H * W rows.  `listed()` holds representative sizes, `draw()` more
of the same ranges; `run()` is one pass, by the framework's kernels where `own` is true and in elementary torch operations otherwise;
`exact()` is the same result in 64 bits, written from the definitions.

Definition of the format.  For a block of up to 32 consecutive channels of a row with largest magnitude a:
    scale = the least power of two s = 2^e, e >= -127, for which a / s, rounded to nearest even on the element grid, is no larger than
            the largest finite element (6 for e2m1, 448 for e4m3);  an all-zero block has e = -127
    value = round_to_nearest_even(x / s) * s
"""
import math

import torch

own = False

BLOCK = 32
DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
SIZE = {"bf16": 2, "f32": 4}
#: bits of one element, exponent of the largest finite element, and that element's neighbourhood: magnitudes m * 2^emax with m up to
#: `top` still round to it (`tie`: m == top does too)
GRID = {"e2m1": dict(bits=4, emax=2, top=1.75, tie=False), "e4m3": dict(bits=8, emax=8, top=1.8125, tie=True)}


# ---------------------------------------------------------------------------------------------------------------- the cases
def listed():
    return [
        # a deep 512-channel map of two 128^2 images kept for the backward pass: the launch is what costs
        dict(name="pack e4m3 32x512", op="pack", dtype="bf16", fmt="e4m3", rows=32, k=512),
        # an 80-class map with odd sides, 32-bit parity mode, 4-bit: two and a half blocks a row
        dict(name="pack e2m1 f32 16700x80", op="pack", dtype="f32", fmt="e2m1", rows=16700, k=80),
        # the 64-channel stride-4 map of a training batch of 64 at 512^2: pure bandwidth
        dict(name="pack e4m3 1048576x64", op="pack", dtype="bf16", fmt="e4m3", rows=64 * 128 * 128, k=64),
        # one pixel / one token through a 2048 -> 512 projection: latency
        dict(name="linear 1x2048x512", op="linear", dtype="bf16", rows=1, k=2048, n=512, bias=True, residual=False, relu=False),
        # ragged everything in 32-bit parity mode
        dict(name="linear f32 5883x208x80", op="linear", dtype="f32", rows=3 * 37 * 53, k=208, n=80, bias=True, residual=False, relu=True),
        # bottleneck entry of a ResNet-101 stage 3 at batch 64, 512^2: 1024 -> 256
        dict(name="linear 65536x1024x256", op="linear", dtype="bf16", rows=64 * 32 * 32, k=1024, n=256, bias=True, residual=False, relu=True),
        # bottleneck exit of the same stage with its identity path: 256 -> 1024
        dict(name="linear 65536x256x1024", op="linear", dtype="bf16", rows=64 * 32 * 32, k=256, n=1024, bias=True, residual=True, relu=True),
        # a wide projection of few rows (a small batch, deep in the network)
        dict(name="wgrad 1024x2048x512", op="wgrad", dtype="bf16", rows=4 * 16 * 16, k=2048, n=512, bias=False),
        dict(name="wgrad f32 5883x208x80", op="wgrad", dtype="f32", rows=3 * 37 * 53, k=208, n=80, bias=True),
        # bottleneck entry of stage 2 at batch 64: the sum runs over 262144 pixels
        dict(name="wgrad 262144x256x128", op="wgrad", dtype="bf16", rows=64 * 64 * 64, k=256, n=128, bias=False),
        # a small deep layer, and the bottleneck exit of stage 1's sequel at batch 64 with its identity path
        dict(name="norm 512x512", op="norm", dtype="bf16", rows=2 * 16 * 16, k=512, residual=True, relu=True),
        dict(name="norm 262144x256", op="norm", dtype="bf16", rows=64 * 64 * 64, k=256, residual=True, relu=True),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["pack", "linear", "wgrad", "norm"])
    case = dict(op=op, dtype=rng.choice(["bf16", "bf16", "bf16", "f32"]))
    k = _log(rng, 16, 2048)
    if rng.random() < 0.6:
        k = (k + 15) // 16 * 16                      # the framework's activations have a multiple of 16 channels; odd counts hold too
    n = _log(rng, 2, 2048)
    if op in ("pack", "norm"):
        case.update(rows=_log(rng, 1, max(1, min(262144, 33_000_000 // k))), k=k)
        if op == "pack":
            case.update(fmt=rng.choice(["e2m1", "e4m3"]))
        else:
            case.update(rows=max(2, case["rows"]), residual=rng.random() < 0.5, relu=rng.random() < 0.75)
        return case
    most = min(262144, 33_000_000 // max(k, n), 17_000_000_000 // (k * n))
    case.update(rows=_log(rng, 1, max(1, most)), k=k, n=n, bias=rng.random() < 0.5)
    if op == "linear":
        case.update(residual=rng.random() < 0.4, relu=rng.random() < 0.5)
    return case


# ---------------------------------------------------------------------------------------------------------------- inputs
def _activations(g, rows, k, dtype, positive):
    """Channels of unlike magnitude, a few dead ones, now and then a pixel far above the rest; `positive`: behind a ReLU."""
    x = torch.randn(rows, k, generator=g, device="cuda")
    x *= torch.exp(0.7 * torch.randn(k, generator=g, device="cuda"))
    x *= (torch.rand(k, generator=g, device="cuda") > 0.03).float()
    x *= 1 + 15 * (torch.rand(rows, 1, generator=g, device="cuda") < 0.01).float()
    return (x.clamp_(min=0) if positive else x).to(DTYPES[dtype])


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed) * 1000003 + 17)
    rows, k, dt = case["rows"], case["k"], DTYPES[case["dtype"]]
    s = dict(case=case)
    if case["op"] == "pack":
        s["x"] = _activations(g, rows, k, case["dtype"], False)
    elif case["op"] == "linear":
        n = case["n"]
        s["x"] = _activations(g, rows, k, case["dtype"], True)
        w = torch.randn(n, k, generator=g, device="cuda") / math.sqrt(k)
        s["bias"] = 0.1 * torch.randn(n, generator=g, device="cuda") if case["bias"] else None
        s["residual"] = _activations(g, rows, n, case["dtype"], True) if case["residual"] else None
        s["w"] = w
        # the weights are laid out once, as a program keeps them
        if own:
            from centernet_amd import mx
            s["packed"] = mx.pack_weight(w)
        else:
            s["values"] = _values(w, "e2m1")
    elif case["op"] == "wgrad":
        s["x"] = _activations(g, rows, k, case["dtype"], True)
        s["dy"] = (1e-3 * torch.randn(rows, case["n"], generator=g, device="cuda")).to(dt)
    else:
        s["x"] = _activations(g, rows, k, case["dtype"], False)
        x = s["x"].double()
        var, mean = torch.var_mean(x, dim=0, correction=0)
        s["mean"], s["invstd"] = mean.float(), torch.rsqrt(var + 1e-5).float()
        s["gamma"] = 1 + 0.2 * torch.randn(k, generator=g, device="cuda")
        s["y"] = torch.randn(rows, k, generator=g, device="cuda").clamp_(min=0).to(dt) if case["relu"] else None   # the layer's output
        s["dy"] = (1e-3 * torch.randn(rows, k, generator=g, device="cuda")).to(dt)
    return s


# ---------------------------------------------------------------------------------------------------------------- one pass
def _blocks(x):
    """[rows, k] in 32 bits -> [rows, blocks, 32], the last block filled up with zeros"""
    x = x.float()
    return torch.nn.functional.pad(x, (0, -x.shape[1] % BLOCK)).view(x.shape[0], -1, BLOCK)


def _two_to(e):
    """2^e in 32 bits from its exponent field, -127 <= e <= 127 (2^-127 is subnormal)"""
    return torch.where(e > -127, (e + 127) << 23, torch.full_like(e, 1 << 22)).to(torch.int32).view(torch.float32)


def _values(x, fmt):
    """What x stands for after quantisation, in 32 bits (each step is exact: scaling by powers of two, one rounding to the grid)."""
    f, b = GRID[fmt], _blocks(x)
    m, e = torch.frexp(b.abs().amax(-1, keepdim=True))            # a = m * 2^e with m in [0.5, 1)
    up = (2 * m > f["top"]) if f["tie"] else (2 * m >= f["top"])
    e = torch.where(m == 0, torch.full_like(e, -127), (e - 1 - f["emax"] + up.to(e.dtype)).clamp(min=-127))
    v = b * _two_to(-e)
    if fmt == "e2m1":
        a = v.abs()
        step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
        v = torch.round(v / step) * step
    else:
        v = v.clamp(-448, 448).to(torch.float8_e4m3fn).float()
    return (v * _two_to(e)).view(x.shape[0], -1)[:, :x.shape[1]]


def run(s):
    c = s["case"]
    if own:
        from centernet_amd import mx
        if c["op"] == "pack":
            return mx.dequantize(mx.quantize(s["x"], c["fmt"]))
        if c["op"] == "linear":
            return mx.linear(s["x"], s["packed"], s["bias"], s["residual"], relu=c["relu"])
        if c["op"] == "wgrad":
            return mx.linear_wgrad(s["dy"], mx.checkpoint(s["x"]), bias=c["bias"])
        ck = mx.checkpoint(s["x"], sign_of=s["y"])
        return mx.batch_norm_act_bwd(s["dy"], ck, s["gamma"], s["mean"], s["invstd"], residual=c["residual"])
    dt = s["x"].dtype
    if c["op"] == "pack":
        return _values(s["x"], c["fmt"]).to(dt)
    if c["op"] == "linear":
        y = _values(s["x"], "e2m1") @ s["values"].t()
        if s["bias"] is not None:
            y = y + s["bias"]
        if s["residual"] is not None:
            y = y + s["residual"].float()
        return (y.clamp(min=0) if c["relu"] else y).to(dt)
    dy = s["dy"].float()
    if c["op"] == "wgrad":
        return dy.t() @ _values(s["x"], "e4m3"), dy.sum(0) if c["bias"] else None
    xh = (_values(s["x"], "e4m3") - s["mean"]) * s["invstd"]
    d = dy * (s["y"].float() > 0) if c["relu"] else dy
    dbeta, dgamma = d.sum(0), (d * xh).sum(0)
    dx = s["gamma"] * s["invstd"] * (d - (dbeta + xh * dgamma) / c["rows"])
    return dx.to(dt), dgamma, dbeta, d.to(dt) if c["residual"] else None


# ---------------------------------------------------------------------------------------------------------------- what a pass needs
def _packed_bytes(rows, k, fmt):
    return rows * (k * GRID[fmt]["bits"] / 8 + math.ceil(k / BLOCK))


def work(case):
    rows, k, b = case["rows"], case["k"], SIZE[case["dtype"]]
    if case["op"] == "pack":                       # x in, the packed form out, the values out
        return dict(bytes=2 * rows * k * b + _packed_bytes(rows, k, case["fmt"]), flops=4 * rows * k)
    if case["op"] == "linear":
        n = case["n"]
        return dict(bytes=rows * k * b + _packed_bytes(n, k, "e2m1") + rows * n * b * (2 if case["residual"] else 1) + 4 * n * case["bias"],
                    flops=2 * rows * k * n)
    if case["op"] == "wgrad":                      # x and dy in, the checkpoint out, the gradient out
        n = case["n"]
        return dict(bytes=rows * (k + n) * b + _packed_bytes(rows, k, "e4m3") + 4 * n * (k + case["bias"]), flops=2 * rows * k * n)
    return dict(bytes=rows * k * b * (3 + case["relu"] + case["residual"]) + _packed_bytes(rows, k, "e4m3") + 20 * k, flops=12 * rows * k)


# ---------------------------------------------------------------------------------------------------------------- 64 bits
def _grid64(fmt):
    """The format's non-negative finite elements in order, from its exponent and significand fields."""
    ebits, mbits, bias = (2, 1, 1) if fmt == "e2m1" else (4, 3, 7)
    vals = []
    for e in range(2 ** ebits):
        for m in range(2 ** mbits):
            if fmt == "e4m3" and e == 15 and m == 7:
                continue                                           # not a number
            vals.append((m / 2 ** mbits) * 2.0 ** (1 - bias) if e == 0 else (1 + m / 2 ** mbits) * 2.0 ** (e - bias))
    return vals


def _power64(e):
    return ((e.long() + 1023) << 52).view(torch.float64)            # (pow() on a GPU is an ulp off now and then)


def _values64(x, fmt):
    """Rounding by comparison with the midpoints of the grid (a midpoint goes to the neighbour with the even code)."""
    grid = torch.tensor(_grid64(fmt), dtype=torch.float64, device=x.device)
    mid = (grid[1:] + grid[:-1]) / 2
    rows, k = x.shape
    b = torch.zeros(rows, (k + BLOCK - 1) // BLOCK * BLOCK, dtype=torch.float64, device=x.device)
    b[:, :k] = x.double()
    b = b.view(rows, -1, BLOCK)
    a = b.abs().amax(-1, keepdim=True)
    last, below = grid[-1], grid[-2]
    limit = last + (last - below) / 2                               # where the grid's next element would begin to win
    odd_next = (len(grid) - 1) % 2 == 0                             # an even last code keeps the midpoint
    e = torch.floor(torch.log2(torch.where(a > 0, a, torch.ones_like(a)))) - 9
    for _ in range(12):                                             # the least e that fits, by trial
        fits = (a <= limit * _power64(e)) if odd_next else (a < limit * _power64(e))
        e = torch.where(fits, e, e + 1)
    s = _power64(torch.where(a > 0, e.clamp(min=-127), torch.full_like(e, -127)))
    v = b / s
    up, down = torch.bucketize(v.abs(), mid, right=True), torch.bucketize(v.abs(), mid, right=False)
    code = torch.where(up == down, up, up + (up % 2) * (down - up))  # on a midpoint the two differ: take the even one
    return (torch.copysign(grid[code], v) * s).view(rows, -1)[:, :k]


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "pack":
        return _values64(s["x"], case["fmt"])
    if case["op"] == "linear":
        y = torch.matmul(_values64(s["x"], "e2m1"), _values64(s["w"], "e2m1").t().contiguous())
        if case["bias"]:
            y += s["bias"].double()
        if case["residual"]:
            y += s["residual"].double()
        return torch.relu(y) if case["relu"] else y
    dy, x = s["dy"].double(), _values64(s["x"], "e4m3")
    if case["op"] == "wgrad":
        return torch.matmul(dy.t().contiguous(), x), dy.sum(0) if case["bias"] else None
    mean, invstd, gamma, rows = s["mean"].double(), s["invstd"].double(), s["gamma"].double(), case["rows"]
    if case["relu"]:
        dy = torch.where(s["y"] > 0, dy, torch.zeros_like(dy))
    xh = (x - mean) * invstd
    dgamma, dbeta = torch.einsum("rk,rk->k", dy, xh), dy.sum(dim=0)
    dx = (dy - dbeta / rows - xh * (dgamma / rows)) * (gamma * invstd)
    return dx, dgamma, dbeta, dy if case["residual"] else None
