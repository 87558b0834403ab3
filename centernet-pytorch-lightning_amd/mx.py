"""Block-scaled ("MX") operators: 8- and 4-bit floating-point storage with one power-of-two scale per 32 channels, the 4-bit product
for serving, and the backward passes that read 8-bit activation checkpoints.

    q  = mx.quantize(x, "e4m3" | "e2m1");  y = mx.dequantize(q)
    w4 = mx.pack_weight(weight);           y = mx.linear(x, w4, bias, residual, relu=True)                   # no-grad (serving)
    ck = mx.checkpoint(x, sign_of=y);      dw, db = mx.linear_wgrad(dy, ck, bias=True)
                                           dx, dgamma, dbeta, dres = mx.batch_norm_act_bwd(dy, ck, gamma, mean, invstd)

Tensors are [..., channels] in torch.bfloat16 or torch.float32 (NHWC activations of the other operators, or rows of a linear layer);
any channel count from 1 to 65536 and any number of rows, zero included where a result is defined.  Non-contiguous inputs are copied.
Work is enqueued on the current stream of the tensors' device; nothing synchronises and scratch comes from torch's allocator, so every
call can be captured into a graph and two captured graphs share no scratch.  Results do not depend on the launch (sums have a fixed
order).  Layers use these operators through `nn.use_checkpoints` (training) and `nn.use_mxfp4` (no-grad forward).

Format.  scale = the least power of two (>= 2^-127) for which the block's largest magnitude rounds to a finite element (448 / 6);
value = round-to-nearest-even(x / scale) * scale, in the type asked for (next to 2^128 it may round up to an infinity).  A block that holds an infinity or a NaN stands for 32 NaNs.
"""
import torch

from . import _hip
from ._hip import call, dtype_code

BLOCK = 32
FORMATS = {"e2m1": 0, "e4m3": 1}          # CN_MX_E2M1, CN_MX_E4M3
MAX_CHANNELS = 65536


class MXTensor:
    """A quantised tensor: `codes` uint8 [rows, Cp * bits / 8] (Cp = channels rounded up to 32), `scales` uint8 [rows, Cp / 32], the
    `shape` and `dtype` it was made from, and optionally `signs` uint8 [rows, Cp / 8] (see `checkpoint`)."""
    __slots__ = ("codes", "scales", "signs", "shape", "dtype", "fmt")

    def __init__(self, codes, scales, shape, dtype, fmt, signs=None):
        self.codes, self.scales, self.signs = codes, scales, signs
        self.shape, self.dtype, self.fmt = torch.Size(shape), dtype, fmt

    @property
    def device(self):
        return self.codes.device

    @property
    def rows(self):
        return self.codes.shape[0]

    def nbytes(self):
        return self.codes.numel() + self.scales.numel() + (self.signs.numel() if self.signs is not None else 0)

    def record_stream(self, stream):
        for t in (self.codes, self.scales, self.signs):
            if t is not None:
                t.record_stream(stream)

    def __repr__(self):
        return f"MXTensor({self.fmt}, {tuple(self.shape)}, {self.dtype}{', signs' if self.signs is not None else ''})"


class MXWeight:
    """e2m1 weights of a linear layer / 1x1 convolution in the product's own order (`pack_weight`)."""
    __slots__ = ("packed", "out_features", "in_features")

    def __init__(self, packed, out_features, in_features):
        self.packed, self.out_features, self.in_features = packed, out_features, in_features

    def __repr__(self):
        return f"MXWeight({self.out_features}, {self.in_features})"


def _tensor(t, what):
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{what}: expected a tensor, got {type(t).__name__}")
    dtype_code(t.dtype)                                    # bf16 / fp32, else TypeError
    if t.dim() < 1 or not 1 <= t.shape[-1] <= MAX_CHANNELS:
        raise ValueError(f"{what}: expected [..., 1 .. {MAX_CHANNELS} channels], got {tuple(t.shape)}")
    if not t.is_cuda:
        raise RuntimeError(f"{what}: tensor is not on the GPU (no CPU path exists)")
    return t.detach().contiguous()


def _like(t, ref, what, shape=None, dtype=None):
    """`t` as a contiguous tensor with ref's device and the wanted shape / dtype, or an error"""
    shape, dtype = ref.shape if shape is None else shape, dtype or ref.dtype
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{what}: expected a tensor, got {type(t).__name__}")
    if tuple(t.shape) != tuple(shape) or t.dtype != dtype or t.device != ref.device:
        raise ValueError(f"{what}: expected {tuple(shape)} {dtype} on {ref.device}, got {tuple(t.shape)} {t.dtype} on {t.device}")
    return t.detach().contiguous()


def _fmt(fmt):
    if fmt not in FORMATS:
        raise ValueError(f"unknown format {fmt!r}: one of {sorted(FORMATS)}")
    return FORMATS[fmt]


def _rows(t):
    return t.numel() // t.shape[-1]


def _empty(n, dtype, device):
    return torch.empty(n, dtype=dtype, device=device)


def quantize(x, fmt="e4m3"):
    """x [..., C] -> MXTensor.  One pass: x is read once, codes and scales are written."""
    return _quantize(x, fmt, None)


def checkpoint(x, sign_of=None):
    """x [..., C] -> e4m3 MXTensor for the backward pass: 8.25 bits a value instead of 16 or 32.  sign_of: the tensor (x's shape and
    dtype) whose positive entries a ReLU let through; one bit of each is kept with the codes."""
    return _quantize(x, "e4m3", sign_of)


def _quantize(x, fmt, sign_of):
    code = _fmt(fmt)
    x = _tensor(x, "mx.quantize")
    if sign_of is not None:
        sign_of = _like(sign_of, x, "mx.checkpoint: sign_of")
    rows, C = _rows(x), x.shape[-1]
    blocks = (C + BLOCK - 1) // BLOCK
    with torch.cuda.device(x.device):
        codes = _empty((rows, blocks * (32 if code else 16)), torch.uint8, x.device)
        scales = _empty((rows, blocks), torch.uint8, x.device)
        signs = _empty((rows, blocks * 4), torch.uint8, x.device) if sign_of is not None else None
        if rows:
            call("cn_mx_quantize", x, codes, scales, sign_of, signs, rows, C, code, dtype_code(x.dtype))
    return MXTensor(codes, scales, x.shape, x.dtype, fmt, signs)


def dequantize(q, dtype=None):
    """MXTensor -> the values it stands for, in `dtype` (default: the type it was made from)"""
    if not isinstance(q, MXTensor):
        raise TypeError(f"mx.dequantize: expected an MXTensor, got {type(q).__name__}")
    dtype = dtype or q.dtype
    code = dtype_code(dtype)
    with torch.cuda.device(q.device):
        out = _empty(q.shape, dtype, q.device)
        if out.numel():
            call("cn_mx_dequantize", q.codes, q.scales, out, q.rows, q.shape[-1], _fmt(q.fmt), code)
    return out


def pack_weight(weight):
    """weight [N, K] (or a 1x1 convolution's [N, K, 1, 1]), fp32 or bf16 -> MXWeight; done once per weight version"""
    if isinstance(weight, torch.Tensor) and weight.dim() == 4:
        if tuple(weight.shape[2:]) != (1, 1):
            raise ValueError(f"mx.pack_weight: only 1x1 kernels, got {tuple(weight.shape)}")
        weight = weight.reshape(weight.shape[0], weight.shape[1])
    if not isinstance(weight, torch.Tensor) or weight.dim() != 2:
        raise ValueError("mx.pack_weight: expected [out_features, in_features]")
    w = _tensor(weight, "mx.pack_weight")
    N, K = w.shape
    if not 1 <= N <= MAX_CHANNELS:
        raise ValueError(f"mx.pack_weight: out_features {N} not in 1 .. {MAX_CHANNELS}")
    with torch.cuda.device(w.device):
        packed = _empty(int(_hip.query("cn_mx_weight_bytes", N, K)), torch.uint8, w.device)
        call("cn_mx_pack_weight", w, packed, N, K, dtype_code(w.dtype))
    return MXWeight(packed, N, K)


def linear(x, weight, bias=None, residual=None, relu=False):
    """act(e2m1(x) @ weight^T + bias + residual) in x's type: x [..., K], weight an MXWeight [N, K], bias fp32 [N], residual [..., N] in
    x's type.  Serving only: an input that wants a gradient is refused (train in bf16, pack the result)."""
    if not isinstance(weight, MXWeight):
        raise TypeError("mx.linear: weight must come from mx.pack_weight")
    if torch.is_grad_enabled() and any(isinstance(t, torch.Tensor) and t.requires_grad for t in (x, bias, residual)):
        raise RuntimeError("mx.linear has no backward pass: call it under torch.no_grad()")
    x = _tensor(x, "mx.linear")
    N, K = weight.out_features, weight.in_features
    if x.shape[-1] != K:
        raise ValueError(f"mx.linear: x has {x.shape[-1]} channels, weight expects {K}")
    if weight.packed.device != x.device:
        raise ValueError(f"mx.linear: weight on {weight.packed.device}, x on {x.device}")
    shape = (*x.shape[:-1], N)
    if bias is not None:
        bias = _like(bias, x, "mx.linear: bias", (N,), torch.float32)
    if residual is not None:
        residual = _like(residual, x, "mx.linear: residual", shape)
    with torch.cuda.device(x.device):
        y = _empty(shape, x.dtype, x.device)
        if y.numel():
            call("cn_mx_linear_fwd", x, weight.packed, bias, residual, y, _rows(x), K, N, int(bool(relu)), dtype_code(x.dtype))
    return y


def _checkpoint_of(ck, dy, what):
    if not isinstance(ck, MXTensor) or ck.fmt != "e4m3":
        raise TypeError(f"{what}: expected a checkpoint (mx.checkpoint)")
    if ck.device != dy.device:
        raise ValueError(f"{what}: checkpoint on {ck.device}, gradient on {dy.device}")


def linear_wgrad(dy, ck, bias=False, into=None, bias_into=None):
    """Gradients of a linear layer / 1x1 convolution whose input was kept as `ck`: -> (dw fp32 [N, K], db fp32 [N] | None) for
    dy [..., N].  into / bias_into: contiguous fp32 tensors (of N * K / N values) the gradients are added to instead."""
    dy = _tensor(dy, "mx.linear_wgrad")
    _checkpoint_of(ck, dy, "mx.linear_wgrad")
    if dy.shape[:-1] != ck.shape[:-1]:
        raise ValueError(f"mx.linear_wgrad: gradient {tuple(dy.shape)} and checkpoint {tuple(ck.shape)} have different rows")
    rows, N, K = ck.rows, dy.shape[-1], ck.shape[-1]
    for t, n, what in ((into, N * K, "into"), (bias_into, N, "bias_into")):
        if t is not None and (t.dtype != torch.float32 or t.numel() != n or t.device != dy.device or not t.is_contiguous()):
            raise ValueError(f"mx.linear_wgrad: {what} must be contiguous fp32 with {n} values on {dy.device}")
    if bias_into is not None and into is None or into is not None and bias and bias_into is None:
        raise ValueError("mx.linear_wgrad: into and bias_into come together when a bias gradient is wanted")
    want_b = bool(bias) or bias_into is not None
    dt = dtype_code(dy.dtype)
    with torch.cuda.device(dy.device):
        dw = into if into is not None else _empty((N, K), torch.float32, dy.device)
        db = bias_into if bias_into is not None else (_empty((N,), torch.float32, dy.device) if want_b else None)
        if rows == 0:
            if into is None:
                dw.zero_()
                if db is not None:
                    db.zero_()
        else:
            n = int(_hip.query("cn_mx_linear_wgrad_bytes", rows, K, N, dt))
            ws = _empty(n, torch.uint8, dy.device)
            call("cn_mx_linear_wgrad", dy, ck.codes, ck.scales, dw, db, int(into is not None), rows, K, N, dt, ws, n)
    return dw, db


def batch_norm_act_bwd(dy, ck, gamma, mean, invstd, residual=False, racc=None, into=None):
    """Backward of y = [relu](gamma * (x - mean) * invstd + beta [+ residual]) with batch statistics over the rows, from ck =
    mx.checkpoint(x, sign_of=y) (sign_of=None: no ReLU): -> (dx, dgamma, dbeta, dres).  residual: also return the residual input's
    gradient (racc: a tensor to add to it), else dres is None.  into: (gamma.grad, beta.grad) to add to instead of new tensors."""
    dy = _tensor(dy, "mx.batch_norm_act_bwd")
    _checkpoint_of(ck, dy, "mx.batch_norm_act_bwd")
    if dy.shape != ck.shape or dy.dtype != ck.dtype:
        raise ValueError(f"mx.batch_norm_act_bwd: gradient {tuple(dy.shape)} {dy.dtype}, checkpoint of {tuple(ck.shape)} {ck.dtype}")
    rows, C = ck.rows, ck.shape[-1]
    if rows == 0:
        raise ValueError("mx.batch_norm_act_bwd: no rows (batch statistics are undefined)")
    if racc is not None and not residual:
        raise ValueError("mx.batch_norm_act_bwd: racc without residual")
    gamma, mean, invstd = (_like(t, dy, f"mx.batch_norm_act_bwd: {n}", (C,), torch.float32)
                           for t, n in ((gamma, "gamma"), (mean, "mean"), (invstd, "invstd")))
    if racc is not None:
        racc = _like(racc, dy, "mx.batch_norm_act_bwd: racc")
    if into is not None:
        for t in into:
            if _like(t, dy, "mx.batch_norm_act_bwd: into", (C,), torch.float32).data_ptr() != t.data_ptr():
                raise ValueError("mx.batch_norm_act_bwd: into must be contiguous")
    with torch.cuda.device(dy.device):
        dx = torch.empty_like(dy)
        dres = torch.empty_like(dy) if residual else None
        dgamma, dbeta = into if into is not None else (_empty((C,), torch.float32, dy.device) for _ in range(2))
        n = int(_hip.query("cn_mx_bn_bwd_bytes", rows, C))
        ws = _empty(n, torch.uint8, dy.device)
        call("cn_mx_bn_bwd", dy, ck.codes, ck.scales, ck.signs, gamma, mean, invstd, dx, dres, racc, dgamma, dbeta,
             int(into is not None), rows, C, dtype_code(dy.dtype), ws, n)
    return dx, dgamma, dbeta, dres
