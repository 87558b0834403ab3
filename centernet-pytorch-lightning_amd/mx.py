"""Block-scaled ("MX") operators: 8- and 4-bit floating-point storage with one power-of-two scale per 32 channels, the 4-bit product
for serving, and the backward passes that read 8-bit activation checkpoints.

    q  = mx.quantize(x, "e4m3" | "e2m1");  y = mx.dequantize(q)
    w4 = mx.pack_weight(weight);           y = mx.linear(x, w4, bias, residual, relu=True)                   # no-grad (serving)
    ck = mx.checkpoint(x, sign_of=y);      dw, db = mx.linear_wgrad(dy, ck, bias=True)
    y, ck = mx.scale_shift_act(x, scale, shift, residual, relu=True)                                          # y and x's checkpoint at once
                                           dx, dgamma, dbeta, dres = mx.batch_norm_act_bwd(dy, ck, gamma, mean, invstd)

Tensors are [..., channels] in torch.bfloat16 or torch.float32 (NHWC activations of the other operators, or rows of a linear layer);
any channel count from 1 to 65536 and any number of rows, zero included where a result is defined (what one launch's 2^32 threads do not
cover is refused: from 2^32 blocks of 32 channels when quantising, from 2^29 rows of a product).  Nothing here is recorded by autograd
(the layers' autograd functions call these): `quantize`, `scale_shift_act` and `linear` refuse inputs that want a gradient while autograd
records, a checkpoint and the results of the backward passes are constants to it.  Non-contiguous inputs are copied.
Work is enqueued on the current stream of the tensors' device; nothing synchronises and scratch comes from torch's allocator, so every
call can be captured into a graph and two captured graphs share no scratch.  Results do not depend on the launch (sums have a fixed
order).  Layers use these operators through `nn.use_checkpoints` (training) and `nn.use_mxfp4` (no-grad forward).

Format.  scale = the least power of two (>= 2^-127) for which the block's largest magnitude rounds to a finite element (448 / 6): nothing
saturates.  (The rule that the OCP specification of these formats recommends, 2^(floor(log2 max) - emax), is half of that for the blocks
whose largest magnitude would round past the last element, and saturates there; both decode alike.)
value = round-to-nearest-even(x / scale) * scale, in the type asked for (next to 2^128 it may round up to an infinity).  A block that holds an infinity or a NaN stands for 32 NaNs.
"""
import torch

from . import _hip
from ._hip import launch

BLOCK = 32
FORMATS = {"e2m1": 0, "e4m3": 1}          # CN_MX_E2M1, CN_MX_E4M3
MAX_CHANNELS = 65536
_DTYPES = {torch.float32: _hip.CN_F32, torch.bfloat16: _hip.CN_BF16}


class MXTensor:
    """A quantised tensor: `codes` uint8 [rows, Cp * bits / 8] (Cp = channels rounded up to 32), `scales` uint8 [rows, Cp / 32], the
    `shape` and `dtype` it was made from, and optionally `signs` uint8 [rows, Cp / 8] (see `checkpoint`) — three views of one buffer."""
    __slots__ = ("buffer", "shape", "dtype", "fmt", "rows", "blocks", "has_signs", "_n")

    def __init__(self, shape, dtype, fmt, device, signs=False, buffer=None):
        self.shape, self.dtype, self.fmt, self.has_signs = shape, dtype, fmt, signs
        self.blocks = (shape[-1] + BLOCK - 1) // BLOCK
        self.rows = shape[:-1].numel()
        self._n = self.rows * self.blocks                  # blocks in all
        n = self._n * ((33 if fmt == "e4m3" else 17) + (4 if signs else 0))
        if buffer is None:
            buffer = torch.empty(n, dtype=torch.uint8, device=device)
        elif buffer.numel() != n or buffer.dtype != torch.uint8 or not buffer.is_contiguous():
            raise ValueError(f"MXTensor: a contiguous uint8 buffer of {n} bytes is needed, got {tuple(buffer.shape)} {buffer.dtype}")
        self.buffer = buffer

    @property
    def meta(self):
        """what makes the tensor again from its buffer: `MXTensor.of(buffer, meta)` (an autograd node saves the buffer)"""
        return self.shape, self.dtype, self.fmt, self.has_signs

    @classmethod
    def of(cls, buffer, meta):
        shape, dtype, fmt, signs = meta
        return cls(shape, dtype, fmt, buffer.device, signs, buffer)

    def _pointers(self):
        """codes, scales, signs (None without)"""
        p = self.buffer.data_ptr()
        s = p + self._n * (32 if self.fmt == "e4m3" else 16)
        return p, s, s + self._n if self.has_signs else None

    def _part(self, first, width):
        return self.buffer[self._n * first:self._n * (first + width)].view(self.rows, self.blocks * width)

    @property
    def codes(self):
        return self._part(0, 32 if self.fmt == "e4m3" else 16)

    @property
    def scales(self):
        return self._part(32 if self.fmt == "e4m3" else 16, 1)

    @property
    def signs(self):
        return self._part(33 if self.fmt == "e4m3" else 17, 4) if self.has_signs else None

    @property
    def device(self):
        return self.buffer.device

    def nbytes(self):
        return self.buffer.numel()

    def record_stream(self, stream):
        self.buffer.record_stream(stream)

    def __repr__(self):
        return f"MXTensor({self.fmt}, {tuple(self.shape)}, {self.dtype}{', signs' if self.has_signs else ''})"


class MXWeight:
    """e2m1 weights of a linear layer / 1x1 convolution in the product's own order (`pack_weight`)."""
    __slots__ = ("packed", "out_features", "in_features", "_n")

    def __init__(self, packed, out_features, in_features):
        if packed.dtype != torch.uint8 or not packed.is_contiguous():
            raise ValueError("MXWeight: packed must be contiguous uint8")
        self.packed, self.out_features, self.in_features = packed, out_features, in_features
        self._n = _hip.query("cn_mx_weight_bytes", out_features, in_features)

    def __repr__(self):
        return f"MXWeight({self.out_features}, {self.in_features})"


def _tensor(t, what):
    """-> (t contiguous, dtype code), or an error"""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{what}: expected a tensor, got {type(t).__name__}")
    code = _DTYPES.get(t.dtype)
    if code is None:
        raise TypeError(f"{what}: unsupported dtype {t.dtype} (bfloat16 or float32)")
    if t.dim() < 1 or not 1 <= t.shape[-1] <= MAX_CHANNELS:
        raise ValueError(f"{what}: expected [..., 1 .. {MAX_CHANNELS} channels], got {tuple(t.shape)}")
    if not t.is_cuda:
        raise RuntimeError(f"{what}: tensor is not on the GPU (no CPU path exists)")
    return (t if t.is_contiguous() else t.contiguous()), code


def _unrecorded(what, *tensors):
    """an error where autograd would record the call and a tensor wants a gradient: the result would be a constant, without a word"""
    if torch.is_grad_enabled() and any(getattr(t, "requires_grad", False) for t in tensors):
        raise RuntimeError(f"{what} has no backward pass: call it under torch.no_grad(), or on detached tensors")


def _like(t, device, shape, dtype, what):
    """t contiguous if it is a tensor of that device, shape and type, else an error"""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{what}: expected a tensor, got {type(t).__name__}")
    if t.shape != shape or t.dtype != dtype or t.device != device:
        raise ValueError(f"{what}: expected {tuple(shape)} {dtype} on {device}, got {tuple(t.shape)} {t.dtype} on {t.device}")
    return t if t.is_contiguous() else t.contiguous()


def _ptr(t):
    return None if t is None else t.data_ptr()


def _fmt(fmt):
    if fmt not in FORMATS:
        raise ValueError(f"unknown format {fmt!r}: one of {sorted(FORMATS)}")
    return FORMATS[fmt]


def quantize(x, fmt="e4m3"):
    """x [..., C] -> MXTensor.  One pass: x is read once, codes and scales are written."""
    _unrecorded("mx.quantize", x)
    return _quantize(x, fmt, None, "mx.quantize")


def checkpoint(x, sign_of=None):
    """x [..., C] -> e4m3 MXTensor for the backward pass: 8.25 bits a value instead of 16 or 32.  sign_of: the tensor (x's shape and
    dtype) whose positive entries a ReLU let through; one bit of each is kept with the codes.  A copy: no gradient comes back through it."""
    return _quantize(x, "e4m3", sign_of, "mx.checkpoint")


def scale_shift_act(x, scale, shift, residual=None, relu=False):
    """-> (y, ck): y = act(x * scale + shift + residual) per channel (scale, shift fp32 [C]) and ck = checkpoint(x, sign_of=y if relu), in one
    pass over x: a normalisation's forward apply that keeps what its backward (`batch_norm_act_bwd`) needs."""
    _unrecorded("mx.scale_shift_act", x, scale, shift, residual)
    x, dt = _tensor(x, "mx.scale_shift_act")
    dev, one = x.device, (x.shape[-1],)
    scale = _like(scale, dev, one, torch.float32, "mx.scale_shift_act: scale")
    shift = _like(shift, dev, one, torch.float32, "mx.scale_shift_act: shift")
    if residual is not None:
        residual = _like(residual, dev, x.shape, x.dtype, "mx.scale_shift_act: residual")
    y, q = torch.empty_like(x), MXTensor(x.shape, x.dtype, "e4m3", dev, bool(relu))
    codes, scales, signs = q._pointers()
    launch("cn_mx_scale_shift_act", x.get_device(), x.data_ptr(), _ptr(residual), scale.data_ptr(), shift.data_ptr(), y.data_ptr(), codes,
           scales, signs, q.rows, x.shape[-1], 1 if relu else 0, dt)
    return y, q


def _quantize(x, fmt, sign_of, what):
    code = _fmt(fmt)
    x, dt = _tensor(x, what)
    if sign_of is not None:
        sign_of = _like(sign_of, x.device, x.shape, x.dtype, "mx.checkpoint: sign_of")
    q = MXTensor(x.shape, x.dtype, fmt, x.device, sign_of is not None)
    codes, scales, signs = q._pointers()
    launch("cn_mx_quantize", x.get_device(), x.data_ptr(), codes, scales, _ptr(sign_of), signs, q.rows, x.shape[-1], code, dt)
    return q


def dequantize(q, dtype=None):
    """MXTensor -> the values it stands for, in `dtype` (default: the type it was made from); to autograd a constant"""
    if not isinstance(q, MXTensor):
        raise TypeError(f"mx.dequantize: expected an MXTensor, got {type(q).__name__}")
    dtype = dtype or q.dtype
    if dtype not in _DTYPES:
        raise TypeError(f"mx.dequantize: unsupported dtype {dtype} (bfloat16 or float32)")
    if not q.buffer.is_cuda:
        raise RuntimeError("mx.dequantize: tensor is not on the GPU (no CPU path exists)")
    out = q.buffer.new_empty(*q.shape, dtype=dtype)
    codes, scales, _ = q._pointers()
    launch("cn_mx_dequantize", out.get_device(), codes, scales, out.data_ptr(), q.rows, q.shape[-1], FORMATS[q.fmt], _DTYPES[dtype])
    return out


def pack_weight(weight):
    """weight [N, K] (or a 1x1 convolution's [N, K, 1, 1]), fp32 or bf16 -> MXWeight; done once per weight version"""
    if isinstance(weight, torch.Tensor) and weight.dim() == 4:
        if tuple(weight.shape[2:]) != (1, 1):
            raise ValueError(f"mx.pack_weight: only 1x1 kernels, got {tuple(weight.shape)}")
        weight = weight.reshape(weight.shape[0], weight.shape[1])
    if not isinstance(weight, torch.Tensor) or weight.dim() != 2:
        raise ValueError("mx.pack_weight: expected [out_features, in_features]")
    w, dt = _tensor(weight, "mx.pack_weight")
    N, K = w.shape
    if not 1 <= N <= MAX_CHANNELS:
        raise ValueError(f"mx.pack_weight: out_features {N} not in 1 .. {MAX_CHANNELS}")
    packed = torch.empty(_hip.query("cn_mx_weight_bytes", N, K), dtype=torch.uint8, device=w.device)
    launch("cn_mx_pack_weight", w.get_device(), w.data_ptr(), packed.data_ptr(), N, K, dt)
    return MXWeight(packed, N, K)


def linear(x, weight, bias=None, residual=None, relu=False):
    """act(e2m1(x) @ weight^T + bias + residual) in x's type: x [..., K], weight an MXWeight [N, K], bias fp32 [N], residual [..., N] in
    x's type.  Serving only: an input that wants a gradient is refused (train in bf16, pack the result)."""
    if not isinstance(weight, MXWeight):
        raise TypeError("mx.linear: weight must come from mx.pack_weight")
    _unrecorded("mx.linear", x, bias, residual)
    x, dt = _tensor(x, "mx.linear")
    N, K, dev = weight.out_features, weight.in_features, x.device
    if x.shape[-1] != K:
        raise ValueError(f"mx.linear: x has {x.shape[-1]} channels, weight expects {K}")
    if weight.packed.device != dev:
        raise ValueError(f"mx.linear: weight on {weight.packed.device}, x on {dev}")
    if weight.packed.numel() != weight._n:
        raise ValueError(f"mx.linear: packed weights of {weight._n} bytes are needed, got {weight.packed.numel()}")
    lead = x.shape[:-1]
    shape = (*lead, N)
    if bias is not None:
        bias = _like(bias, dev, (N,), torch.float32, "mx.linear: bias")
    if residual is not None:
        residual = _like(residual, dev, shape, x.dtype, "mx.linear: residual")
    y = x.new_empty(*shape) if residual is None else torch.empty_like(residual)
    launch("cn_mx_linear_fwd", x.get_device(), x.data_ptr(), weight.packed.data_ptr(), _ptr(bias), _ptr(residual), y.data_ptr(), lead.numel(),
           K, N, 1 if relu else 0, dt)
    return y


def _checkpoint_of(ck, dy, what):
    if not isinstance(ck, MXTensor) or ck.fmt != "e4m3":
        raise TypeError(f"{what}: expected a checkpoint (mx.checkpoint)")
    if ck.device != dy.device:
        raise ValueError(f"{what}: checkpoint on {ck.device}, gradient on {dy.device}")


def linear_wgrad(dy, ck, bias=False, into=None, bias_into=None):
    """Gradients of a linear layer / 1x1 convolution whose input was kept as `ck`: -> (dw fp32 [N, K], db fp32 [N] | None) for
    dy [..., N].  into / bias_into: contiguous fp32 tensors (of N * K / N values) the gradients are added to instead.  N and K of which
    more than 65535 output tiles (of 64 x 64 up to 128 x 128 values) would be needed are refused.  Sums are 32-bit; what the checkpoint holds
    below 2^-126 counts as zero, and of a 32-bit dy below 2^-110 what lies under 2^-133."""
    dy, dt = _tensor(dy, "mx.linear_wgrad")
    _checkpoint_of(ck, dy, "mx.linear_wgrad")
    if dy.shape[:-1] != ck.shape[:-1]:
        raise ValueError(f"mx.linear_wgrad: gradient {tuple(dy.shape)} and checkpoint {tuple(ck.shape)} have different rows")
    rows, N, K, dev = ck.rows, dy.shape[-1], ck.shape[-1], dy.device
    for t, n, what in ((into, N * K, "into"), (bias_into, N, "bias_into")):
        if t is not None and (t.dtype != torch.float32 or t.numel() != n or t.device != dev or not t.is_contiguous()):
            raise ValueError(f"mx.linear_wgrad: {what} must be contiguous fp32 with {n} values on {dev}")
    if bias_into is not None and into is None or into is not None and bias and bias_into is None:
        raise ValueError("mx.linear_wgrad: into and bias_into come together when a bias gradient is wanted")
    dw = into if into is not None else dy.new_empty(N, K, dtype=torch.float32)
    db = bias_into if bias_into is not None else (dy.new_empty(N, dtype=torch.float32) if bias else None)
    if rows == 0:
        if into is None:
            dw.zero_()
            if db is not None:
                db.zero_()
        return dw, db
    n = _hip.query("cn_mx_linear_wgrad_bytes", rows, K, N, dt)
    ws = torch.empty(n, dtype=torch.uint8, device=dev) if n else None
    codes, scales, _ = ck._pointers()
    launch("cn_mx_linear_wgrad", dy.get_device(), dy.data_ptr(), codes, scales, dw.data_ptr(), _ptr(db), 0 if into is None else 1, rows, K, N,
           dt, _ptr(ws), n)
    return dw, db


def batch_norm_act_bwd(dy, ck, gamma, mean, invstd, residual=False, racc=None, into=None):
    """Backward of y = [relu](gamma * (x - mean) * invstd + beta [+ residual]) with batch statistics over the rows, from ck =
    mx.checkpoint(x, sign_of=y) (sign_of=None: no ReLU; mean, invstd and the mask are the unrounded input's): -> (dx, dgamma, dbeta, dres).  residual: also return the residual input's
    gradient (racc: a tensor to add to it), else dres is None.  into: (gamma.grad, beta.grad) to add to instead of new tensors."""
    dy, dt = _tensor(dy, "mx.batch_norm_act_bwd")
    _checkpoint_of(ck, dy, "mx.batch_norm_act_bwd")
    if dy.shape != ck.shape or dy.dtype != ck.dtype:
        raise ValueError(f"mx.batch_norm_act_bwd: gradient {tuple(dy.shape)} {dy.dtype}, checkpoint of {tuple(ck.shape)} {ck.dtype}")
    rows, C, dev, one = ck.rows, ck.shape[-1], dy.device, (ck.shape[-1],)
    if rows == 0:
        raise ValueError("mx.batch_norm_act_bwd: no rows (batch statistics are undefined)")
    if racc is not None and not residual:
        raise ValueError("mx.batch_norm_act_bwd: racc without residual")
    gamma = _like(gamma, dev, one, torch.float32, "mx.batch_norm_act_bwd: gamma")
    mean = _like(mean, dev, one, torch.float32, "mx.batch_norm_act_bwd: mean")
    invstd = _like(invstd, dev, one, torch.float32, "mx.batch_norm_act_bwd: invstd")
    if racc is not None:
        racc = _like(racc, dev, dy.shape, dy.dtype, "mx.batch_norm_act_bwd: racc")
    if into is not None:
        dgamma, dbeta = into
        for t in into:
            if _like(t, dev, one, torch.float32, "mx.batch_norm_act_bwd: into") is not t:
                raise ValueError("mx.batch_norm_act_bwd: into must be contiguous")
        if dgamma.data_ptr() == dbeta.data_ptr():
            raise ValueError("mx.batch_norm_act_bwd: into needs two tensors")
    else:
        dgamma, dbeta = torch.empty_like(gamma), torch.empty_like(gamma)       # (half the host time of torch.empty with a torch.Size)
    dx = torch.empty_like(dy)
    dres = torch.empty_like(dy) if residual else None
    n = _hip.query("cn_mx_bn_bwd_bytes", rows, C, dt)
    ws = torch.empty(n, dtype=torch.uint8, device=dev) if n else None
    codes, scales, signs = ck._pointers()
    launch("cn_mx_bn_bwd", dy.get_device(), dy.data_ptr(), codes, scales, signs, gamma.data_ptr(), mean.data_ptr(), invstd.data_ptr(),
           dx.data_ptr(), _ptr(dres), _ptr(racc), dgamma.data_ptr(), dbeta.data_ptr(), 0 if into is None else 1, rows, C, dt, _ptr(ws), n)
    return dx, dgamma, dbeta, dres
