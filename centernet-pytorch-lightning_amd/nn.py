"""Layer modules over the HIP operators.  Parameters keep the reference's names/shapes (NCHW fp32),
so `state_dict`s are interchangeable with the reference; activations flowing between layers are NHWC in the
backbone's compute dtype.

Training: conv -> (batch-stat BN + residual + ReLU) as separate HBM passes (statistics need the whole
conv output first).  Inference: BN is folded into the packed conv weights and residual/ReLU ride in the conv
epilogue, so a conv+BN+ReLU(+add) block is ONE kernel; folded weights are cached per parameter version.
"""
import math

import torch
import torch.nn as nn

import os

from . import mx, ops

STEM_BN_FUSED = not (os.environ.get("CN_DISABLE_STEM_BN_FUSED") or os.environ.get("CN_DISABLE_WGRAD_C16"))   # stem conv + BN as one autograd node
# training-mode BN of the 16-channel 512^2 layers applied by the consuming conv: needs the kernels with the pre-affine hook, so the
# switches that turn those kernels off turn this off too (they used to end in CN_EUNSUPPORTED instead of the unfused chain)
BN_DEFER = not (os.environ.get("CN_DISABLE_BN_DEFER") or os.environ.get("CN_DISABLE_CONV_C16R") or os.environ.get("CN_DISABLE_WGRAD_C16"))


def _capturing(device):
    """the current stream of CUDA device index `device` (-1: the CPU) is being captured into a graph"""
    return device >= 0 and torch._C._cuda_isCurrentStreamCapturing()


def _state(key, a, b, c, d):
    """what a value made from these tensors (b, c, d may be None) goes by, next to their identity"""
    return (key, ops.WeightsEpoch.value, a._version, a.data_ptr(), None if b is None else (b._version, b.data_ptr()),
            None if c is None else (c._version, c.data_ptr()), None if d is None else (d._version, d.data_ptr()))


class _Entry:
    """one value of a `Derived` and what makes it safe to hand out"""
    __slots__ = ("state", "value", "a", "b", "c", "d", "memory", "tensors", "device", "streams", "done")

    def __init__(self, state, value, made):
        self.state, self.value = state, value
        self.a, self.b, self.c, self.d = made
        self.memory = [None if t is None else t.detach() for t in made]        # (the memory of `made`: no other tensor gets their addresses)
        self.tensors = [getattr(t, "packed", t) for t in (value.values() if isinstance(value, dict) else value) if t is not None]
        self.device = made[0].get_device()
        if self.device >= 0:
            self.streams = {torch._C._cuda_getCurrentRawStream(self.device)}       # that may use the value as it is
            self.done = torch.cuda.current_stream(self.device).record_event()

    def follow(self):
        """The first call on another stream than the one that makes the value: what this stream does from now on waits for that, and the memory is
        not given away before this stream is done with it."""
        here = torch.cuda.current_stream(self.device)
        here.wait_event(self.done)
        for t in self.tensors:
            t.record_stream(here)
        self.streams.add(here.cuda_stream)


class Derived:
    """What a layer makes of its parameters for the no-grad path, kept until they change: an entry answers for the tensors it was made from
    (it holds them and their memory, so no other takes their place) at their versions and addresses (`.data` assigned anew keeps the
    version), in its `ops.WeightsEpoch`, on any stream.

    The replays of a graph read what its capture was given, so that stays for the layer's life (a capture at other weights keeps one more).
    What a capture itself makes exists only once the graph has run: it lies in the graph's memory and is not kept here.  (A capture does not
    wait for the stream that made an entry: `torch.cuda.graph` has synchronised before it begins.)

    `find` runs for every layer of an eager forward pass, whose host time is what a small batch takes: it is written for that."""
    __slots__ = ("entry", "captured")

    def __init__(self):
        self.entry = None
        self.captured = []           # what captured graphs read: entries, tensors

    def __reduce__(self):
        """a copy of the layer begins anew: its parameters are others, and start at version 0 again"""
        return Derived, ()

    @classmethod
    def of(cls, layer, name):
        d = layer.__dict__.get(name)
        if d is None:
            d = layer.__dict__[name] = cls()
        return d

    def find(self, key, a, b, c, d, held=False):
        """the value kept for `key` and these tensors (b, c, d may be None), or None.  held: the caller's own entry holds the value for the graph"""
        e = self.entry
        if e is None or a is not e.a or b is not e.b or c is not e.c or d is not e.d or e.state != _state(key, a, b, c, d):
            return None
        if not held and _capturing(e.device):
            if all(k is not e for k in self.captured):
                self.captured.append(e)
        elif e.device >= 0 and torch._C._cuda_getCurrentRawStream(e.device) not in e.streams and not (held and _capturing(e.device)):
            e.follow()
        return e.value

    def keep(self, key, made, value):
        """value (a tuple or dict of tensors, packed weights or None) is what the four tensors `made` give -> value"""
        if _capturing(made[0].get_device()):
            self.captured.append(made)             # (the graph makes the value again in every replay: what it reads stays)
        else:
            self.entry = _Entry(_state(key, *made), value, made)
        return value


class Conv2d(nn.Module):
    ckpt8 = False           # `use_checkpoints`: keep the input in 8 bits for the backward pass
    mx4 = False             # `use_mxfp4`: the no-grad forward as a 4-bit product (1x1, stride 1)

    def __init__(self, cin, cout, k, stride=1, padding=0, bias=False):
        super().__init__()
        self.stride, self.padding, self.k = stride, padding, k
        self.weight = nn.Parameter(torch.empty(cout, cin, k, k))
        nn.init.kaiming_uniform_(self.weight, a=math.sqrt(5))
        if bias:
            bound = 1 / math.sqrt(cin * k * k)
            self.bias = nn.Parameter(torch.empty(cout).uniform_(-bound, bound))
        else:
            self.register_parameter("bias", None)

    def __getstate__(self):
        """copies and pickles pack their 4-bit weights again: a copied parameter starts at version 0"""
        state = self.__dict__.copy()
        state.pop("_mx_cache", None)
        return state

    def extra_repr(self):
        co, ci, k, _ = self.weight.shape
        return f"{ci}, {co}, kernel_size={k}, stride={self.stride}, padding={self.padding}, bias={self.bias is not None}"

    def forward(self, x, relu=False, mask_dx=False, defer_relu_bwd=False, bn_stats=False):
        """bn_stats: the output goes straight into a training-mode BatchNorm2d (ops.BnStats: statistics from the conv epilogue)"""
        pre = getattr(x, "_cn_pre", None)           # x is a raw conv output whose BN (+ ReLU) is applied by this conv's kernels (ops.BnDeferFn)
        if torch.is_grad_enabled() and (self.weight.requires_grad or x.requires_grad or (self.bias is not None and self.bias.requires_grad)):
            if self.ckpt8 and pre is None and not (relu or mask_dx or defer_relu_bwd):
                return ops.conv2d_ckpt(x, self.weight, self.bias, self.stride, self.padding, bn_stats)
            return ops.conv2d(x, self.weight, self.bias, self.stride, self.padding, relu, mask_dx, defer_relu_bwd, bn_stats=bn_stats, pre=pre)
        if pre is not None:
            c = self.infer_key(x)
            Co, _, KH, KW = self.weight.shape
            OH, OW = ops.conv_out(x.shape[1], KH, self.stride, self.padding), ops.conv_out(x.shape[2], KW, self.stride, self.padding)
            y = ops._igemm(x, c["wp"], c["b"], None, Co, KH, KW, self.stride, self.padding, False, relu, OH, OW, bn_stats=bn_stats, pre=pre)
            return ops.BnStats.pop(y) if bn_stats else y
        return self.infer(x, None, None, None, relu)

    def with_skip(self, x, bn_stats=False):
        """-> (conv(x), x) for a residual connection around this conv: the skip path's gradient is added in the epilogue of this
        conv's data-gradient kernel (training; otherwise just the pair)."""
        if torch.is_grad_enabled() and x.requires_grad and self.stride == 1:
            if self.ckpt8:
                return ops.conv2d_ckpt(x, self.weight, self.bias, self.stride, self.padding, bn_stats, passthrough=True)
            return ops.conv2d(x, self.weight, self.bias, self.stride, self.padding, False, False, False, True, bn_stats=bn_stats)
        return self.forward(x), x

    def infer_key(self, x, scale=None, shift=None):
        """-> the cache entry {wp: packed (folded) weights, b: folded bias} for x's dtype and the current parameter versions"""
        p = self._parameters                        # (an attribute of a Module takes several times as long)
        weight, bias = p["weight"] if "weight" in p else self.weight, p["bias"] if "bias" in p else self.bias
        kept = Derived.of(self, "_packed")
        hit = kept.find(x.dtype, weight, bias, scale, shift)
        if hit is not None:
            return hit
        wp = ops.pack_weight(weight, 1, x.dtype, scale)
        b = bias.detach() if bias is not None else None
        if shift is not None:
            b = shift if b is None else (b * scale + shift)   # tiny [Co] host-side fold (once per weight version)
        return kept.keep(x.dtype, (weight, bias, scale, shift), {"wp": wp, "b": b})

    def infer(self, x, scale, shift, residual, relu, out_dtype=None):
        """No-grad path: y = act(conv(x)*scale + shift + residual); packed (folded) weights are cached."""
        if self.mx4 and out_dtype in (None, x.dtype):
            w, b = self._mx_weight(x, scale, shift)
            return mx.linear(x, w, b, residual, relu)
        c, p, stride, padding = self.infer_key(x, scale, shift), self._parameters, self.stride, self.padding
        Co, _, KH, KW = (p["weight"] if "weight" in p else self.weight).shape
        N, H, W, _ = x.shape
        OH, OW = ops.conv_out(H, KH, stride, padding), ops.conv_out(W, KW, stride, padding)
        return ops._igemm(x, c["wp"], c["b"], residual, Co, KH, KW, stride, padding, False, relu, OH, OW, out_dtype)

    def _mx_weight(self, x, scale, shift):
        """(4-bit weights, fp32 bias) with the following BN folded in, for x's channels and this layer's padded output channels"""
        p = self._parameters
        weight, bias = p["weight"] if "weight" in p else self.weight, p["bias"] if "bias" in p else self.bias
        key, kept = (x.shape[-1], x.get_device()), Derived.of(self, "_mx_cache")
        hit = kept.find(key, weight, bias, scale, shift)
        if hit is not None:
            return hit
        Co, Ci = weight.shape[:2]
        with torch.no_grad():
            w = torch.zeros(ops.rup(Co, 16), x.shape[-1], dtype=torch.float32, device=x.device)
            w[:Co, :Ci] = weight.view(Co, Ci) if scale is None else weight.view(Co, Ci) * scale[:, None]
            b = torch.zeros(w.shape[0], dtype=torch.float32, device=x.device)
            if bias is not None:
                b[:Co] = bias if scale is None else bias * scale
            if shift is not None:
                b[:Co] += shift
        return kept.keep(key, (weight, bias, scale, shift), (mx.pack_weight(w), b))

    def infer_nchw(self, x):
        """No-grad 1x1 conv + bias straight into the public fp32 NCHW layout (a head's last layer); packed weights cached as in `infer`."""
        if self.mx4:
            y = self.infer(x, None, None, None, False)
            N, H, W, ld = y.shape
            out = torch.empty((N, self.weight.shape[0], H, W), dtype=torch.float32, device=x.device)
            ops.call("cn_nhwc_to_nchw", y, out, N, self.weight.shape[0], H, W, ld, ops.dtype_code(y.dtype))
            return out
        c = self.infer_key(x)
        return ops.conv1x1_to_nchw(x, c["wp"], c["b"], self.weight.shape[0])


class BatchNorm2d(nn.BatchNorm2d):
    """Parameter/buffer holder with nn.BatchNorm2d's state_dict; the arithmetic lives in ops.BatchNormActFn."""
    ckpt8 = False           # `use_checkpoints`: keep the input in 8 bits for the backward pass

    def __init__(self, c):
        super().__init__(c, momentum=ops.BN_MOMENTUM)
        self._pending = 0

    def _save_to_state_dict(self, destination, prefix, keep_vars):
        if self._pending:
            self.num_batches_tracked += self._pending
            self._pending = 0
        super()._save_to_state_dict(destination, prefix, keep_vars)

    def folded(self, held=False):
        """(scale, shift) fp32 of the eval-mode affine; cached per buffer/parameter version and per `ops.WeightsEpoch` (the
        optimizer and the training-mode kernel update parameters / running statistics behind `_version`'s back).  held: only for a layer that
        packs them into its own (`Derived.find`)"""
        p, q = self._parameters, self._buffers
        made = (p["weight"] if "weight" in p else self.weight, p["bias"] if "bias" in p else self.bias, q["running_mean"], q["running_var"])
        kept = Derived.of(self, "_folded")
        hit = kept.find(self.eps, *made, held)
        if hit is not None:
            return hit
        with torch.no_grad():
            scale = self.weight * torch.rsqrt(self.running_var + self.eps)   # [C] vectors, once per weight version
            shift = self.bias - self.running_mean * scale
        return kept.keep(self.eps, made, (scale.contiguous(), shift.contiguous()))

    def forward(self, x, residual=None, relu=True, defer=False):
        """defer: the caller guarantees that the ONLY consumer of the result is a 3x3 Conv2d with 16 input channels (DLA base_layer ->
        level0 -> level1): the apply pass is then left to that conv's kernels (ops.BnDeferFn) when x carries its producer's statistics"""
        if self.training:
            self._pending += 1
            ops.WeightsEpoch.bump()              # running_mean / running_var are about to change through raw pointers
            if (defer and BN_DEFER and residual is None and x.dtype == torch.bfloat16 and x.shape[-1] == 16
                    and getattr(x, "_bn_part", None) is not None and getattr(x, "_cn_pre", None) is None):
                return ops.batch_norm_defer(x, self, relu)         # (keeps x once for this layer and its consumer: less than two checkpoints)
            if self.ckpt8 and torch.is_grad_enabled():
                return ops.batch_norm_act(x, self, residual, relu, ckpt=True)
            return ops.batch_norm_act(x, self, residual, relu)
        s, b = self.folded()
        return ops.scale_shift_act(x, s, b, residual, relu)


def conv_bn_act_skip(conv, bn, x):
    """(ReLU(BN(conv(x))), x) — the first half of a residual block whose identity path is its own input."""
    if bn.training and torch.is_grad_enabled() and x.requires_grad and conv.stride == 1:
        c, skip = conv.with_skip(x, bn_stats=True)
        return bn(c, None, True), skip
    return conv_bn_act(conv, bn, x), x


def cat_conv_bn_act(conv, bn, xs, residual=None, relu=True):
    """conv1x1(cat(xs, channel)) -> BN -> (+residual) -> ReLU without building the concatenation (DLA Root).  Falls back to
    concat + conv for anything that is not a bias-free 1x1 / stride-1 conv over 32-channel-aligned sources."""
    ok = (conv.k == 1 and conv.stride == 1 and conv.padding == 0 and conv.bias is None and 1 <= len(xs) <= 6
          and all(t.shape[-1] % 32 == 0 for t in xs))      # the data-gradient GEMM of a source reads rup32(C_s) operand rows
    if not ok or len(xs) == 1:
        return conv_bn_act(conv, bn, ops.concat(list(xs)), residual, relu)
    grad = torch.is_grad_enabled() and (conv.weight.requires_grad or any(t.requires_grad for t in xs))
    if bn.training or grad:
        return bn(ops.conv1x1_cat(xs, conv.weight, bn_stats=bn.training, ckpt=conv.ckpt8), residual, relu)
    s, b = bn.folded(held=True)                     # eval: BN folded into the packed weights, one launch
    if conv.mx4:
        return conv.infer(ops.concat(list(xs)), s, b, residual, relu)
    c = conv.infer_key(xs[0], s, b)
    return ops.conv1x1_cat_raw([t.contiguous() for t in xs], c["wp"], c["b"], residual, conv.weight.shape[0], relu)


def conv_bn_act(conv, bn, x, residual=None, relu=True, defer=False):
    """conv -> BN -> (+residual) -> ReLU.  One fused kernel in eval/no-grad mode.  defer: see BatchNorm2d.forward."""
    if bn.training:
        return bn(conv(x, bn_stats=True), residual, relu, defer)      # statistics from the conv kernel's epilogue where it has the hook
    if torch.is_grad_enabled() and (conv.weight.requires_grad or x.requires_grad):
        return bn(conv(x), residual, relu)          # eval-mode BN but gradients wanted: unfused affine pass
    s, b = bn.folded(held=True)
    return conv.infer(x, s, b, residual, relu)


class StemConv(nn.Module):
    """7x7 conv on the NCHW fp32 image -> NHWC activations in `dtype`."""

    def __init__(self, cin, cout, k, stride, padding):
        super().__init__()
        self.stride, self.padding = stride, padding
        self.weight = nn.Parameter(torch.empty(cout, cin, k, k))
        nn.init.kaiming_uniform_(self.weight, a=math.sqrt(5))

    def forward(self, img, dtype, bn_stats=False):
        y = ops.StemConvFn.apply(img, self.weight, self.stride, self.padding, dtype, bn_stats)
        return ops.BnStats.pop(y) if bn_stats else y

    def infer(self, img, dtype, scale, shift, relu):
        """no-grad path with the following eval-mode BN (+ReLU) folded into the kernel's epilogue"""
        return ops.stem_conv_infer(img, self.weight, scale, shift, self.stride, self.padding, relu, dtype)


def stem_bn_act(stem, bn, img, dtype, relu=True, defer=False):
    """stem conv -> BN -> ReLU; one fused kernel in eval / no-grad mode.  defer: see BatchNorm2d.forward."""
    if (defer and BN_DEFER and STEM_BN_FUSED and bn.training and dtype == torch.bfloat16 and stem.weight.shape[0] == 16
            and stem.weight.shape[2] == 7 and stem.padding == 3 and stem.weight.shape[1] <= 3 and ops.BnStats.enabled):
        # the BN behind the stem lives entirely in the neighbouring kernels (ops.StemBnDeferFn)
        bn._pending += 1
        ops.WeightsEpoch.bump()
        return ops.stem_bn_defer(img, stem.weight, bn, stem.stride, stem.padding, dtype, relu)
    if bn.training or (torch.is_grad_enabled() and stem.weight.requires_grad):
        return bn(stem(img, dtype, bn_stats=bn.training), None, relu, defer)
    s, b = bn.folded()
    return stem.infer(img, dtype, s, b, relu)


class ConvTranspose2d(nn.Module):
    def __init__(self, cin, cout, k, stride, padding):
        super().__init__()
        self.stride, self.padding = stride, padding
        self.weight = nn.Parameter(torch.empty(cin, cout, k, k))
        nn.init.kaiming_uniform_(self.weight, a=math.sqrt(5))

    def forward(self, x):
        return ops.conv_transpose2d(x, self.weight, self.stride, self.padding)


class DepthwiseUp(nn.Module):
    """ConvTranspose2d(o, o, 2f, stride=f, padding=f//2, groups=o, bias=False), bilinear init (pose_dla_dcn.py:424-432,466-476)."""

    def __init__(self, c, f):
        super().__init__()
        self.stride, self.padding = f, f // 2
        k = 2 * f
        fc = math.ceil(k / 2)
        cc = (2 * fc - 1 - fc % 2) / (2.0 * fc)
        g = torch.tensor([1 - abs(i / fc - cc) for i in range(k)])
        self.weight = nn.Parameter(torch.outer(g, g).expand(c, 1, k, k).clone())

    def forward(self, x, residual=None):
        """up(x) (+ residual, fused into the store)"""
        return ops.DwDeconvFn.apply(x, self.weight, self.stride, self.padding, residual)


class DCN(nn.Module):
    """Drop-in for DCN.dcn_v2.DCN(chi, cho, (3,3), stride=1, padding=1, dilation=1, deformable_groups=1)."""

    def __init__(self, cin, cout, kernel_size=(3, 3), stride=1, padding=1, dilation=1, deformable_groups=1):
        super().__init__()
        if tuple(kernel_size) != (3, 3) or stride != 1 or padding != 1 or dilation != 1 or deformable_groups != 1:
            raise NotImplementedError("DCN: only the 3x3/s1/p1/d1/g1 configuration the reference uses is implemented")
        self.weight = nn.Parameter(torch.empty(cout, cin, 3, 3))
        bound = 1.0 / math.sqrt(cin * 9)
        nn.init.uniform_(self.weight, -bound, bound)
        self.bias = nn.Parameter(torch.zeros(cout))
        self.conv_offset_mask = Conv2d(cin, 27, 3, 1, 1, bias=True)
        nn.init.zeros_(self.conv_offset_mask.weight)
        nn.init.zeros_(self.conv_offset_mask.bias)

    def forward(self, x, bn_stats=False):
        y = ops.DCNv2Fn.apply(x, self.weight, self.bias, self.conv_offset_mask.weight, self.conv_offset_mask.bias, bn_stats)
        return ops.BnStats.pop(y) if bn_stats else y

    def infer(self, x, scale, shift, relu):
        """No-grad path with the following BN folded in: offset conv -> sampling -> ONE 1x1 GEMM (+shift, ReLU)."""
        p = self._parameters
        weight, bias = p["weight"] if "weight" in p else self.weight, p["bias"] if "bias" in p else self.bias
        kept = Derived.of(self, "_packed")
        hit = kept.find(x.dtype, weight, bias, scale, shift)
        if hit is None:
            hit = kept.keep(x.dtype, (weight, bias, scale, shift), (ops.pack_weight(weight, 1, x.dtype, scale), (bias.detach() * scale + shift).contiguous()))
        wp, b = hit
        N, H, W, Ci = x.shape
        om = self.conv_offset_mask.infer(x, None, None, None, False, out_dtype=torch.float32)
        Co = weight.shape[0]
        cp = ops.rup(Co, 16)
        y = torch.empty((N, H, W, cp), dtype=x.dtype, device=x.device) if cp == Co else ops.zeros((N, H, W, cp), x.dtype, x.device)
        ops.call("cn_dcn_fwd", x, om, wp, b, y, N, H, W, Ci, Ci, Co, cp, om.shape[-1], int(relu),
                 ops.dtype_code(x.dtype))
        return y


class MaxPool2d(nn.Module):
    def __init__(self, k, stride, padding=0):
        super().__init__()
        self.k, self.stride, self.padding = k, stride, padding

    def forward(self, x):
        return ops.max_pool(x, self.k, self.stride, self.padding)


def use_checkpoints(module, on=True):
    """Training with 8-bit activation checkpoints: every Conv2d and BatchNorm2d under `module` keeps its input in e4m3 (one scale per 32
    channels) and a ReLU's mask in bits, instead of the bf16 / fp32 tensors.  The forward pass is unchanged.  A convolution's weight gradient is
    the one at the rounded input, its other gradients are exact.  A batch norm puts the rounded input into its backward formula next to the
    mean, variance and mask of the unrounded one, so dgamma and dx are off by that rounding, and dx sums to zero over the rows only up to it.
    (The task heads, DCN and transposed convolutions keep what they kept, and so do the bf16 layers
    whose batch norm is applied by their consumer: they keep one tensor between the two.)  -> layers switched"""
    n = 0
    for m in module.modules():
        if isinstance(m, (Conv2d, BatchNorm2d)):
            m.ckpt8 = bool(on)
            n += 1
    return n


def use_mxfp4(module, on=True):
    """No-grad forward with 4-bit products: every 1x1 / stride-1 Conv2d under `module` quantises its input and its (BN-folded) weights to
    e2m1 with one scale per 32 channels (mx.linear).  Training is not affected.  Pass the whole model or only its backbone: a head's
    last convolution is a 1x1 too.  -> layers switched"""
    n = 0
    for m in module.modules():
        if isinstance(m, Conv2d) and m.k == 1 and m.stride == 1 and m.padding == 0:
            m.mx4 = bool(on)
            n += 1
    return n
