"""8-bit activation checkpoints and 4-bit inference through the layers (nn.use_checkpoints, nn.use_mxfp4) on the GPU."""
import copy
import gc

import numpy as np
import pytest
import torch
import torch.nn.functional as F

from oracle import mx_ref
from tests.test_gpu_mx import BF, DEV, F32, U, f64, half_step, rnd, within

pytestmark = pytest.mark.gpu


def hnn():
    from centernet_amd import nn
    return nn


def ops():
    from centernet_amd import ops
    return ops


def img(shape, seed, dt, scale=1.0):
    return rnd(shape, seed, dt, scale=scale)


def q8(x):
    """what an e4m3 checkpoint of the NHWC tensor stands for, float64"""
    return torch.tensor(mx_ref.quantize(f64(x).reshape(-1, x.shape[-1]), "e4m3")[0]).view(x.shape)


@pytest.mark.parametrize("dt", [BF, F32])
@pytest.mark.parametrize("relu,residual", [(True, True), (True, False), (False, True), (False, False)])
@pytest.mark.parametrize("shape", [(2, 8, 8, 64), (1, 5, 7, 48), (3, 16, 16, 256)])
def test_batch_norm_layer(dt, relu, residual, shape):
    C = shape[-1]
    bn = hnn().BatchNorm2d(C).to(DEV).train()
    with torch.no_grad():
        bn.weight.copy_(rnd((C,), 1, F32, spread=0) * 0.2 + 1)
        bn.bias.copy_(rnd((C,), 2, F32, spread=0) * 0.3)
    plain = copy.deepcopy(bn)
    assert hnn().use_checkpoints(bn) == 1
    x, dy = img(shape, 3, dt), img(shape, 4, dt, 1e-2)
    res = img(shape, 5, dt) if residual else None
    grads = {}
    for name, m in (("ck", bn), ("plain", plain)):
        xi = x.clone().requires_grad_()
        ri = res.clone().requires_grad_() if residual else None
        y = m(xi, ri, relu)
        if name == "ck":
            stats = y.grad_fn.saved_tensors[2]
            kept = sum(t.numel() * t.element_size() for t in y.grad_fn.saved_tensors)
            mean, invstd = f64(stats[0]), f64(stats[1])
        y.backward(dy)
        grads[name] = (y.detach(), xi.grad, m.weight.grad, m.bias.grad, ri.grad if residual else None)
    rows = x.numel() // C
    blocks = -(-C // 32)
    assert kept == rows * blocks * (33 + (4 if relu else 0)) + 4 * C + 16 * C        # codes, scales, bits; gamma; statistics
    assert torch.equal(grads["ck"][0], grads["plain"][0])                              # the forward pass is the same
    assert torch.equal(bn.running_mean, plain.running_mean) and torch.equal(bn.running_var, plain.running_var)
    y = grads["ck"][0]
    want = mx_ref.batch_norm_act_bwd(f64(dy).reshape(rows, C), f64(x).reshape(rows, C), f64(y).reshape(rows, C) if relu else None,
                                     f64(bn.weight), mean, invstd)
    within(grads["ck"][1].reshape(rows, C), want[0], half_step(dt) * np.abs(want[0]) + U * want[4], "dx")
    within(grads["ck"][2], want[1], U * want[5], "dgamma")
    within(grads["ck"][3], want[2], U * want[6], "dbeta")
    if residual:
        assert np.array_equal(f64(grads["ck"][4]).reshape(rows, C), want[3])


@pytest.mark.parametrize("dt", [BF, F32])
@pytest.mark.parametrize("N,H,W,Ci,Co,k,s,p,bias", [(2, 9, 7, 64, 128, 1, 1, 0, False), (1, 8, 8, 32, 27, 1, 1, 0, True), (2, 8, 8, 48, 16, 1, 1, 0, True),
                                                    (2, 8, 8, 64, 64, 1, 2, 0, False), (2, 12, 12, 32, 48, 3, 1, 1, False), (1, 16, 16, 64, 64, 3, 2, 1, True)])
def test_conv_layer(dt, N, H, W, Ci, Co, k, s, p, bias):
    conv = hnn().Conv2d(Ci, Co, k, s, p, bias=bias).to(DEV)
    plain = copy.deepcopy(conv)
    assert hnn().use_checkpoints(conv) == 1
    x = img((N, H, W, Ci), 1, dt)
    out = {}
    for name, m in (("ck", conv), ("plain", plain)):
        xi = x.clone().requires_grad_()
        y = m(xi)
        dy = img(tuple(y.shape), 2, dt, 1e-2)
        if y.shape[-1] > Co:
            dy[..., Co:] = 0
        y.backward(dy)
        out[name] = (y.detach(), xi.grad, m.weight.grad, m.bias.grad if bias else None)
    assert torch.equal(out["ck"][0], out["plain"][0])
    assert torch.equal(out["ck"][1], out["plain"][1])                                  # the data gradient does not read the input
    xq, d = q8(x).permute(0, 3, 1, 2), torch.tensor(f64(dy))[..., :Co].permute(0, 3, 1, 2)

    def wgrad(a, b):
        w = torch.zeros(Co, Ci, k, k, dtype=torch.float64, requires_grad=True)
        F.conv2d(a, w, None, s, p).backward(b)
        return w.grad.numpy()

    rows = dy.numel() // dy.shape[-1]
    terms = (1 if dt == BF else 3) * rows + 16
    within(out["ck"][2], wgrad(xq, d), terms * U * wgrad(xq.abs(), d.abs()), "dw")
    if bias:
        within(out["ck"][3], d.sum((0, 2, 3)).numpy(), terms * U * d.abs().sum((0, 2, 3)).numpy(), "db")


@pytest.mark.parametrize("k,p", [(1, 0), (3, 1)])
def test_conv_layer_with_frozen_parameters(k, p):
    """a bias trains above a frozen weight; a layer that is frozen altogether passes the gradient on and keeps nothing"""
    conv = hnn().Conv2d(32, 24, k, 1, p, bias=True).to(DEV)
    hnn().use_checkpoints(conv)
    conv.weight.requires_grad_(False)
    x = img((2, 6, 6, 32), 1, F32).requires_grad_()
    y = conv(x)
    dy = img(tuple(y.shape), 2, F32, 1e-2)
    dy[..., 24:] = 0
    y.backward(dy)
    dx = x.grad.clone()
    d = f64(dy)[..., :24].reshape(-1, 24)
    within(conv.bias.grad, d.sum(0), (3 * 72 + 16) * U * np.abs(d).sum(0), "db")
    assert conv.weight.grad is None
    want = torch.zeros(2, 32, 6, 6, dtype=torch.float64, requires_grad=True)
    F.conv2d(want, conv.weight.detach().double().cpu(), None, 1, p).backward(torch.tensor(f64(dy)[..., :24]).permute(0, 3, 1, 2))
    s = 24 * k * k * np.abs(f64(conv.weight)).max() * np.abs(d).max()
    within(dx, want.grad.permute(0, 2, 3, 1).numpy(), np.full(dx.shape, (24 * k * k + 16) * U * s), "dx")
    conv.bias.requires_grad_(False)
    x.grad = None
    y = conv(x)
    assert y.grad_fn.saved_tensors[0] is None
    y.backward(dy)
    assert torch.equal(x.grad, dx)


@pytest.mark.parametrize("dt", [BF, F32])
def test_root_over_several_sources(dt):
    """conv1x1 over a concatenation that is never built, its sources shared with other layers and kept once"""
    o = ops()
    w = (rnd((48, 160, 1, 1), 1, F32, spread=0) * 0.1).requires_grad_()
    xs = [img((2, 6, 6, c), 2 + c, dt) for c in (64, 32, 64)]
    out = {}
    for ck in (True, False):
        leaves = [t.clone().requires_grad_() for t in xs]
        shared = [o.share(t * 1) for t in leaves]
        y = o.conv1x1_cat(shared, w, ckpt=ck)
        side = o.conv2d_ckpt(shared[0], rnd((16, 64, 1, 1), 9, F32, spread=0).requires_grad_()) if ck else None
        if ck:
            assert side.grad_fn.saved_tensors[0].data_ptr() == y.grad_fn.saved_tensors[1].data_ptr()      # one checkpoint for both readers
        dy = img(tuple(y.shape), 5, dt, 1e-2)
        w.grad = None
        y.backward(dy)
        out[ck] = (y.detach(), w.grad.clone(), [t.grad for t in leaves])
    assert torch.equal(out[True][0], out[False][0])
    assert all(torch.equal(a, b) for a, b in zip(out[True][2], out[False][2]))
    want, _, s, _ = mx_ref.linear_wgrad(f64(dy).reshape(-1, 48), f64(xs[0]).reshape(-1, 64))
    terms = (1 if dt == BF else 3) * 72 + 16
    within(out[True][1].view(48, 160)[:, :64], want, terms * U * s, "dw of the first source")
    want, _, s, _ = mx_ref.linear_wgrad(f64(dy).reshape(-1, 48), f64(xs[2]).reshape(-1, 64))
    within(out[True][1].view(48, 160)[:, 96:], want, terms * U * s, "dw of the last source")


def test_layers_in_a_row_against_64_bits():
    """conv1x1 -> BN -> ReLU -> conv1x1 -> BN + identity -> ReLU, every gradient against the chain of the definitions in 64 bits, fed
    with the activations of the run itself.  Tolerance: four operators, each within 2e-5 of its output's largest value in 32 bits."""
    n = hnn()
    torch.manual_seed(0)
    c1, b1, c2, b2 = n.Conv2d(64, 32, 1).to(DEV), n.BatchNorm2d(32).to(DEV), n.Conv2d(32, 64, 1).to(DEV), n.BatchNorm2d(64).to(DEV)
    layers = torch.nn.ModuleList([c1, b1, c2, b2]).train()
    assert n.use_checkpoints(layers) == 4
    x = img((2, 10, 10, 64), 1, F32).clamp_(min=0).requires_grad_()
    a1 = c1(x)
    y1 = b1(a1, None, True)
    a2 = c2(y1)
    y2 = b2(a2, x, True)
    dy = img((2, 10, 10, 64), 2, F32, 1e-2)
    saved = {k: [f64(t) for t in m.grad_fn.saved_tensors[2][:2]] for k, m in (("b1", y1), ("b2", y2))}
    y2.backward(dy)
    flat = lambda t: f64(t).reshape(-1, t.shape[-1])     # noqa: E731
    w1, w2 = f64(c1.weight)[:, :, 0, 0], f64(c2.weight)[:, :, 0, 0]
    d2, g2, h2, r2 = mx_ref.batch_norm_act_bwd(flat(dy), flat(a2), flat(y2), f64(b2.weight), *saved["b2"])[:4]
    dw2 = mx_ref.linear_wgrad(d2, flat(y1))[0]
    d1, g1, h1, _ = mx_ref.batch_norm_act_bwd(d2 @ w2, flat(a1), flat(y1), f64(b1.weight), *saved["b1"])[:4]
    dw1 = mx_ref.linear_wgrad(d1, flat(x))[0]
    dx = d1 @ w1 + r2
    for what, got, want in (("dx", flat(x.grad), dx), ("dw1", f64(c1.weight.grad)[:, :, 0, 0], dw1), ("dw2", f64(c2.weight.grad)[:, :, 0, 0], dw2),
                            ("dgamma1", f64(b1.weight.grad), g1), ("dbeta1", f64(b1.bias.grad), h1), ("dgamma2", f64(b2.weight.grad), g2),
                            ("dbeta2", f64(b2.bias.grad), h2)):
        assert np.abs(got - want).max() <= 8e-5 * np.abs(want).max(), what


def _detector(arch, ck, dt):
    from centernet_amd.centernet_detection import CenterNetDetection
    torch.manual_seed(0)
    model = CenterNetDetection(arch, compute_dtype=dt).to(DEV).train()
    if ck:
        assert hnn().use_checkpoints(model) > 50
    return model


def _batch():
    from centernet_amd import synth
    x, tgt = synth.ctdet_batch(11, 4, 256, 256)
    return x.to(DEV), {k: v.to(DEV) for k, v in tgt.items()}


@pytest.mark.parametrize("arch", ["dla_34", "res_101"])
def test_model_with_checkpoints(arch):
    """32-bit compute (whose sums have a fixed order): the loss is the plain model's bit for bit, every parameter gets a finite gradient,
    and between forward and backward a good part of the memory is free"""
    x, tgt = _batch()
    loss, kept, names = {}, {}, {}
    for ck in (False, True):
        model = _detector(arch, ck, F32)
        for rep in range(2):                                       # (the first pass allocates what the layers keep for good)
            model.zero_grad(set_to_none=True)
            gc.collect()
            base = torch.cuda.memory_allocated()
            total, _ = model.loss(model(x), tgt)
            gc.collect()
            kept[ck] = torch.cuda.memory_allocated() - base
            if rep == 0:
                loss[ck] = total.detach().clone()
            total.backward()
        names[ck] = {k for k, p in model.named_parameters() if p.grad is not None}
        assert all(torch.isfinite(p.grad).all() for p in model.parameters() if p.grad is not None)
        del model, total
    print(f"{arch}: kept between forward and backward {kept[False] / 2 ** 20:.0f} -> {kept[True] / 2 ** 20:.0f} MiB")
    assert torch.equal(loss[True], loss[False])
    assert names[True] == names[False]
    assert kept[True] < 0.8 * kept[False]


def test_which_layers_keep_checkpoints():
    """bf16 layers whose batch norm is applied by their consumer keep one tensor between the two, all others checkpoints"""
    x, tgt = _batch()
    names = {}
    for ck in (False, True):
        total, _ = (model := _detector("dla_34", ck, BF)).loss(model(x), tgt)
        seen, todo, names[ck] = set(), [total.grad_fn], []
        while todo:
            node = todo.pop()
            if node is not None and node not in seen:
                seen.add(node)
                names[ck].append(type(node).__name__)
                todo += [n for n, _ in node.next_functions]
    count = lambda ck, what: names[ck].count(what + "Backward")     # noqa: E731
    for kind in ("BnDeferFn", "StemBnDeferFn"):
        assert count(True, kind) == count(False, kind) > 0
    assert count(True, "BatchNormCkptFn") == count(False, "BatchNormActFn") > 30 and count(True, "BatchNormActFn") == 0
    assert count(True, "Conv2dCkptFn") > 20


@pytest.mark.parametrize("arch", ["dla_34", "res_101"])
def test_training_steps_with_checkpoints(arch):
    """captured bf16 training steps: replays stay finite and the weights that move are the plain model's (a model may own unused ones)"""
    from centernet_amd.engine import TrainStep
    batch, moved = _batch(), {}
    for ck in (False, True):
        model = _detector(arch, ck, BF)
        before = {k: p.detach().clone() for k, p in model.named_parameters()}
        step = TrainStep(model, lr=1e-4, distributed=False)
        losses = [float(step(batch).detach()) for _ in range(5)]
        assert np.isfinite(losses).all()
        assert all(torch.isfinite(p).all() for p in model.parameters())
        moved[ck] = {k for k, p in model.named_parameters() if p.dim() > 1 and not torch.equal(p, before[k])}
        del step, model
    assert moved[True] == moved[False] and len(moved[True]) > 50


# ------------------------------------------------------------------------------------------------ 4-bit inference
@pytest.mark.parametrize("dt", [BF, F32])
@pytest.mark.parametrize("Ci,Co", [(64, 64), (48, 27), (256, 128)])
def test_conv_bn_inference_in_4_bits(dt, Ci, Co):
    n = hnn()
    conv, bn = n.Conv2d(Ci, Co, 1, bias=False).to(DEV), n.BatchNorm2d(Co).to(DEV).eval()
    with torch.no_grad():
        bn.running_var.copy_(rnd((Co,), 1, F32).abs() + 0.5)
        bn.running_mean.copy_(rnd((Co,), 2, F32))
    x = img((2, 5, 6, Ci), 3, dt)
    cp = -(-Co // 16) * 16
    res = img((2, 5, 6, cp), 4, dt)
    if Co < cp:
        res[..., Co:] = 0
    with torch.no_grad():
        before = n.conv_bn_act(conv, bn, x, res if Co == cp else None)
        assert n.use_mxfp4(conv) == 1
        got = n.conv_bn_act(conv, bn, x, res if Co == cp else None)
        s, b = bn.folded()
        w = f64(conv.weight.view(Co, Ci) * s[:, None])
        want, m = mx_ref.linear(f64(x).reshape(-1, Ci), w, f64(b), f64(res).reshape(-1, cp) if Co == cp else None, relu=True)
        within(got.reshape(-1, cp)[:, :Co], want, half_step(dt) * np.abs(want) + (Ci + 8) * U * m, "y")
        assert not got.reshape(-1, cp)[:, Co:].any()
        conv.weight.mul_(2)                                        # a new weight version is packed anew
        bn.running_mean.mul_(2)
        two = n.conv_bn_act(conv, bn, x, None)
        s, b = bn.folded()
        want, m = mx_ref.linear(f64(x).reshape(-1, Ci), f64(conv.weight.view(Co, Ci) * s[:, None]), f64(b), None, relu=True)
        within(two.reshape(-1, cp)[:, :Co], want, half_step(dt) * np.abs(want) + (Ci + 8) * U * m, "y of the new weights")
        conv.weight.div_(2)
        bn.running_mean.div_(2)
        n.use_mxfp4(conv, False)
        assert torch.equal(before, n.conv_bn_act(conv, bn, x, res if Co == cp else None))


def test_root_and_head_inference_in_4_bits():
    n = hnn()
    conv, bn = n.Conv2d(96, 64, 1).to(DEV), n.BatchNorm2d(64).to(DEV).eval()
    xs = [img((1, 6, 6, 64), 1, BF), img((1, 6, 6, 32), 2, BF)]
    n.use_mxfp4(conv)
    with torch.no_grad():
        got = n.cat_conv_bn_act(conv, bn, xs)
        s, b = bn.folded()
        want, m = mx_ref.linear(f64(torch.cat(xs, -1)).reshape(-1, 96), f64(conv.weight.view(64, 96) * s[:, None]), f64(b), relu=True)
        within(got.reshape(-1, 64), want, half_step(BF) * np.abs(want) + 104 * U * m, "root")
        head = n.Conv2d(64, 20, 1, bias=True).to(DEV)
        n.use_mxfp4(head)
        x = img((2, 4, 4, 64), 3, BF)
        y = head.infer_nchw(x)
        assert y.shape == (2, 20, 4, 4) and y.dtype == F32
        want, m = mx_ref.linear(f64(x).reshape(-1, 64), f64(head.weight.view(20, 64)), f64(head.bias))
        within(y.permute(0, 2, 3, 1).reshape(-1, 20), want, half_step(BF) * np.abs(want) + 72 * U * m, "head")


def test_weights_of_a_copy_or_another_parameter_are_packed_anew():
    """a copied parameter starts at version 0, and one put in another's place may have its version: what was packed for the first must not
    answer for the second"""
    n = hnn()
    conv = n.Conv2d(64, 32, 1).to(DEV)
    n.use_mxfp4(conv)
    x = img((1, 4, 4, 64), 1, F32)
    sds = [{"weight": rnd((32, 64, 1, 1), 5 + i, F32)} for i in range(3)]

    def fresh(sd):
        c = n.Conv2d(64, 32, 1).to(DEV)
        n.use_mxfp4(c)
        c.load_state_dict(sd)
        return c(x)

    with torch.no_grad():
        wants = [fresh(sd) for sd in sds]
        conv.load_state_dict(sds[0], assign=True)
        conv.weight.mul_(1)                                        # version 1
        assert conv.weight._version == 1 and torch.equal(conv(x), wants[0])
        other = copy.deepcopy(conv)
        other.load_state_dict(sds[1])                              # version 1 again
        assert other.weight._version == 1 and other.mx4 and torch.equal(other(x), wants[1])
        for i in (2, 1, 0):
            conv.load_state_dict({k: v.clone() for k, v in sds[i].items()}, assign=True)
            assert conv.weight._version == 0 and torch.equal(conv(x), wants[i])


def test_inference_captured_before_any_eager_call():
    """weights packed during a capture are not kept for eager calls (they hold nothing until the graph has run)"""
    n = hnn()
    conv = n.Conv2d(64, 64, 1).to(DEV)
    x = img((2, 8, 8, 64), 1, BF)
    n.use_mxfp4(conv)
    with torch.no_grad():
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            y = conv(x)
        eager = conv(x)
        for _ in range(3):
            y.fill_(float("nan"))
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(y, eager)
            assert torch.equal(conv(x), eager)


def test_model_inference_in_4_bits():
    """the whole detector: only the 1x1 layers of the backbone change, the maps stay finite and keep their shapes, and switching back
    gives the first result"""
    from centernet_amd.centernet_detection import CenterNetDetection
    torch.manual_seed(0)
    model = CenterNetDetection("res_101").to(DEV).eval()
    x = torch.randn(2, 3, 128, 128, generator=torch.Generator().manual_seed(1)).to(DEV)
    with torch.no_grad():
        a = model(x)
        assert hnn().use_mxfp4(model.backbone) > 60
        b = model(x)
        hnn().use_mxfp4(model.backbone, False)
        c = model(x)
    for p, q, r in zip(a, b, c):
        for k in p:
            assert p[k].shape == q[k].shape and torch.isfinite(q[k]).all() and torch.equal(p[k], r[k])
