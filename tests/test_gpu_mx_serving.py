"""What the layers keep for the no-grad path, under captured graphs and streams on the GPU."""
import numpy as np
import pytest
import torch

from tests.test_gpu_mx import BF, DEV, F32, U, f64, rnd, within
from tests.test_gpu_mx_layers import hnn, img, ops

pytestmark = pytest.mark.gpu


def _refill(n=64):
    """take what the allocator has free and fill it with something else"""
    return [torch.full((1 << 14,), 0x7f, dtype=torch.uint8, device=DEV) for _ in range(n)]


def test_replays_read_the_weights_they_were_captured_with():
    """warm-up, capture, then new weights and an eager call, which makes the layer pack again: the graph's own weights stay"""
    n = hnn()
    conv, bn = n.Conv2d(64, 64, 1).to(DEV), n.BatchNorm2d(64).to(DEV).eval()
    x = img((2, 8, 8, 64), 1, BF)
    n.use_mxfp4(conv)
    with torch.no_grad():
        want = n.conv_bn_act(conv, bn, x)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            y = n.conv_bn_act(conv, bn, x)
        for rep in range(3):
            if rep == 1:
                conv.weight.copy_(rnd((64, 64, 1, 1), 5, F32))
            else:
                ops().WeightsEpoch.bump()
            eager = n.conv_bn_act(conv, bn, x)
            assert torch.equal(eager, want) == (rep < 1)
            junk = _refill()
            y.fill_(float("nan"))
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(y, want), rep
            del junk


def _delay():
    """some milliseconds of the current stream"""
    torch.cuda._sleep(20_000_000)


def test_weights_packed_on_one_stream_are_used_on_another():
    """the layer packs on a stream that is far behind; another stream's call waits for that, and its own work may outlive the entry"""
    n = hnn()
    conv = n.Conv2d(256, 256, 1, bias=True).to(DEV)
    n.use_mxfp4(conv)
    x = img((1, 16, 16, 256), 1, BF)
    ws = [rnd((256, 256, 1, 1), 5 + i, F32) for i in range(3)]
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    with torch.no_grad():
        wants = []
        for w in ws:
            conv.weight.copy_(w)
            wants.append(conv(x))
        for i in (0, 1, 2, 1):
            conv.weight.copy_(ws[i])
            torch.cuda.synchronize()
            with torch.cuda.stream(a):
                _delay()
                first = conv(x)
            with torch.cuda.stream(b):
                second = conv(x)
                _delay()
                third = conv(x)                                    # queued when the entry goes
            with torch.cuda.stream(a):
                ops().WeightsEpoch.bump()
                conv(x)
                junk = _refill()
            torch.cuda.synchronize()
            del junk
            assert all(torch.equal(y, wants[i]) for y in (first, second, third)), i


@pytest.mark.parametrize("dt", [BF, F32])
def test_replays_of_the_plain_path_read_the_weights_they_were_captured_with(dt):
    """convolution + batch norm, a root over several sources and a deformable convolution, in bf16 / fp32"""
    n = hnn()
    torch.manual_seed(0)
    conv, root, bn, dcn = n.Conv2d(64, 64, 3, 1, 1).to(DEV), n.Conv2d(128, 64, 1).to(DEV), n.BatchNorm2d(64).to(DEV).eval(), n.DCN(64, 64).to(DEV)
    x = img((2, 16, 16, 64), 1, dt)
    one, zero = torch.ones(64, device=DEV), torch.zeros(64, device=DEV)

    def forward():
        y = n.conv_bn_act(conv, bn, x)
        return n.cat_conv_bn_act(root, bn, [x, y]), bn(y), dcn.infer(x, one, zero, True)

    with torch.no_grad():
        wants = forward()
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            ys = forward()
        for rep in range(3):
            if rep == 1:
                for m in (conv, root, dcn):
                    m.weight.mul_(2)
                bn.running_mean.add_(1)
            else:
                ops().WeightsEpoch.bump()
            eager = forward()
            assert all(torch.equal(a, b) == (rep < 1) for a, b in zip(eager, wants))
            junk = _refill()
            for y in ys:
                y.fill_(float("nan"))
            g.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(ys, wants)), rep
            del junk


def test_the_plain_path_captured_before_any_eager_call():
    n = hnn()
    conv, bn = n.Conv2d(64, 64, 3, 1, 1).to(DEV), n.BatchNorm2d(64).to(DEV).eval()
    x = img((2, 8, 8, 64), 1, BF)
    with torch.no_grad():
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            y = n.conv_bn_act(conv, bn, x)
        eager = n.conv_bn_act(conv, bn, x)
        for _ in range(3):
            y.fill_(float("nan"))
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(y, eager)
            assert torch.equal(n.conv_bn_act(conv, bn, x), eager)


def test_the_plain_path_on_two_streams():
    n = hnn()
    conv, bn = n.Conv2d(64, 64, 3, 1, 1).to(DEV), n.BatchNorm2d(64).to(DEV).eval()
    x = img((1, 16, 16, 64), 1, BF)
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    with torch.no_grad():
        for i in range(3):
            conv.weight.mul_(1.5)
            bn.running_mean.add_(0.25)
            torch.cuda.synchronize()
            with torch.cuda.stream(a):
                _delay()
                first = n.conv_bn_act(conv, bn, x)
            with torch.cuda.stream(b):
                second = n.conv_bn_act(conv, bn, x)
            torch.cuda.synchronize()
            assert torch.equal(first, second) and torch.equal(first, n.conv_bn_act(conv, bn, x))


@pytest.mark.parametrize("dt", [BF, F32])
def test_scale_shift_act_of_no_rows(dt):
    from centernet_amd import mx
    v = torch.ones(48, device=DEV)
    for relu in (False, True):
        x = torch.empty(2, 0, 48, dtype=dt, device=DEV)
        y, ck = mx.scale_shift_act(x, v, v, x, relu)
        assert y.shape == (2, 0, 48) and ck.has_signs == relu and ck.nbytes() == 0


@pytest.mark.parametrize("dt", [BF, F32])
@pytest.mark.parametrize("k,p", [(1, 0), (3, 1)])
@pytest.mark.parametrize("shared", [False, True])
def test_identity_around_a_checkpointed_convolution(dt, k, p, shared):
    """the skip path's gradient joins in the data gradient's epilogue (one rounding in all), as without checkpoints"""
    n = hnn()
    conv = n.Conv2d(64, 64, k, 1, p).to(DEV)
    x = img((2, 8, 8, 64), 1, dt)
    dy, ds = img((2, 8, 8, 64), 2, dt, 1e-2), img((2, 8, 8, 64), 3, dt, 1e-2)
    out = {}
    for ck in (False, True):
        n.use_checkpoints(conv, ck)
        xi = x.clone().requires_grad_()
        xs = ops().share(xi * 1) if shared else xi
        y, skip = conv.with_skip(xs)
        assert torch.equal(skip, x) and type(y.grad_fn).__name__.startswith("Conv2dCkptFn") == ck
        torch.autograd.backward([y, skip], [dy, ds], retain_graph=True)
        both = xi.grad.clone()
        xi.grad = None
        torch.autograd.backward([skip], [ds])                      # the convolution's output unused
        out[ck] = (y.detach(), both, xi.grad)
    assert all(torch.equal(a, b) for a, b in zip(out[True], out[False]))
    assert torch.equal(out[True][2], ds)


@pytest.mark.parametrize("dt", [BF, F32])
@pytest.mark.parametrize("ck", [False, True])
@pytest.mark.parametrize("k,p,Co", [(1, 0, 24), (3, 1, 32), (1, 0, 2)])
def test_a_bias_trains_above_a_frozen_weight(dt, ck, k, p, Co):
    """its gradient is dy's column sums and nothing of the input is kept for it.  Tolerance: 2^-24 of the magnitudes for each of at most
    72 + 16 additions, whatever their order"""
    conv = hnn().Conv2d(32, Co, k, 1, p, bias=True).to(DEV)
    hnn().use_checkpoints(conv, ck)
    conv.weight.requires_grad_(False)
    x = img((2, 6, 6, 32), 1, dt).requires_grad_()
    y = conv(x)
    assert not ck or y.grad_fn.saved_tensors[0] is None
    dy = img(tuple(y.shape), 2, dt, 1e-2)
    dy[..., Co:] = 0
    y.backward(dy)
    d = f64(dy)[..., :Co].reshape(-1, Co)
    within(conv.bias.grad, d.sum(0), 88 * U * np.abs(d).sum(0), "db")
    assert conv.weight.grad is None and x.grad is not None
    first, conv.bias.grad = conv.bias.grad, None
    conv(x.detach()).backward(dy)                                  # nothing but the bias wants a gradient
    within(conv.bias.grad, f64(first), 2 * 88 * U * np.abs(d).sum(0), "db alone")


@pytest.mark.parametrize("rows", [False, True])
def test_biases_of_a_head_train_above_frozen_weights(rows):
    """for a loss over the whole map and for one that gathers a few rows"""
    from centernet_amd import ops as o
    torch.manual_seed(0)
    x = img((2, 16, 16, 64), 1, BF)
    w1, b1, w2, b2 = rnd((64, 64, 3, 3), 2, F32) * 0.05, rnd((64,), 3, F32), rnd((2, 64, 1, 1), 4, F32), rnd((2,), 5, F32)
    ind = torch.randint(0, 256, (2, 5), generator=torch.Generator().manual_seed(1)).to(DEV)
    got = {}
    for frozen in (False, True):
        ps = [t.clone().requires_grad_(not (frozen and t.dim() == 4)) for t in (w1, b1, w2, b2)]
        out = o.HeadFn.apply(x.clone().requires_grad_(), *ps)
        if rows:
            o.GatherL1Fn.apply(out, torch.ones(2, 5, dtype=torch.uint8, device=DEV), ind, torch.zeros(2, 5, 2, device=DEV)).backward()
        else:
            (out * out).sum().backward()
        got[frozen] = [p.grad for p in ps]
    assert got[True][0] is None and got[True][2] is None
    for i in (1, 3):
        assert got[True][i] is not None and torch.allclose(got[True][i], got[False][i], rtol=1e-4, atol=1e-4 * float(got[False][i].abs().max()))


def test_graphs_of_checkpointed_batch_norms_side_by_side(monkeypatch):
    """two layers' forward and backward passes, captured on one stream, replayed at once on two: they share no scratch"""
    n = hnn()
    bns = [n.BatchNorm2d(96).to(DEV).train() for _ in range(2)]
    xs = [img((4, 40, 40, 96), 1 + i, F32, 2.0 ** i) for i in range(2)]
    dys = [img((4, 40, 40, 96), 5 + i, F32, 1e-2) for i in range(2)]

    def step(i):
        xi = xs[i].detach().requires_grad_()
        y = bns[i](xi, None, True)
        return (y.detach(), *torch.autograd.grad(y, (xi, bns[i].weight, bns[i].bias), dys[i]))

    for bn in bns:
        n.use_checkpoints(bn)
    wants = [step(i) for i in range(2)]
    torch.cuda.synchronize()
    from centernet_amd import _hip
    monkeypatch.setattr(_hip, "workspace", None)                   # the stream's own scratch is not asked for
    graphs, outs = [], []
    for i in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step(i))
        graphs.append(g)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for rep in range(6):
        for o in outs:
            for t in o:
                t.fill_(float("nan"))
        torch.cuda.synchronize()
        for s, g in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for o, w in zip(outs, wants):
            assert all(torch.equal(a, b) for a, b in zip(o, w)), rep
