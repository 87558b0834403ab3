"""What the layers keep for the no-grad path, under captured graphs and streams on the GPU."""
import pytest
import torch

from tests.test_gpu_mx import BF, DEV, F32, rnd
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
