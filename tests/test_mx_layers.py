"""What the layers keep of their packed weights (nn.Derived), without a GPU."""
import gc
import os
import weakref

import numpy as np
import pytest
import torch


@pytest.fixture(scope="module")
def lib():
    from centernet_amd import _hip
    if not os.path.exists(_hip.LIB_PATH):
        import __graft_entry__ as g
        g.build()
    return _hip.lib()


def hnn():
    from centernet_amd import nn
    return nn


@pytest.fixture
def packing(lib, monkeypatch):
    """packing without a GPU: -> a dict whose "capturing" says whether the current stream is; packed weights are any bytes"""
    from centernet_amd import mx
    state = {"capturing": False}
    monkeypatch.setattr(hnn(), "_capturing", lambda device: state["capturing"])
    monkeypatch.setattr(mx, "pack_weight", lambda w: mx.MXWeight(w.reshape(-1).view(torch.uint8).clone(), *w.shape))
    return state


def test_a_captured_graph_keeps_the_weights_it_reads(packing):
    """replays read the buffers that the capture was handed: the layer may not let go of them when its weights change"""
    conv, x = hnn().Conv2d(32, 16, 1, bias=True), torch.zeros(1, 1, 1, 32)
    conv._mx_weight(x, None, None)                                 # the warm-up
    packing["capturing"] = True
    w, b = conv._mx_weight(x, None, None)
    assert conv._mx_weight(x, None, None)[0] is w                  # (a layer used twice)
    packing["capturing"] = False
    kept = [weakref.ref(w.packed), weakref.ref(b)]
    were = w.packed.clone()
    del w, b
    for _ in range(2):
        with torch.no_grad():
            conv.weight.add_(1)
        assert not torch.equal(conv._mx_weight(x, None, None)[0].packed, were)
        gc.collect()
        assert all(r() is not None for r in kept) and torch.equal(kept[0](), were)
    eager = weakref.ref(conv._mx_weight(x, None, None)[0].packed)
    with torch.no_grad():
        conv.weight.add_(1)
    conv._mx_weight(x, None, None)
    gc.collect()
    assert eager() is None                                         # what no graph reads goes


def test_what_a_capture_packs_is_not_kept(packing):
    conv, x = hnn().Conv2d(32, 16, 1), torch.zeros(1, 1, 1, 32)
    packing["capturing"] = True
    first = conv._mx_weight(x, None, None)[0]
    packing["capturing"] = False
    assert conv._mx_weight(x, None, None)[0] is not first


def test_new_data_in_the_same_parameter_is_packed_anew(packing):
    """`p.data = t` (what `module.to` does) changes neither the parameter nor its version"""
    conv, x = hnn().Conv2d(32, 16, 1, bias=True), torch.zeros(1, 1, 1, 32)
    w, b = conv._mx_weight(x, None, None)
    assert conv._mx_weight(x, None, None)[0] is w
    conv.weight.data = conv.weight.data + 1
    w2, b2 = conv._mx_weight(x, None, None)
    assert not torch.equal(w2.packed, w.packed)
    conv.bias.data = conv.bias.data + 1
    assert torch.equal(conv._mx_weight(x, None, None)[1], b2 + 1)
    data = np.zeros((16, 32, 1, 1), np.float32)
    first = weakref.ref(data)
    conv.weight.data = torch.from_numpy(data)
    del data
    conv._mx_weight(x, None, None)
    conv.weight.data = torch.ones(16, 32, 1, 1)
    gc.collect()
    assert first() is not None                                     # or the next data could lie where the first did
    conv._mx_weight(x, None, None)
    gc.collect()
    assert first() is None


# ------------------------------------------------------------------------------------------------ the bf16 / fp32 path
def _fill(bn, seed):
    g = torch.Generator().manual_seed(seed)
    return {k: v if k == "num_batches_tracked" else torch.rand(v.shape, generator=g) + 0.5 for k, v in bn.state_dict().items()}


def _folded(sd):
    scale = sd["weight"] / torch.sqrt(sd["running_var"] + 1e-5)
    return scale, sd["bias"] - sd["running_mean"] * scale


def test_a_copy_folds_its_own_batch_norm():
    """copied parameters start at version 0; loading a state dict brings them to the version at which the first was folded"""
    import copy
    import pickle
    bn = hnn().BatchNorm2d(8)
    bn.load_state_dict(_fill(bn, 1), assign=True)
    with torch.no_grad():
        for t in (bn.weight, bn.bias, bn.running_mean, bn.running_var):
            t.mul_(1)                                              # version 1
    bn.folded()
    for other in (copy.deepcopy(bn), pickle.loads(pickle.dumps(bn))):
        sd = _fill(bn, 2)
        other.load_state_dict(sd)
        for got, want in zip(other.folded(), _folded(sd)):
            assert torch.allclose(got, want, rtol=1e-5)
    for seed in (3, 4):                                            # another parameter in the old one's place, and other data in the same
        sd = _fill(bn, seed)
        bn.load_state_dict(sd, assign=True)
        for got, want in zip(bn.folded(), _folded(sd)):
            assert torch.allclose(got, want, rtol=1e-5)
    sd = {k: v.clone() for k, v in bn.state_dict().items()}
    bn.running_mean.data = bn.running_mean.data + 1
    sd["running_mean"] += 1
    for got, want in zip(bn.folded(), _folded(sd)):
        assert torch.allclose(got, want, rtol=1e-5)


def _packs(monkeypatch):
    from centernet_amd import ops
    monkeypatch.setattr(ops, "pack_weight", lambda w, mode, dtype, scale=None: w.detach().clone() if scale is None else w.detach() * scale.view(-1, 1, 1, 1))


def test_a_copy_packs_its_own_weights(monkeypatch):
    import copy
    _packs(monkeypatch)
    conv, x = hnn().Conv2d(4, 6, 3), torch.zeros(1)
    with torch.no_grad():
        conv.load_state_dict({"weight": torch.randn(6, 4, 3, 3)}, assign=True)
        conv.weight.mul_(1)
    assert torch.equal(conv.infer_key(x)["wp"], conv.weight) and conv.infer_key(x)["wp"] is conv.infer_key(x)["wp"]
    other, new = copy.deepcopy(conv), torch.randn(6, 4, 3, 3)
    other.load_state_dict({"weight": new})
    assert other.weight._version == conv.weight._version and torch.equal(other.infer_key(x)["wp"], new)
    for _ in range(2):
        new = torch.randn(6, 4, 3, 3)
        conv.load_state_dict({"weight": new}, assign=True)
        assert torch.equal(conv.infer_key(x)["wp"], new)
    conv.weight.data = new + 1
    assert torch.equal(conv.infer_key(x)["wp"], new + 1)


def test_graphs_keep_packed_and_folded_weights_too(packing, monkeypatch):
    _packs(monkeypatch)
    conv, bn, x = hnn().Conv2d(4, 6, 3), hnn().BatchNorm2d(6), torch.zeros(1)
    packing["capturing"] = True
    made = bn.folded()                                             # without a warm-up: in the graph's memory, not for eager calls
    packing["capturing"] = False
    s, b = bn.folded()
    assert s is not made[0]
    wp = conv.infer_key(x, s, b)["wp"]
    packing["capturing"] = True
    assert bn.folded()[0] is s and conv.infer_key(x, s, b)["wp"] is wp
    packing["capturing"] = False
    kept = [weakref.ref(t) for t in (s, b, wp)]
    del s, b, wp, made
    with torch.no_grad():
        conv.weight.add_(1)
        bn.weight.add_(1)
    conv.infer_key(x, *bn.folded())
    gc.collect()
    assert all(r() is not None for r in kept)


# ------------------------------------------------------------------------------------------------ entry points
def test_scale_shift_act_of_no_rows(lib):
    """an empty checkpoint's buffers are null, those of its sign bits too"""
    for relu in (0, 1):
        assert lib.cn_mx_scale_shift_act(None, None, None, None, None, None, None, None, 0, 32, relu, 1, None) == 0


P = 4096                            # never dereferenced: every call below is refused on the host


@pytest.mark.parametrize("name,args", [
    ("cn_mx_quantize", (P, P, P, None, None, 1 << 33, 1, 1, 1, None)),
    ("cn_mx_dequantize", (P, P, P, 1 << 33, 1, 0, 1, None)),
    ("cn_mx_linear_fwd", (P, P, None, None, P, 1 << 30, 16, 8, 0, 1, None)),
    ("cn_mx_linear_fwd", (P, P, None, None, P, 1 << 33, 64, 64, 0, 0, None)),
    ("cn_mx_bn_bwd", (P, P, P, None, P, P, P, P, None, None, P, P, 0, 1 << 36, 1, 1, P, 1 << 30, None)),
    ("cn_mx_scale_shift_act", (P, None, P, P, P, P, P, P, 1 << 36, 1, 1, 1, None)),
])
def test_more_threads_than_a_launch_has_are_refused(lib, name, args):
    assert getattr(lib, name)(*args) == -1
    error = lib.cn_last_error().decode()
    assert name in error and "one launch" in error


def test_inputs_that_want_a_gradient_are_refused():
    """where autograd records, a result that is a constant to it would cut the gradient without a word"""
    from centernet_amd import mx
    x, v = torch.zeros(4, 32), torch.zeros(32)
    xg, vg = torch.zeros(4, 32, requires_grad=True), torch.zeros(32, requires_grad=True)
    calls = [lambda: mx.quantize(xg), lambda: mx.quantize(xg * 2, "e2m1"), lambda: mx.scale_shift_act(xg, v, v), lambda: mx.scale_shift_act(x, vg, v),
             lambda: mx.scale_shift_act(x, v, vg), lambda: mx.scale_shift_act(x, v, v, xg, True)]
    for call in calls:
        with pytest.raises(RuntimeError, match="no backward pass"):
            call()
        with torch.no_grad(), pytest.raises(RuntimeError, match="not on the GPU|expected"):       # (taken: the next check speaks)
            call()
    for call in (lambda: mx.quantize(xg.detach()), lambda: mx.checkpoint(xg), lambda: mx.checkpoint(x, sign_of=xg)):
        with pytest.raises(RuntimeError, match="not on the GPU"):
            call()


def test_a_capture_that_packs_keeps_the_folded_batch_norm_it_reads(packing, monkeypatch):
    """the batch norm was folded before the capture, the convolution is packed in it: every replay reads scale and shift again"""
    _packs(monkeypatch)
    monkeypatch.setattr(hnn().Conv2d, "infer", lambda self, x, s, b, res, relu: self.infer_key(x, s, b)["wp"])
    conv, bn, x = hnn().Conv2d(4, 6, 3), hnn().BatchNorm2d(6).eval(), torch.zeros(1)
    kept = [weakref.ref(t) for t in bn.folded()]
    packing["capturing"] = True
    with torch.no_grad():
        hnn().conv_bn_act(conv, bn, x)
    packing["capturing"] = False
    with torch.no_grad():
        bn.weight.add_(1)
        hnn().conv_bn_act(conv, bn, x)
    gc.collect()
    assert all(r() is not None for r in kept)
