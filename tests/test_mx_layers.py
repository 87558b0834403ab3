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
    monkeypatch.setattr(torch.cuda, "is_initialized", lambda: True)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: state["capturing"])
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
