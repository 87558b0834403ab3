"""Block-scaled operators without a GPU: what they refuse, and the 64-bit oracle against definitions and finite differences."""
import ctypes
import os

import numpy as np
import pytest
import torch

from oracle import mx_ref


@pytest.fixture(scope="module")
def lib():
    from centernet_amd import _hip
    if not os.path.exists(_hip.LIB_PATH):
        import __graft_entry__ as g
        g.build()
    return _hip.lib()


def mx():
    from centernet_amd import mx as m
    return m


P = ctypes.c_void_p(4096)          # never dereferenced: every call below is refused (or has nothing to do) on the host
ODD = ctypes.c_void_p(4100)


@pytest.mark.parametrize("name,args", [
    ("cn_mx_quantize", (P, P, P, None, None, -1, 32, 1, 1, None)),
    ("cn_mx_quantize", (P, P, P, None, None, 4, 0, 1, 1, None)),
    ("cn_mx_quantize", (P, P, P, None, None, 4, 65537, 1, 1, None)),
    ("cn_mx_quantize", (P, P, P, None, None, 4, 32, 2, 1, None)),
    ("cn_mx_quantize", (P, P, P, None, None, 4, 32, 1, 3, None)),
    ("cn_mx_quantize", (None, P, P, None, None, 4, 32, 1, 1, None)),
    ("cn_mx_quantize", (P, ODD, P, None, None, 4, 32, 1, 1, None)),
    ("cn_mx_quantize", (P, P, P, P, None, 4, 32, 1, 1, None)),
    ("cn_mx_quantize", (P, P, P, None, None, 1 << 60, 32, 1, 1, None)),
    ("cn_mx_dequantize", (P, None, P, 4, 32, 1, 1, None)),
    ("cn_mx_dequantize", (ODD, P, P, 4, 32, 1, 1, None)),
    ("cn_mx_dequantize", (P, P, P, 4, 32, 7, 1, None)),
    ("cn_mx_pack_weight", (P, P, 0, 32, 0, None)),
    ("cn_mx_pack_weight", (P, P, 8, 65537, 0, None)),
    ("cn_mx_pack_weight", (P, ODD, 8, 32, 0, None)),
    ("cn_mx_linear_fwd", (P, P, None, None, P, -1, 32, 32, 0, 1, None)),
    ("cn_mx_linear_fwd", (P, P, None, None, P, 1, 0, 32, 0, 1, None)),
    ("cn_mx_linear_fwd", (P, P, None, None, P, 1, 32, 70000, 0, 1, None)),
    ("cn_mx_linear_fwd", (P, ODD, None, None, P, 1, 32, 32, 0, 1, None)),
    ("cn_mx_linear_fwd", (P, P, None, None, None, 1, 32, 32, 0, 1, None)),
    ("cn_mx_linear_fwd", (P, P, None, None, P, 1, 32, 32, 0, 9, None)),
    ("cn_mx_linear_wgrad", (P, P, P, P, None, 0, 0, 32, 32, 1, P, 1 << 30, None)),
    ("cn_mx_linear_wgrad", (P, P, P, None, None, 0, 8, 32, 32, 1, P, 1 << 30, None)),
    ("cn_mx_linear_wgrad", (P, ODD, P, P, None, 0, 8, 32, 32, 1, P, 1 << 30, None)),
    ("cn_mx_bn_bwd", (P, P, P, None, P, P, P, P, None, None, P, P, 0, 0, 32, 1, P, 1 << 30, None)),
    ("cn_mx_scale_shift_act", (P, None, P, P, P, P, P, None, -1, 32, 0, 1, None)),
    ("cn_mx_scale_shift_act", (P, None, P, P, P, P, P, None, 4, 65537, 0, 1, None)),
    ("cn_mx_scale_shift_act", (P, None, P, P, P, P, P, None, 4, 32, 1, 1, None)),
    ("cn_mx_scale_shift_act", (P, None, P, P, P, P, P, P, 4, 32, 0, 1, None)),
    ("cn_mx_scale_shift_act", (P, None, P, P, P, ODD, P, None, 4, 32, 0, 1, None)),
    ("cn_mx_scale_shift_act", (P, None, P, None, P, P, P, None, 4, 32, 0, 1, None)),
    ("cn_mx_scale_shift_act", (P, None, P, P, P, P, P, None, 4, 32, 0, 5, None)),
    ("cn_bn_train_stats", (P, P, P, None, None, P, P, P, 0, 32, 0.1, 1e-5, 1, P, 1 << 30, None)),
    ("cn_bn_train_stats", (P, P, P, None, None, P, P, P, 64, 20, 0.1, 1e-5, 1, P, 1 << 30, None)),
    ("cn_bn_train_stats", (P, P, P, None, None, P, P, None, 64, 32, 0.1, 1e-5, 1, P, 1 << 30, None)),
    ("cn_mx_bn_bwd", (P, P, P, None, P, P, P, P, None, P, P, P, 0, 8, 32, 1, P, 1 << 30, None)),
    ("cn_mx_bn_bwd", (P, P, P, None, None, P, P, P, None, None, P, P, 0, 8, 32, 1, P, 1 << 30, None)),
])
def test_entry_points_refuse(lib, name, args):
    assert getattr(lib, name)(*args) == -1
    assert name in lib.cn_last_error().decode()


def test_entry_points_ask_for_workspace(lib):
    n = lib.cn_mx_linear_wgrad_bytes(100000, 64, 64, 1)
    assert n > 4 * 64 * 64
    assert lib.cn_mx_linear_wgrad(P, P, P, P, None, 0, 100000, 64, 64, 1, P, n - 1, None) == -3
    assert lib.cn_mx_linear_wgrad(P, P, P, P, None, 0, 100000, 64, 64, 1, None, n, None) == -3
    n = lib.cn_mx_bn_bwd_bytes(100000, 64, 1)
    assert n > 4 * 64
    assert lib.cn_mx_bn_bwd(P, P, P, None, P, P, P, P, None, None, P, P, 0, 100000, 64, 1, P, n - 1, None) == -3
    for bad in ((0, 64, 1), (100000, 0, 1), (100000, 65537, 0)):
        assert lib.cn_mx_bn_bwd_bytes(*bad) == 0
    assert lib.cn_mx_weight_bytes(0, 8) == 0 and lib.cn_mx_weight_bytes(8, 70000) == 0
    assert lib.cn_mx_weight_bytes(33, 65) == 2 * 2 * 1024 + 2 * 256


def test_no_rows_is_no_work(lib):
    assert lib.cn_mx_quantize(None, None, None, None, None, 0, 32, 1, 1, None) == 0
    assert lib.cn_mx_dequantize(None, None, None, 0, 32, 1, 1, None) == 0
    assert lib.cn_mx_linear_fwd(None, None, None, None, None, 0, 32, 32, 0, 1, None) == 0


def test_python_refusals(lib):
    m, x = mx(), torch.zeros(4, 32)
    for f in (m.quantize, m.checkpoint, m.pack_weight):
        with pytest.raises(RuntimeError, match="not on the GPU"):
            f(x)
        with pytest.raises(TypeError):
            f(x.half()) if f is not m.pack_weight else f(x.double())
    with pytest.raises(ValueError, match="unknown format"):
        m.quantize(x, "int8")
    with pytest.raises(TypeError):
        m.quantize([1.0], "e4m3")
    with pytest.raises(ValueError):
        m.quantize(torch.zeros(()), "e4m3")
    with pytest.raises(ValueError):
        m.quantize(torch.zeros(4, 0), "e4m3")
    with pytest.raises(ValueError, match="1x1"):
        m.pack_weight(torch.zeros(4, 4, 3, 3))
    with pytest.raises(ValueError):
        m.pack_weight(torch.zeros(4))
    with pytest.raises(TypeError):
        m.dequantize(x)
    with pytest.raises(TypeError, match="pack_weight"):
        m.linear(x, x)
    with pytest.raises(RuntimeError, match="no backward"):
        m.linear(x.requires_grad_(), m.MXWeight(torch.zeros(1, dtype=torch.uint8), 8, 32))


def test_buffers_of_the_wrong_kind_are_refused(lib):
    """a buffer that came back from a file or another device is checked before a kernel could read beyond it"""
    m, shape = mx(), torch.Size((4, 40))
    meta = (shape, torch.float32, "e4m3", False)
    n = 4 * 2 * 33
    assert m.MXTensor.of(torch.zeros(n, dtype=torch.uint8), meta).nbytes() == n
    for bad in (torch.zeros(n - 1, dtype=torch.uint8), torch.zeros(n), torch.zeros(1, dtype=torch.uint8).expand(n), torch.zeros(2 * n, dtype=torch.uint8)[::2]):
        with pytest.raises(ValueError, match="uint8 buffer"):
            m.MXTensor.of(bad, meta)
    with pytest.raises(RuntimeError, match="not on the GPU"):
        m.dequantize(m.MXTensor.of(torch.zeros(n, dtype=torch.uint8), meta))
    for bad in (torch.zeros(1 * 1024 + 256), torch.zeros(1, dtype=torch.uint8).expand(1280)):
        with pytest.raises(ValueError, match="contiguous uint8"):
            m.MXWeight(bad, 8, 32)


def test_copies_of_a_layer_leave_packed_weights_behind():
    import copy
    import pickle
    from centernet_amd import nn as hnn
    conv = hnn.Conv2d(32, 16, 1)
    conv._mx_cache = ("key", "weights", "bias", ())
    for c in (copy.deepcopy(conv), copy.copy(conv), pickle.loads(pickle.dumps(conv))):
        assert "_mx_cache" not in c.__dict__ and torch.equal(c.weight, conv.weight)
    assert conv._mx_cache[0] == "key"


# ---- the oracle -----------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("fmt,largest,tie", [("e2m1", 6.0, 7.0), ("e4m3", 448.0, 464.0)])
def test_oracle_scale_rule(fmt, largest, tie):
    """the least power of two for which the largest magnitude rounds to a finite element, hand-checked around the border"""
    up = fmt == "e2m1"                                             # e2m1: the tie goes to the next power of two; e4m3: it stays
    x = np.array([[largest], [np.nextafter(tie, 0)], [tie], [np.nextafter(tie, 1e9)], [2.0 ** -140], [0.0]])
    val, codes, scale = mx_ref.quantize(x, fmt)
    assert scale[:, 0].tolist() == [127, 127, 128 if up else 127, 128, 0, 0]
    assert val[:4, 0].tolist() == [largest, largest, 8.0 if up else largest, 8.0 if up else 480.0]


@pytest.mark.parametrize("fmt", ["e2m1", "e4m3"])
def test_oracle_is_idempotent_and_nearest(fmt):
    x = np.random.RandomState(0).randn(20, 70) * np.exp(np.random.RandomState(1).randn(20, 1) * 5)
    val, _, scale = mx_ref.quantize(x, fmt)
    again = mx_ref.quantize(val, fmt)
    assert np.array_equal(again[0], val) and np.array_equal(again[2], scale)
    s = 2.0 ** (np.repeat(scale, 32, 1)[:, :70] - 127.0)
    g = np.concatenate([-mx_ref.grid(fmt)[::-1], mx_ref.grid(fmt)])
    best = np.abs(x[..., None] / s[..., None] - g).min(-1)
    assert np.allclose(np.abs(x - val) / s, best, rtol=1e-12, atol=0)


def test_oracle_gradients_by_differences():
    """at a point that e4m3 holds exactly the checkpointed backward passes are the layers' own: central differences in 64 bits"""
    r = np.random.RandomState(3)
    x = mx_ref.quantize(r.randn(9, 5), "e4m3")[0]
    gamma, beta, cot, res = r.rand(5) + .5, r.randn(5), r.randn(9, 5), r.randn(9, 5)

    def bn(x, gamma, beta, res):
        mu, var = x.mean(0), x.var(0)
        return np.maximum(gamma * (x - mu) / np.sqrt(var + 1e-5) + beta + res, 0)

    def diff(f, a, h=1e-6):
        g = np.zeros_like(a)
        for i in np.ndindex(a.shape):
            p, m = a.copy(), a.copy()
            p[i] += h
            m[i] -= h
            g[i] = (f(p) - f(m)) / (2 * h)
        return g

    y = bn(x, gamma, beta, res)
    dx, dgamma, dbeta, d = mx_ref.batch_norm_act_bwd(cot, x, y, gamma, x.mean(0), 1 / np.sqrt(x.var(0) + 1e-5))[:4]
    loss = lambda *a: (bn(*a) * cot).sum()      # noqa: E731
    for got, want in ((dx, diff(lambda v: loss(v, gamma, beta, res), x)), (dgamma, diff(lambda v: loss(x, v, beta, res), gamma)),
                      (dbeta, diff(lambda v: loss(x, gamma, v, res), beta)), (d, diff(lambda v: loss(x, gamma, beta, v), res))):
        assert np.allclose(got, want, rtol=1e-6, atol=1e-7)

    w, dy = r.randn(3, 5), r.randn(9, 3)
    assert np.allclose(mx_ref.linear_wgrad(dy, x)[0], diff(lambda v: ((x @ v.T) * dy).sum(), w), rtol=1e-7, atol=1e-8)
