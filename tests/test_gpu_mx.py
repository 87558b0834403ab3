"""Block-scaled operators on the GPU against the 64-bit oracle (oracle/mx_ref.py).  Quantisation is compared bit for bit; sums are held to
bounds counted from the roundings they contain (u = 2^-24 for fp32 steps, eps / 2 of the output type once)."""
import numpy as np
import pytest
import torch

from oracle import mx_ref

pytestmark = pytest.mark.gpu

DEV = "cuda"
BF, F32 = torch.bfloat16, torch.float32
U = 2.0 ** -24


def mx():
    from centernet_amd import mx as m
    return m


def f64(t):
    return t.detach().double().cpu().numpy()


def rnd(shape, seed, dt, scale=1.0, spread=0.5):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(shape, generator=g) * torch.exp(spread * torch.randn(shape[-1], generator=g)) * scale
    return x.to(dt).to(DEV)


def half_step(dt):
    return torch.finfo(dt).eps / 2


def within(got, want, tol, what):
    got = f64(got)
    assert got.shape == want.shape, what
    bad = ~((np.abs(got - want) <= tol) | (np.isnan(got) & np.isnan(want)) | (got == want))
    assert not bad.any(), f"{what}: {bad.sum()} of {bad.size} off, worst {np.nanmax((np.abs(got - want) / np.maximum(tol, 1e-300))[bad])} of the bound"


def codes_of(q):
    c = q.codes.cpu().numpy().astype(np.int64)
    return c if q.fmt == "e4m3" else np.stack([c & 15, c >> 4], -1).reshape(c.shape[0], -1)


def same_quantised(q, x, fmt, what=""):
    val, codes, scale = mx_ref.quantize(f64(x).reshape(-1, x.shape[-1]), fmt)
    assert np.array_equal(q.scales.cpu().numpy(), scale), f"{what} scales"
    got = codes_of(q)
    assert got.shape == codes.shape
    if not np.array_equal(got, codes):
        i = np.argwhere(got != codes)[0]
        raise AssertionError(f"{what}: code {got[tuple(i)]} for {codes[tuple(i)]} at {i}, {np.sum(got != codes)} in all")
    back = f64(mx().dequantize(q, F32)).reshape(val.shape)
    with np.errstate(over="ignore"):
        val = val.astype(np.float32).astype(np.float64)            # (a magnitude just below 2^128 rounds up to it: an infinity in 32 bits)
    assert np.array_equal(back, val, equal_nan=True), f"{what} values"
    return val


# ------------------------------------------------------------------------------------------------ quantisation
@pytest.mark.parametrize("fmt", ["e2m1", "e4m3"])
@pytest.mark.parametrize("dt", [BF, F32])
@pytest.mark.parametrize("rows,C", [(1, 1), (1, 7), (3, 8), (2, 16), (5, 31), (257, 32), (2, 33), (67, 80), (4, 208), (3, 515), (2, 2048),
                                    (1031, 64), (1, 65536)])
def test_quantise_matches_the_definition(fmt, dt, rows, C):
    same_quantised(mx().quantize(rnd((rows, C), rows * C, dt), fmt), rnd((rows, C), rows * C, dt), fmt)


@pytest.mark.parametrize("fmt", ["e2m1", "e4m3"])
@pytest.mark.parametrize("dt", [BF, F32])
def test_quantise_ties_and_extremes(fmt, dt):
    """every midpoint of the grid with its neighbours, scale borders, subnormal blocks, zeros of both signs, the largest values, and
    blocks with an infinity or a NaN (which stand for 32 NaNs)"""
    g = mx_ref.grid(fmt)
    mid = (g[1:] + g[:-1]) / 2
    v = np.concatenate([g, mid, np.nextafter(mid.astype(np.float32), np.float32(1e9)), np.nextafter(mid.astype(np.float32), np.float32(0))])
    v = np.concatenate([v, -v]).astype(np.float32)
    v = np.resize(v, (len(v) // 31 + 1, 31))
    blocks = np.concatenate([np.full((len(v), 1), g[-1], np.float32), v], 1)            # the block's maximum fixes scale 1
    rows = [blocks * np.float32(2.0 ** e) for e in (0, 60, -60, -118, -125, -133)]
    top = np.float32({"e2m1": 7, "e4m3": 464}[fmt])
    border = np.zeros((8, 32), np.float32)
    border[:, 3] = [top, np.nextafter(top, np.float32(0)), np.nextafter(top, np.float32(1e9)), -top, 1e-45, 2 ** -126, 3.3e38, -3.38e38]
    special = np.zeros((6, 32), np.float32)
    special[0, 5], special[1, 31], special[2, 0] = np.inf, np.nan, -np.inf
    special[3], special[4, :2], special[5] = -0.0, [np.nan, np.inf], 1.0
    x = torch.tensor(np.concatenate(rows + [border, special])).to(dt).to(DEV)
    val = same_quantised(mx().quantize(x, fmt), x, fmt)
    assert np.isnan(val).all(1).sum() == 4
    y = x.reshape(-1, 64)[: x.shape[0] // 2]                                           # a NaN block leaves its neighbour alone
    same_quantised(mx().quantize(y, fmt), y, fmt)


@pytest.mark.parametrize("dt", [BF, F32])
@pytest.mark.parametrize("C", [8, 77, 96])
def test_quantise_any_address_and_order(dt, C):
    flat = rnd((40 * C + 3,), 5, dt, spread=0)
    for ofs in (1, 2, 3):                                                              # rows that start off a 16-byte border
        x = flat[ofs:ofs + 39 * C].view(39, C)
        q = mx().quantize(x, "e4m3")
        same_quantised(q, x, "e4m3", f"offset {ofs}")
    x = flat[:40 * C].view(C, 40).t()                                                  # transposed, and every other row
    same_quantised(mx().quantize(x, "e2m1"), x, "e2m1")
    same_quantised(mx().quantize(x[::2], "e4m3"), x[::2], "e4m3")
    x = flat[:40 * C].view(2, 4, 5, C)
    q = mx().quantize(x, "e4m3")
    assert mx().dequantize(q).shape == x.shape and mx().dequantize(q).dtype == dt
    same_quantised(q, x, "e4m3")


def test_one_dimension():
    m, x, w = mx(), rnd((96,), 1, BF, spread=0), rnd((40, 96), 2, F32)
    same_quantised(m.quantize(x, "e4m3"), x, "e4m3")
    assert m.dequantize(m.quantize(x, "e2m1")).shape == (96,)
    assert torch.equal(m.linear(x, m.pack_weight(w)), m.linear(x.view(1, 96), m.pack_weight(w))[0])
    dy = rnd((40,), 3, BF, spread=0)
    assert torch.equal(m.linear_wgrad(dy, m.checkpoint(x))[0], m.linear_wgrad(dy.view(1, 40), m.checkpoint(x.view(1, 96)))[0])


def test_dequantise_writes_its_rows_only():
    x = rnd((7, 77), 3, BF)
    q = mx().quantize(x, "e4m3")
    buf = torch.full((9 * 77 + 16,), 5.0, dtype=BF, device=DEV)
    from centernet_amd._hip import call
    call("cn_mx_dequantize", q.codes, q.scales, buf[77:], 7, 77, 1, 1)
    assert (buf[:77] == 5).all() and (buf[8 * 77:] == 5).all()
    assert torch.equal(buf[77:8 * 77].view(7, 77), mx().dequantize(q))


def test_no_rows():
    m = mx()
    q = m.quantize(torch.empty(0, 48, dtype=BF, device=DEV), "e2m1")
    assert m.dequantize(q).shape == (0, 48)
    w = m.pack_weight(rnd((16, 48), 1, F32))
    assert m.linear(torch.empty(2, 0, 48, dtype=BF, device=DEV), w).shape == (2, 0, 16)
    dw, db = m.linear_wgrad(torch.empty(0, 16, dtype=BF, device=DEV), m.checkpoint(torch.empty(0, 48, dtype=BF, device=DEV)), bias=True)
    assert dw.shape == (16, 48) and not dw.any() and not db.any()
    with pytest.raises(ValueError, match="no rows"):
        v = torch.ones(48, device=DEV)
        m.batch_norm_act_bwd(torch.empty(0, 48, dtype=BF, device=DEV), m.checkpoint(torch.empty(0, 48, dtype=BF, device=DEV)), v, v, v)


def test_more_than_2_to_31_elements():
    rows, C = (1 << 25) + 3, 72                                                        # 2.4e9 elements, filler in every row
    x = torch.zeros(rows, C, dtype=BF, device=DEV)
    tail = rnd((5, C), 8, BF)
    x[-5:] = tail
    q = mx().quantize(x, "e2m1")
    y = mx().dequantize(q)
    val = mx_ref.quantize(f64(tail), "e2m1")[0]
    assert np.array_equal(f64(y[-5:]), val)
    assert not y[:-5].any()
    del y
    w = rnd((3, C), 9, F32)
    out = mx().linear(x, mx().pack_weight(w))
    want, s = mx_ref.linear(f64(tail), f64(w))
    within(out[-5:], want, half_step(BF) * np.abs(want) + C * U * s, "linear tail")
    assert not out[:-5].any()
    ck = mx().checkpoint(x)
    dy = torch.zeros(rows, 3, dtype=BF, device=DEV)
    dy[-5:] = rnd((5, 3), 10, BF)
    want, _, s, _ = mx_ref.linear_wgrad(f64(dy[-5:]), f64(tail))
    within(mx().linear_wgrad(dy, ck)[0], want, 64 * U * s, "wgrad tail")
    one = torch.ones(C, device=DEV)
    dz = torch.zeros(rows, C, dtype=BF, device=DEV)
    dz[-5:] = tail
    dx, dgamma, dbeta, _ = mx().batch_norm_act_bwd(dz, ck, one, 0 * one, one)
    dz64, x64 = f64(tail), mx_ref.quantize(f64(tail), "e4m3")[0]
    within(dbeta, dz64.sum(0), 32 * U * np.abs(dz64).sum(0), "dbeta")
    want = dz64 - (dz64.sum(0) + x64 * (dz64 * x64).sum(0)) / rows
    within(dx[-5:], want, half_step(BF) * np.abs(want) + 1e-5 * np.abs(dz64).sum(0), "dx tail")


# ------------------------------------------------------------------------------------------------ checkpoints
@pytest.mark.parametrize("dt", [BF, F32])
@pytest.mark.parametrize("rows,C", [(1, 1), (3, 8), (65, 80), (9, 77), (300, 64)])
def test_checkpoint_signs(dt, rows, C):
    x, y = rnd((rows, C), 1, dt), rnd((rows, C), 2, dt)
    y[0, 0] = float("nan")
    y[-1, -1] = 0.0
    y[rows // 2, C // 2] = -0.0
    ck = mx().checkpoint(x, sign_of=y)
    same_quantised(ck, x, "e4m3")
    bits = np.unpackbits(ck.signs.cpu().numpy(), axis=1, bitorder="little")
    assert np.array_equal(bits[:, :C], (f64(y) > 0).astype(np.uint8)) and not bits[:, C:].any()
    assert ck.nbytes() == rows * (-(-C // 32)) * (32 + 1 + 4)


@pytest.mark.parametrize("dt", [BF, F32])
@pytest.mark.parametrize("relu,residual", [(True, True), (True, False), (False, True), (False, False)])
@pytest.mark.parametrize("rows,C", [(1, 1), (3, 8), (65, 80), (9, 77), (300, 64), (2000, 264), (5003, 12), (2, 3000), (40000, 32)])
def test_scale_shift_act(dt, relu, residual, rows, C):
    """y within its roundings (a product and a sum at once, a sum, the result's), and the checkpoint mx.checkpoint would have made of x and y"""
    x, res = rnd((rows, C), 1, dt), rnd((rows, C), 2, dt) if residual else None
    scale, shift = rnd((C,), 3, F32), rnd((C,), 4, F32)
    y, ck = mx().scale_shift_act(x, scale, shift, res, relu)
    terms = [f64(x) * f64(scale), np.broadcast_to(f64(shift), x.shape), f64(res) if residual else np.zeros(x.shape)]
    want = terms[0] + terms[1] + terms[2]
    want = np.maximum(want, 0) if relu else want
    within(y, want, half_step(dt) * np.abs(want) + 3 * U * sum(np.abs(t) for t in terms), "y")
    again = mx().checkpoint(x, sign_of=y if relu else None)
    assert ck.meta == again.meta and torch.equal(ck.buffer, again.buffer)
    x[0, 0], x[-1, -1] = float("nan"), float("inf")                        # what is no number stays in its block
    y2, ck = mx().scale_shift_act(x, scale, shift, res, relu)
    again = mx().checkpoint(x, sign_of=y2 if relu else None)
    assert torch.equal(ck.buffer, again.buffer)
    same = torch.ones(rows, C, dtype=torch.bool, device=DEV)
    same[0, 0] = same[-1, -1] = False
    assert torch.equal(y2[same], y[same])
    if C % 8 == 0:                                                         # the layers' own kernel
        from centernet_amd import ops
        assert np.array_equal(f64(ops.scale_shift_act(x, scale, shift, res, relu)), f64(y2), equal_nan=True)


def test_scale_shift_act_tiny_values_and_refusals():
    x = torch.full((4, 64), 2.0 ** -130, device=DEV)
    y, ck = mx().scale_shift_act(x, torch.full((64,), 2.0 ** -18, device=DEV), torch.zeros(64, device=DEV), None, True)
    assert torch.equal(ck.buffer, mx().checkpoint(x, sign_of=y).buffer)   # subnormal outputs, kept or flushed, agree with their signs
    xb = torch.full((4, 64), 2.0 ** -126, device=DEV, dtype=BF)
    y, ck = mx().scale_shift_act(xb, torch.full((64,), 2.0 ** -20, device=DEV), torch.zeros(64, device=DEV), None, True)
    assert torch.equal(ck.buffer, mx().checkpoint(xb, sign_of=y).buffer)   # 2^-146 is nothing in 16 bits: not positive
    y, ck = mx().scale_shift_act(x[:0], x[0], x[0])
    assert y.shape == (0, 64) and ck.nbytes() == 0
    v = torch.ones(64, device=DEV)
    for bad in (lambda: mx().scale_shift_act(x, v[:32], v), lambda: mx().scale_shift_act(x, v, v.bfloat16()), lambda: mx().scale_shift_act(x, v, v.cpu()),
                lambda: mx().scale_shift_act(x, v, v, x[:2]), lambda: mx().scale_shift_act(x, v, v, x.bfloat16())):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(RuntimeError, match="not on the GPU"):
        mx().scale_shift_act(x.cpu(), v, v)


# ------------------------------------------------------------------------------------------------ product
LINEAR = [(1, 1, 1), (1, 32, 32), (1, 2048, 512), (2, 64, 80), (31, 16, 64), (33, 77, 5), (64, 100, 200), (65, 513, 130), (129, 208, 65),
          (200, 1100, 300), (130, 4096, 260), (67, 4500, 70), (300, 2100, 100), (5, 9000, 40), (128, 512, 1024), (1000, 64, 64), (257, 256, 2048), (20000, 72, 4), (40, 2056, 3), (50001, 200, 264), (49153, 33, 130)]


@pytest.mark.parametrize("dt", [BF, F32])
@pytest.mark.parametrize("M,K,N", LINEAR)
def test_linear(dt, M, K, N):
    x, w = rnd((M, K), M + K, dt), rnd((N, K), N + K, F32, spread=0)
    bias, res = rnd((N,), 7, F32, spread=0), rnd((M, N), 8, dt, scale=K ** 0.5)
    w4 = mx().pack_weight(w)
    x64, w64 = f64(x), f64(w)
    for b, r, relu in ((None, None, False), (bias, None, True), (None, res, False), (bias, res, True)):
        y = mx().linear(x, w4, b, r, relu=relu)
        want, s = mx_ref.linear(x64, w64, None if b is None else f64(b), None if r is None else f64(r), relu)
        assert y.dtype == dt
        within(y, want, half_step(dt) * np.abs(want) + (K + 8) * U * s, f"bias {b is not None} res {r is not None} relu {relu}")


def test_linear_weight_types_and_shapes():
    m, w = mx(), rnd((48, 96), 1, BF)
    x = rnd((2, 3, 5, 96), 2, BF)
    a = m.linear(x, m.pack_weight(w))
    assert a.shape == (2, 3, 5, 48)
    for v in (w.float(), w.view(48, 96, 1, 1), torch.nn.Parameter(w.float()), w.t().contiguous().t()):
        assert torch.equal(a, m.linear(x, m.pack_weight(v)))
    assert torch.equal(a, m.linear(x.permute(3, 0, 1, 2).contiguous().permute(1, 2, 3, 0), m.pack_weight(w)))
    flat = rnd((97 * 96 + 1,), 3, BF, spread=0)
    for ofs in (0, 1):                                             # rows off a 16-byte border give the same bits
        v = flat[ofs:ofs + 97 * 96].view(97, 96)
        assert torch.equal(m.linear(v, m.pack_weight(w)), m.linear(v.clone(), m.pack_weight(w)))


@pytest.mark.parametrize("M,K,N", [(5, 96, 70), (200, 96, 70), (200, 96, 300)])
def test_linear_keeps_nans_where_they_are(M, K, N):
    x, w = rnd((M, K), 1, BF), rnd((N, K), 2, F32)
    x[2, 40], x[3, 95] = float("inf"), float("nan")
    w[4, 0] = float("nan")
    y = f64(mx().linear(x, mx().pack_weight(w), relu=True))
    bad = np.isnan(y)
    assert bad[2].all() and bad[3].all() and bad[:, 4].all()
    bad[[2, 3]], bad[:, 4] = False, False
    assert not bad.any()
    want, s = mx_ref.linear(f64(x), f64(w), relu=True)
    within(torch.tensor(y), want, half_step(BF) * np.abs(want) + (K + 8) * U * s, "the rest")


def test_linear_refusals():
    m = mx()
    w, x = m.pack_weight(rnd((8, 32), 1, F32)), rnd((4, 32), 2, BF)
    for bad in (lambda: m.linear(rnd((4, 33), 2, BF), w), lambda: m.linear(x, w, torch.zeros(9, device=DEV)),
                lambda: m.linear(x, w, torch.zeros(8, dtype=BF, device=DEV)), lambda: m.linear(x, w, None, torch.zeros(4, 8, device=DEV)),
                lambda: m.linear(x, w, None, torch.zeros(3, 8, dtype=BF, device=DEV)), lambda: m.linear(x, w, torch.zeros(8))):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(RuntimeError, match="no backward"):
        m.linear(x.requires_grad_(), w)
    with torch.no_grad():
        assert m.linear(x, w).shape == (4, 8)


# ------------------------------------------------------------------------------------------------ weight gradient
WGRAD = [(1, 1, 1), (1, 32, 8), (3, 16, 7), (63, 64, 64), (65, 77, 65), (64, 33, 130), (1000, 80, 208), (5000, 64, 16), (700, 515, 129),
         (40000, 16, 24), (128, 2048, 130), (200, 808, 732), (4000, 7, 3), (17000, 424, 420)]


@pytest.mark.parametrize("dt", [BF, F32])
@pytest.mark.parametrize("rows,K,N", WGRAD)
def test_linear_wgrad(dt, rows, K, N):
    x, dy = rnd((rows, K), rows + K, dt).clamp_(min=0), rnd((rows, N), rows + N, dt, scale=1e-3)
    ck = mx().checkpoint(x)
    dw, db = mx().linear_wgrad(dy, ck, bias=True)
    w64, b64, sw, sb = mx_ref.linear_wgrad(f64(dy), f64(x))
    terms = (1 if dt == BF else 3) * rows + 16                     # a 32-bit dy counts as three terms
    within(dw, w64, terms * U * sw, "dw")
    within(db, b64, (rows + 16) * U * sb, "db")
    again = mx().linear_wgrad(dy, ck, bias=True)
    assert torch.equal(dw, again[0]) and torch.equal(db, again[1])
    only, none = mx().linear_wgrad(dy, ck)
    assert none is None and torch.equal(only, dw)
    gw, gb = rnd((N, K, 1, 1), 5, F32), rnd((N,), 6, F32)
    want = (f64(gw).reshape(N, K) + f64(dw), f64(gb) + f64(db))
    got = mx().linear_wgrad(dy, ck, bias=True, into=gw, bias_into=gb)
    assert got[0] is gw and got[1] is gb
    within(gw.view(N, K), want[0], U * np.abs(want[0]), "dw into")
    within(gb, want[1], U * np.abs(want[1]), "db into")


@pytest.mark.parametrize("dt", [BF, F32])
def test_linear_wgrad_nans_and_infinities(dt):
    x, dy = rnd((300, 96), 1, dt), rnd((300, 72), 2, dt)
    x[7, 40] = float("nan")
    dy[9, 3], dy[10, 5] = float("inf"), float("nan")
    dw = f64(mx().linear_wgrad(dy, mx().checkpoint(x))[0])
    with np.errstate(invalid="ignore"):
        want = mx_ref.linear_wgrad(f64(dy), f64(x))[0]
    assert np.array_equal(np.isnan(dw), np.isnan(want)) and np.array_equal(dw[np.isinf(want)], want[np.isinf(want)])


def test_linear_wgrad_odd_addresses():
    flat, x = rnd((301 * 72 + 1,), 1, BF, spread=0), rnd((301, 48), 2, BF)
    ck = mx().checkpoint(x)
    for n in (72, 8):
        dy = flat[1:1 + 301 * n].view(301, n)
        assert torch.equal(mx().linear_wgrad(dy, ck)[0], mx().linear_wgrad(dy.clone(), ck)[0])


def test_linear_wgrad_refusals():
    m = mx()
    ck, dy = m.checkpoint(rnd((6, 32), 1, BF)), rnd((6, 8), 2, BF)
    for bad in (lambda: m.linear_wgrad(rnd((5, 8), 2, BF), ck), lambda: m.linear_wgrad(dy, ck, into=torch.zeros(8, 31, device=DEV)),
                lambda: m.linear_wgrad(dy, ck, into=torch.zeros(8, 32, device=DEV, dtype=BF)),
                lambda: m.linear_wgrad(dy, ck, bias=True, into=torch.zeros(8, 32, device=DEV)),
                lambda: m.linear_wgrad(dy, ck, bias_into=torch.zeros(8, device=DEV)),
                lambda: m.linear_wgrad(dy, ck, into=torch.zeros(32, 8, device=DEV).t())):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(TypeError, match="checkpoint"):
        m.linear_wgrad(dy, m.quantize(rnd((6, 32), 1, BF), "e2m1"))


# ------------------------------------------------------------------------------------------------ batch norm
NORM = [(2, 1), (3, 8), (5, 33), (64, 80), (300, 64), (129, 515), (2000, 256), (7, 2048), (30000, 16), (11, 4100), (512, 100), (513, 24), (1024, 24), (1025, 72),
        (2049, 72), (2100, 13), (9000, 520), (70000, 7)]


@pytest.mark.parametrize("dt", [BF, F32])
@pytest.mark.parametrize("relu,residual", [(True, True), (True, False), (False, False), (False, True)])
@pytest.mark.parametrize("rows,C", NORM)
def test_batch_norm_act_bwd(dt, relu, residual, rows, C):
    x, dy = rnd((rows, C), rows + C, dt), rnd((rows, C), rows, dt, scale=1e-2)
    y = rnd((rows, C), 3, dt).clamp_(min=0) if relu else None
    x64 = f64(x)
    gamma, mean = rnd((C,), 4, F32, spread=0) + 1, torch.tensor(x64.mean(0), dtype=F32, device=DEV)
    invstd = torch.tensor(1 / np.sqrt(x64.var(0) + 1e-5), dtype=F32, device=DEV)
    ck = mx().checkpoint(x, sign_of=y)
    dx, dgamma, dbeta, dres = mx().batch_norm_act_bwd(dy, ck, gamma, mean, invstd, residual=residual)
    want = mx_ref.batch_norm_act_bwd(f64(dy), x64, None if y is None else f64(y), f64(gamma), f64(mean), f64(invstd))
    within(dx, want[0], half_step(dt) * np.abs(want[0]) + U * want[4], "dx")
    within(dgamma, want[1], U * want[5], "dgamma")
    within(dbeta, want[2], U * want[6], "dbeta")
    assert (dres is None) if not residual else np.array_equal(f64(dres), want[3])
    again = mx().batch_norm_act_bwd(dy, ck, gamma, mean, invstd, residual=residual)
    assert all(torch.equal(a, b) for a, b in zip((dx, dgamma, dbeta), again))
    if residual:
        gg, gb, racc = rnd((C,), 5, F32), rnd((C,), 6, F32), rnd((rows, C), 7, dt)
        sums = (f64(gg) + f64(dgamma), f64(gb) + f64(dbeta))
        got = mx().batch_norm_act_bwd(dy, ck, gamma, mean, invstd, residual=True, racc=racc, into=(gg, gb))
        assert torch.equal(got[0], dx) and got[1] is gg and got[2] is gb
        within(gg, sums[0], U * np.abs(sums[0]), "dgamma into")
        within(gb, sums[1], U * np.abs(sums[1]), "dbeta into")
        tot = want[3] + f64(racc)
        within(got[3], tot, (half_step(dt) + U) * np.abs(tot), "dres + racc")


def test_batch_norm_nothing_passed_the_relu():
    """a layer whose ReLU let nothing through has zero gradients, whatever dy holds there"""
    x, dy = rnd((50, 40), 1, BF), rnd((50, 40), 2, BF)
    dy[3, 4] = float("nan")
    one = torch.ones(40, device=DEV)
    out = mx().batch_norm_act_bwd(dy, mx().checkpoint(x, sign_of=torch.zeros_like(x)), one, 0 * one, one, residual=True)
    assert all(not t.any() for t in out)


def test_batch_norm_refusals():
    m = mx()
    ck, dy, v = m.checkpoint(rnd((6, 32), 1, BF)), rnd((6, 32), 2, BF), torch.ones(32, device=DEV)
    for bad in (lambda: m.batch_norm_act_bwd(dy.float(), ck, v, v, v), lambda: m.batch_norm_act_bwd(dy[:5], ck, v, v, v),
                lambda: m.batch_norm_act_bwd(dy, ck, v[:31], v, v), lambda: m.batch_norm_act_bwd(dy, ck, v, v.to(BF), v),
                lambda: m.batch_norm_act_bwd(dy, ck, v, v, v, racc=dy), lambda: m.batch_norm_act_bwd(dy, ck, v, v, v.cpu()),
                lambda: m.batch_norm_act_bwd(dy, ck, v, v, v, residual=True, racc=dy[:5]),
                lambda: m.batch_norm_act_bwd(dy, ck, v, v, v, into=(v, torch.ones(64, device=DEV)[::2])),
                lambda: m.batch_norm_act_bwd(dy, ck, v, v, v, into=(v, v))):
        with pytest.raises(ValueError):
            bad()


# ------------------------------------------------------------------------------------------------ together, streams, graphs
def _pass(x, w4, bias, dy, gamma, mean, invstd):
    m = mx()
    y = m.linear(x, w4, bias, relu=True)
    ck = m.checkpoint(x, sign_of=x)
    a, cka = m.scale_shift_act(y, bias, bias, y, relu=True)
    return (y, a, m.dequantize(cka), m.dequantize(m.quantize(y, "e4m3")), *m.linear_wgrad(dy, ck, bias=True), *m.batch_norm_act_bwd(x, ck, gamma, mean, invstd, residual=True))


def _inputs(seed, rows=3000, K=96, N=72):
    x, dy = rnd((rows, K), seed, BF), rnd((rows, N), seed + 1, BF)
    w4 = mx().pack_weight(rnd((N, K), seed + 2, F32))
    return x, w4, rnd((N,), seed + 3, F32), dy, rnd((K,), seed + 4, F32), rnd((K,), seed + 5, F32), rnd((K,), seed + 6, F32).abs() + 0.1


def test_on_another_stream():
    a = _inputs(1)
    want = _pass(*a)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got = _pass(*a)
        junk = _pass(*_inputs(50))
    s.synchronize()
    del junk
    assert all(torch.equal(p, q) for p, q in zip(want, got))


def test_captured_and_replayed():
    """two graphs of the same operators replayed alternately and side by side on two streams, with eager work between the replays"""
    ins = [_inputs(1), _inputs(30)]
    wants = [_pass(*a) for a in ins]
    torch.cuda.synchronize()
    graphs, outs = [], []
    for a in ins:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(_pass(*a))
        graphs.append(g)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for rep in range(4):
        for o in outs:
            for t in o:
                t.fill_(float("nan"))
        eager = _pass(*ins[rep % 2])
        torch.cuda.synchronize()
        for s, g in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(eager, wants[rep % 2]))
        for o, w in zip(outs, wants):
            assert all(torch.equal(p, q) for p, q in zip(o, w)), rep


def test_two_threads():
    """two host threads, a stream each, call everything at once"""
    import threading
    ins = [_inputs(1), _inputs(30)]
    wants = [_pass(*a) for a in ins]
    torch.cuda.synchronize()
    errors = []

    def work(k):
        try:
            s = torch.cuda.Stream()
            with torch.cuda.stream(s):
                for _ in range(10):
                    got = _pass(*ins[k])
                    s.synchronize()
                    assert all(torch.equal(p, q) for p, q in zip(got, wants[k]))
        except BaseException as e:      # noqa: BLE001 - reported by the main thread
            errors.append(e)

    threads = [threading.Thread(target=work, args=(k,)) for k in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors


@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="needs two GPUs")
def test_on_a_device_that_is_not_the_current_one():
    a = _inputs(1)
    want = _pass(*a)
    with torch.cuda.device(0):
        b = [t.to("cuda:1") if isinstance(t, torch.Tensor) else mx().MXWeight(t.packed.to("cuda:1"), t.out_features, t.in_features) for t in a]
        torch.cuda.synchronize(1)
        got = _pass(*b)
        torch.cuda.synchronize(1)
    assert all(t.device.index == 1 for t in got)
    assert all(torch.equal(p, q.to(p.device)) for p, q in zip(want, got))


def test_packed_weights_of_another_size_are_refused():
    w = mx().pack_weight(torch.randn(40, 70, device="cuda"))
    x = torch.randn(3, 70, device="cuda")
    again = mx().MXWeight(w.packed.clone(), 40, 70)
    assert torch.equal(mx().linear(x, w), mx().linear(x, again))
    with pytest.raises(ValueError, match="packed weights"):
        mx().linear(x, mx().MXWeight(w.packed[:-256], 40, 70))
    with pytest.raises(ValueError, match="packed weights"):
        mx().linear(torch.randn(3, 200, device="cuda"), mx().MXWeight(w.packed, 40, 200))
