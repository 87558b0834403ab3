"""Every form that the block-scaled product, weight gradient and batch norm backward choose by size, on data whose results are exact.

Values are small integers (or e2m1 elements) times powers of two: quantisation loses nothing, every product and every partial sum is a
multiple of one unit below 2^24 of them, so 32-bit sums are exact in any order and the only rounding left is the one to the output's type.
A row, channel or block left out, doubled or scaled by its neighbour's scale shows at any size."""
import numpy as np
import pytest
import torch

from tests.test_gpu_mx import BF, DEV, F32, U, f64, half_step, mx, within

pytestmark = pytest.mark.gpu


def ints(shape, lo, hi, seed):
    return torch.randint(lo, hi + 1, shape, generator=torch.Generator().manual_seed(seed)).double()


def blocks_scaled(x, most, seed):
    """x [rows, C] with every block of 32 channels times a power of two of its own, 1 .. 2^most"""
    rows, C = x.shape
    e = ints((rows, -(-C // 32)), 0, most, seed)
    return x * (2.0 ** e).repeat_interleave(32, 1)[:, :C]


def exactly(got, want, what):
    """got is the float64 result rounded once to got's type"""
    want = want.to(F32).to(got.dtype)
    bad = ~(got.cpu() == want)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, the first at {bad.nonzero()[0].tolist()}"


# ------------------------------------------------------------------------------------------------ product
#: M, K, N and the kernel (cn_mx_linear_variant): even sizes, then channels and columns that are no multiples of eight
LINEAR = [(5, 70, 40, 11114), (9, 2056, 40, 11118), (200, 1100, 200, 11118), (201, 1104, 203, 11118), (600, 520, 504, 11114), (20000, 72, 20, 11114),
          (5, 7616, 40, 111118), (5, 7617, 37, 111118), (550, 8008, 504, 111114), (550, 8009, 499, 111114),
          (8300, 72, 64, 12411), (8300, 77, 61, 12411), (8301, 256, 40, 12411), (4200, 200, 128, 12221), (4201, 77, 101, 12221),
          (700, 1104, 760, 12141), (701, 1023, 757, 12141), (700, 264, 760, 12141), (33000, 312, 520, 12141), (700, 8008, 760, 112141),
          (701, 8009, 757, 112141), (49160, 200, 264, 22141), (49201, 77, 301, 22141), (49160, 256, 136, 22141)]


@pytest.mark.parametrize("dt", [BF, F32])
@pytest.mark.parametrize("M,K,N,form", LINEAR)
def test_linear(dt, M, K, N, form):
    grid = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64)
    x = blocks_scaled(grid[ints((M, K), 0, 7, 1).long()] * (2 * ints((M, K), 0, 1, 2) - 1), 2, 3)
    w = blocks_scaled(grid[ints((N, K), 0, 7, 4).long()] * (2 * ints((N, K), 0, 1, 5) - 1), 2, 6)
    bias, res = ints((N,), -64, 64, 7) / 4, ints((M, N), -64, 64, 8) / 4              # (bf16 holds 7 bits and a sign)
    acc = x @ w.t()
    # a partial sum has at most this many units of 1/4 (magnitudes by their largest: 6 * 4 each)
    assert K * (24 * 24 * 4) + 256 < 1 << 26 and float((x[:64].abs() @ w[:64].abs().t()).max()) * 4 < 1 << 24
    xd, w4 = x.to(dt).to(DEV), mx().pack_weight(w.to(F32).to(DEV))
    assert torch.equal(xd.double().cpu(), x) and torch.equal(mx().dequantize(mx().quantize(xd, "e2m1")), xd)
    exactly(mx().linear(xd, w4), acc, "alone")
    exactly(mx().linear(xd, w4, bias.to(F32).to(DEV), res.to(dt).to(DEV), relu=True), (acc + bias + res).clamp(min=0), "bias, residual, relu")


# ------------------------------------------------------------------------------------------------ weight gradient
#: rows, K, N, type and the kernel (cn_mx_linear_wgrad_variant; splits apart)
WGRAD = [(7, 40, 24, BF, 64064), (1000, 64, 64, BF, 64064), (1003, 77, 101, BF, 64064), (900, 808, 736, BF, 64064), (40003, 16, 24, BF, 64064),
         (40003, 13, 21, BF, 64064), (70001, 96, 72, BF, 64064), (17001, 424, 424, BF, 128128), (17001, 424, 420, BF, 128128),
         (24577, 200, 696, BF, 128128), (100003, 136, 328, BF, 128128), (262147, 128, 96, BF, 128128), (7, 40, 24, F32, 64064),
         (1003, 80, 104, F32, 64064), (40003, 13, 21, F32, 64064), (3001, 424, 424, F32, 64128), (3001, 421, 420, F32, 64128),
         (24577, 200, 696, F32, 64128), (100003, 72, 80, F32, 64128)]


@pytest.mark.parametrize("rows,K,N,dt,form", WGRAD)
def test_linear_wgrad(rows, K, N, dt, form):
    x, dy = blocks_scaled(ints((rows, K), -15, 15, 1), 1, 2), ints((rows, N), -4, 4, 3)
    assert rows * 30 * 4 <= 1 << 25 and float(x[:, :8].abs().t().matmul(dy[:, :8].abs()).max()) < 1 << 24
    want, db = x.t().matmul(dy).t(), dy.sum(0)
    xd, dyd = x.to(dt).to(DEV), dy.to(dt).to(DEV)
    ck = mx().checkpoint(xd)
    assert torch.equal(mx().dequantize(ck), xd)
    got = mx().linear_wgrad(dyd, ck, bias=True)
    exactly(got[0], want, "dw")
    exactly(got[1], db, "db")
    exactly(mx().linear_wgrad(dyd, ck)[0], want, "dw without a bias")
    gw, gb = ints((N, K), -9, 9, 4), ints((N,), -9, 9, 5)
    into = gw.to(F32).to(DEV), gb.to(F32).to(DEV)
    mx().linear_wgrad(dyd, ck, bias=True, into=into[0], bias_into=into[1])
    exactly(into[0], want + gw, "dw into")
    exactly(into[1], db + gb, "db into")


@pytest.mark.parametrize("rows,K,N", [(70, 40, 24), (1003, 80, 104), (40003, 13, 21), (3001, 424, 424), (3001, 421, 420), (24577, 200, 696)])
def test_linear_wgrad_keeps_all_bits_of_a_32_bit_gradient(rows, K, N):
    """one row per output column carries a gradient of 24 significant bits, x is powers of two: the result is their product, to the last
    bit (rows are spread over the whole range, the first and the last among them)"""
    g = torch.Generator().manual_seed(1)
    at = torch.linspace(0, rows - 1, N).round().long()
    v = (ints((N,), 1 << 23, (1 << 24) - 1, 2) / (1 << 23)) * 2.0 ** ints((N,), -20, 20, 3) * (2 * ints((N,), 0, 1, 4) - 1)
    dy = torch.zeros(rows, N, dtype=torch.float64)
    dy[at, torch.arange(N)] = v[torch.randperm(N, generator=g)]
    x = 2.0 ** ints((rows, K), -4, 4, 5)
    got, db = mx().linear_wgrad(dy.to(F32).to(DEV), mx().checkpoint(x.to(F32).to(DEV)), bias=True)
    exactly(got, dy[at, torch.arange(N)][:, None] * x[at], "dw")
    exactly(db, dy.sum(0), "db")


# ------------------------------------------------------------------------------------------------ batch norm
NORM = [(2, 24), (100, 40), (128, 61), (129, 264), (400, 77), (513, 48), (1024, 29), (1025, 72), (1500, 13), (5003, 520), (5003, 133), (30000, 16), (70000, 7),
        (70000, 64), (300007, 24), (16384, 512)]


@pytest.mark.parametrize("dt", [BF, F32])
@pytest.mark.parametrize("relu", [False, True])
@pytest.mark.parametrize("rows,C", NORM)
def test_batch_norm_act_bwd(dt, relu, rows, C):
    """sums over whole numbers are exact; what is left of dx are the roundings of its three terms (eight each) and the output's"""
    x, dy = blocks_scaled(ints((rows, C), -15, 15, 1), 1, 2), ints((rows, C), -4, 4, 3)
    y = ints((rows, C), -1, 1, 4).clamp(min=0)
    mean, invstd, gamma = ints((C,), -3, 3, 5), 2.0 ** ints((C,), -6, -3, 6), ints((C,), 1, 7, 7)
    assert rows * 33 * 4 < 1 << 26
    d = dy * y if relu else dy
    s0, s1 = d.sum(0), (d * (x - mean)).sum(0)
    assert float((d * (x - mean)).abs().sum(0).max()) < 1 << 24
    xd, f = x.to(dt).to(DEV), lambda t: t.to(F32).to(DEV)      # noqa: E731
    ck = mx().checkpoint(xd, sign_of=y.to(dt).to(DEV) if relu else None)
    dx, dgamma, dbeta, dres = mx().batch_norm_act_bwd(dy.to(dt).to(DEV), ck, f(gamma), f(mean), f(invstd), residual=True)
    exactly(dbeta, s0, "dbeta")
    exactly(dgamma, s1 * invstd, "dgamma")
    exactly(dres, d, "dres")
    a, t0, t1 = (gamma * invstd).numpy(), (s0 / rows).numpy(), ((x - mean) * invstd ** 2 * s1 / rows).numpy()
    want = a * (d.numpy() - t0 - t1)
    within(dx, want, half_step(dt) * np.abs(want) + 8 * U * a * (np.abs(d.numpy()) + np.abs(t0) + np.abs(t1)), "dx")
    gg, gb = ints((C,), -9, 9, 8), ints((C,), -9, 9, 9)
    into = f(gg), f(gb)
    again = mx().batch_norm_act_bwd(dy.to(dt).to(DEV), ck, f(gamma), f(mean), f(invstd), residual=True, racc=xd, into=into)
    assert torch.equal(again[0], dx)
    exactly(into[0], gg + s1 * invstd, "dgamma into")
    exactly(into[1], gb + s0, "dbeta into")
    exactly(again[3], d + x, "dres + racc")
