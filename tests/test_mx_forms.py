"""The cases of test_gpu_mx_forms.py reach every kernel that the sizes choose between (no GPU needed)."""
import os

import pytest
import torch

from tests import test_gpu_mx_forms as forms


@pytest.fixture(scope="module")
def lib():
    from centernet_amd import _hip
    if not os.path.exists(_hip.LIB_PATH):
        import __graft_entry__ as g
        g.build()
    return _hip.lib()


def test_linear_forms(lib):
    seen = set()
    for M, K, N, form in forms.LINEAR:
        assert lib.cn_mx_linear_variant(M, K, N) == form, (M, K, N)
        seen.add((form, K % 8 == 0, N % 8 == 0))
    # every form that any size takes, sampled over the whole range
    every = {lib.cn_mx_linear_variant(M, K, N) for M in (1, 5, 33, 600, 4200, 9000, 20000, 33000, 49152, 1 << 20)
             for K in (1, 64, 200, 256, 257, 600, 3000, 7600, 7700, 7900, 8000, 20000, 65536) for N in (1, 32, 33, 64, 65, 128, 129, 300, 800, 5000, 65536)}
    assert {f for f, _, _ in seen} == every
    for f in every:
        assert (f, True, True) in seen and {k for g, k, _ in seen if g == f} == {True, False} and {n for g, _, n in seen if g == f} == {True, False}, f
    assert lib.cn_mx_linear_variant(0, 8, 8) == 0 and lib.cn_mx_linear_variant(1, 8, 65537) == 0


def test_wgrad_forms(lib):
    seen = set()
    for rows, K, N, dt, form in forms.WGRAD:
        v = lib.cn_mx_linear_wgrad_variant(rows, K, N, 1 if dt == torch.bfloat16 else 0)
        splits = v % 1000
        assert v // 1000 % 1000 + v // 1000000 * 1000 == form, (rows, K, N, dt)
        assert lib.cn_mx_linear_wgrad_bytes(rows, K, N, 1 if dt == torch.bfloat16 else 0) == (4 * splits * (N * K + N) if splits > 1 else 0)
        join = 0 if splits == 1 else 64 if splits >= 64 and N * K <= 2048 else 16 if splits >= 16 else 1
        seen.add((dt, form, N % 8 == 0, join))
    for dt in (torch.bfloat16, torch.float32):
        tiles = {f for t, f, _, _ in seen if t == dt}
        assert tiles == ({64064, 128128} if dt == torch.bfloat16 else {64064, 64128})
        for f in tiles:
            assert {n for t, g, n, _ in seen if (t, g) == (dt, f)} == {True, False}
    assert {j for *_, j in seen} == {0, 1, 16, 64}
    assert lib.cn_mx_linear_wgrad_variant(0, 8, 8, 1) == 0
