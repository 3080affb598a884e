"""Which kernel each MXFP4 product takes (no GPU: 256 CUs assumed): the shapes that the GPU tests run cover
every variant that any shape takes."""
import ctypes
import random

import pytest
import torch

from kb_nano_amd._lib import lib
from tests._mx_util import assert_product, random_mx, values
from tests.test_gpu_mxfp4_tiles import SHAPES

# few rows: weight rows of a workgroup in 16s, activation rows in 16s
FEW = {(rf, cg) for rf in (1, 2, 3, 4) for cg in (1, 2, 3, 4)} - {(4, 4)}
# tiles and K splits
TILES = {(bm, bn, s) for bm, bn in ((64, 64), (64, 128), (128, 128), (128, 256), (256, 256)) for s in (1, 2, 3, 4)} \
    - {(256, 256, 2), (256, 256, 4)}
# few rows of 16-bit values quantized by the product's launch: weight rows in 16s, rows that the variant holds
VALUES = {(rf, n) for rf in (1, 2, 3, 4) for n in (2, 4, 8, 16)} - {(4, 8), (4, 16)}
# 64x128 in two splits, and few rows of one group in 16 and 32 weight rows, which SHAPES has none of
MORE = [(42, 10888, 25216), (3, 515, 1152), (7, 4357, 640)]


def plan(M, N, K, x_dtype=-1):
    out = (ctypes.c_int64 * 6)()
    assert lib().kbn_debug_mxfp4_plan(M, N, K, x_dtype, out) == 0, lib().kbn_last_error().decode()
    return tuple(out)


def variant(M, N, K):
    bm, bn, splits, rf, _, _ = plan(M, N, K)
    return (rf, -(-M // 16)) if rf else (bm, bn, splits)


def test_every_variant_has_a_shape():
    got = {}
    for s in SHAPES + MORE:
        got.setdefault(variant(*s), []).append(s)
    assert set(got) == FEW | TILES, (FEW | TILES) ^ set(got)
    assert variant(*MORE[0]) == (64, 128, 2)


def test_every_variant_of_the_fused_linear_has_a_shape():
    """Those of test_gpu_mxfp4_tiles.test_linear_of_few_rows."""
    got = set()
    for M in (*range(1, 10), 13, 16, 17):
        for N, K in ((67, 128), (515, 1152), (4357, 640), (9001, 1408), (12999, 384)):
            for dt in (0, 1):
                _, _, _, rf, n, ws = plan(M, N, K, dt)
                assert (n > 0) == (ws == 0) and (not n or n // 2 < M <= n or n == 2)
                if n:
                    got.add((rf, n))
            assert plan(M, N, K, 2)[4] == 0     # fp32 values always have a launch of their own
    assert got == VALUES, VALUES ^ got


def test_no_shape_takes_another_variant():
    rng = random.Random(5)

    def spread(lo, hi):
        return round(lo * (hi / lo) ** rng.random())

    taken, fused = set(), set()
    for _ in range(40000):
        M, N, K = spread(1, 8192), spread(1, 200000), 128 * spread(1, 256)
        v = variant(M, N, K)
        taken.add(v)
        bm, bn, splits, rf, _, ws = plan(M, N, K)
        if rf:
            assert splits == 1 and ws == 0 and M <= 64 and (bm, bn) == (0, 0)
        else:
            groups = -(-K // 512)
            assert ws == (splits > 1) * -(-M // bm) * -(-N // bn) * bm * bn * 4 * splits
            assert -(-groups // -(-groups // splits)) == splits      # no split without K
        _, _, _, rf, n, _ = plan(M, N, K, 0)
        if n:
            fused.add((rf, n))
    assert taken <= FEW | TILES, taken - (FEW | TILES)
    assert fused <= VALUES, fused - VALUES


def test_refusals():
    out = (ctypes.c_int64 * 6)()
    for args in ((0, 1, 128, -1), (1, 0, 128, -1), (1, 1, 128, 3), (1, 1, 128, -2), (1, 1, 96, 0), (1, 1, 0, 0)):
        assert lib().kbn_debug_mxfp4_plan(*args, out) == 1
    assert lib().kbn_debug_mxfp4_plan(1, 1, 128, 0, None) == 1


@pytest.mark.gpu
@pytest.mark.parametrize("M,N,K", MORE)
def test_product_of_the_others(gpu_device, M, N, K):
    from kb_nano_amd import _ops
    print(f"mxfp4 product {M}x{N}x{K}", flush=True)
    a, sa = random_mx((M, K), M + K, gpu_device)
    w, sw = random_mx((N, K), N + K + 1, gpu_device)
    out = torch.full((M + 1, N + 3), float("nan"), dtype=torch.bfloat16, device=gpu_device)
    out[M], out[:, N:] = 5.0, 5.0
    _ops.mxfp4_gemm_nt(a, sa, w, sw, out[:M, :N])
    va = values(a, sa)
    for n in range(0, N, 4096):
        assert_product(out[:M, n:min(n + 4096, N)], va, values(w[n:n + 4096], sw[n:n + 4096]), f"{M}x{N}x{K} from {n}")
    assert bool((out[M] == 5).all() and (out[:, N:] == 5).all())
