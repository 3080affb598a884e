"""The MXFP4 product at a shape for each tile, split count and few-rows variant,
what lies behind K in wider buffers, and sizes past 32-bit offsets."""
import pytest
import torch

from tests._mx_util import assert_product, random_mx, values

pytestmark = pytest.mark.gpu

# odd widths and K that ends inside a stage (256), a pair (512) or a scale chunk (1024)
SHAPES = [(17, 67, 640), (33, 65, 640), (51, 67, 1152), (17, 4141, 640), (34, 4183, 1152), (49, 4331, 1152),   # few rows:
          (18, 8295, 1664), (35, 8213, 1664), (16, 8195, 1408), (1, 8209, 1152), (54, 8235, 1664),   # 16, 32, 48
          (2, 12305, 640), (17, 12841, 1664), (34, 12677, 1664), (64, 9001, 2176),        # and 64 wide
          # 64 x 64, 64 x 128, 128 x 128, 128 x 256 and 256 x 256 in 1 to 4 splits
          (65, 130, 2176), (2858, 67, 7808), (75, 67, 4352), (75, 67, 3712), (74, 67, 3200), (2930, 65, 6784), (2765, 73, 7296),
          (17, 16627, 128), (129, 24579, 1152), (17, 8227, 18432), (2793, 65, 11904),
          (1025, 2051, 640), (65, 16571, 1152), (1100, 2050, 2432), (65, 16401, 8832), (139, 11375, 12032), (3714, 261, 16256),
          (2143, 449, 7296), (3637, 131, 17280),
          (258, 13153, 128), (816, 5399, 16000), (3300, 1185, 10368), (2704, 907, 19072), (66, 17429, 12160), (69, 11363, 13440),
          (913, 12331, 640), (3410, 2319, 1408), (129, 17445, 22912)]


@pytest.mark.parametrize("M,N,K", SHAPES)
def test_product_by_every_variant(gpu_device, M, N, K):
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


@pytest.mark.parametrize("K", [128, 384, 640, 1152, 1664])
@pytest.mark.parametrize("M,N", [(1, 48), (20, 100), (65, 130), (140, 17000), (1100, 8300)])
def test_nothing_behind_k_counts(gpu_device, M, N, K):
    """Rows inside wider buffers whose other bytes are NaN scales and codes of 6."""
    from kb_nano_amd import Mxfp4Linear, _ops
    print(f"mxfp4 product {M}x{N}x{K} in wider rows", flush=True)

    def wide(rows, seed):
        c, s = random_mx((rows, K), seed, gpu_device)
        cw = torch.full((rows + 1, K // 2 + 160), 0x77, dtype=torch.uint8, device=gpu_device)
        sw = torch.full((rows + 1, K // 32 + 40), 255, dtype=torch.uint8, device=gpu_device)
        cw[:rows, 16:16 + K // 2], sw[:rows, 4:4 + K // 32] = c, s
        return cw[:rows, 16:16 + K // 2], sw[:rows, 4:4 + K // 32], c, s

    a, sa, ac, sac = wide(M, 1)
    w, sw, wc, swc = wide(N, 2)
    out, ref = (torch.empty(M, N, dtype=torch.bfloat16, device=gpu_device) for _ in range(2))
    _ops.mxfp4_gemm_nt(a, sa, w, sw, out)
    _ops.mxfp4_gemm_nt(ac, sac, wc, swc, ref)
    assert torch.equal(out, ref)
    for n in range(0, N, 4096):
        assert_product(out[:, n:min(n + 4096, N)], values(ac, sac), values(wc[n:n + 4096], swc[n:n + 4096]), f"{M}x{N}x{K}")
    x = torch.full((M, K + 64), float("nan"), dtype=torch.bfloat16, device=gpu_device)
    x[:, 8:8 + K] = torch.randn(M, K, generator=torch.Generator().manual_seed(3)).to(torch.bfloat16).to(gpu_device)
    lin = Mxfp4Linear()
    assert torch.equal(lin(x[:, 8:8 + K], w, sw), lin(x[:, 8:8 + K].contiguous(), wc, swc))


def test_past_32_bit_offsets(gpu_device):
    """Values, outputs and weight bytes past 2^31: the last rows and columns agree with the formulas."""
    from kb_nano_amd import Mxfp4Quant, _ops, dequantize_mxfp4
    print("mxfp4 past 32 bits", flush=True)
    M, K = 70001, 32768
    x = torch.ones(M, K, dtype=torch.bfloat16, device=gpu_device)
    x[-1] = torch.arange(K, device=gpu_device) % 7 - 3
    codes, scales = Mxfp4Quant()(x)
    tail_c, tail_s = Mxfp4Quant()(x[-2:].contiguous())
    assert torch.equal(codes[-2:], tail_c) and torch.equal(scales[-2:].view(torch.uint8), tail_s.view(torch.uint8))
    assert torch.equal(dequantize_mxfp4(codes, scales)[-2:], x[-2:])
    del x
    N = 128 * 512
    w, sw = random_mx((N, 128), 5, gpu_device)
    a, sa = codes[:, :64], scales[:, :4]
    out = torch.empty(M, N, dtype=torch.bfloat16, device=gpu_device)
    _ops.mxfp4_gemm_nt(a, sa, w, sw, out)
    for rows in (slice(0, 64), slice(M - 64, M)):
        assert_product(out[rows], values(a[rows], sa[rows]), values(w, sw), f"rows {rows}")
    del out
    # the codes as a weight of 1.1 GB and scales, many rows; then one of 2.3 GB
    w2 = torch.cat((codes, codes))
    s2 = torch.cat((scales.view(torch.uint8), scales.view(torch.uint8)))
    for m in (1, 20, 70):
        a, sa = random_mx((m, K), m, gpu_device)
        out = torch.empty(m, 2 * M, dtype=torch.bfloat16, device=gpu_device)
        _ops.mxfp4_gemm_nt(a, sa, w2, s2, out)
        assert_product(out[:, -64:], values(a, sa), values(w2[-64:], s2[-64:]), f"{m} rows, a weight of 2.3 GB")
        assert_product(out[:, :64], values(a, sa), values(w2[:64], s2[:64]), f"{m} rows, a weight of 2.3 GB")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("M", [*range(1, 10), 13, 16, 17])
@pytest.mark.parametrize("N,K", [(67, 128), (515, 1152), (4357, 640), (9001, 1408), (12999, 384)])
def test_linear_of_few_rows(gpu_device, M, N, K, dtype):
    """One launch or two: the bits of the quantization and the product apart, in strided rows, with values
    over the type's range and a NaN that makes its own row NaN."""
    from kb_nano_amd import Mxfp4Linear, Mxfp4Quant, _ops
    print(f"mxfp4 linear {M}x{N}x{K} {dtype}", flush=True)
    g = torch.Generator().manual_seed(M)
    lim = 8 if dtype is torch.float16 else 30
    x = torch.randn(M, K, generator=g) * torch.exp2(torch.randint(-lim, lim, (M, K // 32), generator=g).float()).repeat_interleave(32, 1)
    wide = torch.full((M, K + 24), float("nan"), dtype=dtype, device=gpu_device)
    wide[:, 16:16 + K] = x.to(dtype).to(gpu_device)
    x = wide[:, 16:16 + K]
    w, sw = random_mx((N, K), 4, gpu_device)
    for nan in (False, True):
        if nan:
            x[M - 1, K - 1] = float("nan")
        y = Mxfp4Linear()(x, w, sw)
        codes, scales = Mxfp4Quant()(x)
        ref = torch.empty_like(y)
        _ops.mxfp4_gemm_nt(codes, scales, w, sw, ref)
        assert_product(y, values(codes, scales), values(w, sw), f"{M}x{N}x{K}")
        assert torch.equal(y.view(torch.int16), ref.view(torch.int16)) or (nan and torch.equal(y[:-1], ref[:-1]))
