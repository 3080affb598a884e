"""MXFP4 on the GPU: quantization and back equal the format's definition bit for
bit; the product and the linear agree with 64-bit sums within the fp32 sums'
and one bf16 rounding's error (tests/_mx_util.py derives the bound)."""
import pytest
import torch

from tests._mx_util import assert_product, quant_plain, random_mx, values

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def _rows(M, K, dtype, seed, dev, wide=False):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(M, K, generator=g)
    if wide:   # groups over the types' range
        lim = 12 if dtype is torch.float16 else 100
        x = x * torch.exp2(torch.randint(-lim, lim, (M, K // 32), generator=g).float()).repeat_interleave(32, 1)
    return x.to(dtype).to(dev)


def _same_quant(x, codes, scales):
    c, s = quant_plain(x.float() if x.dtype is not torch.float32 else x)
    assert torch.equal(scales.view(torch.uint8).cpu(), s)
    assert torch.equal(codes.view(torch.uint8).cpu(), c)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,K", [(1, 32), (1, 7168), (3, 96), (61, 2080), (130, 4096), (700, 288)])
def test_quant_and_back(gpu_device, M, K, dtype):
    from kb_nano_amd import Mxfp4Quant, dequantize_mxfp4
    print(f"mxfp4 quant {M}x{K} {dtype}", flush=True)
    for wide in (False, True):
        x = _rows(M, K, dtype, M + K, gpu_device, wide)
        codes, scales = Mxfp4Quant()(x)
        assert codes.dtype is torch.uint8 and scales.dtype is torch.float8_e8m0fnu
        _same_quant(x, codes, scales)
        ref = values(codes, scales)
        for out in DTYPES:
            assert torch.equal(dequantize_mxfp4(codes, scales, out), ref.to(out)), out


@pytest.mark.parametrize("dtype", DTYPES)
def test_quant_special_values(gpu_device, dtype):
    """Ties and borders of codes and scales, signed zeros, subnormals, the largest numbers, and
    infinities and NaN, which make their own group NaN and no other."""
    from kb_nano_amd import Mxfp4Quant, dequantize_mxfp4
    print(f"mxfp4 special values {dtype}", flush=True)
    fi = torch.finfo(dtype)
    rows = []
    edges = [0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 0.2, 0.3, 0.74, 0.76, 4.9, 5.1, 6.0]
    for top in (6.0, 4.0, 3.5, 6.9, 6.96875, 7.0, 5.0):
        r = torch.tensor([top] + [e for e in edges if e <= top])
        rows.append(torch.cat([r, -r, torch.zeros(32)])[:32])
    rows += [torch.zeros(32), -torch.zeros(32), torch.full((32,), float(fi.max)), torch.full((32,), -float(fi.max))]
    rows += [torch.full((32,), float(fi.tiny)), torch.full((32,), float(fi.smallest_normal) * float(fi.eps)),
             torch.arange(32) * float(fi.smallest_normal) * float(fi.eps)]
    for bad in (float("inf"), float("-inf"), float("nan")):
        r = torch.arange(32.0)
        r[17] = bad
        rows += [r, torch.arange(32.0)]
    # every row at several scales, two groups side by side
    x = torch.cat([torch.stack(rows), torch.stack(rows[::-1])], 1).to(dtype).to(gpu_device)
    codes, scales = Mxfp4Quant()(x)
    _same_quant(x, codes, scales)
    back = dequantize_mxfp4(codes, scales, torch.float32)
    bad = ~torch.isfinite(x.float()).reshape(-1, 32).all(1)
    assert torch.equal(torch.isnan(back).reshape(-1, 32).all(1), bad)
    assert torch.equal(torch.isnan(back).reshape(-1, 32).any(1), bad)


def test_dequant_every_code_and_scale(gpu_device):
    from kb_nano_amd import dequantize_mxfp4
    print("mxfp4 dequant codes x scales", flush=True)
    codes = torch.arange(256, dtype=torch.uint8).repeat(256, 1)
    byte = torch.arange(256, dtype=torch.uint8).view(256, 1).repeat(1, 16)
    codes, byte = codes.to(gpu_device), byte.to(gpu_device)
    ref = values(codes, byte)
    for dtype in DTYPES:
        got = dequantize_mxfp4(codes, byte.view(torch.float8_e8m0fnu), dtype)
        assert torch.equal(torch.isnan(got), torch.isnan(ref))
        keep = ~torch.isnan(ref)
        assert torch.equal(got[keep], ref.to(dtype)[keep]), dtype


def test_strided_rows_and_untouched_rest(gpu_device):
    """Rows of a wider buffer in and out; what lies between and behind them stays."""
    from kb_nano_amd import _ops
    print("mxfp4 strides", flush=True)
    big = _rows(9, 512, torch.bfloat16, 5, gpu_device)
    x = big[1:8, 64:64 + 320]
    codes = torch.full((8, 200), 7, dtype=torch.uint8, device=gpu_device)
    scales = torch.full((8, 23), 9, dtype=torch.uint8, device=gpu_device)
    _ops.mxfp4_quant(x, codes[:7, 8:168], scales[:7, 3:13])
    _same_quant(x, codes[:7, 8:168].contiguous(), scales[:7, 3:13].contiguous())
    assert bool((codes[7] == 7).all() and (codes[:, :8] == 7).all() and (codes[:, 168:] == 7).all())
    assert bool((scales[7] == 9).all() and (scales[:, :3] == 9).all() and (scales[:, 13:] == 9).all())
    out = torch.full((8, 400), -3.0, dtype=torch.float16, device=gpu_device)
    _ops.mxfp4_dequant(codes[:7, 8:168], scales[:7, 3:13], out[:7, 16:336])
    assert torch.equal(out[:7, 16:336], values(codes[:7, 8:168].contiguous(), scales[:7, 3:13].contiguous()).half())
    assert bool((out[7] == -3).all() and (out[:, :16] == -3).all() and (out[:, 336:] == -3).all())


# rows from one token over every tile height's edges; widths odd, below a tile and past several
SHAPES = [(1, 1, 128), (1, 7, 256), (1, 515, 1152), (2, 128, 128), (5, 100, 640), (15, 16, 384), (16, 4096, 512),
          (17, 33, 256), (31, 2050, 896), (33, 130, 1024), (63, 257, 2048), (64, 2048, 2048), (65, 64, 128),
          (100, 515, 768), (127, 1000, 384), (128, 128, 1280), (129, 385, 512), (200, 1030, 4096), (255, 512, 256),
          (257, 770, 640), (513, 300, 128), (777, 1153, 1024), (1025, 2051, 384)]


@pytest.mark.parametrize("M,N,K", SHAPES)
def test_product(gpu_device, M, N, K):
    from kb_nano_amd import _ops
    print(f"mxfp4 product {M}x{N}x{K}", flush=True)
    a, sa = random_mx((M, K), M + K, gpu_device)
    w, sw = random_mx((N, K), N + K + 1, gpu_device)
    out = torch.full((M + 1, N + 3), float("nan"), dtype=torch.bfloat16, device=gpu_device)
    out[M], out[:, N:] = 5.0, 5.0
    _ops.mxfp4_gemm_nt(a, sa, w, sw, out[:M, :N])
    assert_product(out[:M, :N], values(a, sa), values(w, sw), f"{M}x{N}x{K}")
    assert bool((out[M] == 5).all() and (out[:, N:] == 5).all())   # nothing past the output
    again = torch.empty(M, N, dtype=torch.bfloat16, device=gpu_device)
    _ops.mxfp4_gemm_nt(a, sa, w, sw, again)
    assert torch.equal(again, out[:M, :N])                         # the same bits every time, aligned rows or not


@pytest.mark.parametrize("M,N,K", [(1, 36864, 7168), (8, 8192, 28672), (48, 7168, 16384), (300, 7168, 18432),
                                   (2048, 4608, 7168)])
def test_product_of_real_layers(gpu_device, M, N, K):
    from kb_nano_amd import _ops
    print(f"mxfp4 product {M}x{N}x{K}", flush=True)
    a, sa = random_mx((M, K), 3, gpu_device)
    w, sw = random_mx((N, K), 4, gpu_device)
    out = torch.empty(M, N, dtype=torch.bfloat16, device=gpu_device)
    _ops.mxfp4_gemm_nt(a, sa, w, sw, out)
    va = values(a, sa)
    for n in range(0, N, 2048):
        assert_product(out[:, n:n + 2048], va, values(w[n:n + 2048], sw[n:n + 2048]), f"{M}x{N}x{K} from {n}")


@pytest.mark.parametrize("M", [3, 40, 300])
def test_product_strides_and_special_scales(gpu_device, M):
    """Operands inside wider buffers; a NaN group in a row of either operand makes that row's (column's)
    outputs NaN and no others; scales of 2^-127."""
    from kb_nano_amd import _ops
    N, K = 200, 512
    print(f"mxfp4 product strides M={M}", flush=True)
    a, sa = random_mx((M, 1024), 1, gpu_device)
    w, sw = random_mx((N, 2048), 2, gpu_device)
    a, sa, w, sw = a[:, 16:16 + K // 2], sa[:, 4:4 + K // 32], w[:, 32:32 + K // 2], sw[:, 8:8 + K // 32]
    for nan in (False, True):
        if nan:
            sa[M // 2, 3], sw[N // 3, 5], sw[N - 1, 0] = 255, 255, 255
            sa[0, 1], sw[1, 2] = 0, 0
        out = torch.empty(M, N, dtype=torch.bfloat16, device=gpu_device)
        _ops.mxfp4_gemm_nt(a, sa, w, sw, out)
        assert_product(out, values(a.contiguous(), sa.contiguous()), values(w.contiguous(), sw.contiguous()), f"M={M}")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,N,K", [(1, 1000, 1024), (2, 64, 128), (9, 515, 384), (16, 2048, 2048), (17, 130, 640),
                                   (50, 777, 512), (130, 256, 1152), (300, 900, 1024)])
def test_linear_is_quant_then_product(gpu_device, M, N, K, dtype):
    from kb_nano_amd import Mxfp4Linear, Mxfp4Quant, _ops
    print(f"mxfp4 linear {M}x{N}x{K} {dtype}", flush=True)
    x = _rows(M, K, dtype, M, gpu_device, wide=dtype is torch.float32)
    w, sw = random_mx((N, K), 4, gpu_device)
    y = Mxfp4Linear()(x, w, sw.view(torch.float8_e8m0fnu))
    codes, scales = Mxfp4Quant()(x)
    assert y.dtype is torch.bfloat16 and y.shape == (M, N)
    assert_product(y, values(codes, scales), values(w, sw), f"{M}x{N}x{K}")
    ref = torch.empty_like(y)
    _ops.mxfp4_gemm_nt(codes, scales, w, sw, ref)
    assert torch.equal(y, ref)


def test_linear_module(gpu_device):
    """Leading dimensions, bias, no rows at all, rows of a wider buffer, a non-finite activation (its own row
    only), a single row with a stride of its own, and torch.compile."""
    from kb_nano_amd import Mxfp4Linear, Mxfp4Quant, dequantize_mxfp4
    print("mxfp4 linear module", flush=True)
    N, K = 96, 256
    lin, quant = Mxfp4Linear(), Mxfp4Quant()
    w, sw = quant(_rows(N, K, torch.float32, 1, gpu_device) * 0.02)
    x = _rows(12, K, torch.bfloat16, 2, gpu_device)
    bias = _rows(1, N, torch.bfloat16, 3, gpu_device)[0]
    y = lin(x, w, sw)
    assert torch.equal(lin(x.view(3, 4, K), w, sw, bias), (y + bias).view(3, 4, N))
    assert torch.equal(lin(x[0], w, sw), y[0])
    assert lin(x[:0], w, sw).shape == (0, N) and quant(x[:0])[0].shape == (0, K // 2)
    wide = torch.zeros(12, 2 * K, dtype=torch.bfloat16, device=gpu_device)
    wide[:, K:] = x
    assert torch.equal(lin(wide[:, K:], w, sw), y)
    assert torch.equal(lin(x[:1].t().contiguous().t(), w, sw), y[:1])
    bad = x.clone()
    bad[5, 7] = float("inf")
    z = lin(bad, w, sw)
    assert bool(torch.isnan(z[5]).all()) and torch.equal(z[:5], y[:5]) and torch.equal(z[6:], y[6:])
    e, s3 = quant(torch.stack([dequantize_mxfp4(w, sw)] * 2))      # a batch of weights; exact values stay
    assert e.shape == (2, N, K // 2) and torch.equal(e[1], w) and torch.equal(s3[0].view(torch.uint8), sw.view(torch.uint8))
    torch._dynamo.reset()
    f = torch.compile(lambda a: dequantize_mxfp4(*quant(lin(a, w, sw, bias))), fullgraph=True, backend="aot_eager")
    assert torch.equal(f(x), dequantize_mxfp4(*quant(lin(x, w, sw, bias))))


@pytest.mark.parametrize("M", [1, 30, 200])
def test_linear_graph_and_streams(gpu_device, M):
    """Captured calls replayed on new inputs with eager ones between, two graphs that share inputs, and
    calls on two streams at once give the eager bits."""
    from kb_nano_amd import Mxfp4Linear
    print(f"mxfp4 graphs M={M}", flush=True)
    N, K = 640, 2048
    lin = Mxfp4Linear()
    w, sw = random_mx((N, K), 8, gpu_device)
    xs = [_rows(M, K, torch.bfloat16, 10 + i, gpu_device) for i in range(4)]
    refs = [lin(x, w, sw).clone() for x in xs]
    x = xs[0].clone()
    graphs = []
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=side):
                y = lin(x, w, sw)
                y2 = lin(x, w, sw)
            graphs.append((g, y, y2))
    torch.cuda.synchronize()
    for i in range(4):
        x.copy_(xs[i])
        for g, y, y2 in graphs:
            g.replay()
            eager = lin(xs[(i + 1) % 4], w, sw)
        torch.cuda.synchronize()
        assert torch.equal(eager, refs[(i + 1) % 4])
        for g, y, y2 in graphs:
            assert torch.equal(y, refs[i]) and torch.equal(y2, refs[i])
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    for i in range(8):
        with torch.cuda.stream(streams[i % 2]):
            outs.append(lin(xs[i % 4], w, sw))
    torch.cuda.synchronize()
    assert all(torch.equal(o, refs[i % 4]) for i, o in enumerate(outs))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,K", [(1153, 8192), (4611, 2080), (131073, 96)])
def test_quant_of_many_rows(gpu_device, M, K, dtype):
    """Rows in numbers that no group of rows divides, inside wider buffers, with a NaN in the last row."""
    from kb_nano_amd import _ops
    print(f"mxfp4 quant {M}x{K} {dtype}", flush=True)
    x = torch.zeros(M, K + 64, dtype=dtype, device=gpu_device)
    x[:, 8:8 + K] = torch.randn(M, K, generator=torch.Generator(gpu_device).manual_seed(M), device=gpu_device)
    x = x[:, 8:8 + K]
    x[M - 1, 40] = float("nan")
    codes = torch.full((M + 1, K // 2 + 8), 7, dtype=torch.uint8, device=gpu_device)
    scales = torch.full((M + 1, K // 32 + 3), 9, dtype=torch.uint8, device=gpu_device)
    _ops.mxfp4_quant(x, codes[:M, :K // 2], scales[:M, :K // 32])
    rows = torch.cat((torch.arange(0, 64), torch.arange(M - 64, M)))
    _same_quant(x[rows], codes[rows, :K // 2].contiguous(), scales[rows, :K // 32].contiguous())
    small = [torch.empty(512, n, dtype=torch.uint8, device=gpu_device) for n in (K // 2, K // 32)]
    for at in range(0, M, 512):   # the same bits as in small calls
        n = min(512, M - at)
        _ops.mxfp4_quant(x[at:at + n], small[0][:n], small[1][:n])
        assert torch.equal(codes[at:at + n, :K // 2], small[0][:n]) and torch.equal(scales[at:at + n, :K // 32], small[1][:n])
    assert bool((codes[M] == 7).all() and (codes[:, K // 2:] == 7).all())
    assert bool((scales[M] == 9).all() and (scales[:, K // 32:] == 9).all())
