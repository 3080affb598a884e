"""MXFP4 and few-token calls on rows that lie far apart (the last token of each of some long sequences, a
column of a wide output): the bits of the same rows side by side."""
import pytest
import torch

from tests._mx_util import random_mx

pytestmark = pytest.mark.gpu
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
FAR = (1 << 23) + 64     # elements from row to row


def _far(x, step=FAR, at=8):
    """x's rows `step` elements apart; NaN around them."""
    M, K = x.shape
    b = torch.empty((M - 1) * step + at + K + 8, dtype=x.dtype, device=x.device)
    v = b.as_strided((M, K + 16), (step, 1), at - 8)
    v.fill_(float("nan"))
    v[:, 8:8 + K] = x
    return v[:, 8:8 + K]


def _rows(M, K, dtype, dev):
    return torch.randn(M, K, generator=torch.Generator().manual_seed(M + K)).to(dtype).to(dev)


def _same(a, b):
    return torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8))


@pytest.mark.parametrize("dtype,step", [(BF16, FAR), (F16, FAR), (F32, FAR), (BF16, (1 << 30) + 64)])
def test_quant_and_back(gpu_device, dtype, step):
    from kb_nano_amd import Mxfp4Quant, _ops
    print(f"mxfp4 far rows quant {dtype} {step}", flush=True)
    x = _rows(3, 544, dtype, gpu_device)
    far = _far(x, step)
    quant = Mxfp4Quant()
    c, s = quant(x)
    for a, b in zip(quant(far), (c, s)):
        assert _same(a, b)
    wide = _far(torch.zeros_like(x), step)
    _ops.mxfp4_dequant(c, s, wide)
    ref = torch.empty_like(x)
    _ops.mxfp4_dequant(c, s, ref)
    assert _same(wide, ref)
    fc = torch.empty(2 * step + 400, dtype=torch.uint8, device=gpu_device).as_strided((3, 272), (step, 1), 16)
    _ops.mxfp4_quant(x, fc, s)
    assert _same(fc, c)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("M", [2, 7, 20, 70])
def test_linear(gpu_device, M, dtype):
    """Quantized by the product's launch (2 and 7 rows of 16 bits) or by its own; eager, captured, and into
    an output with rows far apart."""
    from kb_nano_amd import Mxfp4Linear, _ops
    print(f"mxfp4 far rows linear M={M} {dtype}", flush=True)
    N, K = 515, 640
    x, (w, sw) = _rows(M, K, dtype, gpu_device), random_mx((N, K), 1, gpu_device)
    far, lin = _far(x), Mxfp4Linear()
    y = lin(x, w, sw)
    assert _same(lin(far, w, sw), y)
    assert _same(lin(far.unsqueeze(1), w, sw).squeeze(1), y)     # [B, 1, K]: x[:, -1:] of a long batch
    wide = _far(torch.zeros(M, N, dtype=BF16, device=gpu_device), FAR + 1)
    _ops.mxfp4_linear(far, w, sw, wide)
    assert _same(wide, y)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        z = lin(far, w, sw)
    for i in range(3):
        far.copy_(x.flip(0) if i % 2 else x)
        g.replay()
        torch.cuda.synchronize()
        assert _same(z, y.flip(0) if i % 2 else y)
        assert _same(lin(x, w, sw), y)


@pytest.mark.parametrize("fmt", ["fp8", "mxfp4"])
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("step", [FAR, (1 << 24) + 64])
def test_experts(gpu_device, step, dtype, fmt):
    from tests.test_gpu_few_token_experts import call, make
    print(f"few-token experts far rows {step} {dtype} {fmt}", flush=True)
    d = make(5, 8, 256, 128, 2, fmt, dtype, 1, gpu_device)
    y = call(d)
    assert _same(call(d, x=_far(d["x"], step)), y)
    from kb_nano_amd import _ops
    wide = _far(torch.zeros_like(y), step)
    _ops.few_token_experts(d["x"], d["w13"], d["s13"], d["w2"], d["s2"], d["tw"], d["ids"], wide)
    assert _same(wide, y)
