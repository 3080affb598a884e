"""The native host path of the MXFP4 and few-token calls against the Python path it stands for: the same
bytes, shapes and strides, and None (so the Python path, which handles the call or refuses it) otherwise."""
import pytest
import torch

from kb_nano_amd import FewTokenExperts, Mxfp4Linear, Mxfp4Quant, _ops, dequantize_mxfp4
from tests._mx_util import random_mx

pytestmark = pytest.mark.gpu
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def _both(monkeypatch, call):
    assert _ops._host is not None, "csrc/host_calls.cpp is not built"
    a = call()
    monkeypatch.setattr(_ops, "_host", None)
    b = call()
    monkeypatch.undo()
    return a, b


def _same(a, b):
    for x, y in zip(a, b, strict=True):
        assert x.dtype == y.dtype and x.shape == y.shape and x.stride() == y.stride()
        assert torch.equal(x.reshape(-1).view(torch.uint8), y.reshape(-1).view(torch.uint8))


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("shape", [(1, 32), (61, 7168), (3, 5, 96), (64,)])
def test_quant_and_back(gpu_device, monkeypatch, shape, dtype):
    g = torch.Generator(device=gpu_device).manual_seed(1)
    x = torch.randn(shape, device=gpu_device, generator=g).to(dtype)
    assert _ops._host.mx_quant(x) is not None
    _same(*_both(monkeypatch, lambda: Mxfp4Quant()(x)))
    c, s = Mxfp4Quant()(x)
    assert _ops._host.mx_dequant(c, s, 1) is not None
    for out in (BF16, F16, F32):
        _same(*_both(monkeypatch, lambda: (dequantize_mxfp4(c, s, out), dequantize_mxfp4(c, s.view(torch.uint8), out))))


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("M", [1, 2, 3, 40, 300])
def test_linear(gpu_device, monkeypatch, M, dtype):
    N, K = 515, 1024
    g = torch.Generator(device=gpu_device).manual_seed(M)
    x = torch.randn(M, K + 64, device=gpu_device, generator=g).to(dtype)[:, :K]
    w, s = random_mx((N, K), 3, gpu_device)
    bias = torch.randn(N, device=gpu_device, generator=g).to(BF16)
    lin = Mxfp4Linear()
    assert _ops._host.mx_linear(x, w, s) is not None
    _same(*_both(monkeypatch, lambda: (lin(x, w, s), lin(x, w, s.view(torch.float8_e8m0fnu), bias),
                                       lin(x.contiguous().view(M, 1, K), w, s))))


@pytest.mark.parametrize("fmt", ["fp8", "mxfp4"])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_experts(gpu_device, monkeypatch, fmt, dtype):
    from tests.test_gpu_few_token_experts import make
    d = make(7, 16, 256, 128, 4, fmt, dtype, 3, gpu_device)
    wide = torch.zeros(7, 512, dtype=dtype, device=gpu_device)
    wide[:, :256] = d["x"]
    layer = FewTokenExperts()

    def call():
        a = (d["w13"], d["w2"], d["tw"])
        b = (16, d["s13"], d["s2"], d["block"])
        return layer(d["x"], *a, d["ids"], *b), layer(wide[:, :256], *a, d["ids"].long(), *b)
    assert _ops._host.few_experts(d["x"], d["w13"], d["s13"], d["w2"], d["s2"], d["tw"], d["ids"]) is not None
    _same(*_both(monkeypatch, call))


def test_anything_but_the_plain_case_is_left_to_python(gpu_device):
    h = _ops._host
    x = torch.randn(4, 256, device=gpu_device).to(BF16)
    c, s = h.mx_quant(x)
    w, sw = random_mx((64, 256), 1, gpu_device)
    assert h.mx_quant(x.cpu()) is None and h.mx_quant(x.double()) is None and h.mx_quant(x[:, :200]) is None
    assert h.mx_quant(x[:0]) is None and h.mx_quant(x.t()) is None and h.mx_quant(x[:, 1:33]) is None   # misaligned: refused
    assert h.mx_dequant(c, s, -1) is None and h.mx_dequant(c, s[:2], 0) is None and h.mx_dequant(c.int(), s, 0) is None
    assert h.mx_linear(x, w[:, :64], sw) is None and h.mx_linear(x, w, sw[:, :4]) is None and h.mx_linear(x, w.t(), sw) is None
    assert h.mx_linear(x[:0], w, sw) is None
    for bad in ([], [x], [x, 1, 2]):
        assert h.mx_linear(*bad) is None
    g = torch.cuda.CUDAGraph()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        with torch.cuda.graph(g, stream=side):
            assert h.mx_quant(x) is None and h.mx_linear(x, w, sw) is None
            y = Mxfp4Linear()(x, w, sw)
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, Mxfp4Linear()(x, w, sw))


def test_refusals_reach_the_caller(gpu_device):
    x = torch.randn(4, 256, device=gpu_device).to(BF16)
    w, sw = random_mx((64, 256), 1, gpu_device)
    lin, quant = Mxfp4Linear(), Mxfp4Quant()
    with pytest.raises(TypeError, match="bfloat16, float16 or float32"):
        quant(x.double())
    with pytest.raises(ValueError, match="multiple of 32"):
        quant(x[:, :200])
    with pytest.raises(RuntimeError, match="16-byte aligned"):
        quant(x[:, 1:33])
    with pytest.raises(ValueError, match="contiguous rows"):
        quant(x.t().contiguous().t())
    with pytest.raises(ValueError, match="multiple of 128"):
        lin(x[:, :64], w[:, :32], sw[:, :2])
    with pytest.raises(ValueError, match="weight codes"):
        lin(x, w[:, :64], sw)
    with pytest.raises(ValueError, match="weight scales"):
        lin(x, w, sw[:, :4])
    with pytest.raises(TypeError, match="weight codes"):
        lin(x, w.int(), sw)
    with pytest.raises(TypeError, match="scales"):
        lin(x, w, sw.float())
    with pytest.raises(RuntimeError, match="same|must be on"):
        lin(x, w.cpu(), sw)
    with pytest.raises(ValueError, match="codes must be|scales must be"):
        dequantize_mxfp4(w, sw[:, :3])
    with pytest.raises(TypeError, match="values must be"):
        dequantize_mxfp4(w, sw, torch.float64)
    from tests.test_gpu_few_token_experts import call, make
    d = make(5, 8, 256, 128, 2, "fp8", BF16, 1, gpu_device)
    many = make(65, 8, 256, 128, 2, "fp8", BF16, 1, gpu_device)
    with pytest.raises(ValueError, match="at most 64"):
        call(d, x=many["x"], ids=many["ids"], tw=many["tw"])
    with pytest.raises(TypeError, match="bfloat16 or float16"):
        call(d, x=d["x"].float())
    with pytest.raises(TypeError, match="topk_weights"):
        call(d, tw=d["tw"].half())
    with pytest.raises(TypeError, match="int32 or int64"):
        call(d, ids=d["ids"].short())
    with pytest.raises(ValueError, match="w2 must be"):
        call(d, w2=d["w2"].transpose(1, 2))
    with pytest.raises(ValueError, match="w13_scale"):
        call(d, s13=d["s13"][:, :1])
    with pytest.raises(ValueError, match="block_shape"):
        call(d, block=[128, 64])
    with pytest.raises(RuntimeError, match="top_k=33"):
        call(d, ids=d["ids"][:, :1].repeat(1, 33), tw=d["tw"][:, :1].repeat(1, 33))


def test_threads_at_once_and_packed_dtype(gpu_device):
    """Calls of several threads on one stream and on their own, and codes as float4_e2m1fn_x2: the bits of
    one call alone."""
    import threading
    from kb_nano_amd import FewTokenExperts, Mxfp4Linear, Mxfp4Quant, dequantize_mxfp4
    print("mxfp4 threads", flush=True)
    quant, lin, few = Mxfp4Quant(), Mxfp4Linear(), FewTokenExperts()
    g = torch.Generator().manual_seed(1)
    x = torch.randn(40, 512, generator=g).bfloat16().to(gpu_device)
    w, sw = quant((torch.randn(4, 512, 512, generator=g) * 0.05).to(gpu_device))
    w13, s13, w2, s2 = w, sw, w[:, :, :128].contiguous(), sw[:, :, :8].contiguous()
    ids = torch.randint(0, 4, (40, 2), generator=g).to(torch.int32).to(gpu_device)
    tw = torch.rand(40, 2, generator=g).to(gpu_device)

    def calls(n):
        return lin(x[:n], w[0], sw[0]), few(x[:n], w13, w2, tw[:n], ids[:n], 4, s13, s2, [1, 32]), *quant(x[:n])

    rows = (1, 7, 30, 40)
    refs = [calls(n) for n in rows]
    f4 = torch.float4_e2m1fn_x2
    assert torch.equal(lin(x, w[0].view(f4), sw[0]), refs[3][0])
    assert torch.equal(dequantize_mxfp4(refs[3][2].view(f4), refs[3][3]), dequantize_mxfp4(refs[3][2], refs[3][3]))
    torch.cuda.synchronize()
    wrong = []

    def work(k, own):
        stream = torch.cuda.Stream() if own else torch.cuda.current_stream()
        with torch.cuda.stream(stream):
            for _ in range(30):
                for a, b in zip(calls(rows[k]), refs[k]):
                    if not torch.equal(a.view(torch.uint8), b.view(torch.uint8)):
                        wrong.append((k, own))

    for own in (False, True):
        threads = [threading.Thread(target=work, args=(k, own)) for k in range(4)]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
    torch.cuda.synchronize()
    assert not wrong, wrong
