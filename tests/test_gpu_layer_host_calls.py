"""The native host path of the router, the gated norms and the adapters against the Python path it stands for:
the same bytes, shapes and strides, and None (so the Python path handles the call or refuses it) otherwise."""
import pytest
import torch

from kb_nano_amd import GatedAddRMSNorm, GatedAddRMSNormFP8Quant, LoraAdd, MoeRouterGemm, MoeRouterTopk, _ops
from tests.test_gpu_lora import args, make
from tests.test_gpu_mx_host_calls import _both, _same

pytestmark = pytest.mark.gpu
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def randn(shape, dtype, seed, dev):
    return torch.randn(shape, device=dev, generator=torch.Generator(device=dev).manual_seed(seed)).to(dtype)


@pytest.mark.parametrize("x_dtype,w_dtype", [(BF16, BF16), (F16, F32), (F32, F32)])
@pytest.mark.parametrize("shape", [(1, 256), (40, 256), (3, 5, 256), (256,)])
def test_router_gemm(gpu_device, monkeypatch, shape, x_dtype, w_dtype):
    x, w = randn(shape, x_dtype, 1, gpu_device), randn((20, 264), w_dtype, 2, gpu_device)[:, :256]
    assert _ops._host.router_gemm(x, w) is not None
    _same(*_both(monkeypatch, lambda: (MoeRouterGemm()(x, w),)))


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("shape", [(1, 64), (40, 64), (3, 5, 64)])
def test_router_topk(gpu_device, monkeypatch, shape, dtype):
    l, bias = randn(shape, dtype, 1, gpu_device), randn(64, F32, 2, gpu_device)
    assert _ops._host.router_topk(l, 4, "softmax", None, 1, 1, True, 1.0, torch.int32) is not None
    topk = MoeRouterTopk()
    _same(*_both(monkeypatch, lambda: (*topk(l, 4), *topk(l, 8, "sigmoid", bias, 8, 4, False, 2, torch.int64))))


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("shape", [(1, 256), (40, 256), (3, 5, 256)])
def test_gated_norm(gpu_device, monkeypatch, shape, dtype):
    x, r, w = randn(shape, dtype, 1, gpu_device), randn(shape, dtype, 2, gpu_device), randn(256, dtype, 3, gpu_device)
    for gate in (None, w, x, x[..., :1].contiguous()):
        assert _ops._host.gated_norm(x, r, w, None, gate, 1.0, 1e-6, True, False) is not None
        for post in (None, w):
            a = (x, r, w, post, gate, 1, 1e-6)
            _same(*_both(monkeypatch, lambda: (*GatedAddRMSNorm()(*a), *GatedAddRMSNormFP8Quant()(*a, with_rows=True))))
    wide = randn((7, 304), dtype, 4, gpu_device)
    a = (wide[:, :256], wide[:, 8:264], w, None, wide[:, 290:291])
    _same(*_both(monkeypatch, lambda: GatedAddRMSNorm()(*a)))


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("T", [1, 30, 200])
def test_lora_add(gpu_device, monkeypatch, T, dtype):
    d = make(T, 130, 264, 4, 16, dtype, 2, gpu_device, pad=8)
    x, base, a, b, ids, s = args(d)
    assert _ops._host.lora_add(x, base, a, b, ids, s) is not None
    c = base.contiguous().view(T, 1, 130)
    _same(*_both(monkeypatch, lambda: (LoraAdd()(x, base, a, b, ids, s), LoraAdd()(x, base, a, b, ids.long()),
                                       LoraAdd()(x.contiguous().view(T, 1, 264), c, a, b, ids.view(T, 1), s))))


def test_anything_but_the_plain_case_is_left_to_python(gpu_device):
    h = _ops._host
    x, w, l = randn((4, 256), BF16, 1, gpu_device), randn((8, 256), BF16, 2, gpu_device), randn((4, 64), F32, 3, gpu_device)
    for bad in ((x.cpu(), w), (x, w.half()), (x.double(), w), (x[:0], w), (x.t(), w), (x[:, :252], w[:, :252]), (x, w[0]), (x, w.cpu()),
                (x[:, 4:252], w[:, :248]), (x,)):
        assert h.router_gemm(*bad) is None
    ok = [l, 4, "softmax", None, 1, 1, True, 1.0, torch.int32]
    assert h.router_topk(*ok) is not None
    for i, v in ((0, l.double()), (0, l[:0]), (0, l.t()), (1, 0), (1, 65), (1, 4.0), (1, 2 ** 70), (2, "tanh"), (2, b"softmax"), (3, l[0].cpu()),
                 (3, l[0, :63]), (3, x[0]), (4, 5), (5, 2), (5, None), (6, 1), (7, "1"), (8, torch.int16), (8, None)):
        assert h.router_topk(*[v if j == i else o for j, o in enumerate(ok)]) is None, (i, v)
    ok = [x, x, x[0], None, None, 1.0, 1e-6, True, True]
    assert h.gated_norm(*ok) is not None
    for i, v in ((0, x.double()), (0, x[:0]), (1, x[:3]), (1, x.float()), (1, x.cpu()), (2, x[0, :128]), (2, x[0].float()), (3, x[0, :8]), (3, 1),
                 (4, x[0, :8]), (4, x.float()), (4, x[:3]), (5, "1"), (6, None)):
        assert h.gated_norm(*[v if j == i else o for j, o in enumerate(ok)]) is None, (i, v)
    assert h.gated_norm(*ok[:7], False, False) is None
    d = make(4, 64, 256, 3, 16, BF16, 2, gpu_device)
    ok = list(args(d))
    assert h.lora_add(*ok) is not None
    for i, v in ((0, ok[0].float()), (0, ok[0][:3]), (0, ok[0][:, :128]), (1, ok[1].half()), (1, ok[1][:0]), (2, ok[2][:, :12]), (2, ok[2][0]),
                 (3, ok[3][:2]), (3, ok[3].half()), (4, ok[4][:3]), (4, ok[4].to(torch.int16)), (4, ok[4].cpu()), (5, ok[5][:2]), (5, 1.0)):
        assert h.lora_add(*[v if j == i else o for j, o in enumerate(ok)]) is None, (i, v)
    g = torch.cuda.CUDAGraph()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        with torch.cuda.graph(g, stream=side):
            assert h.router_gemm(x, w) is None and h.lora_add(*ok) is None
            y = MoeRouterGemm()(x, w)
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, MoeRouterGemm()(x, w))
