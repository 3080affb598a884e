"""MXFP4 and the few-token experts layer without a GPU: the entry points refuse bad arguments before they
touch a device, and the host layer's checks and tracing."""
import ctypes

import pytest
import torch

from tests._mx_util import quant_plain, values

P = ctypes.c_void_p(4096)       # never dereferenced: refused first
ODD = ctypes.c_void_p(4098)


def _lib():
    from kb_nano_amd._lib import lib
    return lib()


def _refused(rc, text):
    assert rc == 1
    assert text in _lib().kbn_last_error().decode(), _lib().kbn_last_error().decode()


def test_quant_refusals():
    L = _lib()
    _refused(L.kbn_mxfp4_quant(P, 3, 4, 64, 64, P, 32, P, 2, None), "dtype code 3")
    _refused(L.kbn_mxfp4_quant(P, 0, 4, 48, 48, P, 32, P, 2, None), "multiple of 32")
    _refused(L.kbn_mxfp4_quant(P, 0, -1, 64, 64, P, 32, P, 2, None), "bad size")
    _refused(L.kbn_mxfp4_quant(P, 0, 4, 64, 60, P, 32, P, 2, None), "input row stride")
    _refused(L.kbn_mxfp4_quant(P, 0, 4, 64, 68, P, 32, P, 2, None), "input row stride")
    _refused(L.kbn_mxfp4_quant(ODD, 0, 4, 64, 64, P, 32, P, 2, None), "input must be 16-byte aligned")
    _refused(L.kbn_mxfp4_quant(None, 0, 4, 64, 64, P, 32, P, 2, None), "input must be")
    _refused(L.kbn_mxfp4_quant(P, 0, 4, 64, 64, P, 34, P, 2, None), "codes row stride")
    _refused(L.kbn_mxfp4_quant(P, 0, 4, 64, 64, ODD, 32, P, 2, None), "codes must be")
    _refused(L.kbn_mxfp4_quant(P, 0, 4, 64, 64, P, 32, P, 1, None), "scales row stride")
    _refused(L.kbn_mxfp4_quant(P, 0, 4, 64, 64, P, 32, None, 2, None), "scales must be")
    _refused(L.kbn_mxfp4_dequant(P, 32, P, 2, 4, 64, P, 9, 64, None), "dtype code 9")
    _refused(L.kbn_mxfp4_dequant(P, 32, P, 2, 4, 64, P, 0, 63, None), "output row stride")
    assert L.kbn_mxfp4_quant(None, 0, 0, 64, 64, None, 32, None, 2, None) == 0
    assert L.kbn_mxfp4_dequant(None, 32, None, 2, 4, 0, None, 0, 64, None) == 0


def test_product_refusals():
    L = _lib()

    def gemm(A=P, lda=64, sA=P, lsa=4, W=P, ldw=64, sW=P, lsw=4, D=P, ldd=256, M=8, N=256, K=128, ws=None, n=0):
        return L.kbn_mxfp4_gemm_nt(A, lda, sA, lsa, W, ldw, sW, lsw, D, ldd, M, N, K, ws, n, None)

    _refused(gemm(K=96), "multiple of 128")
    _refused(gemm(K=0), "bad size")
    _refused(gemm(M=-1), "bad size")
    _refused(gemm(N=1 << 31), "bad size")
    _refused(gemm(lda=48), "A row stride")
    _refused(gemm(lda=72), "A row stride")
    _refused(gemm(A=ctypes.c_void_p(4104)), "A must be 16-byte aligned")
    _refused(gemm(ldw=32), "W row stride")
    _refused(gemm(W=None), "W must be")
    _refused(gemm(lsa=6), "A scales row stride")
    _refused(gemm(sA=ODD), "A scales must be 4-byte aligned")
    _refused(gemm(lsw=3), "W scales row stride")
    _refused(gemm(ldd=255), "output row stride")
    _refused(gemm(D=None), "output must be")
    assert gemm(M=0, A=None) == 0 and gemm(N=0, W=None, ldd=0) == 0
    for M, N, K in ((128, 7168, 18432), (8, 8192, 8192), (300, 256, 16384)):
        need = L.kbn_mxfp4_gemm_nt_workspace_bytes(M, N, K)
        assert need >= 0 and need % 16 == 0
        if need:
            _refused(gemm(M=M, N=N, K=K, lda=K // 2, lsa=K // 32, ldw=K // 2, lsw=K // 32, ldd=N, ws=P, n=need - 1),
                     "workspace")

    def linear(x=P, dt=0, ldx=128, W=P, ldw=64, sW=P, lsw=4, D=P, ldd=256, M=100, N=256, K=128, ws=P, n=1 << 30):
        return L.kbn_mxfp4_linear(x, dt, ldx, W, ldw, sW, lsw, D, ldd, M, N, K, ws, n, None)

    _refused(linear(dt=5), "dtype code 5")
    _refused(linear(K=64), "multiple of 128")
    _refused(linear(ldx=127), "input row stride")
    _refused(linear(x=ODD), "input must be")
    _refused(linear(ldw=60), "W row stride")
    _refused(linear(sW=ODD), "W scales must be")
    _refused(linear(n=0), "workspace")
    _refused(linear(ws=ctypes.c_void_p(4104)), "workspace")
    assert linear(M=0, x=None, ws=None, n=0) == 0


def test_experts_refusals():
    L = _lib()

    def experts(x=P, dt=0, ldx=256, w13=P, s13=P, w2=P, s2=P, fmt=0, tw=P, ids=P, idb=4, T=4, topk=2, E=8, H=256, I=128,
                out=P, ldo=256, ws=P, n=1 << 30):
        return L.kbn_few_token_experts(x, dt, ldx, w13, s13, w2, s2, fmt, tw, ids, idb, T, topk, E, H, I, out, ldo, ws, n, None)

    _refused(experts(dt=2), "dtype code 2")
    _refused(experts(fmt=2), "weight format 2")
    _refused(experts(idb=2), "ids of 2 bytes")
    _refused(experts(T=65), "at most 64")
    _refused(experts(T=-1), "at most 64")
    _refused(experts(topk=0), "top_k=0")
    _refused(experts(topk=33), "top_k=33")
    _refused(experts(E=0), "num_experts=0")
    _refused(experts(E=1025), "num_experts=1025")
    _refused(experts(H=192), "multiples of 128")
    _refused(experts(I=64), "multiples of 128")
    _refused(experts(ldx=248), "input rows")
    _refused(experts(ldx=260), "input rows")
    _refused(experts(x=ODD), "input rows")
    _refused(experts(ldo=128), "output row stride")
    _refused(experts(out=None), "output")
    _refused(experts(w13=None), "null")
    _refused(experts(ids=None), "null")
    _refused(experts(w2=ODD), "weights must be 16-byte aligned")
    _refused(experts(s2=ODD), "scales must be 4-byte aligned")
    need = L.kbn_few_token_experts_workspace_bytes(4, 2, 128)
    assert need > 0
    _refused(experts(n=need - 1), "workspace")
    _refused(experts(ws=None), "workspace")
    assert experts(T=0, x=None, out=None, ws=None, n=0) == 0


def test_host_layer_refuses_cpu_tensors_and_bad_shapes():
    from kb_nano_amd import FewTokenExperts, Mxfp4Linear, Mxfp4Quant, dequantize_mxfp4
    u8, e8 = torch.uint8, torch.float8_e8m0fnu
    with pytest.raises(RuntimeError, match="no CPU path"):
        Mxfp4Quant()(torch.zeros(2, 64))
    with pytest.raises(RuntimeError, match="no CPU path"):
        dequantize_mxfp4(torch.zeros(2, 32, dtype=u8), torch.zeros(2, 2, dtype=u8))
    with pytest.raises(RuntimeError, match="no CPU path"):
        Mxfp4Linear()(torch.zeros(2, 128), torch.zeros(8, 64, dtype=u8), torch.zeros(8, 4, dtype=u8).view(e8))
    layer = FewTokenExperts()
    w13, w2 = torch.zeros(4, 256, 128, dtype=torch.float8_e4m3fn), torch.zeros(4, 128, 128, dtype=torch.float8_e4m3fn)
    x, tw, ids = torch.zeros(2, 128).bfloat16(), torch.zeros(2, 2), torch.zeros(2, 2, dtype=torch.int32)
    s13, s2 = torch.zeros(4, 2, 1), torch.zeros(4, 1, 1)
    with pytest.raises(RuntimeError, match="no CPU path"):
        layer(x, w13, w2, tw, ids, 4, s13, s2, [128, 128])
    with pytest.raises(ValueError, match="block_shape"):
        layer(x, w13, w2, tw, ids, 4, s13, s2, [1, 32])
    with pytest.raises(ValueError, match="num_experts"):
        layer(x, w13, w2, tw, ids, 5, s13, s2, [128, 128])


def test_ops_trace_without_a_device():
    from torch._subclasses.fake_tensor import FakeTensorMode

    from kb_nano_amd import FewTokenExperts, Mxfp4Linear, Mxfp4Quant, dequantize_mxfp4  # noqa: F401  (registers the ops)
    with FakeTensorMode():
        x = torch.empty(4, 256, device="meta", dtype=torch.bfloat16)
        c, s = torch.empty(4, 128, device="meta", dtype=torch.uint8), torch.empty(4, 8, device="meta", dtype=torch.uint8)
        torch.ops.kb_nano_mxfp4.quant(x, c, s)
        torch.ops.kb_nano_mxfp4.dequant(c, s, x)
        torch.ops.kb_nano_mxfp4.gemm_nt(c, s, c, s, torch.empty(4, 4, device="meta", dtype=torch.bfloat16))
        torch.ops.kb_nano_mxfp4.linear(x, c, s, torch.empty(4, 4, device="meta", dtype=torch.bfloat16))
        torch.ops.kb_nano_fp8_moe.few_token_experts(x, c, s, c, s, x, c, x)


def test_plain_quantization_is_the_nearest():
    """The tests' own reference: no other code is nearer, the top of each group lies in [3.5, 7) scales, and
    one code's spacing there bounds the error."""
    g = torch.Generator().manual_seed(0)
    x = torch.randn(64, 128, generator=g) * torch.exp2(torch.randint(-40, 40, (64, 1), generator=g).float())
    codes, byte = quant_plain(x)
    v, s = values(codes, byte), torch.exp2(byte.double() - 127).repeat_interleave(32, 1)
    top = (x.double().abs() / s).reshape(-1, 32).amax(1)
    assert bool(((top >= 3.5) & (top < 7)).all())
    every = torch.tensor([0.0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64)
    best = (x.double().abs().unsqueeze(-1) / s.unsqueeze(-1) - every).abs().amin(-1)
    assert torch.equal((v - x.double()).abs() / s, best)
    assert float(best.max()) <= 1.0


def test_dequantize_refuses_other_rows():
    """As many rows in another arrangement are other rows."""
    from kb_nano_amd import dequantize_mxfp4
    for shape in ((3, 2, 2), (6, 2), (2, 4, 2)):
        with pytest.raises(ValueError, match="other rows"):
            dequantize_mxfp4(torch.zeros(2, 3, 32, dtype=torch.uint8), torch.zeros(shape, dtype=torch.uint8))
