"""Sizes and strides that the MXFP4 and few-token C entries refuse, before they touch a device."""
import ctypes

from kb_nano_amd._lib import lib

P = ctypes.c_void_p(4096)       # never dereferenced: refused first


def _refused(rc, text):
    assert rc == 1
    assert text in lib().kbn_last_error().decode(), lib().kbn_last_error().decode()


def test_rows_far_apart():
    """A product's operands are read at 32-bit offsets."""
    L, far = lib(), 1 << 23
    for a in range(4):
        ld = [64, 4, 64, 4]
        ld[a] = far
        _refused(L.kbn_mxfp4_gemm_nt(P, ld[0], P, ld[1], P, ld[2], P, ld[3], P, 256, 8, 256, 128, None, 0, None),
                 f"row stride {far} is too large")
    for M, dt in ((2, 0), (4, 1)):
        assert L.kbn_mxfp4_linear_workspace_bytes(M, 256, 128, dt) == 0
        _refused(L.kbn_mxfp4_linear(P, dt, far, P, 64, P, 4, P, 256, M, 256, 128, None, 0, None), "input row stride")
    _refused(L.kbn_few_token_experts(P, 0, 1 << 24, P, P, P, P, 0, P, P, 4, 4, 2, 8, 256, 128, P, 256, P, 1 << 30, None),
             f"input row stride {1 << 24} is too large")


def test_rows_past_32_bits():
    L, many = lib(), (1 << 30) + 1
    for M, N in ((many, 256), (8, many), ((1 << 31) - 1, 256)):
        _refused(L.kbn_mxfp4_gemm_nt(P, 64, P, 4, P, 64, P, 4, P, N, M, N, 128, P, 1 << 60, None), "bad size")
        _refused(L.kbn_mxfp4_linear(P, 0, 128, P, 64, P, 4, P, N, M, N, 128, P, 1 << 60, None), "bad size")
