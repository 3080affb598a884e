"""The C entries of the router, the gated norms and the adapters refuse before any device call (no GPU needed)."""
import ctypes

import pytest

P = ctypes.c_void_p(4096)   # never dereferenced
ODD = ctypes.c_void_p(4098)


def refused(rc, words):
    from kb_nano_amd._lib import lib
    msg = lib().kbn_last_error().decode()
    assert rc == 1 and words in msg, (rc, msg)


GEMM = dict(x=P, xd=0, ldx=256, w=P, wd=0, ldw=256, out=P, ldo=8, T=4, E=8, H=256, ws=None, wsb=0)


@pytest.mark.parametrize("over,words", [
    (dict(xd=3), "dtype codes"), (dict(wd=1), "rows' dtype"), (dict(xd=2), "rows' dtype"), (dict(H=252), "multiple of 8"),
    (dict(H=0), "multiple of 8"), (dict(E=0), "bad sizes"), (dict(T=-1), "bad sizes"), (dict(x=None), "null"), (dict(out=None), "null"),
    (dict(x=ODD), "16-byte"), (dict(ldx=248), "16-byte"), (dict(ldw=260), "16-byte"), (dict(ldx=1 << 23), "2^23"), (dict(ldo=7), "output rows"),
    (dict(T=20, H=4096, ldx=4096, ldw=4096), "workspace"), (dict(T=20, H=4096, ldx=4096, ldw=4096, ws=P, wsb=16), "workspace")])
def test_router_gemm(over, words):
    from kb_nano_amd._lib import lib
    a = {**GEMM, **over}
    refused(lib().kbn_moe_router_gemm(a["x"], a["xd"], a["ldx"], a["w"], a["wd"], a["ldw"], a["out"], a["ldo"], a["T"], a["E"], a["H"],
                                      a["ws"], a["wsb"], None), words)


TOPK = dict(l=P, d=2, ld=64, bias=None, T=4, E=64, k=4, sig=0, G=1, kept=1, renorm=1, w=P, ids=P, b=4)


@pytest.mark.parametrize("over,words", [
    (dict(d=3), "dtype code"), (dict(b=2), "ids of 2"), (dict(E=0), "outside"), (dict(E=1025, ld=1025), "outside"), (dict(G=5), "divide"),
    (dict(G=0), "divide"), (dict(G=65, E=65, ld=65), "at most 64"), (dict(kept=2), "topk_groups"), (dict(kept=0), "topk_groups"),
    (dict(k=0), "top_k"), (dict(k=65), "top_k"), (dict(G=16, kept=1, k=5), "top_k"), (dict(ld=63), "row stride"), (dict(l=None), "null"),
    (dict(T=-1), "bad T")])
def test_router_topk(over, words):
    from kb_nano_amd._lib import lib
    a = {**TOPK, **over}
    refused(lib().kbn_moe_router_topk(a["l"], a["d"], a["ld"], a["bias"], a["T"], a["E"], a["k"], a["sig"], a["G"], a["kept"], a["renorm"], 1.0,
                                      a["w"], a["ids"], a["b"], None), words)


NORM = dict(x=P, d=0, ldx=256, r=P, ldr=256, w=P, post=None, g=None, gr=0, gc=0, T=4, H=256, ro=P, ldro=256, n=P, ldn=256, q=None, ldq=0,
            s=None, sm=1, sg=4)


@pytest.mark.parametrize("over,words", [
    (dict(d=3), "dtype code"), (dict(H=252), "multiple of 8"), (dict(T=-1), "bad T"), (dict(x=None), "null"), (dict(ro=None), "null"),
    (dict(n=None), "null"), (dict(x=ODD), "16-byte"), (dict(ldr=248), "16-byte"), (dict(post=ODD), "weights"), (dict(g=ODD, gc=1), "gate"),
    (dict(g=P, gc=2), "gate"), (dict(g=P, gc=1, gr=12), "gate"), (dict(q=P, ldq=256), "scales"), (dict(q=P, ldq=250, s=P), "code rows"),
    (dict(q=P, ldq=256, s=P, sm=1 << 31), "2 GiB")])
def test_gated_add_rmsnorm(over, words):
    from kb_nano_amd._lib import lib
    a = {**NORM, **over}
    refused(lib().kbn_gated_add_rmsnorm(a["x"], a["d"], a["ldx"], a["r"], a["ldr"], a["w"], a["post"], a["g"], a["gr"], a["gc"], 1.0, 1e-6, a["T"],
                                        a["H"], a["ro"], a["ldro"], a["n"], a["ldn"], a["q"], a["ldq"], a["s"], a["sm"], a["sg"], None), words)


LORA = dict(x=P, d=0, ldx=256, base=P, ldb=64, a=P, b=P, ids=P, ib=4, T=4, N=64, K=256, L=3, R=16, out=P, ldo=64, ws=P, wsb=1 << 20)


@pytest.mark.parametrize("over,words", [
    (dict(d=2), "dtype code"), (dict(ib=1), "ids of 1"), (dict(N=0), "bad sizes"), (dict(L=0), "bad sizes"), (dict(K=252), "multiple of 8"),
    (dict(R=12), "rank 12"), (dict(R=264), "rank 264"), (dict(x=None), "null"), (dict(ids=None), "null"), (dict(x=ODD), "16-byte"),
    (dict(ldx=250), "16-byte"), (dict(ldx=1 << 22), "2^22"), (dict(ldb=63), "strides"), (dict(ldo=80), "in place"), (dict(wsb=16), "workspace"),
    (dict(ws=None), "workspace"), (dict(N=1 << 23, R=256, ldb=1 << 23, ldo=1 << 23), "too large")])
def test_lora_add(over, words):
    from kb_nano_amd._lib import lib
    a = {**LORA, **over}
    refused(lib().kbn_lora_add(a["x"], a["d"], a["ldx"], a["base"], a["ldb"], a["a"], a["b"], a["ids"], a["ib"], None, a["T"], a["N"], a["K"],
                               a["L"], a["R"], a["out"], a["ldo"], a["ws"], a["wsb"], None), words)


def test_empty_batches_are_noops_and_workspaces_are_told():
    from kb_nano_amd._lib import lib
    L = lib()
    assert L.kbn_moe_router_gemm(None, 0, 0, None, 0, 0, None, 0, 0, 8, 256, None, 0, None) == 0
    assert L.kbn_moe_router_gemm_workspace_bytes(4, 8, 252, 0, 0) == -1 and L.kbn_moe_router_gemm_workspace_bytes(4, 8, 256, 0, 1) == -1
    assert L.kbn_moe_router_gemm_workspace_bytes(1, 8, 256, 0, 0) == 0
    assert L.kbn_moe_router_topk(None, 2, 0, None, 0, 64, 4, 0, 1, 1, 1, 1.0, None, None, 4, None) == 0
    assert L.kbn_gated_add_rmsnorm(None, 0, 0, None, 0, None, None, None, 0, 0, 1.0, 1e-6, 0, 256, None, 0, None, 0, None, 0, None, 0, 0, None) == 0
    assert L.kbn_lora_add(None, 0, 0, None, 0, None, None, None, 4, None, 0, 64, 256, 3, 16, None, 0, None, 0, None) == 0
    assert L.kbn_lora_add_workspace_bytes(4, 256, 3, 12) == -1 and L.kbn_lora_add_workspace_bytes(4, 4, 3, 16) == -1
    assert L.kbn_lora_add_workspace_bytes(0, 256, 3, 16) == 0
    for T in (1, 64, 65, 4096):
        n = L.kbn_lora_add_workspace_bytes(T, 4096, 8, 32)
        assert n >= T * 32 * 4 and n % (T * 32 * 4) == 0


def test_modules_have_no_cpu_path():
    import torch

    from kb_nano_amd import GatedAddRMSNorm, LoraAdd, MoeRouterGemm, MoeRouterTopk
    x = torch.zeros(4, 64, dtype=torch.bfloat16)
    for call in (lambda: MoeRouterGemm()(x, x), lambda: MoeRouterTopk()(x, 4), lambda: GatedAddRMSNorm()(x, x, x[0]),
                 lambda: LoraAdd()(x, x, x.view(1, 4, 64), x.view(1, 64, 4), torch.zeros(4, dtype=torch.int32))):
        with pytest.raises(RuntimeError, match="no CPU path"):
            call()
