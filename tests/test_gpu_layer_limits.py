"""The router, the gated norms and the adapters at the edges of their variants: every way the adapters' chunks
are found, every tile width and split of the router's product, threads, padded batches, compiled calls."""
import pytest
import torch

from tests._layer_util import assert_gate, assert_lora, assert_routing, routing_plain
from tests.test_gpu_lora import args, make
from tests.test_gpu_mx_threads import together

pytestmark = pytest.mark.gpu
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def randn(shape, dtype, seed, dev, std=1.0):
    return (torch.randn(shape, device=dev, generator=torch.Generator(device=dev).manual_seed(seed)) * std).to(dtype)


# ---------------------------------------------------------------- adapters

@pytest.mark.parametrize("L", [1, 2, 62, 63, 64, 65, 300])
@pytest.mark.parametrize("T", [1, 8, 9, 63, 64, 65, 255, 256, 257, 520])
def test_every_way_to_find_a_window_s_chunks(gpu_device, T, L):
    """63 adapters and more, windows that end inside a batch, adapters of one token beside ones of hundreds."""
    from kb_nano_amd import LoraAdd
    print(f"lora {T} tokens of {L} adapters", flush=True)
    d = make(T, 72, 136, L, 8, BF16, T + L, gpu_device)
    g = torch.Generator().manual_seed(T * L)
    few = torch.randint(-1, L, (T,), generator=g)
    few[torch.rand(T, generator=g) < 0.6] = L - 1          # most tokens name one adapter
    for ids in (d["ids"], few.to(torch.int32).to(gpu_device), torch.arange(T, device=gpu_device, dtype=torch.int32) % L,
                torch.full((T,), -1, dtype=torch.int32, device=gpu_device)):
        d["ids"] = ids
        assert_lora(LoraAdd()(*args(d)), *args(d), f"{T} of {L}")


@pytest.mark.parametrize("T,N,K,R", [(700, 5000, 128, 16), (3000, 1030, 64, 64), (2500, 4096, 256, 256), (1025, 36, 2056, 48)])
def test_strips_and_splits(gpu_device, T, N, K, R):
    """Several strips a workgroup, widths that end inside one, ranks of every variant."""
    from kb_nano_amd import LoraAdd
    print(f"lora strips {T} x {N} x {K} rank {R}", flush=True)
    for dtype in (BF16, F16):
        for ids in ("runs", "random"):
            d = make(T, N, K, 5, R, dtype, N, gpu_device, ids=ids)
            assert_lora(LoraAdd()(*args(d)), *args(d), f"{T}x{N}")


def test_in_place_reads_its_input_first_and_tells_autograd(gpu_device):
    """base may be x itself (the first launch has read it all); what is saved of base counts as changed."""
    from kb_nano_amd import LoraAdd
    d = make(70, 256, 256, 4, 16, BF16, 5, gpu_device)
    want = LoraAdd()(d["x"], d["x"], d["a"], d["b"], d["ids"], d["s"])
    x = d["x"].clone()
    before = x._version
    assert LoraAdd()(x, x, d["a"], d["b"], d["ids"], d["s"], inplace=True) is x
    assert torch.equal(x, want) and x._version == before + 1
    with torch.inference_mode():   # which keeps no versions
        x = d["x"].clone()
        assert torch.equal(LoraAdd()(x, x, d["a"], d["b"], d["ids"], d["s"], inplace=True), want)
    # B, ids and scaling are read while the output is written
    both = torch.zeros(4 * 256 * 16, dtype=BF16, device=gpu_device)
    with pytest.raises(ValueError, match="overlaps lora_b"):
        LoraAdd()(d["x"][:8], both[:2048].view(8, 256), d["a"], both.view(4, 256, 16), d["ids"][:8], d["s"], inplace=True)


def test_zeros_keep_their_signs_in_rows_without_an_adapter(gpu_device):
    from kb_nano_amd import LoraAdd
    d = make(70, 64, 64, 2, 8, BF16, 1, gpu_device)
    d["base"][::2] = -0.0
    d["base"][1] = float("nan")
    d["ids"][:40] = -1
    out = LoraAdd()(*args(d))
    assert torch.equal(out[:40].view(torch.int16), d["base"][:40].view(torch.int16))


def test_adapters_read_only_what_they_name(gpu_device):
    """NaN in adapters that nobody names, in x of tokens without one, and in B and A of others reaches nothing."""
    from kb_nano_amd import LoraAdd
    d = make(100, 96, 192, 6, 16, BF16, 4, gpu_device)
    ref = LoraAdd()(*args(d))
    nan = float("nan")
    d["ids"] = torch.where(d["ids"] == 3, torch.full_like(d["ids"], -1), d["ids"])
    keep = d["ids"] >= 0
    d["a"][3], d["b"][3], d["s"][3] = nan, nan, nan
    d["x"][~keep] = nan
    out = LoraAdd()(*args(d))
    assert torch.equal(out[keep], ref[keep]) and torch.equal(out[~keep], d["base"][~keep])


# ------------------------------------------------------------------ router

@pytest.mark.parametrize("x_dtype,w_dtype", [(BF16, BF16), (BF16, F32), (F32, F32), (F16, F32)])
@pytest.mark.parametrize("E", [8, 16, 17, 40, 256])
@pytest.mark.parametrize("T", [12, 13, 16, 17, 130, 600, 2100])
def test_every_tile_and_split(gpu_device, T, E, x_dtype, w_dtype):
    from kb_nano_amd import MoeRouterGemm
    print(f"router tiles {T} x {E} {x_dtype} {w_dtype}", flush=True)
    x, w = randn((T, 2056), x_dtype, T, gpu_device), randn((E, 2056), w_dtype, E, gpu_device, 0.02)
    assert_gate(MoeRouterGemm()(x, w), x, w, f"{T}x{E}")


@pytest.mark.parametrize("T,E,H,x_dtype", [(1101, 250, 7176, F32), (1101, 250, 7176, BF16), (1101, 250, 7176, F16), (2051, 129, 7168, F32),
                                           (2049, 256, 7168, BF16), (4096, 320, 2056, F16), (20000, 256, 520, F32)])
def test_many_tokens_and_weights_in_fp32(gpu_device, T, E, H, x_dtype):
    """Tiles of 128 x 128 that end inside tokens, experts and K; with and without splits; rows with gaps; NaN behind the rows."""
    from kb_nano_amd import MoeRouterGemm
    print(f"router wide {T} x {E} x {H} {x_dtype}", flush=True)
    gap = 24
    x, w = randn((T + 1, H + gap), x_dtype, T, gpu_device), randn((E + 1, H + gap), F32, E, gpu_device, 0.02)
    x[T], w[E], x[:, H:], w[:, H:] = float("nan"), float("nan"), float("nan"), float("nan")
    x, w = x[:T, :H], w[:E, :H]
    out = MoeRouterGemm()(x, w)
    assert_gate(out, x, w, f"{T}x{E}x{H}")
    assert all(torch.equal(out, MoeRouterGemm()(x, w)) for _ in range(3))
    small = MoeRouterGemm()(x[:61], w)   # other tiles: the same sums in another order
    assert_gate(small, x[:61], w, "first rows")


def test_weights_far_apart(gpu_device):
    """Weight rows further apart than 128 of them fit into 32-bit offsets."""
    from kb_nano_amd import MoeRouterGemm
    H, ld = 7168, (1 << 22) + 8
    x, buf = randn((2051, H), BF16, 1, gpu_device), torch.empty(129 * ld, dtype=F32, device=gpu_device)
    w = buf.view(129, ld)[:, :H]
    w.copy_(randn((129, H), F32, 2, gpu_device, 0.02))
    assert_gate(MoeRouterGemm()(x, w), x, w, "far")


def test_product_does_not_depend_on_the_run(gpu_device):
    """Splits meet in one order: the same bits on every run, beside other work."""
    from kb_nano_amd import MoeRouterGemm
    x, w = randn((61, 7168), BF16, 1, gpu_device), randn((256, 7168), F32, 2, gpu_device, 0.02)
    ref = MoeRouterGemm()(x, w)
    side = torch.cuda.Stream()
    for _ in range(20):
        with torch.cuda.stream(side):
            torch.matmul(x, x.t())
        assert torch.equal(MoeRouterGemm()(x, w), ref)
    torch.cuda.synchronize()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("k", [1, 7, 8, 9])
@pytest.mark.parametrize("E", [8, 63, 64, 128, 255, 256, 500, 512])
def test_many_tokens_with_near_and_equal_values(gpu_device, E, k, dtype):
    """Logits on a coarse grid, moved by up to some units in the last place: ties, near ties and rows of one value in
    the four-token kernel, next to its switch to 64 bits, and past it (nine experts)."""
    from kb_nano_amd import MoeRouterTopk
    k = min(k, E)
    g = torch.Generator().manual_seed(E + k)
    l = torch.randint(-6, 7, (203, E), generator=g) * 0.5
    l = l * (1 + torch.randint(-2, 3, l.shape, generator=g) * 2.0 ** -23)
    l[5] = 0.25
    l[6] = -1e-30
    l[7, : E // 2] = float("-inf")
    l[8] = float("-inf")
    l[9, 3] = float("nan")
    l[10, E - 1] = 3.4e38
    l = l.to(dtype).to(gpu_device)
    bias = (torch.randint(-1, 2, (E,), generator=g) * 2.0 ** -20).to(gpu_device)
    for scoring in ("softmax", "sigmoid"):
        for b in (None, bias, bias * 0):
            w, i = MoeRouterTopk()(l, k, scoring, b)
            assert_routing(w, i, routing_plain(l, k, scoring, b), f"{E} top {k} {scoring}")


@pytest.mark.parametrize("E,groups,kept", [(64, 16, 5), (256, 16, 3), (512, 8, 2), (96, 6, 3), (160, 8, 3), (32, 8, 8), (320, 5, 1)])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_groups_with_near_and_equal_ranks(gpu_device, E, groups, kept, scoring):
    from kb_nano_amd import MoeRouterTopk
    g = torch.Generator().manual_seed(E)
    l = torch.randint(-3, 4, (90, E), generator=g) * 0.75
    l = l * (1 + torch.randint(-1, 2, l.shape, generator=g) * 2.0 ** -23)
    l[3] = 1.0
    l[4, : E // groups] = float("-inf")
    l[5] = float("-inf")
    l = l.to(gpu_device)
    for bias in (None, torch.zeros(E, device=gpu_device), (torch.randint(0, 3, (E,), generator=g) * 0.125).to(gpu_device),
                 torch.where(torch.rand(E, generator=g) < 0.5, 1000.0, -999.5).to(gpu_device)):
        w, i = MoeRouterTopk()(l, 4, scoring, bias, groups, kept)
        assert_routing(w, i, routing_plain(l, 4, scoring, bias, groups, kept), f"{E} in {groups}")


# --------------------------------------------------------------- all of them

@pytest.mark.parametrize("own", [False, True])
def test_calls_of_threads(gpu_device, own):
    from kb_nano_amd import GatedAddRMSNorm, GatedAddRMSNormFP8Quant, LoraAdd, MoeRouterGemm, MoeRouterTopk
    print(f"layer threads own={own}", flush=True)
    gemm, topk, norm, norm8, lora = MoeRouterGemm(), MoeRouterTopk(), GatedAddRMSNorm(), GatedAddRMSNormFP8Quant(), LoraAdd()
    x, w, bias = randn((300, 1024), BF16, 1, gpu_device), randn((64, 1024), F32, 2, gpu_device, 0.05), randn(64, F32, 3, gpu_device, 0.02)
    nw = randn(1024, BF16, 4, gpu_device)
    d = make(300, 256, 1024, 6, 16, BF16, 5, gpu_device)

    def calls(n):
        rows, res = norm(x[:n], x[:n], nw, nw)
        q, s, _ = norm8(x[:n], x[:n], nw, nw)
        logits = gemm(rows, w)
        tw, ids = topk(logits, 6, "sigmoid", bias, 8, 4)
        y = lora(rows, d["base"][:n], d["a"], d["b"], d["ids"][:n], d["s"])
        return rows, res, q, s.t(), logits, tw, ids, y

    sizes = (1, 14, 90, 300)
    refs = [calls(n) for n in sizes]
    torch.cuda.synchronize()

    def work(k):
        made = 0
        stream = torch.cuda.Stream() if own else torch.cuda.current_stream()
        with torch.cuda.stream(stream):
            for _ in range(25):
                outs = calls(sizes[k])
                assert all(torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8))
                           for a, b in zip(outs, refs[k], strict=True))
                made += len(outs)
        return made

    assert together(work, len(sizes)) == [25 * 8] * len(sizes)
    torch.cuda.synchronize()


def test_outputs_carry_no_gradient(gpu_device):
    from kb_nano_amd import GatedAddRMSNorm, LoraAdd, MoeRouterGemm, MoeRouterTopk
    d = make(4, 64, 128, 2, 8, BF16, 5, gpu_device)
    x = d["x"].requires_grad_()
    w = randn((16, 128), BF16, 2, gpu_device).requires_grad_()
    assert not MoeRouterGemm()(x, w).requires_grad
    assert not MoeRouterTopk()(randn((4, 16), F32, 1, gpu_device).requires_grad_(), 2)[0].requires_grad
    assert not any(t.requires_grad for t in GatedAddRMSNorm()(x, x, w[0]))
    assert not LoraAdd()(x, d["base"], d["a"], d["b"], d["ids"], d["s"]).requires_grad


def test_a_layer_s_run(gpu_device):
    """Gated norm with rows and codes, the codes through the FP8 product, the rows through the router and the adapters
    added to that product, the experts on the rows: each step against its own reference."""
    from kb_nano_amd import GatedAddRMSNormFP8Quant, LoraAdd, MoeRouterGemm, MoeRouterTopk, VllmFusedExperts
    from kb_nano_amd.fp8_linear import _block_requant
    from tests.test_gpu_few_token_experts import make as experts
    T, H, N = 48, 512, 384
    e = experts(T, 16, H, 256, 4, "fp8", BF16, 5, gpu_device)
    d = make(T, N, H, 4, 16, BF16, 5, gpu_device)
    w, sw = _block_requant(randn((N, H), F32, 1, gpu_device, 0.05), True)
    nw, pw = randn(H, BF16, 2, gpu_device, 0.1) + 1, randn(H, BF16, 3, gpu_device, 0.1) + 1
    q, s, res, rows = GatedAddRMSNormFP8Quant()(e["x"], d["x"], nw, pw, None, 0.5, with_rows=True)
    y = torch.empty(T, N, dtype=BF16, device=gpu_device)
    torch.ops.kb_nano_fp8.fp8_gemm_nt(q, s, w, sw, y)
    out = LoraAdd()(rows, y, d["a"], d["b"], d["ids"], d["s"])
    assert_lora(out, rows, y, d["a"], d["b"], d["ids"], d["s"], "run")
    # the product of the codes is near that of the rows: e4m3 on one side, half a step 2^-4 at most
    dense = rows.double() @ (w.double() * sw.double().repeat_interleave(128, 0).repeat_interleave(128, 1)[:N, :H]).t()
    assert float((y.double() - dense).norm() / dense.norm()) < 2.0 ** -4
    wr = randn((16, H), F32, 9, gpu_device, 0.05)
    logits = MoeRouterGemm()(rows, wr)
    assert_gate(logits, rows, wr, "run")
    tw, ids = MoeRouterTopk()(logits, 4)
    assert_routing(tw, ids, routing_plain(logits, 4), "run")
    moe = VllmFusedExperts()(rows, e["w13"], e["w2"], tw, ids, 16, e["s13"], e["s2"], e["block"])
    assert moe.shape == rows.shape and bool(torch.isfinite(moe).all())


def test_compiled_calls_make_the_same_launches(gpu_device):
    """The opaque ops trace and give the eager results."""
    from kb_nano_amd import GatedAddRMSNormFP8Quant, LoraAdd, MoeRouterGemm, MoeRouterTopk
    gemm, topk, norm, lora = MoeRouterGemm(), MoeRouterTopk(), GatedAddRMSNormFP8Quant(), LoraAdd()
    d = make(20, 64, 256, 3, 16, BF16, 5, gpu_device)
    w, nw = randn((32, 256), F32, 2, gpu_device, 0.05), randn(256, BF16, 4, gpu_device)

    def run(x, base):
        q, s, res, rows = norm(x, x, nw, with_rows=True)
        tw, ids = topk(gemm(rows, w), 4, "sigmoid", None, 4, 2)
        return q, s, res, tw, ids, lora(rows, base, d["a"], d["b"], d["ids"], d["s"])

    refs = run(d["x"], d["base"])
    outs = torch.compile(run, backend="aot_eager", fullgraph=True)(d["x"], d["base"])
    for a, b in zip(outs, refs, strict=True):
        assert torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8))
