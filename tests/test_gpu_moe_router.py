"""The router's product and the choice of experts against plain forms in 64 bits."""
import pytest
import torch

from tests._layer_util import assert_gate, assert_routing, replayed, routing_plain

pytestmark = pytest.mark.gpu
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def rows(T, H, dtype, seed, dev, pad=0, std=1.0):
    g = torch.Generator(device=dev).manual_seed(seed)
    return (torch.randn(T, H + pad, device=dev, generator=g) * std).to(dtype)[:, :H]


# ------------------------------------------------------------------ product

@pytest.mark.parametrize("x_dtype,w_dtype", [(BF16, BF16), (F16, F16), (F32, F32), (BF16, F32), (F16, F32)])
@pytest.mark.parametrize("T,E,H", [(1, 1, 8), (1, 16, 2048), (2, 5, 72), (3, 49, 840), (7, 128, 4096), (8, 8, 512), (9, 17, 136),
                                   (16, 64, 2056), (61, 256, 7168), (65, 33, 1000), (200, 160, 512), (513, 300, 264)])
def test_product(gpu_device, T, E, H, x_dtype, w_dtype):
    from kb_nano_amd import MoeRouterGemm
    print(f"router product {T} x {E} x {H} {x_dtype} {w_dtype}", flush=True)
    x = rows(T, H, x_dtype, T, gpu_device)
    w = rows(E, H, w_dtype, E + 1, gpu_device, std=0.02)
    assert_gate(MoeRouterGemm()(x, w), x, w, f"{T}x{E}x{H}")


@pytest.mark.parametrize("T,E", [(1111, 256), (2500, 130), (4096, 256), (4099, 512)])
@pytest.mark.parametrize("w_dtype", [BF16, F32])
def test_product_of_many_tokens(gpu_device, T, E, w_dtype):
    from kb_nano_amd import MoeRouterGemm
    print(f"router product {T} x {E} {w_dtype}", flush=True)
    x, w = rows(T, 1032, BF16, 1, gpu_device), rows(E, 1032, w_dtype, 2, gpu_device, std=0.02)
    assert_gate(MoeRouterGemm()(x, w), x, w, f"{T}x{E}")


@pytest.mark.parametrize("T", [3, 20, 300])
def test_product_of_strided_rows_and_leading_dimensions(gpu_device, T):
    from kb_nano_amd import MoeRouterGemm
    gate = MoeRouterGemm()
    x, w = rows(T, 520, BF16, 1, gpu_device, pad=56), rows(40, 520, BF16, 2, gpu_device, pad=24, std=0.02)
    out = gate(x, w)
    assert_gate(out, x, w, "strided")
    assert torch.equal(out, gate(x.contiguous(), w.contiguous()))
    assert torch.equal(out, gate(x.view(T, 1, 520), w).view(T, 40))
    assert gate(x[:0], w).shape == (0, 40)
    back = gate(x.flip(1).contiguous(), w.flip(1).contiguous())   # another order of the same products
    assert_gate(back, x, w, "reversed")


def test_product_of_rows_far_apart(gpu_device):
    """Every 2^23-th element: the last tokens of long sequences, a row stride that 32-bit offsets do not reach."""
    from kb_nano_amd import MoeRouterGemm
    store = torch.zeros(11 * (1 << 23) + 256, dtype=BF16, device=gpu_device)
    x = store.as_strided((12, 256), (1 << 23, 1))
    x.copy_(rows(12, 256, BF16, 3, gpu_device))
    w = rows(19, 256, BF16, 4, gpu_device, std=0.02)
    assert torch.equal(MoeRouterGemm()(x, w), MoeRouterGemm()(x.contiguous(), w))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("T", [2, 40])
def test_product_of_infinities_and_large_values(gpu_device, T, dtype):
    """An infinity leaves no finite logit in its row (the pieces may make it a NaN) and touches no other;
    values near the type's largest do not overflow in pieces."""
    from kb_nano_amd import MoeRouterGemm
    x, w = rows(T, 256, dtype, 5, gpu_device), rows(24, 256, F32, 6, gpu_device).abs() + 0.1
    ref = MoeRouterGemm()(x, w)
    x[1, 77] = float("inf")
    out = MoeRouterGemm()(x, w)
    assert not bool(torch.isfinite(out[1]).any()) and torch.equal(out[0], ref[0])
    x[1, 77] = 3.0e38
    w2 = w * 1e-3
    assert_gate(MoeRouterGemm()(x, w2), x, w2, "large")


def test_product_captured_and_on_a_stream(gpu_device):
    from kb_nano_amd import MoeRouterGemm
    gate = MoeRouterGemm()
    sets = [(rows(T, 1024, BF16, T, gpu_device), rows(64, 1024, F32, 9, gpu_device)) for T in (4, 70)]
    refs = [gate(*s) for s in sets]
    replayed(lambda: [gate(*s) for s in sets], refs, lambda: (gate(*sets[0]), torch.cuda.synchronize()))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        outs = [gate(*s) for s in sets]
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(outs, refs))


def test_product_refusals(gpu_device):
    from kb_nano_amd import MoeRouterGemm
    gate = MoeRouterGemm()
    x, w = rows(4, 256, BF16, 1, gpu_device), rows(8, 256, BF16, 2, gpu_device)
    with pytest.raises(TypeError, match="hidden states"):
        gate(x.double(), w)
    with pytest.raises(TypeError, match="weight"):
        gate(x, w.half())
    with pytest.raises(TypeError, match="weight"):
        gate(x.float(), w)
    with pytest.raises(ValueError, match="multiple of 8"):
        gate(x[:, :252], w[:, :252])
    with pytest.raises(ValueError, match="weight must be"):
        gate(x, w[:, :128])
    with pytest.raises(ValueError, match="contiguous rows"):
        gate(x.t().contiguous().t(), w)
    with pytest.raises(RuntimeError, match="16-byte"):
        gate(x[:, 4:252], w[:, :248])
    with pytest.raises(RuntimeError, match="must be on"):
        gate(x, w.cpu())


# ------------------------------------------------------------------- choice

SIZES = [(1, 1, 1), (3, 2, 2), (5, 8, 2), (7, 49, 5), (64, 64, 6), (33, 65, 8), (40, 128, 8), (9, 160, 6), (50, 256, 8), (4, 384, 64),
         (3, 513, 10), (2, 1000, 33), (2, 1024, 64)]


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("biased", [False, True])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("T,E,k", SIZES)
def test_choice(gpu_device, T, E, k, dtype, biased, scoring):
    from kb_nano_amd import MoeRouterTopk
    l = rows(T, E, dtype, E, gpu_device, std=1.5)
    bias = rows(1, E, F32, 7, gpu_device, std=0.05)[0] if biased else None
    for renormalize in (True, False):
        w, i = MoeRouterTopk()(l, k, scoring=scoring, bias=bias, renormalize=renormalize, scale=2.5)
        assert w.dtype == F32 and i.dtype == torch.int32
        assert_routing(w, i, routing_plain(l, k, scoring, bias, renormalize=renormalize, scale=2.5), f"{T}x{E} top {k}")


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("biased", [False, True])
@pytest.mark.parametrize("E,groups,kept,k", [(256, 8, 4, 8), (160, 8, 3, 6), (60, 4, 2, 8), (64, 64, 6, 6), (72, 8, 1, 9), (96, 6, 6, 4),
                                             (512, 16, 4, 8), (1000, 40, 7, 12), (24, 24, 24, 24), (6, 3, 1, 1), (128, 2, 1, 64)])
def test_choice_among_groups(gpu_device, E, groups, kept, k, biased, scoring):
    from kb_nano_amd import MoeRouterTopk
    l = rows(37, E, F32, E + groups, gpu_device, std=1.5)
    bias = rows(1, E, F32, 7, gpu_device, std=0.05)[0] if biased else None
    w, i = MoeRouterTopk()(l, k, scoring, bias, groups, kept, index_dtype=torch.int64)
    assert i.dtype == torch.int64
    assert_routing(w, i, routing_plain(l, k, scoring, bias, groups, kept), f"{E} in {groups}")


@pytest.mark.parametrize("biased", [False, True])
@pytest.mark.parametrize("groups,kept", [(1, 1), (8, 4)])
def test_equal_values_go_to_the_lower_index(gpu_device, biased, groups, kept):
    """Few distinct logits (and biases), -0 beside 0, whole rows of one value."""
    from kb_nano_amd import MoeRouterTopk
    g = torch.Generator().manual_seed(1)
    l = torch.randint(-2, 3, (64, 128), generator=g).float()
    l[0] = 0.0
    l[1] = -3.0
    l[2, ::2], l[2, 1::2] = -0.0, 0.0
    l = l.to(gpu_device)
    bias = (torch.randint(0, 2, (128,), generator=g).float() * 0.25).to(gpu_device) if biased else None
    for scoring in ("softmax", "sigmoid"):
        w, i = MoeRouterTopk()(l, 8, scoring, bias, groups, kept)
        assert_routing(w, i, routing_plain(l, 8, scoring, bias, groups, kept), f"{scoring} ties")


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_scores_next_to_a_border(gpu_device, scoring):
    """Biases that undo the scores up to 64-bit roundings would tie; 1e-9 beside that decides, far below fp32's."""
    from kb_nano_amd import MoeRouterTopk
    l = torch.tensor([[0.0, 1e-7, -1e-7, 5e-8] * 16], device=gpu_device)
    bias = torch.zeros(64, device=gpu_device)
    bias[2::4] = 2e-8
    w, i = MoeRouterTopk()(l, 16, scoring, bias)
    assert_routing(w, i, routing_plain(l, 16, scoring, bias), "near ties")


@pytest.mark.parametrize("biased", [False, True])
@pytest.mark.parametrize("groups,kept", [(1, 1), (4, 2)])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_masked_experts_and_extreme_logits(gpu_device, scoring, groups, kept, biased):
    """-inf and NaN logits, rows that have nothing else, +inf, the types' largest and smallest values, scores that
    underflow: experts in range and distinct, weights finite, masked ones 0."""
    from kb_nano_amd import MoeRouterTopk
    inf, nan = float("inf"), float("nan")
    l = rows(12, 32, F32, 3, gpu_device)
    l[0] = -inf
    l[1] = nan
    l[2] = -inf
    l[2, 17] = 1.0
    l[3, ::2] = nan
    l[4, :30] = -inf
    l[5, 9] = inf
    l[6] = torch.finfo(F32).min
    l[7, 4] = torch.finfo(F32).max
    l[8] = -200.0
    l[9] = -750.0
    l[10, 8:] = -inf
    l[11] = 90.0
    bias = rows(1, 32, F32, 7, gpu_device, std=0.05)[0] if biased else None
    for renormalize in (True, False):
        w, i = MoeRouterTopk()(l, 8, scoring, bias, groups, kept, renormalize)
        ids = i.cpu()
        assert int(ids.min()) >= 0 and int(ids.max()) < 32 and all(len(set(r)) == 8 for r in ids.tolist())
        assert bool(torch.isfinite(w).all())
        assert_routing(w, i, routing_plain(l, 8, scoring, bias, groups, kept, renormalize), "masked")
        assert bool((w[:2] == 0).all())


def test_choice_from_strided_rows_and_leading_dimensions(gpu_device):
    from kb_nano_amd import MoeRouterTopk
    topk = MoeRouterTopk()
    wide = rows(30, 70, F32, 3, gpu_device, pad=3)
    l = wide[:, 3:67]    # rows at odd addresses
    w, i = topk(l, 6)
    assert_routing(w, i, routing_plain(l, 6), "strided")
    w3, i3 = topk(l.contiguous().view(5, 6, 64), 6)
    assert w3.shape == i3.shape == (5, 6, 6) and torch.equal(w3.view(30, 6), w) and torch.equal(i3.view(30, 6), i)
    w0, i0 = topk(l[:0], 6)
    assert w0.shape == i0.shape == (0, 6)


def test_choice_captured_and_on_a_stream(gpu_device):
    from kb_nano_amd import MoeRouterTopk
    topk = MoeRouterTopk()
    l, bias = rows(100, 256, F32, 3, gpu_device), rows(1, 256, F32, 7, gpu_device, std=0.05)[0]

    def call():
        return [*topk(l, 8, "sigmoid", bias, 8, 4), *topk(l, 8)]
    refs = call()
    replayed(call, refs, lambda: (call(), torch.cuda.synchronize()))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        outs = call()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(outs, refs))


def test_choice_refusals(gpu_device):
    from kb_nano_amd import MoeRouterTopk
    topk = MoeRouterTopk()
    l = rows(4, 64, F32, 1, gpu_device)
    with pytest.raises(TypeError, match="logits"):
        topk(l.double(), 4)
    with pytest.raises(ValueError, match="scoring"):
        topk(l, 4, "tanh")
    for k in (0, 65):
        with pytest.raises(ValueError, match="top_k"):
            topk(l, k)
    with pytest.raises(ValueError, match="top_k=9"):
        topk(l, 9, num_groups=8, topk_groups=1)
    with pytest.raises(ValueError, match="num_groups"):
        topk(l, 4, num_groups=5)
    with pytest.raises(ValueError, match="topk_groups"):
        topk(l, 4, num_groups=4, topk_groups=5)
    with pytest.raises(ValueError, match="outside"):
        topk(rows(2, 1025, F32, 1, gpu_device), 4)
    with pytest.raises(ValueError, match="bias"):
        topk(l, 4, bias=torch.zeros(63, device=gpu_device))
    with pytest.raises(TypeError, match="bias"):
        topk(l, 4, bias=torch.zeros(64, device=gpu_device, dtype=BF16))
    with pytest.raises(TypeError, match="ids"):
        topk(l, 4, index_dtype=torch.int16)
    with pytest.raises(RuntimeError, match="must be on"):
        topk(l, 4, bias=torch.zeros(64))


# ------------------------------------------------------------------ together

def test_router_and_experts(gpu_device):
    """Product, choice and both experts layers, as a decoder layer calls them."""
    from kb_nano_amd import FewTokenExperts, MoeRouterGemm, MoeRouterTopk, VllmFusedExperts
    from tests.test_gpu_few_token_experts import make
    d = make(48, 16, 512, 256, 4, "fp8", BF16, 5, gpu_device)
    wr, bias = rows(16, 512, F32, 9, gpu_device, std=0.05), rows(1, 16, F32, 8, gpu_device, std=0.02)[0]
    logits = MoeRouterGemm()(d["x"], wr)
    tw, ids = MoeRouterTopk()(logits, 4, "sigmoid", bias, 4, 2, scale=1.5)
    assert_gate(logits, d["x"], wr, "logits")
    assert_routing(tw, ids, routing_plain(logits, 4, "sigmoid", bias, 4, 2, scale=1.5), "routing")
    few = FewTokenExperts()(d["x"], d["w13"], d["w2"], tw, ids, 16, d["s13"], d["s2"], d["block"])
    more = VllmFusedExperts()(d["x"], d["w13"], d["w2"], tw, ids, 16, d["s13"], d["s2"], d["block"])
    rel = float((few.float() - more.float()).norm() / few.float().norm())
    # the FP8 x FP8 layer quantizes its activations twice (e4m3, half a step 2^-4 each at most)
    assert rel < 2 * 2.0 ** -4
