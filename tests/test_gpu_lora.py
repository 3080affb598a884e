"""Adapters of many requests beside a shared projection, against the formula in 64 bits."""
import pytest
import torch

from tests._layer_util import assert_lora, replayed

pytestmark = pytest.mark.gpu
BF16, F16 = torch.bfloat16, torch.float16


def make(T, N, K, L, R, dtype, seed, dev, pad=0, ids="random"):
    g = torch.Generator(device=dev).manual_seed(seed)

    def randn(*shape):
        return torch.randn(shape, device=dev, generator=g)
    which = {"random": lambda: torch.randint(-1, L, (T,), device=dev, generator=g), "one": lambda: torch.full((T,), L - 1, device=dev),
             "none": lambda: torch.full((T,), -1, device=dev),
             "runs": lambda: torch.randint(-1, L, (T // 40 + 1,), device=dev, generator=g).repeat_interleave(40)[:T]}[ids]()
    return {"x": randn(T, K + pad).to(dtype)[:, :K], "base": randn(T, N + pad).to(dtype)[:, :N], "a": (randn(L, R, K) * K ** -0.5).to(dtype),
            "b": (randn(L, N, R) * R ** -0.5).to(dtype), "ids": which.to(torch.int32), "s": 0.25 + torch.rand(L, device=dev, generator=g)}


def args(d):
    return d["x"], d["base"], d["a"], d["b"], d["ids"], d["s"]


def check(d, what):
    from kb_nano_amd import LoraAdd
    base = d["base"].clone()
    out = LoraAdd()(*args(d))
    assert torch.equal(d["base"], base)
    assert_lora(out, *args(d), what)
    return out


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("T,N,K,L,R", [(1, 8, 8, 1, 8), (1, 4096, 4096, 3, 16), (2, 100, 64, 2, 8), (5, 257, 520, 4, 24), (16, 640, 1032, 7, 64),
                                       (17, 63, 200, 1, 72), (64, 513, 2048, 64, 16), (65, 512, 512, 100, 40), (130, 1000, 776, 5, 128),
                                       (33, 300, 264, 2, 256), (300, 1536, 1024, 12, 32), (40, 1, 128, 3, 136)])
@pytest.mark.parametrize("ids", ["random", "one"])
def test_adapters(gpu_device, T, N, K, L, R, ids, dtype):
    print(f"lora {T} x {N} x {K}, {L} of rank {R}, {ids} {dtype}", flush=True)
    check(make(T, N, K, L, R, dtype, T + N, gpu_device, ids=ids), f"{T}x{N}x{K} {L} of {R}")


@pytest.mark.parametrize("ids", ["runs", "random", "none"])
def test_many_tokens(gpu_device, ids):
    print(f"lora many tokens {ids}", flush=True)
    check(make(2100, 768, 1536, 6, 16, BF16, 3, gpu_device, ids=ids), ids)


@pytest.mark.parametrize("T", [7, 200])
def test_strides_ids_and_scaling(gpu_device, T):
    from kb_nano_amd import LoraAdd
    lora = LoraAdd()
    d = make(T, 264, 520, 5, 16, BF16, 2, gpu_device, pad=8)
    assert d["x"].stride(0) == 528
    out = check(d, "strided")
    d["base"] = make(T, 264, 520, 5, 16, BF16, 2, gpu_device, pad=5)["base"]      # rows at odd addresses
    check(d, "odd strides")
    d = make(T, 264, 520, 5, 16, BF16, 2, gpu_device, pad=8)
    assert torch.equal(lora(d["x"], d["base"], d["a"], d["b"], d["ids"].long(), d["s"]), out)
    x3, b3 = d["x"].contiguous().view(T, 1, 520), d["base"].contiguous().view(T, 1, 264)
    assert torch.equal(lora(x3, b3, d["a"], d["b"], d["ids"].view(T, 1), d["s"]).view(T, 264), out)
    assert_lora(lora(*args(d)[:5]), *args(d)[:5], None, "no scaling")
    d["ids"] = torch.where(d["ids"] < 0, torch.full_like(d["ids"], 2 ** 31 - 1), d["ids"])   # outside on the other side
    assert torch.equal(lora(*args(d)), out)
    assert torch.equal(lora(d["x"], d["base"], d["a"], d["b"], d["ids"].long() * 2 ** 32 + d["ids"], d["s"])[d["ids"] > 0],
                       d["base"][d["ids"] > 0])   # ids past 32 bits are outside, whatever their low words
    assert lora(d["x"][:0], d["base"][:0], d["a"], d["b"], d["ids"][:0], d["s"]).shape == (0, 264)


@pytest.mark.parametrize("T", [5, 150])
def test_in_place(gpu_device, T):
    """Only base's own columns are written, rows without an adapter and the columns beside stay as they were."""
    from kb_nano_amd import LoraAdd
    d = make(T, 264, 520, 5, 16, BF16, 2, gpu_device)
    out = LoraAdd()(*args(d))
    wide = torch.randn(T + 2, 400, device=gpu_device).to(BF16)
    kept = wide.clone()
    part = wide[1:T + 1, 64:328]
    part.copy_(d["base"])
    got = LoraAdd()(d["x"], part, d["a"], d["b"], d["ids"], d["s"], inplace=True)
    assert got.data_ptr() == part.data_ptr() and torch.equal(part, out)
    assert torch.equal(wide[:, :64], kept[:, :64]) and torch.equal(wide[:, 328:], kept[:, 328:])
    assert torch.equal(wide[0], kept[0]) and torch.equal(wide[-1], kept[-1])


def test_rows_far_apart(gpu_device):
    from kb_nano_amd import LoraAdd
    d = make(6, 64, 256, 3, 8, BF16, 2, gpu_device)
    out = LoraAdd()(*args(d))
    store = torch.zeros(5 * (1 << 23) + 256, dtype=BF16, device=gpu_device)
    x = store.as_strided((6, 256), (1 << 23, 1))
    x.copy_(d["x"])
    base = torch.zeros(5 * (1 << 23) + 64, dtype=BF16, device=gpu_device).as_strided((6, 64), (1 << 23, 1))
    base.copy_(d["base"])
    assert torch.equal(LoraAdd()(x, base, *args(d)[2:]), out)


def test_large_values_in_between(gpu_device):
    """A x past fp16's range, brought back by the scaling; infinities stay in their rows."""
    from kb_nano_amd import LoraAdd
    d = make(20, 128, 256, 2, 16, F16, 2, gpu_device, ids="one")
    d["x"] *= 1000
    d["a"] *= 100
    d["s"] *= 1e-5
    out = check(d, "large")
    d["x"][3, 5] = float("inf")
    got = LoraAdd()(*args(d))
    assert not bool(torch.isfinite(got[3]).any())
    keep = torch.arange(20, device=gpu_device) != 3
    assert torch.equal(got[keep], out[keep])


def test_captured_and_on_a_stream(gpu_device):
    from kb_nano_amd import LoraAdd
    sets = [args(make(T, 264, 520, 5, 16, BF16, T, gpu_device)) for T in (3, 90, 400)]

    def call():
        return [LoraAdd()(*s) for s in sets]
    refs = call()
    replayed(call, refs, lambda: (call(), torch.cuda.synchronize()))
    streams = [torch.cuda.Stream() for _ in range(3)]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    outs = []
    for _ in range(10):      # at once, on streams of their own
        for s in streams:
            with torch.cuda.stream(s):
                outs.append(call())
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for o in outs for a, b in zip(o, refs))


def test_refusals(gpu_device):
    from kb_nano_amd import LoraAdd
    lora = LoraAdd()
    d = make(4, 64, 256, 3, 16, BF16, 2, gpu_device)
    x, base, a, b, ids, s = args(d)
    with pytest.raises(TypeError, match="input must be"):
        lora(x.float(), base, a, b, ids, s)
    for other in ((x, base.half(), a, b, ids, s), (x, base, a.half(), b, ids, s), (x, base, a, b.half(), ids, s)):
        with pytest.raises(TypeError, match="must be torch.bfloat16"):
            lora(*other)
    with pytest.raises(TypeError, match="adapter_ids"):
        lora(x, base, a, b, ids.to(torch.int16), s)
    with pytest.raises(TypeError, match="scaling"):
        lora(x, base, a, b, ids, s.to(BF16))
    with pytest.raises(ValueError, match="other rows"):
        lora(x, base[:3], a, b, ids, s)
    with pytest.raises(ValueError, match="rank 12"):
        lora(x, base, a[:, :12].contiguous(), b[:, :, :12].contiguous(), ids, s)
    with pytest.raises(ValueError, match="lora_b must be"):
        lora(x, base, a, b[:2], ids, s)
    with pytest.raises(ValueError, match="lora_a must be"):
        lora(x[:, :128], base, a, b, ids, s)
    with pytest.raises(ValueError, match="adapter_ids must be"):
        lora(x, base, a, b, ids[:3], s)
    with pytest.raises(ValueError, match="scaling must be"):
        lora(x, base, a, b, ids, s[:2])
    with pytest.raises(ValueError, match="contiguous rows"):
        lora(x, base.t().contiguous().t(), a, b, ids, s)
    with pytest.raises(RuntimeError, match="16-byte"):
        lora(x[:, 4:252], base, a[:, :, :248].contiguous(), b, ids, s)
    with pytest.raises(RuntimeError, match="must be on"):
        lora(x, base, a, b, ids.cpu(), s)


@pytest.mark.parametrize("T", [3, 100])
def test_linear_with_adapters(gpu_device, T):
    """Norm, FP8 linear and adapters as a layer calls them: the adapters on the linear's own output, bit for bit."""
    from kb_nano_amd import Fp8Linear, GatedAddRMSNorm, LoraAdd, LoraFp8Linear
    from kb_nano_amd.fp8_linear import _block_requant
    d = make(T, 384, 512, 4, 16, BF16, 5, gpu_device)
    n, _ = GatedAddRMSNorm()(d["x"], d["x"], torch.ones(512, dtype=BF16, device=gpu_device))
    w, sw = _block_requant(torch.randn(384, 512, device=gpu_device, generator=torch.Generator(device=gpu_device).manual_seed(1)) * 0.05, True)
    base = Fp8Linear()(n, w, sw)
    out = LoraFp8Linear()(n, w, sw, d["a"], d["b"], d["ids"], d["s"])
    assert torch.equal(out, LoraAdd()(n, base, d["a"], d["b"], d["ids"], d["s"]))
    assert_lora(out, n, base, d["a"], d["b"], d["ids"], d["s"], "linear")
    bias = torch.randn(384, device=gpu_device).to(BF16)
    layer = LoraFp8Linear()
    layer.linear._ensure_buffers(128, 512, 384, gpu_device)
    got = layer(n.view(T, 1, 512), w, sw, d["a"], d["b"], d["ids"], d["s"])
    assert got.shape == (T, 1, 384) and torch.equal(got.view(T, 384), out)
    assert_lora(LoraFp8Linear()(n, w, sw, d["a"], d["b"], d["ids"], d["s"], bias), n, base + bias, d["a"], d["b"], d["ids"], d["s"], "bias")
