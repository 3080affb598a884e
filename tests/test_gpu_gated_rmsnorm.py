"""The norms after and before a block with gate and scaled residual, against the formula in 64 bits."""
import pytest
import torch

from tests._layer_util import assert_codes, assert_gated, norm_error, replayed, rms

pytestmark = pytest.mark.gpu
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def make(T, H, dtype, post, gate, seed, dev, pad=0):
    g = torch.Generator(device=dev).manual_seed(seed)

    def randn(*shape):
        return torch.randn(shape, device=dev, generator=g)
    d = {"x": randn(T, H + pad).to(dtype)[:, :H], "r": randn(T, H + pad).to(dtype)[:, :H], "w": (1 + 0.1 * randn(H)).to(dtype),
         "post": (1 + 0.1 * randn(H)).to(dtype) if post else None}
    shape = {"none": None, "channel": (H,), "token": (T, 1), "full": (T, H + pad), "row": (1, H), "one": ()}[gate]
    d["g"] = None if shape is None else (0.7 + 0.2 * randn(*shape)).to(dtype)
    if gate == "full":
        d["g"] = d["g"][:, :H]
    return d


def check(d, rs, eps, what):
    from kb_nano_amd import GatedAddRMSNorm, GatedAddRMSNormFP8Quant
    args = (d["x"], d["r"], d["w"], d["post"], d["g"], rs, eps)
    before = d["x"].clone(), d["r"].clone()
    normed, res = GatedAddRMSNorm()(*args)
    gate = d["g"]
    assert_gated(res, normed, d["x"], d["r"], d["w"], d["post"], gate, rs, eps, what)
    q, s, res2, rows = GatedAddRMSNormFP8Quant()(*args, with_rows=True)
    q3, s3, res3 = GatedAddRMSNormFP8Quant()(*args)
    assert torch.equal(res, res2) and torch.equal(res, res3) and torch.equal(rows, normed)
    assert torch.equal(q.view(torch.uint8), q3.view(torch.uint8)) and torch.equal(s, s3)
    T, H = d["x"].shape
    assert q.dtype == torch.float8_e4m3fn and s.stride() == (1, T)
    assert_codes(q, s, rms(res.double(), d["w"].double(), eps), norm_error(H), what)
    assert torch.equal(d["x"], before[0]) and torch.equal(d["r"], before[1])


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("post,gate", [(True, "none"), (True, "channel"), (False, "token"), (True, "full"), (False, "none"), (True, "row"),
                                       (False, "one")])
@pytest.mark.parametrize("T,H", [(1, 8), (1, 7168), (2, 128), (3, 520), (5, 2048), (4, 2056), (37, 4096), (3, 8200), (2, 16384)])
def test_step(gpu_device, T, H, post, gate, dtype):
    print(f"gated norm {T} x {H} {dtype} {post} {gate}", flush=True)
    check(make(T, H, dtype, post, gate, T + H, gpu_device), 0.875, 1e-6, f"{T}x{H} {gate}")


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("H", [16392, 40960])
def test_long_rows(gpu_device, H, dtype):
    print(f"gated norm long {H} {dtype}", flush=True)
    for post, gate in ((True, "full"), (False, "token"), (True, "none")):
        check(make(3, H, dtype, post, gate, H, gpu_device), 1.0, 1e-5, f"{H}")


def test_many_tokens(gpu_device):
    check(make(3001, 1536, BF16, True, "channel", 1, gpu_device), 0.5, 1e-6, "many")


def test_strided_rows(gpu_device):
    d = make(33, 1000, BF16, True, "full", 4, gpu_device, pad=24)
    assert d["g"].stride(0) == 1024
    check(d, 1.25, 1e-6, "strided")
    d["g"] = d["g"].t().contiguous().t()     # columns in memory: copied
    check(d, 1.25, 1e-6, "transposed gate")


def test_leading_dimensions_and_empty(gpu_device):
    from kb_nano_amd import GatedAddRMSNorm, GatedAddRMSNormFP8Quant
    d = make(12, 256, BF16, True, "full", 2, gpu_device)
    n, r = GatedAddRMSNorm()(d["x"], d["r"], d["w"], d["post"], d["g"])
    x3, r3, g3 = (t.view(3, 4, 256) for t in (d["x"], d["r"], d["g"]))
    n3, res3 = GatedAddRMSNorm()(x3, r3, d["w"], d["post"], g3)
    assert n3.shape == x3.shape and torch.equal(n3.view(12, 256), n) and torch.equal(res3.view(12, 256), r)
    per = g3[:, :1]     # a gate for each sequence
    n4, res4 = GatedAddRMSNorm()(x3, r3, d["w"], d["post"], per)
    n5, res5 = GatedAddRMSNorm()(d["x"], d["r"], d["w"], d["post"], per.expand(3, 4, 256).reshape(12, 256))
    assert torch.equal(n4.view(12, 256), n5) and torch.equal(res4.view(12, 256), res5)
    q, s, res = GatedAddRMSNormFP8Quant()(x3, r3, d["w"], d["post"], g3)
    assert q.shape == (12, 256) and s.shape == (12, 2) and res.shape == x3.shape
    n0, r0 = GatedAddRMSNorm()(d["x"][:0], d["r"][:0], d["w"])
    assert n0.shape == r0.shape == (0, 256)


def test_in_place_residual(gpu_device):
    from kb_nano_amd import GatedAddRMSNorm, _ops
    for H in (1024, 16392):
        d = make(9, H, BF16, True, "full", 3, gpu_device)
        n, r = GatedAddRMSNorm()(d["x"], d["r"], d["w"], d["post"], d["g"], 0.5)
        own, out = d["r"].clone(), torch.empty_like(d["x"])
        _ops.gated_add_rmsnorm(d["x"], own, d["w"], d["post"], d["g"], 0.5, 1e-6, own, out, None, None)
        assert torch.equal(own, r) and torch.equal(out, n)


def test_zeros_infinities_and_small_values(gpu_device):
    """Rows of zeros, rows with an infinity or a NaN, subnormal rows: each row by itself, the others as ever."""
    from kb_nano_amd import GatedAddRMSNorm, GatedAddRMSNormFP8Quant
    d = make(6, 520, BF16, True, "channel", 8, gpu_device)
    args = (d["w"], d["post"], d["g"], 1.0, 1e-6)
    ref = GatedAddRMSNorm()(d["x"], d["r"], *args)
    d["x"][0], d["r"][0] = 0, 0
    d["x"][2, 7] = float("inf")
    d["r"][3, 9] = float("nan")
    d["x"][4], d["r"][4] = 1e-39, 1e-39
    n, r = GatedAddRMSNorm()(d["x"], d["r"], *args)
    q, s, r2 = GatedAddRMSNormFP8Quant()(d["x"], d["r"], *args)
    for row in (1, 5):
        assert torch.equal(n[row], ref[0][row]) and torch.equal(r[row], ref[1][row])
    assert bool((n[0] == 0).all()) and bool((q[0].float() == 0).all()) and bool((r[0] == 0).all())
    assert bool(torch.isnan(r[2, 7])) and bool((r[2, :7] == d["r"][2, :7]).all())      # inf / inf, and x / inf = 0
    assert bool(torch.isnan(n[3]).all()) and bool(torch.isnan(r[3, 9])) and int(torch.isnan(r[3]).sum()) == 1
    assert bool(torch.isfinite(n[4]).all())
    assert torch.equal(r.view(torch.int16), r2.view(torch.int16))


def test_captured_and_on_a_stream(gpu_device):
    from kb_nano_amd import GatedAddRMSNorm, GatedAddRMSNormFP8Quant
    d = make(50, 1024, BF16, True, "token", 8, gpu_device)
    args = (d["x"], d["r"], d["w"], d["post"], d["g"], 0.75)

    def call():
        return [*GatedAddRMSNorm()(*args), *GatedAddRMSNormFP8Quant()(*args)]
    refs = call()
    replayed(lambda: [t if t.is_contiguous() else t.t() for t in call()], [t if t.is_contiguous() else t.t() for t in refs],
             lambda: (call(), torch.cuda.synchronize()))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        outs = call()
    side.synchronize()
    assert all(torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8)) for a, b in zip(outs, refs))


def test_as_the_rmsnorm_module_where_they_meet(gpu_device):
    """Nothing added: the normed rows of the residual itself, as RMSNormFP8Quant's codes up to their own rounding."""
    from kb_nano_amd import GatedAddRMSNormFP8Quant, RMSNormFP8Quant
    d = make(20, 2048, BF16, False, "none", 8, gpu_device)
    q, s, r = GatedAddRMSNormFP8Quant()(torch.zeros_like(d["x"]), d["r"], d["w"])
    q2, s2 = RMSNormFP8Quant()(d["r"], d["w"])
    assert torch.equal(r, d["r"]) and s.stride() == s2.stride()
    v = rms(r.double(), d["w"].double(), 1e-6)
    assert_codes(q, s, v, norm_error(2048), "gated")
    assert_codes(q2, s2, v, norm_error(2048), "plain")


def test_refusals(gpu_device):
    from kb_nano_amd import GatedAddRMSNorm, GatedAddRMSNormFP8Quant
    norm = GatedAddRMSNorm()
    d = make(4, 256, BF16, True, "channel", 8, gpu_device)
    x, r, w = d["x"], d["r"], d["w"]
    with pytest.raises(TypeError, match="input must be"):
        norm(x.double(), r.double(), w.double())
    for other in ((x, r.float(), w), (x, r, w.float()), (x, r, w, w.float()), (x, r, w, None, w.float())):
        with pytest.raises(TypeError, match="must be torch.bfloat16"):
            norm(*other)
    with pytest.raises(ValueError, match="differ"):
        norm(x, r[:3], w)
    with pytest.raises(ValueError, match="multiple of 8"):
        norm(x[:, :252], r[:, :252], w[:252])
    with pytest.raises(ValueError, match="weight must be"):
        norm(x, r, w[:128])
    with pytest.raises(ValueError, match="broadcast"):
        norm(x, r, w, None, w[:128])
    with pytest.raises(ValueError, match="contiguous rows"):
        norm(x.t().contiguous().t(), r, w)
    with pytest.raises(RuntimeError, match="16-byte"):
        norm(x[:, 4:252], r[:, 4:252], w[:248])
    with pytest.raises(RuntimeError, match="must be on"):
        GatedAddRMSNormFP8Quant()(x, r.cpu(), w)
