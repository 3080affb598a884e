"""FewTokenExperts on the GPU against the layer's formula in 64 bits."""
import pytest
import torch

from tests._mx_util import random_mx, values

pytestmark = pytest.mark.gpu

FP8 = torch.float8_e4m3fn


def make(T, E, H, I, topk, w, dtype, seed, dev, spread=True):
    """Inputs, and the weights' float64 values."""
    g = torch.Generator().manual_seed(seed)
    d = {"x": torch.randn(T, H, generator=g).to(dtype).to(dev)}
    ids = torch.stack([torch.randperm(E, generator=g)[:topk] for _ in range(T)]) if spread else \
        torch.randperm(E, generator=g)[:topk].repeat(T, 1)
    d["ids"] = ids.to(torch.int32).to(dev)
    d["tw"] = torch.softmax(torch.randn(T, topk, generator=g), -1).to(dev)
    for name, rows, K in (("13", 2 * I, H), ("2", H, I)):
        if w == "fp8":
            codes = (torch.randn(E, rows, K, generator=g) * 100).clamp(-448, 448).to(FP8).to(dev)
            s = (torch.rand(E, rows // 128, K // 128, generator=g) * 3e-4 + 1e-4).to(dev)
            v = codes.double() * s.double().repeat_interleave(128, 1).repeat_interleave(128, 2)
        else:
            codes, s = random_mx((E, rows, K), seed + rows, dev, 2)
            s -= 3
            v = values(codes, s)
        d["w" + name], d["s" + name], d["v" + name] = codes, s, v
    d["E"], d["block"] = E, [128, 128] if w == "fp8" else [1, 32]
    return d


def call(d, **over):
    from kb_nano_amd import FewTokenExperts
    a = {**d, **over}
    return FewTokenExperts()(a["x"], a["w13"], a["w2"], a["tw"], a["ids"], a["E"], a["s13"], a["s2"], a["block"])


def check(d, out, what):
    """Bound: each fp32 sum of n products is off by at most (n / 32 + 16) 2^-23 of the sum of magnitudes
    (32 products a matrix instruction, and the joins); |silu'| < 1.1, the exponential and the quotient
    add 2^-18 of h; h as two bf16 values is off by 2^-16; the result is rounded once (half a step of its type)."""
    x, I = d["x"].double(), d["v13"].shape[1] // 2
    T, H = x.shape
    ref, err = torch.zeros(T, H, dtype=torch.float64, device=x.device), torch.zeros(T, H, dtype=torch.float64, device=x.device)
    for t in range(T):
        for j in range(d["ids"].shape[1]):
            e = int(d["ids"][t, j])
            if not 0 <= e < d["E"]:
                continue
            w13, w2, c = d["v13"][e], d["v2"][e], d["tw"][t, j].double()
            gu, mag = w13 @ x[t], w13.abs() @ x[t].abs()
            gate, up = gu[:I], gu[I:]
            act = gate / (1 + torch.exp(-gate))
            h = act * up
            eh = (H / 32 + 16) * 2.0 ** -23 * (1.1 * mag[:I] * up.abs() + act.abs() * mag[I:]) + (2.0 ** -18 + 2.0 ** -16) * h.abs()
            ref[t] += c * (w2 @ h)
            err[t] += c.abs() * (w2.abs() @ (eh + (I / 32 + 16) * 2.0 ** -23 * h.abs()))
    got = out.double()
    err += torch.finfo(out.dtype).eps / 2 * ref.abs()
    if out.dtype is torch.float16:
        err += 2.0 ** -25   # half a subnormal step
    bad = ~((got - ref).abs() <= err)
    assert not bool(bad.any()), f"{what}: {int(bad.sum())} of {bad.numel()} outside, first at {tuple(bad.nonzero()[0].tolist())}"


SHAPES = [(1, 8, 256, 128, 2), (1, 256, 512, 256, 8), (2, 16, 128, 384, 4), (5, 128, 1024, 256, 8), (15, 4, 256, 256, 1),
          (16, 64, 512, 128, 8), (17, 32, 256, 512, 6), (31, 8, 384, 128, 8), (33, 256, 256, 128, 8), (48, 3, 128, 128, 3),
          (64, 100, 256, 256, 8), (64, 1024, 128, 128, 32)]


@pytest.mark.parametrize("w", ["fp8", "mxfp4"])
@pytest.mark.parametrize("T,E,H,I,topk", SHAPES)
def test_layer(gpu_device, T, E, H, I, topk, w):
    print(f"few-token experts T={T} E={E} H={H} I={I} topk={topk} {w}", flush=True)
    dtype = torch.float16 if T % 3 == 0 else torch.bfloat16
    for dt in {dtype, torch.bfloat16} if T < 20 else {dtype}:
        d = make(T, E, H, I, topk, w, dt, T + E, gpu_device)
        out = call(d)
        assert out.dtype is dt and out.shape == (T, H)
        check(d, out, f"T={T} E={E} {w} {dt}")
        assert torch.equal(out, call(d, ids=d["ids"].long()))     # int64 ids; the same bits every time


@pytest.mark.parametrize("w", ["fp8", "mxfp4"])
@pytest.mark.parametrize("T", [3, 20, 64])
def test_every_token_on_the_same_experts(gpu_device, T, w):
    print(f"few-token experts, all on the same, T={T} {w}", flush=True)
    d = make(T, 32, 256, 128, 4, w, torch.bfloat16, T, gpu_device, spread=False)
    check(d, call(d), f"T={T} {w}")


@pytest.mark.parametrize("w", ["fp8", "mxfp4"])
@pytest.mark.parametrize("T", [4, 40])
def test_ids_twice_outside_and_none(gpu_device, T, w):
    """An expert named twice by a token, ids of other ranks, a token that names none, weights of zero
    and below; and a whole batch without an expert."""
    print(f"few-token experts odd ids T={T} {w}", flush=True)
    d = make(T, 16, 256, 256, 4, w, torch.bfloat16, 3, gpu_device)
    d["ids"][0, 1] = d["ids"][0, 0]
    d["ids"][1] = d["ids"][1, 2]
    d["ids"][2, 0], d["ids"][2, 3] = -1, 16
    d["ids"][3] = torch.tensor([-1, 99, 2 ** 31 - 1, -2 ** 31], dtype=torch.int32)
    d["tw"][0, 2], d["tw"][0, 3] = 0.0, -0.7
    out = call(d)
    check(d, out, f"T={T}")
    assert bool((out[3] == 0).all())
    d["ids"].fill_(-1)
    assert bool((call(d) == 0).all())


@pytest.mark.parametrize("w", ["fp8", "mxfp4"])
def test_nonfinite_values_stay_with_their_tokens(gpu_device, w):
    """An infinite activation, a NaN weight and a NaN scale reach the tokens that use them and no others."""
    print(f"few-token experts nonfinite {w}", flush=True)
    d = make(9, 8, 256, 128, 2, w, torch.bfloat16, 5, gpu_device)
    d["ids"] = torch.tensor([[0, 1], [1, 2], [2, 3], [3, 4], [4, 5], [5, 0], [1, 3], [0, 2], [4, 1]], dtype=torch.int32,
                            device=gpu_device)
    base = call(d)
    x = d["x"].clone()
    x[4, 100] = float("inf")
    out = call(d, x=x)
    assert not bool(torch.isfinite(out[4]).any())
    keep = torch.arange(9, device=gpu_device) != 4
    assert torch.equal(out[keep], base[keep])
    for name in ("2", "13"):
        wt, s = d["w" + name].clone(), d["s" + name].clone()
        if w == "fp8":
            wt.view(torch.uint8)[5, 7, 3] = 0x7F
        else:
            s[5, 7, 1] = 255
        out = call(d, **{"w" + name: wt, "s" + name: s})
        hit = (d["ids"] == 5).any(1)
        assert torch.equal(out[~hit], base[~hit])
        assert bool(torch.isnan(out[hit]).any(1).all())
    if w == "fp8":
        s = d["s2"].clone()
        s[5, 0, 0] = float("inf")
        out = call(d, s2=s)
        assert torch.equal(out[~hit], base[~hit]) and not bool(torch.isfinite(out[hit][:, :128]).any())


def test_strided_inputs_no_tokens_and_compile(gpu_device):
    from kb_nano_amd import FewTokenExperts
    print("few-token experts strides", flush=True)
    d = make(6, 16, 256, 128, 4, "fp8", torch.bfloat16, 11, gpu_device)
    ref = call(d)
    wide = torch.full((6, 512), float("nan"), dtype=torch.bfloat16, device=gpu_device)
    wide[:, 128:384] = d["x"]
    routing = torch.stack([d["ids"], d["ids"]], -1)[..., 0]
    assert torch.equal(call(d, x=wide[:, 128:384], ids=routing), ref)
    assert call(d, x=d["x"][:0], ids=d["ids"][:0], tw=d["tw"][:0]).shape == (0, 256)
    layer = FewTokenExperts()
    torch._dynamo.reset()
    f = torch.compile(lambda x: layer(x, d["w13"], d["w2"], d["tw"], d["ids"], 16, d["s13"], d["s2"], [128, 128]),
                      fullgraph=True, backend="aot_eager")
    assert torch.equal(f(d["x"]), ref)


@pytest.mark.parametrize("w", ["fp8", "mxfp4"])
def test_graphs_and_streams(gpu_device, w):
    """Replays with other tokens and routing, eager calls between, two graphs, two streams at once."""
    print(f"few-token experts graphs {w}", flush=True)
    ds = [make(7, 32, 256, 256, 4, w, torch.bfloat16, 1, gpu_device)]
    for seed in (21, 22, 23):
        o = make(7, 32, 256, 256, 4, w, torch.bfloat16, seed, gpu_device)
        ds.append({**ds[0], "x": o["x"], "ids": o["ids"], "tw": o["tw"]})
    refs = [call(d).clone() for d in ds]
    live = {**ds[0], "x": ds[0]["x"].clone(), "ids": ds[0]["ids"].clone(), "tw": ds[0]["tw"].clone()}
    graphs = []
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=side):
                out = call(live)
                out2 = call(live)
            graphs.append((g, out, out2))
    torch.cuda.synchronize()
    for i, d in enumerate(ds):
        for k in ("x", "ids", "tw"):
            live[k].copy_(d[k])
        for g, _, _ in graphs:
            g.replay()
            eager = call(ds[(i + 1) % 4])
        torch.cuda.synchronize()
        assert torch.equal(eager, refs[(i + 1) % 4])
        assert all(torch.equal(o, refs[i]) and torch.equal(o2, refs[i]) for _, o, o2 in graphs)
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    for i in range(8):
        with torch.cuda.stream(streams[i % 2]):
            outs.append(call(ds[i % 4]))
    torch.cuda.synchronize()
    assert all(torch.equal(o, refs[i % 4]) for i, o in enumerate(outs))


def test_a_decode_step_together(gpu_device):
    """Projection, experts quantized by Mxfp4Quant and projection back, as a decode step chains them, with
    the weights' values read back for the reference; the experts also near VllmFusedExperts' FP8 chain,
    whose activations have 4 significant bits (2^-4 of each, independent over hundreds of terms)."""
    from kb_nano_amd import FewTokenExperts, Mxfp4Linear, Mxfp4Quant, VllmFusedExperts, dequantize_mxfp4
    print("decode step with MXFP4", flush=True)
    T, E, H, I, topk = 6, 8, 512, 256, 2
    g = torch.Generator().manual_seed(9)
    quant, lin = Mxfp4Quant(), Mxfp4Linear()
    x = torch.randn(T, H, generator=g).bfloat16().to(gpu_device)
    wp, sp = quant((torch.randn(H, H, generator=g) * 0.05).to(gpu_device))
    d = {"E": E, "block": [1, 32]}
    d["w13"], d["s13"] = quant((torch.randn(E, 2 * I, H, generator=g) * 0.05).to(gpu_device))
    d["w2"], d["s2"] = quant((torch.randn(E, H, I, generator=g) * 0.05).to(gpu_device))
    d["v13"], d["v2"] = dequantize_mxfp4(d["w13"], d["s13"], torch.float32).double(), dequantize_mxfp4(d["w2"], d["s2"], torch.float32).double()
    d["x"] = lin(x, wp, sp)
    tw, ids = torch.topk(torch.softmax(torch.randn(T, E, generator=g), -1), topk)
    d["tw"], d["ids"] = tw.to(gpu_device), ids.to(gpu_device)
    y = call(d)
    check(d, y, "chained")
    z = lin(y, wp, sp)
    assert z.shape == (T, H) and bool(torch.isfinite(z).all())
    f = make(T, E, H, I, topk, "fp8", torch.bfloat16, 2, gpu_device)
    f["s13"], f["s2"] = f["s13"] * 0 + 2.0 ** -12, f["s2"] * 0 + 2.0 ** -12
    a = call(f).double()
    b = VllmFusedExperts()(f["x"], f["w13"], f["w2"], f["tw"], f["ids"], E, f["s13"], f["s2"], [128, 128]).double()
    assert float((a - b).norm() / a.norm()) < 2.0 ** -4
