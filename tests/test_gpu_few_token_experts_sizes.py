"""FewTokenExperts where a launch takes several tiles of an expert, several
passes of its tokens, a wide hidden size, or weights past 32-bit offsets."""
import pytest
import torch

from tests.test_gpu_few_token_experts import FP8, call, check, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("w", ["fp8", "mxfp4"])
@pytest.mark.parametrize("T,E,H,I,topk,spread", [(40, 96, 128, 640, 8, True), (64, 128, 128, 384, 8, True),
                                                 (64, 128, 256, 384, 8, False), (20, 128, 384, 384, 8, False),
                                                 (2, 64, 6272, 128, 2, True), (1, 64, 7168, 256, 1, True),
                                                 (12, 9, 1152, 1920, 4, True), (64, 12, 640, 128, 12, True)])
def test_tiles_and_passes(gpu_device, T, E, H, I, topk, spread, w):
    print(f"few-token experts T={T} E={E} H={H} I={I} topk={topk} spread={spread} {w}", flush=True)
    for dt in (torch.bfloat16, torch.float16):
        d = make(T, E, H, I, topk, w, dt, T + H, gpu_device, spread)
        check(d, call(d), f"T={T} {w} {dt}")


@pytest.mark.parametrize("w", ["fp8", "mxfp4"])
def test_weights_past_32_bit_offsets(gpu_device, w):
    """1024 experts, 4.3 and 2.1 GB of FP8 weights (half of that in MXFP4): the last ones and one in between."""
    print(f"few-token experts past 32 bits {w}", flush=True)
    T, E, H, I, topk = 6, 1024, 2048, 1024, 3
    some = torch.tensor([0, 700, E - 1])
    d = make(T, 3, H, I, topk, w, torch.bfloat16, 9, gpu_device)
    full = {**d, "E": E, "ids": some.to(torch.int32).to(gpu_device)[d["ids"].long()]}
    for name in ("w13", "s13", "w2", "s2"):
        big = torch.zeros(E, *d[name].shape[1:], dtype=torch.uint8 if d[name].dtype is FP8 else d[name].dtype, device=gpu_device)
        big[some] = d[name].view(big.dtype)
        full[name] = big.view(d[name].dtype)
    check(d, call(full), w)


@pytest.mark.parametrize("w", ["fp8", "mxfp4"])
def test_weights_of_slots_that_name_nobody_are_not_read(gpu_device, w):
    print(f"few-token experts NaN routing weights {w}", flush=True)
    d = make(7, 16, 256, 128, 4, w, torch.bfloat16, 2, gpu_device)
    d["ids"][::2, 1], d["tw"][::2, 1] = -1, float("nan")
    d["ids"][3], d["tw"][3] = 16, float("inf")
    out = call(d)
    check(d, out, w)
    assert bool((out[3] == 0).all())


@pytest.mark.parametrize("w", ["fp8", "mxfp4"])
def test_the_last_rows_of_the_weights_end_the_buffer(gpu_device, w):
    """Weights that end where their storage ends, with NaN codes and scales before their start."""
    print(f"few-token experts at the end of a buffer {w}", flush=True)
    d = make(3, 5, 384, 128, 2, w, torch.bfloat16, 4, gpu_device)
    d["ids"][0, 0] = 4
    d["ids"][0, 1] = 0
    for name in ("w13", "s13", "w2", "s2"):
        t = d[name]
        b = torch.full((256 + t.numel() * t.element_size(),), 0xFF, dtype=torch.uint8, device=gpu_device)
        b[256:] = t.contiguous().view(torch.uint8).flatten()
        d[name] = b[256:].view(t.dtype).view(t.shape)
    check(d, call(d), w)


@pytest.mark.parametrize("w", ["fp8", "mxfp4"])
def test_fp16_subnormal_and_large_activations(gpu_device, w):
    """fp16 activations from its smallest subnormal number to its largest, a row each; weights of E4M3's
    smallest subnormals, so that their products show."""
    print(f"few-token experts fp16 range {w}", flush=True)
    d = make(8, 6, 256, 128, 2, w, torch.float16, 5, gpu_device)
    for t, e in enumerate((-24, -20, -15, -14, -10, 0, 8, 12)):
        d["x"][t] = (d["x"][t].float().clamp(-3, 3) * 2.0 ** e).half()
    d["x"][0] = torch.where(torch.arange(256, device=gpu_device) % 3 == 0, 2.0 ** -24, 0.0).half()
    if w == "fp8":
        small = torch.randint(1, 8, (6, 256, 256), generator=torch.Generator().manual_seed(6), dtype=torch.uint8).to(gpu_device)
        d["w13"][:, :, ::2] = small.view(FP8)[:, :, ::2]
        d["s13"][:] = 2.0 ** 18   # sums that reach h from subnormal activations
        d["s13"][:, :, 1:] = 2.0 ** 17
        d["v13"] = d["w13"].double() * d["s13"].double().repeat_interleave(128, 1).repeat_interleave(128, 2)
        d["s2"][:] = 2.0 ** -40
        d["v2"] = d["w2"].double() * 2.0 ** -40
    out = call(d)
    keep = [t for t in range(8) if t < (7 if w == "mxfp4" else 5)]    # the larger rows leave fp16's range with these weights
    check({**d, "x": d["x"][keep], "ids": d["ids"][keep], "tw": d["tw"][keep]}, out[keep], w)
    if w == "mxfp4":   # 65520 and more round to infinity: 231 outputs of the last row, of up to 2.3e6
        x, ref = d["x"][7].double(), torch.zeros(256, dtype=torch.float64, device=gpu_device)
        for e, c in zip(d["ids"][7].tolist(), d["tw"][7].tolist()):
            gate, up = (d["v13"][e] @ x).chunk(2)
            ref += c * (d["v2"][e] @ (gate / (1 + torch.exp(-gate)) * up))
        over = ref.abs() >= 65520
        assert int(over.sum()) == 231 and bool((out[7][over].double() == torch.inf * ref[over].sign()).all())
        assert bool(out[7][~over].isfinite().all())


def _among(d, E, dev):
    """The same layer with its experts as some of E, the others' weights zeros."""
    n = d["E"]
    some = torch.arange(n) * (E - 1) // max(1, n - 1)
    full = {**d, "E": E, "ids": some.to(torch.int32).to(dev)[d["ids"].long()]}
    for name in ("w13", "s13", "w2", "s2"):
        big = torch.zeros(E, *d[name].shape[1:], dtype=torch.uint8 if d[name].dtype is FP8 else d[name].dtype, device=dev)
        big[some] = d[name].view(big.dtype)
        full[name] = big.view(d[name].dtype)
    return full


@pytest.mark.parametrize("w", ["fp8", "mxfp4"])
@pytest.mark.parametrize("T,n,E,H,I,topk", [(1, 8, 64, 4224, 128, 4), (3, 9, 256, 5120, 384, 3), (16, 20, 64, 5248, 256, 6),
                                            (16, 20, 64, 7168, 128, 6), (40, 6, 9, 8192, 256, 4), (64, 16, 1024, 4224, 128, 8),
                                            (64, 32, 32, 4480, 128, 32), (64, 24, 300, 7040, 256, 8), (64, 32, 900, 4224, 128, 32)])
def test_wide_hidden_sizes(gpu_device, T, n, E, H, I, topk, w):
    """More than 16 columns a CU: workgroups of 20 to 32, across the scales' blocks and past the last column."""
    print(f"few-token experts T={T} {n} of {E} H={H} I={I} topk={topk} {w}", flush=True)
    dt = torch.float16 if T == 16 else torch.bfloat16
    d = make(T, n, H, I, topk, w, dt, T + H, gpu_device)
    wide = torch.full((T, H + 24), 3.0, dtype=dt, device=gpu_device)
    full = _among(d, E, gpu_device)
    out = call(full)
    check(d, out, f"T={T} H={H} {w}")
    from kb_nano_amd import _ops
    _ops.few_token_experts(full["x"], full["w13"], full["s13"], full["w2"], full["s2"], full["tw"], full["ids"], wide[:, 8:8 + H])
    assert torch.equal(wide[:, 8:8 + H], out)
    assert bool((wide[:, :8] == 3).all() and (wide[:, 8 + H:] == 3).all())


@pytest.mark.parametrize("w", ["fp8", "mxfp4"])
@pytest.mark.parametrize("T,E,H,I,topk,spread", [(64, 12, 256, 640, 4, True), (24, 16, 384, 512, 4, True), (37, 9, 4224, 768, 2, True),
                                                 (64, 16, 128, 512, 8, False), (33, 8, 5120, 128, 1, True), (64, 14, 4224, 512, 14, True),
                                                 (20, 4, 1152, 1664, 2, True), (64, 40, 128, 256, 32, True)])
def test_many_rows_an_expert(gpu_device, T, E, H, I, topk, spread, w):
    """Passes of sixteen rows, whole ones and the rest, in both launches."""
    print(f"few-token experts T={T} E={E} H={H} I={I} topk={topk} spread={spread} {w}", flush=True)
    for dt in (torch.bfloat16, torch.float16):
        d = make(T, E, H, I, topk, w, dt, T + H, gpu_device, spread)
        out = call(d)
        check(d, out, f"T={T} {w} {dt}")
        assert torch.equal(out, call(d))
