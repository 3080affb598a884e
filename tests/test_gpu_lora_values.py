"""What the adapters' second product keeps of h: both bf16 numbers it is made of, their products with every bit of B,
and values near fp32's largest."""
import pytest
import torch

from tests._layer_util import half_step

pytestmark = pytest.mark.gpu
BF16, F16, F32, F64 = torch.bfloat16, torch.float16, torch.float32, torch.float64


def of_three(T, L, R, seed, dev, one=False):
    """A [L, R, K] and x [T, K] with h[t, r] = a0 + 2^-8 a1 + 2^-16 a2 of eight-bit a's in [1, 2), exact in fp32 (x is
    16, 2^-4 and 2^-12 and the scaling 1 / 16: nothing is subnormal in fp16).  Odd ranks leave a2 out (16 bits: two
    bf16 numbers hold them) and have the a0 and a1 of the even rank before."""
    g = torch.Generator(device=dev).manual_seed(seed)
    a = 1 + torch.randint(0, 128, (L, R, 3), device=dev, generator=g).double() / 128
    a[..., 0] = 1.0 if one else 1 + torch.randint(0, 100, (L, R), device=dev, generator=g).double() / 128
    a[:, 1::2] = a[:, ::2]
    a[:, 1::2, 2] = 0.0
    full = torch.zeros(L, R, 64, dtype=F64, device=dev)
    full[..., 3], full[..., 40], full[..., 63] = a.unbind(-1)
    x = torch.zeros(T, 64, dtype=F64, device=dev)
    x[:, 3], x[:, 40], x[:, 63] = 16.0, 2.0 ** -4, 2.0 ** -12
    return x, full


def check(x, base, a, b, ids, s, what):
    """Against the formula in 64 bits: h in two bf16 numbers, each rounded to nearest (2^-8 of what is left, so 2^-16
    of h), fp32 sums of at most four products of magnitude |h| |b| each 32 ranks (2^-23), one rounding of the result."""
    from kb_nano_amd import LoraAdd
    out = LoraAdd()(x, base, a, b, ids, s)
    ref, tol = base.double().clone(), torch.zeros(base.shape, dtype=F64, device=base.device)
    R = a.shape[1]
    for l in range(a.shape[0]):
        t = (ids == l).nonzero().flatten()
        h = x[t].double() @ a[l].double().t() * s[l].double()
        ref[t] += h @ b[l].double().t()
        loose = (2.0 ** -16 + (R / 8 + 4) * 2.0 ** -23) * h.abs()
        loose[:, 1::2] -= 2.0 ** -16 * h[:, 1::2].abs()      # odd ranks are two bf16 numbers exactly
        tol[t] = loose @ b[l].double().abs().t()
    tol += half_step(base.dtype) * ref.abs() * (1 + 2.0 ** -10) + 2.0 ** -126
    off = (out.double() - ref).abs()
    assert bool((off <= tol).all()), f"{what}: {int((off > tol).sum())} outside, worst {float((off / tol).max()):.3g} of the bound"


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("T,N,L,R", [(1, 64, 1, 8), (20, 100, 3, 16), (40, 63, 2, 32), (70, 256, 2, 64), (300, 260, 4, 136)])
def test_h_keeps_sixteen_bits(gpu_device, T, N, L, R, dtype):
    """Columns of B in pairs b, -b: the sums of 16-bit numbers cancel and leave the lowest bits of h.  Without the
    lower ones' roundings, 2^-15 of h would be lost; of fp16 B (11 bits) 2^-14 more without the product of both low parts."""
    print(f"lora h bits {T} x {N} rank {R} {dtype}", flush=True)
    for one in (True, False):
        x, a = of_three(T, L, R, T + R, gpu_device, one)
        g = torch.Generator(device=gpu_device).manual_seed(R)
        b = torch.zeros(L, N, R, dtype=F64, device=gpu_device)
        b[..., ::2] = (1 + torch.rand(L, N, R // 2, dtype=F64, device=gpu_device, generator=g)).to(dtype).double()
        b[:, 0] = 1 + 2.0 ** -7 - 2.0 ** -10 if dtype is F16 else 1.0    # a low part as large as it can be
        pick = torch.arange(N, device=gpu_device) * 2 % R                   # one pair a column, or all of them
        keep = (torch.arange(R, device=gpu_device) // 2 * 2 == pick[:, None]) | (torch.arange(N, device=gpu_device)[:, None] % 5 == 4)
        b[..., 1::2] = -b[..., ::2]
        b = torch.where(keep, b, 0.0)
        ids = torch.arange(T, device=gpu_device, dtype=torch.int32) % L
        s = torch.full((L,), 2.0 ** -4, device=gpu_device)
        base = torch.zeros(T, N, dtype=dtype, device=gpu_device)
        check(x.to(dtype), base, a.to(dtype), b.to(dtype), ids, s, f"{T}x{N} rank {R}")


def test_large_h(gpu_device):
    """h next to fp32's largest value, where a bf16 number above it would be an infinity, brought back by B."""
    from kb_nano_amd import LoraAdd
    big = 2.0 ** 127 * (1 + 127 / 128)         # the largest bf16 number; h = big (1 + 2^-8 - 2^-15) and the like
    x = torch.zeros(4, 64, dtype=F64, device=gpu_device)
    x[:, 0], x[1, 1], x[2, 1], x[3, 0] = 2.0 ** 60, 2.0 ** 52, 2.0 ** 51, -2.0 ** 60
    x[3, 1] = -2.0 ** 52
    a = torch.zeros(1, 8, 64, dtype=F64, device=gpu_device)
    a[0, :, 0], a[0, :, 1] = big / 2.0 ** 60, 2.0 ** 67 * (1 + 126 / 128)
    b = torch.zeros(1, 64, 8, dtype=F64, device=gpu_device)
    b[0, torch.arange(64), torch.arange(64) % 8] = 2.0 ** -20
    h = x @ a[0].t()
    assert float(h.abs().max()) < torch.finfo(F32).max and float(h.abs().max()) > big * (1 + 2.0 ** -9)
    ids = torch.zeros(4, dtype=torch.int64, device=gpu_device)
    out = LoraAdd()(x.to(BF16), torch.zeros(4, 64, dtype=BF16, device=gpu_device), a.to(BF16), b.to(BF16), ids)
    ref = h @ b[0].t()
    assert bool(((out.double() - ref).abs() <= half_step(BF16) * (1 + 2.0 ** -6) * ref.abs()).all())
