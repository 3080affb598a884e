"""The router's product where every bit of an fp32 weight counts, and its infinities, in every variant that takes
fp32 operands apart: up to 16 tokens, tiles of 16 and 32 experts with and without splits of K, tiles of 128 x 128."""
import pytest
import torch

pytestmark = pytest.mark.gpu
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32

TYPES = [(BF16, F32), (F16, F32), (F32, F32)]
# (up to 16 tokens; tiles of 16 experts, with splits of K; of 32, with splits; of 128 x 128 with splits and without)
SIZES = [(1, 40, 264), (12, 17, 2056), (16, 129, 520), (17, 8, 264), (33, 16, 2056), (61, 256, 7168), (513, 300, 264), (6000, 40, 264),
         (40, 320, 2056), (200, 129, 7176), (1101, 250, 7176), (9000, 256, 520)]


def full_bits(shape, seed, dev):
    """Multiples of 2^-23 in +-[1, 2): all 24 bits of the significand in use."""
    g = torch.Generator(device=dev).manual_seed(seed)
    m = torch.randint(0, 1 << 23, shape, device=dev, generator=g)
    sign = 1 - 2 * torch.randint(0, 2, shape, device=dev, generator=g)
    return ((m + (1 << 23)) * sign).double().mul_(2.0 ** -23).float()


def places(T, H, dev):
    """Two columns for each row, all of K over the rows."""
    t = torch.arange(T, device=dev)
    return (t * 37 + 5) % H, (t * 101 + H // 2 + 3) % H


@pytest.mark.parametrize("x_dtype,w_dtype", TYPES)
@pytest.mark.parametrize("T,E,H", SIZES)
def test_weights_count_to_their_last_bit(gpu_device, T, E, H, x_dtype, w_dtype):
    """Rows of one power of two give the weight's own bits; rows of two, 1 and -1, the difference of two weights (or
    their sum's negative): multiples of 2^-23 below 4, exact in fp32 as long as every partial sum is below 2."""
    from kb_nano_amd import MoeRouterGemm
    print(f"router bits {T} x {E} x {H} {x_dtype}", flush=True)
    w = full_bits((E, H), T + E, gpu_device)
    one, two = places(T, H, gpu_device)
    two = torch.where(two == one, (one + 1) % H, two)
    rows = torch.arange(T, device=gpu_device)
    p = torch.exp2((rows % 9 - 4).float())
    x = torch.zeros(T, H, device=gpu_device)
    x[rows, one] = p
    x = x.to(x_dtype)
    assert torch.equal(MoeRouterGemm()(x, w), p[:, None] * w[:, one].t())
    w = w.abs()      # the leading pieces cancel
    x = torch.zeros(T, H, device=gpu_device)
    x[rows, one], x[rows, two] = 1.0, -1.0
    x = x.to(x_dtype)
    assert torch.equal(MoeRouterGemm()(x, w), w[:, one].t() - w[:, two].t())


@pytest.mark.parametrize("T,E,H", SIZES)
def test_rows_count_to_their_last_bit(gpu_device, T, E, H):
    from kb_nano_amd import MoeRouterGemm
    print(f"router row bits {T} x {E} x {H}", flush=True)
    x = full_bits((T, H), T, gpu_device)
    one, _ = places(E, H, gpu_device)
    w = torch.zeros(E, H, device=gpu_device)
    w[torch.arange(E, device=gpu_device), one] = 0.25
    assert torch.equal(MoeRouterGemm()(x, w), 0.25 * x[:, one])


@pytest.mark.parametrize("T,E,H", SIZES)
def test_products_of_fp32_values_lose_little(gpu_device, T, E, H):
    """One product a logit: off by the products of pieces that are left out, 2^-21 of it in all, and the roundings of
    at most six sums, 2^-23 each; the largest loss is at significands of 1 + 2^-7 - 2^-23."""
    from kb_nano_amd import MoeRouterGemm
    print(f"router products {T} x {E} x {H}", flush=True)
    worst = 1 + 2.0 ** -7 - 2.0 ** -23
    x, w = full_bits((T, H), T, gpu_device), full_bits((E, H), E, gpu_device)
    x[::2], w[::2] = worst, worst
    one = 77 % H
    keep = torch.zeros(H, device=gpu_device)
    keep[one] = 1.0
    w = w * keep
    out = MoeRouterGemm()(x, w)
    ref = x[:, one].double()[:, None] * w[:, one].double()
    assert bool(((out.double() - ref).abs() <= (2.0 ** -21 + 6 * 2.0 ** -23) * ref.abs()).all())


@pytest.mark.parametrize("x_dtype,w_dtype", [*TYPES, (BF16, BF16), (F16, F16)])
@pytest.mark.parametrize("T,E,H", SIZES)
def test_infinities_are_those_of_the_formula(gpu_device, T, E, H, x_dtype, w_dtype):
    """An infinite value gives infinite logits of its sign (NaN against 0, or against an infinity of the other sign), for
    any number of tokens; weights of few bits among them, whose lower pieces are 0."""
    from kb_nano_amd import MoeRouterGemm
    print(f"router infinities {T} x {E} x {H} {x_dtype} {w_dtype}", flush=True)
    inf = float("inf")
    g = torch.Generator(device=gpu_device).manual_seed(T)
    x, w = torch.randn(T, H, device=gpu_device, generator=g), torch.randn(E, H, device=gpu_device, generator=g) * 0.05
    w[::3] = torch.where(w[::3] < 0, -0.5, 0.25)     # one piece each
    w[1, ::2] = 0.0
    x[0, 78] = inf
    w[E - 1, 5] = -inf
    if T > 2:
        x[1, 131] = -inf
        x[2, 7], x[2, 200] = inf, -inf
        x[T - 1, 5] = 0.0
    x, w = x.to(x_dtype), w.to(w_dtype)
    out = MoeRouterGemm()(x, w).cpu()
    ref = (x.double() @ w.double().t()).cpu()
    assert torch.equal(torch.isnan(out), torch.isnan(ref))
    assert torch.equal(out == inf, ref == inf) and torch.equal(out == -inf, ref == -inf)
    assert int(torch.isinf(ref).sum()) > 0
