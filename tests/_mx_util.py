"""Plain MXFP4 in 64 bits for the tests: quantization, values and products from
the format's definition."""
from __future__ import annotations

import torch

E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def quant_plain(x: torch.Tensor):
    """(codes uint8 [M, K/2], bytes uint8 [M, K/32]) of float rows on the CPU, one group at a time
    in the terms of the definition: the largest magnitude over the scale lies in [3.5, 7)."""
    v = x.detach().cpu().double().reshape(-1, 32)
    fine = torch.isfinite(v).all(1)
    a = torch.where(fine.unsqueeze(1), v.abs(), torch.zeros_like(v))
    m, e = torch.frexp(a.amax(1))                       # in [1/2, 1) times 2^e
    exp = torch.where(a.amax(1) > 0, e - 3 + (m >= 0.875).int(), torch.full_like(e, -200)).clamp(min=-126)
    q = a / torch.ldexp(torch.ones_like(m), exp).unsqueeze(1)
    code = torch.zeros_like(q, dtype=torch.int64)
    for i in range(7):                                  # past the middle (or on it, to the even code): one more
        mid = (E2M1[i] + E2M1[i + 1]) / 2
        code += ((q >= mid) if i % 2 else (q > mid)).long()
    code += 8 * torch.signbit(v).long()
    code = torch.where(fine.unsqueeze(1), code, torch.zeros_like(code)).reshape(x.shape)
    byte = torch.where(fine, exp.long() + 127, torch.full_like(exp.long(), 255))
    return (code[:, ::2] + 16 * code[:, 1::2]).to(torch.uint8), byte.reshape(x.shape[0], -1).to(torch.uint8)


def values(codes: torch.Tensor, byte: torch.Tensor) -> torch.Tensor:
    """float64 [..., K] of packed codes and scale bytes (on their device)."""
    c = codes.view(torch.uint8).long()
    c = torch.stack((c % 16, c // 16), -1).flatten(-2)
    mag = torch.tensor(E2M1, dtype=torch.float64, device=c.device)[c % 8]
    b = byte.view(torch.uint8).double().repeat_interleave(32, -1)
    s = torch.where(b == 255, torch.full_like(b, float("nan")), torch.exp2(b - 127))
    return torch.where(c >= 8, -mag, mag) * s


def random_mx(shape, seed: int, device, spread: int = 6):
    """Random codes [..., K/2] and scale bytes (around 2^-4, `spread` binades)."""
    g = torch.Generator().manual_seed(seed)
    codes = torch.randint(0, 256, (*shape[:-1], shape[-1] // 2), generator=g, dtype=torch.uint8)
    byte = torch.randint(123 - spread // 2, 124 + spread // 2, (*shape[:-1], shape[-1] // 32), generator=g).to(torch.uint8)
    return codes.to(device), byte.to(device)


def assert_product(out: torch.Tensor, a: torch.Tensor, w: torch.Tensor, what: str) -> None:
    """`out` (bf16) against a [M, K] w [N, K]^T in 64 bits.  The products are exact in fp32 (2 + 2 bits
    of significand), each matrix instruction adds at most 128 of them to the running fp32 sum with an
    error of at most a unit in the last place of the sum of magnitudes so far, a few instructions or
    partial sums meet at the end: (K / 128 + 8) 2^-23 sum |a w|.  The result is rounded to bf16 once:
    2^-8 of the value."""
    ref, mag = a @ w.t(), a.abs() @ w.abs().t()
    tol = 2.0 ** -8 * ref.abs() + (a.shape[1] / 128 + 8) * 2.0 ** -23 * mag
    got = out.double()
    nan = torch.isnan(ref)
    assert torch.equal(torch.isnan(got), nan), f"{what}: NaN in other places"
    bad = ((got - ref).abs() > tol) & ~nan
    assert not bool(bad.any()), (f"{what}: {int(bad.sum())} of {bad.numel()} outside, first at "
                                 f"{tuple(bad.nonzero()[0].tolist())}, worst {float(((got - ref).abs() / tol)[~nan].max()):.3g}")
