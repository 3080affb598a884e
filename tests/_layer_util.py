"""Plain forms in 64 bits, from the definitions, for the tests of the router, the gated norms and the
adapters, and how far the kernels may be from them."""
from __future__ import annotations

import math

import torch

F64 = torch.float64


def half_step(dtype) -> float:
    """Largest relative error of one rounding to nearest."""
    return torch.finfo(dtype).eps / 2


def routing_plain(logits, top_k, scoring="softmax", bias=None, num_groups=1, topk_groups=1, renormalize=True, scale=1.0):
    """(weights float64, ids int64), token by token on the CPU: experts sorted by (choice, index)."""
    rows, E = logits.detach().cpu().double().tolist(), logits.shape[1]
    b = None if bias is None else bias.detach().cpu().double().tolist()
    low, per = -math.inf, E // num_groups
    weights, ids = [], []
    for row in rows:
        row = [low if math.isnan(v) else min(v, 3.4028234663852886e38) for v in row]
        if scoring == "softmax":
            top = max(row) if max(row) > low else 0.0
            e = [math.exp(v - top) if v > low else 0.0 for v in row]
            total = math.fsum(e)
            score = [v / total if total > 0 else 0.0 for v in e]
        else:
            score = [0.0 if v < -709 else 1.0 / (1.0 + math.exp(-v)) for v in row]
        c = list(row) if b is None else [low if row[i] == low else score[i] + b[i] for i in range(E)]
        if num_groups > 1:
            def rank(g):
                top2 = sorted(c[g * per:(g + 1) * per], reverse=True)[:2]
                return top2[0] if b is None else sum(top2)
            kept = sorted(range(num_groups), key=lambda g: (-rank(g), g))[:topk_groups]
            c = [c[i] if i // per in kept else low for i in range(E)]
        chosen = sorted(range(E), key=lambda i: (-c[i], i))[:top_k]
        w = [0.0 if c[i] == low else score[i] for i in chosen]
        if renormalize:
            total = math.fsum(w)
            w = [v / total if total > 0 else 0.0 for v in w]
        weights.append([v * scale for v in w])
        ids.append(chosen)
    return torch.tensor(weights, dtype=F64).reshape(-1, top_k), torch.tensor(ids, dtype=torch.int64).reshape(-1, top_k)


def assert_routing(weights, ids, plain, what) -> None:
    """The same experts; weights computed in 64 bits and rounded to fp32 once (2^-24, and 2^-40 for the
    64-bit exponentials, or half of fp32's smallest subnormal step)."""
    w, i = plain
    assert torch.equal(ids.cpu().long(), i), f"{what}: other experts in {int((ids.cpu().long() != i).any(1).sum())} tokens"
    off = (weights.cpu().double() - w).abs()
    tol = w.abs() * (2.0 ** -24 + 2.0 ** -40) + 2.0 ** -149
    assert bool((off <= tol).all()), f"{what}: weights off by {float((off / tol).max()):.3g} of the bound"


def assert_gate(out, x, w, what) -> None:
    """Logits against x w^T in 64 bits.  Every instruction adds at most 32 products to a running fp32 sum,
    off by at most a unit in the last place (2^-23) of the sum of magnitudes; fp32 operands are three bf16
    numbers each, so at most six such sums run over K, and what is left out is three products of pieces
    below 2^-24 of the largest.  16 partial sums meet at the end."""
    x, w = x.double(), w.double()
    ref, mag = x @ w.t(), x.abs() @ w.abs().t()
    tol = (6 * x.shape[1] / 32 + 24) * 2.0 ** -23 * mag + 2.0 ** -126
    off = (out.double() - ref).abs()
    assert out.dtype == torch.float32 and out.shape == ref.shape
    assert bool((off <= tol).all()), f"{what}: {int((off > tol).sum())} outside, worst {float((off / tol).max()):.3g} of the bound"


def norm_error(H: int) -> float:
    """Relative error of x / sqrt(mean(x^2) + eps) * w in fp32: the squares are summed over at most H / 256 + 8
    of a lane's elements, 6 butterfly steps and 8 wavefronts, each step off by 2^-24 of a sum of positive
    terms; the root halves that; mean, eps, root, quotient and the two products add six roundings."""
    return ((H / 256 + 8 + 14) / 2 + 6) * 2.0 ** -24


def rms(x, w, eps):
    return x / torch.sqrt(x.square().mean(-1, keepdim=True) + eps) * w


def assert_gated(res, normed, x, r, w, post, gate, rs, eps, what) -> None:
    """residual' against the formula, normed against the formula of the residual' that was returned."""
    dt = r.dtype
    e = norm_error(x.shape[-1])
    p = x.double() if post is None else rms(x.double(), post.double(), eps)
    gp = p if gate is None else gate.double() * p
    ref = rs * r.double() + gp
    # fp32: the norm's error on p, one rounding of rs (to fp32) and one of rs r, one of the sum; then the type's
    tol = half_step(dt) * ref.abs() * (1 + 2.0 ** -10) + (e + 2.0 ** -23) * gp.abs() + 2.0 ** -22 * (rs * r.double()).abs() + _tiny(dt)
    _near(res, ref, tol, f"{what}: residual")
    if normed is not None:
        ref = rms(res.double(), w.double(), eps)
        _near(normed, ref, (half_step(dt) * (1 + 2.0 ** -10) + e) * ref.abs() + _tiny(dt), f"{what}: normed")


def _tiny(dt) -> float:
    """Half of the type's smallest subnormal step."""
    return {torch.float16: 2.0 ** -25}.get(dt, 2.0 ** -126)


def _near(got, ref, tol, what) -> None:
    assert torch.equal(torch.isnan(got.double()), torch.isnan(ref)), f"{what}: NaN in other places"
    fine = torch.isfinite(ref)
    off = (got.double() - ref).abs()
    bad = fine & ~(off <= tol)
    assert not bool(bad.any()), (f"{what}: {int(bad.sum())} of {bad.numel()} outside, first at {tuple(bad.nonzero()[0].tolist())}, "
                                 f"worst {float((off / tol)[fine].max()):.3g} of the bound")


def assert_codes(q, s, v, err, what) -> None:
    """e4m3 codes and UE8M0 scales of 1x128 groups of v (float64), known to a relative error err: scales are powers
    of two, no less than max |v| / 448 and less than twice that (or the floor of 1e-10); a code is off by half
    a step, 2^-4 of the value or 2^-10 of the scale (e4m3's subnormal step is 2^-9)."""
    T, H = v.shape
    G = -(-H // 128)
    m = torch.nn.functional.pad(v, (0, G * 128 - H)).view(T, G, 128).abs().amax(2).clamp(min=1e-10) / 448
    s = s.double()
    assert s.shape == (T, G) and bool((torch.frexp(s)[0] == 0.5).all()), f"{what}: scales are no powers of two"
    assert bool((s >= m * (1 - err)).all()) and bool((s < 2 * m * (1 + err)).all()), f"{what}: scales of another size"
    each = s.repeat_interleave(128, 1)[:, :H]
    off = (q.double() * each - v).abs()
    tol = (2.0 ** -4 + 2 * err) * v.abs() + 2.0 ** -10 * each
    assert bool((off <= tol).all()), f"{what}: {int((off > tol).sum())} codes outside"


def lora_plain(x, base, a, b, ids, scaling):
    """(out, magnitude of the error's terms) in 64 bits."""
    out, mag = base.double().clone(), torch.zeros(base.shape, dtype=F64, device=base.device)
    K, R = x.shape[1], a.shape[1]
    for l in range(a.shape[0]):
        t = (ids == l).nonzero().flatten()
        if len(t):
            s = 1.0 if scaling is None else float(scaling[l])
            xa, aa, bb = x[t].double(), a[l].double(), b[l].double()
            h, hm = xa @ aa.t(), xa.abs() @ aa.abs().t()
            out[t] += s * (h @ bb.t())
            # h: fp32 sums of 32 products an instruction, 20 partial sums; its two bf16 numbers lose 2^-15 at
            # most; the second product: three instructions for 32 ranks
            err = (K / 32 + 24) * 2.0 ** -23 * hm + 2.0 ** -15 * h.abs() + (R / 8 + 4) * 2.0 ** -23 * h.abs()
            mag[t] = abs(s) * (err @ bb.abs().t())
    return out, mag


def assert_lora(out, x, base, a, b, ids, scaling, what) -> None:
    ref, mag = lora_plain(x, base, a, b, ids, scaling)
    tol = half_step(base.dtype) * ref.abs() * (1 + 2.0 ** -10) + (1 + 2.0 ** -7) * mag + 2.0 ** -23 * base.double().abs() + _tiny(base.dtype)
    _near(out, ref, tol, what)
    none = (ids < 0) | (ids >= a.shape[0])
    assert torch.equal(out[none].view(torch.int16), base[none].view(torch.int16)), f"{what}: rows without an adapter changed"


def replayed(call, refs, eager) -> None:
    """Captures call() and replays it four times with eager work between: every replay gives refs' bits."""
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        call()
        with torch.cuda.graph(g, stream=side):
            outs = call()
    torch.cuda.current_stream().wait_stream(side)
    for _ in range(4):
        for o in outs:
            o.zero_()
        g.replay()
        torch.cuda.synchronize()
        for o, r in zip(outs, refs, strict=True):
            assert torch.equal(o.view(torch.uint8), r.view(torch.uint8))
        eager()
