"""Timed cases of the MXFP4 and few-token operators.

  quant     Mxfp4Quant and back (dequantize_mxfp4): 32-element groups along K with a
            power-of-two scale and 4-bit e2m1 codes
  linear    Mxfp4Linear: activations quantised as above, times an MXFP4 weight
  experts   FewTokenExperts: a whole mixture-of-experts layer (gate/up, SiLU*Mul, down,
            weighted sum) for at most 64 tokens, with 128x128-block-scaled FP8 weights
            or MXFP4 ones

``run`` computes them in elementary torch operations, in fp32 and rounded once at the
end; with ``own`` set it makes the calls of the package's modules.  Inputs are drawn on
the GPU from the seed: activations ~N(0, 1) with a few large ones, weights ~N(0, 0.02)
quantised, routing by the top-k of seeded softmax logits.
"""
import functools
import types

import torch

own = False

FP8 = torch.float8_e4m3fn
E8M0 = torch.float8_e8m0fnu
F64 = torch.float64
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}

# (N, K) of dense layers: prefill and decode layers, their shards over eight GPUs, a small one
DENSE = [(24576, 1536), (36864, 7168), (7168, 18432), (7168, 16384), (10240, 8192), (8192, 8192), (57344, 8192),
         (8192, 28672), (4608, 7168), (7168, 2048), (7168, 2304), (2048, 2048)]
# (experts, hidden, intermediate, top-k): whole layers, their shards, a small generic one
MOE = [(256, 7168, 2048, 8), (256, 7168, 256, 8), (128, 4096, 1536, 8), (128, 4096, 384, 8), (16, 2048, 1024, 4)]


def listed():
    return [
        # a decode step's activations, and back for a check of the error
        {"name": "quant_61x7168", "kind": "quant", "M": 61, "K": 7168, "x": "bf16"},
        # a prefill chunk's MLP activations: bandwidth bound
        {"name": "quant_4096x18432", "kind": "quant", "M": 4096, "K": 18432, "x": "bf16"},
        # a weight at load time, from an fp32 master copy
        {"name": "quant_8192x8192_fp32", "kind": "quant", "M": 8192, "K": 8192, "x": "fp32"},
        # one decoding sequence, attention's input projection: streams the weight
        {"name": "linear_1_10240x8192", "kind": "linear", "M": 1, "N": 10240, "K": 8192, "x": "bf16"},
        # the smallest layer at a decode batch of 64: launches and latency
        {"name": "linear_64_2048x2048", "kind": "linear", "M": 64, "N": 2048, "K": 2048, "x": "bf16"},
        # a decode step of 200 sequences: between streaming and compute
        {"name": "linear_200_8192x8192", "kind": "linear", "M": 200, "N": 8192, "K": 8192, "x": "bf16"},
        # a mixed batch (a prefill chunk's ragged end plus decoding sequences) on one of eight shards
        {"name": "linear_777_4608x7168", "kind": "linear", "M": 777, "N": 4608, "K": 7168, "x": "bf16"},
        # a full prefill chunk through the widest layer: matrix-core bound
        {"name": "linear_4096_36864x7168", "kind": "linear", "M": 4096, "N": 36864, "K": 7168, "x": "bf16"},
        # one decoding sequence on one of eight shards: eight experts' slices, latency
        {"name": "experts_1_of_256_shard", "kind": "experts", "T": 1, "E": 256, "H": 7168, "I": 256, "topk": 8,
         "w": "fp8", "x": "bf16"},
        # a small decode batch over MXFP4 experts
        {"name": "experts_5_of_128_mxfp4", "kind": "experts", "T": 5, "E": 128, "H": 4096, "I": 1536, "topk": 8,
         "w": "mxfp4", "x": "bf16"},
        # a decode batch of 16 in fp16
        {"name": "experts_16_of_128_fp16", "kind": "experts", "T": 16, "E": 128, "H": 4096, "I": 1536, "topk": 8,
         "w": "fp8", "x": "fp16"},
        # the largest batch through a whole layer: streams about 220 experts
        {"name": "experts_64_of_256", "kind": "experts", "T": 64, "E": 256, "H": 7168, "I": 2048, "topk": 8,
         "w": "fp8", "x": "bf16"},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, round(lo * (hi / lo) ** rng.random())))


def draw(rng):
    kind = rng.choice(["quant"] * 2 + ["linear"] * 5 + ["experts"] * 4)
    if kind == "quant":
        return {"kind": kind, "M": _log_int(rng, 1, 4096), "K": 32 * _log_int(rng, 4, 576),
                "x": rng.choice(["bf16", "bf16", "fp16", "fp32"])}
    if kind == "linear":
        if rng.random() < 0.6:
            N, K = rng.choice(DENSE)
        else:   # any width, as of a vocabulary or an odd shard
            N, K = _log_int(rng, 200, 30000), 128 * _log_int(rng, 4, 64)
        most = 4096 * 36864 * 7168 // (N * K)
        return {"kind": kind, "M": _log_int(rng, 1, min(4096, most)), "N": N, "K": K,
                "x": rng.choice(["bf16", "bf16", "bf16", "fp16", "fp32"])}
    E, H, I, topk = rng.choice(MOE)
    return {"kind": kind, "T": _log_int(rng, 1, 64), "E": E, "H": H, "I": I, "topk": topk,
            "w": rng.choice(["fp8", "mxfp4"]), "x": rng.choice(["bf16", "bf16", "fp16"])}


# ------------------------------------------------------------------- inputs

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _activations(shape, dtype, g):
    x = torch.randn(shape, device="cuda", generator=g)
    big = torch.rand(shape, device="cuda", generator=g) < 1e-3   # a few large activations, as models have
    return torch.where(big, x * 20.0, x).to(DTYPES[dtype])


def _fp8_weight(shape, g):
    """Codes and fp32 128x128 block scales of ~N(0, 0.02) weights [E, N, K]."""
    w = torch.empty(shape, dtype=FP8, device="cuda")
    rows, step = w.view(-1, shape[-1]), max(1, (1 << 27) // shape[-1])
    for r in range(0, rows.shape[0], step):
        part = rows[r:r + step]
        part.copy_(torch.randn(part.shape, device="cuda", generator=g).mul_(109.0).clamp_(-448.0, 448.0))
    blocks = shape[:-2] + (-(-shape[-2] // 128), -(-shape[-1] // 128))
    u = torch.rand(blocks, device="cuda", generator=g)
    return w, (1.83e-4 * (0.75 + 0.5 * u)).contiguous()


def _mxfp4_weight(shape, g):
    """Packed codes [..., N, K/2] and scale bytes [..., N, K/32] of ~N(0, 0.02) weights."""
    n, K = 1, shape[-1]
    for d in shape[:-1]:
        n *= d
    codes = torch.empty((n, K // 2), dtype=torch.uint8, device="cuda")
    scales = torch.empty((n, K // 32), dtype=torch.uint8, device="cuda")
    step = max(1, (1 << 26) // K)
    for r in range(0, n, step):
        v, e = _quantise(torch.randn((min(step, n - r), K), device="cuda", generator=g).mul_(0.02))
        a = v.abs()
        c = (2 * a).where(a < 2, (a + 2).where(a < 4, a / 2 + 4)).to(torch.uint8) | ((v < 0).to(torch.uint8) << 3)
        codes[r:r + step] = c[:, 0::2] | (c[:, 1::2] << 4)
        scales[r:r + step] = e
    return codes.view(shape[:-1] + (K // 2,)), scales.view(shape[:-1] + (K // 32,))


def _weight(shape, kind, g):
    return _fp8_weight(shape, g) if kind == "fp8" else _mxfp4_weight(shape, g)


def prepare(case, seed):
    g = _gen(seed)
    kind = case["kind"]
    if kind == "quant":
        return {"kind": kind, "x": _activations((case["M"], case["K"]), case["x"], g)}
    if kind == "linear":
        w, s = _mxfp4_weight((case["N"], case["K"]), g)
        return {"kind": kind, "x": _activations((case["M"], case["K"]), case["x"], g), "w": w, "s": s.view(E8M0)}
    T, E, H, I = case["T"], case["E"], case["H"], case["I"]
    d = {"kind": kind, "x": _activations((T, H), case["x"], g), "E": E, "w": case["w"],
         "block": [128, 128] if case["w"] == "fp8" else [1, 32]}
    d["w13"], d["s13"] = _weight((E, 2 * I, H), case["w"], g)
    d["w2"], d["s2"] = _weight((E, H, I), case["w"], g)
    if case["w"] == "mxfp4":
        d["s13"], d["s2"] = d["s13"].view(E8M0), d["s2"].view(E8M0)
    p = torch.softmax(torch.randn(T, E, device="cuda", generator=g), dim=-1)
    tw, ids = torch.topk(p, case["topk"], dim=-1)
    d["ids"], d["tw"] = ids.to(torch.int32).contiguous(), (tw / tw.sum(dim=-1, keepdim=True)).contiguous()
    return d


# --------------------------------------------------------------- plain forms

def _quantise(x):
    """(e2m1 values, scale bytes) of fp32 rows: the group's largest magnitude, rounded to one
    mantissa bit, gives the exponent; values to nearest, ties to the even code, at most 6."""
    g = x.unflatten(-1, (-1, 32))
    bits = g.abs().amax(-1).view(torch.int32)
    e = (((bits + 0x200000) >> 23) - 2).clamp(1, 254)
    a = (g * ((254 - e) << 23).view(torch.float32).unsqueeze(-1)).clamp(-6.0, 6.0)
    step = torch.where(a.abs() < 2, 0.5, torch.where(a.abs() < 4, 1.0, 2.0))
    return (torch.round(a / step) * step).flatten(-2), e.to(torch.uint8)


def _scaled(v, e):
    """Values [..., K] times the powers of two of their groups' bytes [..., K/32]."""
    return (v.unflatten(-1, (-1, 32)) * (e.to(torch.int32) << 23).view(torch.float32).unsqueeze(-1)).flatten(-2)


def _unpacked(codes):
    """The e2m1 values of packed codes [..., K/2]."""
    c = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).to(torch.int8)
    m = c & 7
    twice = torch.where(m < 4, m, torch.where(m < 6, 2 * m - 4, 4 * m - 16))
    return torch.where(c < 8, twice, -twice).float().mul_(0.5)


def _plain_weight(w, s, kind):
    if kind == "mxfp4":
        return _scaled(_unpacked(w), s.view(torch.uint8))
    E, N, K = w.shape
    return w.float().view(E, N // 128, 128, K // 128, 128).mul_(s.view(E, N // 128, 1, K // 128, 1)).view(E, N, K)


def _plain_experts(s):
    x, ids, tw, E = s["x"].float(), s["ids"].long(), s["tw"], s["E"]
    T, topk = ids.shape
    if T * topk <= E:   # the named experts' weights, one by one
        at = ids.flatten()
        w13 = _plain_weight(s["w13"].view(torch.uint8)[at].view(s["w13"].dtype), s["s13"].view(_bits(s["s13"]))[at].view(s["s13"].dtype), s["w"])
        gu = torch.matmul(w13, x.repeat_interleave(topk, 0).unsqueeze(-1)).squeeze(-1)
        del w13
        gate, up = gu.chunk(2, -1)
        h = gate / (1 + torch.exp(-gate)) * up
        w2 = _plain_weight(s["w2"].view(torch.uint8)[at].view(s["w2"].dtype), s["s2"].view(_bits(s["s2"]))[at].view(s["s2"].dtype), s["w"])
        y = torch.matmul(w2, h.unsqueeze(-1)).squeeze(-1).view(T, topk, -1)
        return (y * tw.unsqueeze(-1)).sum(1).to(s["x"].dtype)
    # more pairs than experts: every expert on every token, weighted by the routing
    c = torch.zeros(T, E, device=x.device).scatter_add_(1, ids, tw)
    w13 = _plain_weight(s["w13"], s["s13"], s["w"])
    gate, up = torch.matmul(w13.flatten(0, 1), x.t()).view(E, -1, T).chunk(2, 1)      # [E, I, T]
    del w13
    h = gate / (1 + torch.exp(-gate)) * up * c.t().unsqueeze(1)
    w2 = _plain_weight(s["w2"], s["s2"], s["w"])
    return torch.matmul(w2, h.contiguous()).sum(0).t().contiguous().to(s["x"].dtype)


def _bits(t):
    return torch.uint8 if t.element_size() == 1 else torch.int32


def _plain(s):
    if s["kind"] == "quant":
        v, e = _quantise(s["x"].float())
        return _scaled(v, e).to(s["x"].dtype), e.view(E8M0)
    if s["kind"] == "linear":
        a = _scaled(*_quantise(s["x"].float()))
        return torch.matmul(a, _scaled(_unpacked(s["w"]), s["s"].view(torch.uint8)).t()).bfloat16()
    return _plain_experts(s)


# ------------------------------------------------------------ the package's

@functools.cache
def _package():
    import kb_nano_amd as k
    return types.SimpleNamespace(quant=k.Mxfp4Quant(), dequant=k.dequantize_mxfp4, linear=k.Mxfp4Linear(),
                                 experts=k.FewTokenExperts())


def run(state):
    if not own:
        return _plain(state)
    k, s = _package(), state
    if s["kind"] == "quant":
        codes, scales = k.quant(s["x"])
        return k.dequant(codes, scales, s["x"].dtype), scales
    if s["kind"] == "linear":
        return k.linear(s["x"], s["w"], s["s"])
    return k.experts(s["x"], s["w13"], s["w2"], s["tw"], s["ids"], s["E"], s["s13"], s["s2"], s["block"])


# --------------------------------------------------------------------- work

def work(case):
    if case["kind"] == "quant":
        n, b = case["M"] * case["K"], DTYPES[case["x"]].itemsize
        # the rows in, codes and scales out; those in again, the values out
        return {"bytes": n * (2 * b + 2 * (0.5 + 1 / 32)), "flops": 4 * n}
    if case["kind"] == "linear":
        M, N, K = case["M"], case["N"], case["K"]
        return {"bytes": DTYPES[case["x"]].itemsize * M * K + (0.5 + 1 / 32) * N * K + 2 * M * N, "flops": 2 * M * N * K}
    T, E, H, I, topk = (case[k] for k in ("T", "E", "H", "I", "topk"))
    active = E * (1 - (1 - topk / E) ** T)   # experts that T tokens name, on average
    per = 1 + 4 / 16384 if case["w"] == "fp8" else 0.5 + 1 / 32
    return {"bytes": active * 3 * I * H * per + 4 * T * H + 8 * T * topk, "flops": 2 * T * topk * 3 * I * H}


# -------------------------------------------------------------------- exact

_POSITIVE = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _exact_quant(x):
    """(values, scales) in 64 bits, from the definition: the scale is the power of two for which the
    largest magnitude lies in [3.5, 7); each value goes to the nearest of the eight, a tie to the even one."""
    v = x.double().reshape(x.shape[0], -1, 32)
    amax = v.abs().amax(2)
    m, e = torch.frexp(amax.clamp(min=2.0 ** -140))        # amax = m 2^e, m in [1/2, 1)
    e = (e - 3 + (m >= 0.875)).clamp(min=-126)
    scale = torch.ldexp(torch.ones_like(amax), e)
    a = v.abs() / scale.unsqueeze(2)
    out = torch.zeros_like(a)
    for i in range(7):
        lo, hi = _POSITIVE[i], _POSITIVE[i + 1]
        mid = (lo + hi) / 2
        out = torch.where((a >= mid) if i % 2 else (a > mid), torch.full_like(a, hi), out)
    return torch.where(v < 0, -out, out) * scale.unsqueeze(2), scale


def _exact_weight(w, s, kind):
    """One expert's (or linear's) weight rows [n, K] in 64 bits."""
    if kind == "fp8":
        return w.double() * s.double().repeat_interleave(128, 0).repeat_interleave(128, 1)[:w.shape[0], :w.shape[1]]
    b = w.to(torch.int64)
    c = torch.empty(w.shape[0], 2 * w.shape[1], dtype=torch.int64, device=w.device)
    c[:, ::2], c[:, 1::2] = b % 16, torch.div(b, 16, rounding_mode="floor")
    mag = torch.tensor(_POSITIVE, dtype=F64, device=w.device)[c % 8]
    e = s.view(torch.uint8).to(F64).repeat_interleave(32, 1) - 127
    return torch.where(c >= 8, -mag, mag) * torch.exp2(e)


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "quant":
        v, scale = _exact_quant(s["x"])
        return v.reshape(s["x"].shape), scale
    if case["kind"] == "linear":
        a = _exact_quant(s["x"])[0].reshape(s["x"].shape)
        out = torch.empty(case["M"], case["N"], dtype=F64, device="cuda")
        for n in range(0, case["N"], 2048):
            out[:, n:n + 2048] = a @ _exact_weight(s["w"][n:n + 2048], s["s"][n:n + 2048], "mxfp4").t()
        return out
    x, ids, tw, I = s["x"].double(), s["ids"], s["tw"].double(), case["I"]
    out = torch.zeros(case["T"], case["H"], dtype=F64, device="cuda")
    for e in torch.unique(ids).tolist():
        t, j = (ids == e).nonzero(as_tuple=True)
        gu = x[t] @ _exact_weight(s["w13"][e], s["s13"][e], case["w"]).t()
        h = torch.nn.functional.silu(gu[:, :I]) * gu[:, I:]
        out.index_add_(0, t, (h @ _exact_weight(s["w2"][e], s["s2"][e], case["w"]).t()) * tw[t, j].unsqueeze(1))
    return out
