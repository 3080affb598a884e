"""Timed cases of the operators between the FP8 products of a decoder layer.

  gate    MoeRouterGemm: the router's product, fp32 logits of bf16 or fp16 rows
  topk    MoeRouterTopk: scores, balance bias, groups, top-k, renormalised weights
  norm    GatedAddRMSNorm and GatedAddRMSNormFP8Quant: the norms after and before a
          block with its gate, its residual and the residual's scale, rows or FP8 codes out
  lora    LoraAdd: low-rank adapters of many requests added to a shared projection

``run`` computes them in elementary torch operations, in fp32 (scores that decide a
choice in 64 bits) and rounded once at the end; with ``own`` set it makes the calls of
the package's modules.  Inputs are drawn on the GPU from the seed: activations ~N(0, 1)
with a few large ones, router weights ~N(0, 0.02), norm weights around 1, adapters that
change the projection by about half of its size.
"""
import functools
import types

import torch

own = False

FP8 = torch.float8_e4m3fn
E8M0 = torch.float8_e8m0fnu
F64 = torch.float64
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}

# (N, K) of dense layers that adapters stand beside: prefill and decode layers, their shards, a small one
DENSE = [(24576, 1536), (7168, 16384), (10240, 8192), (8192, 8192), (4608, 7168), (7168, 2048), (7168, 2304), (2048, 2048)]
# (experts, hidden) of routers
ROUTERS = [(256, 7168), (128, 4096), (16, 2048)]
# (experts, top-k, scoring, groups, kept groups, bias): grouped with a balance bias, plain softmax, small ones
ROUTINGS = [(256, 8, "sigmoid", 8, 4, True), (128, 8, "softmax", 1, 1, False), (160, 6, "softmax", 8, 3, False),
            (64, 6, "sigmoid", 1, 1, True), (16, 4, "softmax", 1, 1, False), (8, 2, "softmax", 1, 1, False)]


def listed():
    return [
        # one decoding sequence's router: launch and latency
        {"name": "gate_1_128x4096", "kind": "gate", "T": 1, "E": 128, "H": 4096, "x": "bf16", "w": "bf16"},
        # a decode batch of 61, the router's weight kept in fp32 as checkpoints have it
        {"name": "gate_61_256x7168_fp32", "kind": "gate", "T": 61, "E": 256, "H": 7168, "x": "bf16", "w": "fp32"},
        # a full prefill chunk: streams the hidden states
        {"name": "gate_4096_256x7168", "kind": "gate", "T": 4096, "E": 256, "H": 7168, "x": "bf16", "w": "bf16"},
        # one decoding sequence, grouped routing with a balance bias: latency
        {"name": "topk_1_of_256_grouped", "kind": "topk", "T": 1, "E": 256, "k": 8, "scoring": "sigmoid", "groups": 8, "kept": 4,
         "bias": True, "l": "fp32"},
        # a mixed batch, plain softmax routing of 16-bit logits
        {"name": "topk_777_of_128", "kind": "topk", "T": 777, "E": 128, "k": 8, "scoring": "softmax", "groups": 1, "kept": 1,
         "bias": False, "l": "bf16"},
        # several prefill chunks at once, grouped
        {"name": "topk_16384_of_256_grouped", "kind": "topk", "T": 16384, "E": 256, "k": 8, "scoring": "sigmoid", "groups": 8,
         "kept": 4, "bias": True, "l": "fp32"},
        # one decoding sequence between two blocks, rows out
        {"name": "norm_1x7168", "kind": "norm", "T": 1, "H": 7168, "x": "bf16", "post": True, "gate": "none", "out": "rows"},
        # a mixed batch in fp16 with a gate for each channel, FP8 codes out
        {"name": "norm_777x8192_fp8", "kind": "norm", "T": 777, "H": 8192, "x": "fp16", "post": True, "gate": "channel", "out": "fp8"},
        # a full prefill chunk with a gate of its own for each value, FP8 codes out: streams the rows
        {"name": "norm_4096x7168_fp8", "kind": "norm", "T": 4096, "H": 7168, "x": "bf16", "post": True, "gate": "full", "out": "fp8"},
        # a decode batch in which nearly every request has an adapter of its own
        {"name": "lora_32_8192x8192", "kind": "lora", "T": 32, "N": 8192, "K": 8192, "L": 24, "R": 16, "run": 1, "x": "bf16"},
        # a prefill chunk's ragged end beside decoding requests, on one of eight shards
        {"name": "lora_777_4608x7168", "kind": "lora", "T": 777, "N": 4608, "K": 7168, "L": 12, "R": 64, "run": 90, "x": "bf16"},
        # a full prefill chunk of a few long prompts, the widest input
        {"name": "lora_4096_7168x16384", "kind": "lora", "T": 4096, "N": 7168, "K": 16384, "L": 8, "R": 32, "run": 700, "x": "bf16"},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, round(lo * (hi / lo) ** rng.random())))


def draw(rng):
    kind = rng.choice(["gate", "topk", "norm", "lora"])
    x = rng.choice(["bf16", "bf16", "fp16"])
    if kind == "gate":
        if rng.random() < 0.6:
            E, H = rng.choice(ROUTERS)
        else:   # any number of experts, any width
            E, H = _log_int(rng, 5, 320), 8 * _log_int(rng, 64, 1024)
        most = 4096 * 256 * 7168 // (E * H)
        return {"kind": kind, "T": _log_int(rng, 1, min(4096, most)), "E": E, "H": H, "x": x, "w": rng.choice([x, x, "fp32"])}
    if kind == "topk":
        if rng.random() < 0.6:
            E, k, scoring, groups, kept, bias = rng.choice(ROUTINGS)
        else:
            groups = rng.choice([1, 1, 4, 6])
            E, kept = groups * _log_int(rng, 8, 40), max(1, groups // 2)
            k, scoring, bias = rng.randint(1, 8), rng.choice(["softmax", "sigmoid"]), rng.random() < 0.5
        return {"kind": kind, "T": _log_int(rng, 1, 16384), "E": E, "k": k, "scoring": scoring, "groups": groups, "kept": kept,
                "bias": bias, "l": rng.choice(["fp32", "fp32", "bf16", "fp16"])}
    if kind == "norm":
        x = rng.choice([x, x, "fp32"])
        return {"kind": kind, "T": _log_int(rng, 1, 2048 if x == "fp32" else 4096), "H": 8 * _log_int(rng, 64, 896), "x": x,
                "post": rng.random() < 0.7, "gate": rng.choice(["none", "channel", "token", "full"]), "out": rng.choice(["rows", "fp8"])}
    if rng.random() < 0.7:
        N, K = rng.choice(DENSE)
    else:   # any output width, any input width in eights
        N, K = _log_int(rng, 200, 8000), 8 * _log_int(rng, 64, 1024)
    T = _log_int(rng, 1, 2048)
    return {"kind": kind, "T": T, "N": N, "K": K, "L": rng.randint(1, 24 if T <= 256 else 8), "R": rng.choice([8, 16, 16, 32, 64]),
            "run": rng.choice([1, 1, 20, 300]), "x": x}


# ------------------------------------------------------------------- inputs

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _randn(shape, g, dtype="fp32", std=1.0):
    return torch.randn(shape, device="cuda", generator=g).mul_(std).to(DTYPES[dtype])


def _activations(shape, dtype, g):
    x = torch.randn(shape, device="cuda", generator=g)
    big = torch.rand(shape, device="cuda", generator=g) < 1e-3   # a few large activations, as models have
    return torch.where(big, x * 20.0, x).to(DTYPES[dtype])


def _adapter_ids(T, L, run, g):
    """One adapter for each run of tokens (runs of `run` on average, at random borders), -1 (none) for one in L + 1."""
    border = torch.rand(T, device="cuda", generator=g) < 1.0 / run
    which = torch.randint(-1, L, (T,), device="cuda", generator=g)
    return which[torch.cumsum(border, 0).clamp(max=T - 1)].to(torch.int32)


def prepare(case, seed):
    g, kind = _gen(seed), case["kind"]
    if kind == "gate":
        return {"kind": kind, "x": _activations((case["T"], case["H"]), case["x"], g),
                "w": _randn((case["E"], case["H"]), g, case["w"], 0.02)}
    if kind == "topk":
        return {"kind": kind, "l": _randn((case["T"], case["E"]), g, case["l"], 1.5),
                "bias": _randn((case["E"],), g, "fp32", 0.05) if case["bias"] else None,
                "k": case["k"], "scoring": case["scoring"], "groups": case["groups"], "kept": case["kept"], "scale": 2.5}
    if kind == "norm":
        T, H, t = case["T"], case["H"], case["x"]
        gate = {"none": None, "channel": (H,), "token": (T, 1), "full": (T, H)}[case["gate"]]
        return {"kind": kind, "x": _activations((T, H), t, g), "r": _activations((T, H), t, g),
                "w": (1 + 0.1 * _randn((H,), g)).to(DTYPES[t]),
                "post": (1 + 0.1 * _randn((H,), g)).to(DTYPES[t]) if case["post"] else None,
                "g": (0.7 + 0.2 * _randn(gate, g)).to(DTYPES[t]) if gate else None, "rs": 0.875, "out": case["out"]}
    T, N, K, L, R, t = (case[k] for k in ("T", "N", "K", "L", "R", "x"))
    return {"kind": kind, "x": _activations((T, K), t, g), "base": _randn((T, N), g, t),
            "a": _randn((L, R, K), g, t, K ** -0.5), "b": _randn((L, N, R), g, t, R ** -0.5),
            "s": 0.25 + 0.5 * torch.rand(L, device="cuda", generator=g), "ids": _adapter_ids(T, L, case["run"], g)}


# --------------------------------------------------------------- plain forms

EPS = 1e-6


def _plain_topk(s):
    l = s["l"].double()
    l = torch.where(torch.isnan(l), -torch.inf, l).clamp(max=torch.finfo(torch.float32).max)
    if s["scoring"] == "softmax":
        e = torch.exp(l - l.amax(1, keepdim=True).clamp(min=-1e300))
        score = e / e.sum(1, keepdim=True).clamp(min=1e-300)
    else:
        score = 1 / (1 + torch.exp(-l))
    T, E = l.shape
    # without a bias scores order as the logits do
    c = l if s["bias"] is None else torch.where(l == -torch.inf, -torch.inf, score + s["bias"].double())
    if s["groups"] > 1:
        members = c.view(T, s["groups"], -1)
        if s["bias"] is None:
            by = members.amax(2)
        else:
            by = members.topk(min(2, E // s["groups"]), dim=2).values.sum(2)
        kept = torch.sort(by, dim=1, descending=True, stable=True).indices[:, :s["kept"]]
        keep = torch.zeros(T, s["groups"], dtype=torch.bool, device=l.device).scatter_(1, kept, True)
        c = torch.where(keep.repeat_interleave(E // s["groups"], 1), c, -torch.inf)
    value, ids = torch.sort(c, dim=1, descending=True, stable=True)
    ids = ids[:, :s["k"]]
    w = torch.where(value[:, :s["k"]] == -torch.inf, 0.0, score.gather(1, ids))
    w = w / w.sum(1, keepdim=True).clamp(min=1e-300) * s["scale"]
    return w.float(), ids.to(torch.int32)


def _rms(x):
    return torch.rsqrt((x * x).mean(1, keepdim=True) + EPS)


def _quantise(v):
    """(e4m3 codes, power-of-two scales) of 1x128 groups: ceil to a power of two of the largest magnitude / 448."""
    T, H = v.shape
    G = -(-H // 128)
    g = torch.nn.functional.pad(v, (0, G * 128 - H)).view(T, G, 128)
    m, e = torch.frexp(g.abs().amax(2).clamp(min=1e-10))
    scale = torch.ldexp(torch.ones_like(m), e - 8 - (m <= 0.875).int())
    q = (g / scale.unsqueeze(2)).clamp(-448.0, 448.0).to(FP8)
    return q.view(T, G * 128)[:, :H].contiguous(), scale.to(E8M0)


def _plain_norm(s):
    p = s["x"].float()
    if s["post"] is not None:
        p = p * _rms(p) * s["post"].float()
    if s["g"] is not None:
        p = p * s["g"].float()
    r = (s["rs"] * s["r"].float() + p).to(s["r"].dtype)
    n = r.float()
    n = n * _rms(n) * s["w"].float()
    return (n.to(r.dtype), r) if s["out"] == "rows" else (*_quantise(n), r)


def _plain_lora(s):
    L, R, K = s["a"].shape
    T = s["x"].shape[0]
    # every adapter on every token, the token's own kept: one product down, one up
    mine = (s["ids"].unsqueeze(1) == torch.arange(L, device=s["ids"].device)).float() * s["s"]
    h = torch.matmul(s["x"].float(), s["a"].view(L * R, K).float().t()).view(T, L, R) * mine.unsqueeze(2)
    up = s["b"].float().transpose(1, 2).reshape(L * R, -1)
    return (s["base"].float() + torch.matmul(h.view(T, L * R), up)).to(s["base"].dtype)


def _plain(s):
    if s["kind"] == "gate":
        return torch.matmul(s["x"].float(), s["w"].float().t())
    return {"topk": _plain_topk, "norm": _plain_norm, "lora": _plain_lora}[s["kind"]](s)


# ------------------------------------------------------------ the package's

@functools.cache
def _package():
    import kb_nano_amd as k
    return types.SimpleNamespace(gate=k.MoeRouterGemm(), topk=k.MoeRouterTopk(), norm=k.GatedAddRMSNorm(),
                                 norm_fp8=k.GatedAddRMSNormFP8Quant(), lora=k.LoraAdd())


def run(state):
    if not own:
        return _plain(state)
    k, s = _package(), state
    if s["kind"] == "gate":
        return k.gate(s["x"], s["w"])
    if s["kind"] == "topk":
        return k.topk(s["l"], s["k"], scoring=s["scoring"], bias=s["bias"], num_groups=s["groups"], topk_groups=s["kept"],
                      renormalize=True, scale=s["scale"])
    if s["kind"] == "norm":
        args = (s["x"], s["r"], s["w"], s["post"], s["g"], s["rs"], EPS)
        if s["out"] == "rows":
            return k.norm(*args)
        codes, scales, r = k.norm_fp8(*args)
        return codes, scales.to(E8M0), r
    return k.lora(s["x"], s["base"], s["a"], s["b"], s["ids"], s["s"])


# --------------------------------------------------------------------- work

def work(case):
    if case["kind"] == "gate":
        T, E, H = case["T"], case["E"], case["H"]
        return {"bytes": DTYPES[case["x"]].itemsize * T * H + DTYPES[case["w"]].itemsize * E * H + 4 * T * E, "flops": 2 * T * E * H}
    if case["kind"] == "topk":
        n = case["T"] * case["E"]
        return {"bytes": DTYPES[case["l"]].itemsize * n + 8 * case["T"] * case["k"] + (4 * case["E"] if case["bias"] else 0),
                "flops": 6 * n}
    if case["kind"] == "norm":
        T, H, b = case["T"], case["H"], DTYPES[case["x"]].itemsize
        gate = {"none": 0, "channel": H, "token": T, "full": T * H}[case["gate"]]
        out = b * T * H if case["out"] == "rows" else T * H + T * -(-H // 128)
        return {"bytes": b * (3 * T * H + gate + H * (2 if case["post"] else 1)) + out, "flops": 10 * T * H}
    T, N, K, L, R = (case[k] for k in ("T", "N", "K", "L", "R"))
    b = DTYPES[case["x"]].itemsize
    runs = 1 + (T - 1) / case["run"]
    used = L * (1 - (1 - 1 / (L + 1)) ** runs)      # adapters that the batch names, on average
    return {"bytes": b * (T * K + 2 * T * N + used * R * (N + K)) + 4 * T, "flops": 2 * T * R * (N + K) * L / (L + 1)}


# -------------------------------------------------------------------- exact

def _exact_topk(s):
    """Weights in 64 bits on the CPU, one token at a time from the definition (the ids have to be equal anyway)."""
    import numpy as np
    logits, E, k = s["l"].double().cpu().numpy(), s["l"].shape[1], s["k"]
    bias = None if s["bias"] is None else s["bias"].double().cpu().numpy()
    per = E // s["groups"]
    out = np.zeros((len(logits), k))
    for t, row in enumerate(logits):
        if s["scoring"] == "softmax":
            score = np.exp(row - row.max())
            score = score / score.sum()
        else:
            score = 1 / (1 + np.exp(-row))
        c = score if bias is None else score + bias
        allowed = np.arange(E)
        if s["groups"] > 1:
            best = -np.sort(-c.reshape(s["groups"], per), axis=1)
            by = best[:, 0] if bias is None else best[:, :2].sum(1)
            kept = np.argsort(-by, kind="stable")[:s["kept"]]
            allowed = np.nonzero(np.isin(np.arange(E) // per, kept))[0]
        top = score[allowed[np.argsort(-c[allowed], kind="stable")[:k]]]
        out[t] = top / top.sum() * s["scale"]
    return torch.from_numpy(out)


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "gate":
        return s["x"].double() @ s["w"].double().t()
    if case["kind"] == "topk":
        return (_exact_topk(s), None)
    if case["kind"] == "norm":
        x, r = s["x"].double(), s["rs"] * s["r"].double()
        y = x
        if s["post"] is not None:
            y = x / torch.sqrt(x.square().sum(1, keepdim=True) / x.shape[1] + EPS) * s["post"].double()
        r = r + y if s["g"] is None else r + s["g"].double() * y
        if s["out"] == "fp8":     # codes and scales are steps of the values: no number in 64 bits
            return None, None, r
        n = r.to(s["r"].dtype).double()      # the second norm is of the residual as it is kept
        return n / torch.sqrt(n.square().sum(1, keepdim=True) / n.shape[1] + EPS) * s["w"].double(), r
    out = s["base"].double()
    for a in range(case["L"]):
        t = (s["ids"] == a).nonzero().flatten()
        if len(t):
            out[t] += (s["x"][t].double() @ s["a"][a].double().t()) @ s["b"][a].double().t() * s["s"][a].double()
    return out
