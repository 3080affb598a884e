"""Calls of the gated norms and the adapters beside their plain ones: truth values that are no bool, ids of
several dimensions, and the compiled forms of the adapters in place."""
import pytest
import torch

from tests.test_gpu_lora import args, make

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


@pytest.mark.parametrize("yes,no", [(True, False), (1, 0), ("rows", "")])
def test_with_rows_goes_by_its_truth_value(gpu_device, yes, no):
    from kb_nano_amd import GatedAddRMSNorm, GatedAddRMSNormFP8Quant
    x = torch.randn(5, 256, device=gpu_device).to(BF16)
    normed, _ = GatedAddRMSNorm()(x, x, x[0])
    *_, rows = got = GatedAddRMSNormFP8Quant()(x, x, x[0], with_rows=yes)
    assert len(got) == 4 and torch.equal(rows, normed)
    assert len(GatedAddRMSNormFP8Quant()(x, x, x[0], with_rows=no)) == 3


def test_ids_of_several_dimensions(gpu_device):
    from kb_nano_amd import LoraAdd
    x, base, a, b, ids, s = args(make(12, 64, 128, 4, 8, BF16, 3, gpu_device))
    out = LoraAdd()(x, base, a, b, ids, s)
    x3, b3 = x.view(3, 4, 128), base.view(3, 4, 64)
    for i in (ids.view(3, 4), ids):
        assert torch.equal(LoraAdd()(x3, b3, a, b, i, s).view(12, 64), out)
    assert torch.equal(LoraAdd()(x, base, a, b, ids.view(3, 4), s), out)
    for i in (ids.view(4, 3), ids.view(3, 4).t(), ids.view(2, 6)):
        for inplace in (False, True):
            with pytest.raises(ValueError, match="adapter_ids"):
                LoraAdd()(x3, b3, a, b, i, s, inplace)


def _compiled(fn):
    torch._dynamo.reset()
    return torch.compile(fn, fullgraph=True, backend="aot_eager")


@pytest.mark.parametrize("lead", [(20,), (4, 5)])
def test_compiled_adapters_in_place(gpu_device, lead):
    """base is written, also where it is x, and only its own columns; work after the call sees it."""
    from kb_nano_amd import LoraAdd
    lora = LoraAdd()
    d = make(20, 64, 256, 3, 16, BF16, 5, gpu_device)
    x, ids = d["x"].view(*lead, 256), d["ids"].view(lead)
    want = lora(x, d["base"].view(*lead, 64), d["a"], d["b"], ids, d["s"])
    wide = torch.zeros(*lead, 96, dtype=BF16, device=gpu_device)
    wide[..., 16:80] = d["base"].view(*lead, 64)

    def run(x, base):
        return lora(x, base, d["a"], d["b"], ids, d["s"], inplace=True) * 2
    if len(lead) == 1:     # (rows of more dimensions in place have to be one block)
        part = wide[..., 16:80]
        got = _compiled(run)(x, part)
        assert torch.equal(part, want) and torch.equal(got, want * 2)
        assert bool((wide[..., :16] == 0).all()) and bool((wide[..., 80:] == 0).all())
    base = d["base"].view(*lead, 64).clone()
    got = _compiled(run)(x, base)
    assert torch.equal(base, want) and torch.equal(got, want * 2)
    e = make(20, 256, 256, 3, 16, BF16, 6, gpu_device)
    want = lora(e["x"], e["x"], e["a"], e["b"], e["ids"], e["s"])
    y = e["x"].clone()

    def same(y):
        lora(y, y, e["a"], e["b"], e["ids"], e["s"], inplace=True)
        return y + 1
    got = _compiled(same)(y)
    assert torch.equal(y, want) and torch.equal(got, want + 1)


@pytest.mark.parametrize("lead", [(20,), (4, 5), (128,)])
def test_compiled_linear_with_adapters(gpu_device, lead):
    from kb_nano_amd import LoraFp8Linear
    from kb_nano_amd.fp8_linear import _block_requant
    T = 1
    for n in lead:
        T *= n
    d = make(T, 384, 512, 4, 16, BF16, 5, gpu_device)
    g = torch.Generator(device=gpu_device).manual_seed(1)
    w, sw = _block_requant(torch.randn(384, 512, device=gpu_device, generator=g) * 0.05, True)
    bias = torch.randn(384, device=gpu_device, generator=g).to(BF16)
    x, ids = d["x"].view(*lead, 512), d["ids"].view(lead)
    for b in (None, bias):
        layer = LoraFp8Linear()
        want = layer(x, w, sw, d["a"], d["b"], ids, d["s"], b).clone()
        got = _compiled(lambda x: layer(x, w, sw, d["a"], d["b"], ids, d["s"], b))(x)
        assert got.shape == want.shape and torch.equal(got, want)
