"""The choice of experts where the last one taken and the only one left out are the row's smallest values, closer
together than fp32 resolves: 7 of 8, 7 of two kept groups of four, rows of k + 1 logits that are not -inf."""
import pytest
import torch

from tests._layer_util import assert_routing, routing_plain

pytestmark = pytest.mark.gpu
F32, F64 = torch.float32, torch.float64


def near_rows(T, E, groups, kept, k, scoring, centre, seed):
    """(logits fp32 [T, E], bias fp32 [E]): k + 1 experts compete, the two smallest biased scores of a row some
    1e-7 apart (as far as fp32 logits can place them); the others are -inf, or in groups that are dropped."""
    g = torch.Generator().manual_seed(seed)

    def rand(*shape):
        return torch.rand(*shape, generator=g, dtype=F64)
    per = E // groups
    competing = torch.arange(kept * per) + (groups - kept) * per if groups > 1 else torch.randperm(E, generator=g)[:k + 1].sort().values
    assert len(competing) == k + 1
    bias = centre + 0.02 * rand(E)
    a, b = competing[torch.randperm(k + 1, generator=g)[:2]].tolist()
    others = [e for e in competing.tolist() if e not in (a, b)]
    bias[others] += 0.2
    if groups > 1:
        bias[:(groups - kept) * per] -= 2.0
    bias = bias.float()
    gap = bias.double()[a] - bias.double()[b]
    off = (rand(T) - 0.5) * 2e-7
    l = torch.full((T, E), -torch.inf, dtype=F64)
    if groups > 1:
        l[:, :(groups - kept) * per] = rand(T, (groups - kept) * per) - 5.0
    l[:, others] = 0.5 + rand(T, len(others))
    l[:, a] = -0.5 * rand(T) if scoring == "sigmoid" else 0.4 * rand(T)
    if scoring == "sigmoid":       # s_b + bias_b = s_a + bias_a + off
        s = torch.sigmoid(l[:, a].float().double()) + gap + off
        l[:, b] = torch.log(s / (1 - s))
    else:                          # e_b / (rest + e_b) = e_a / (rest + e_b) + gap + off
        l = l.float().double()
        rest = torch.exp(l).sum(1)   # (e_b is 0 so far, or the -inf's)
        rest = rest - torch.exp(l[:, b])
        d = gap + off
        l[:, b] = torch.log((torch.exp(l[:, a]) + d * rest) / (1 - d))
    assert bool(torch.isfinite(l[:, b]).all())
    return l.float(), bias


@pytest.mark.parametrize("scoring", ["sigmoid", "softmax"])
@pytest.mark.parametrize("centre", [0.0, 3.0, 30.0])
@pytest.mark.parametrize("E,groups,kept,k", [(3, 1, 1, 2), (8, 1, 1, 7), (16, 4, 2, 7), (8, 2, 2, 7), (64, 1, 1, 8), (100, 1, 1, 5), (300, 1, 1, 8),
                                             (32, 16, 2, 3)])
def test_the_smallest_two_of_a_row_nearly_tie(gpu_device, E, groups, kept, k, centre, scoring):
    from kb_nano_amd import MoeRouterTopk
    print(f"near values {E} in {groups} top {k} {scoring} around {centre}", flush=True)
    for seed in range(4):     # other biases
        l, bias = near_rows(1000, E, groups, kept, k, scoring, centre, 100 * E + seed)
        w, i = MoeRouterTopk()(l.to(gpu_device), k, scoring, bias.to(gpu_device), groups, kept)
        assert_routing(w, i, routing_plain(l, k, scoring, bias, groups, kept), f"{E} in {groups} top {k}")


def test_scores_that_fp32_orders_the_other_way(gpu_device):
    """Both sigmoids are 1 in fp32; with the biases experts 1 and 2 are 0.50000003066 and 0.50000005960."""
    from kb_nano_amd import MoeRouterTopk
    f = float.fromhex
    l = torch.tensor([[40.0, 16.65, 40.0]] * 5, device=gpu_device)
    bias = torch.tensor([0.0, -f("0x1.fffffap-2"), -f("0x1.fffffcp-2")], device=gpu_device)
    w, i = MoeRouterTopk()(l, 2, "sigmoid", bias)
    assert i.tolist() == [[0, 2]] * 5
    assert_routing(w, i, routing_plain(l, 2, "sigmoid", bias), "other order")


@pytest.mark.parametrize("E,k", [(4, 4), (8, 8), (7, 6)])
@pytest.mark.parametrize("scoring", ["sigmoid", "softmax"])
def test_all_or_nearly_all_of_a_row(gpu_device, E, k, scoring):
    from kb_nano_amd import MoeRouterTopk
    g = torch.Generator().manual_seed(E)
    for scale, centre in ((1.5, 0.0), (1e-3, 0.0), (0.1, 3.0), (1.5, -30.0)):
        l = torch.randn(500, E, generator=g) * scale
        bias = centre + 0.01 * torch.randn(E, generator=g)
        for b in (None, bias):
            w, i = MoeRouterTopk()(l.to(gpu_device), k, scoring, None if b is None else b.to(gpu_device))
            assert_routing(w, i, routing_plain(l, k, scoring, b), f"{k} of {E}")
