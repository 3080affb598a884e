"""What the router, the gated norms and the adapters refuse of their tensors before any launch
(no GPU needed: the device check is left out, and no call may reach the library)."""
import pytest
import torch

BF16, F32 = torch.bfloat16, torch.float32


@pytest.fixture
def no_launch(monkeypatch):
    from kb_nano_amd import _ops

    def lib():
        raise AssertionError("launched")
    monkeypatch.setattr(_ops, "_dev_check", lambda what, *t: 0)
    monkeypatch.setattr(_ops, "_host", None)
    monkeypatch.setattr(_ops, "lib", lib)
    return _ops


# ------------------------------------------------------------ adapters' ids

def lora_inputs(*lead):
    n = 1
    for v in lead:
        n *= v
    return (torch.zeros(*lead, 64, dtype=BF16), torch.zeros(*lead, 32, dtype=BF16), torch.zeros(2, 8, 64, dtype=BF16),
            torch.zeros(2, 32, 8, dtype=BF16))


@pytest.mark.parametrize("inplace", [False, True])
@pytest.mark.parametrize("lead,ids", [((2, 3), (3, 2)), ((2, 3, 4), (4, 3, 2)), ((2, 3, 4), (6, 4)), ((2, 1, 3), (3, 2)), ((4,), (3,)), ((2, 3), (5,))])
def test_ids_of_another_shape_are_refused(no_launch, lead, ids, inplace):
    """Ids [S, B] beside x [B, S, K] would give tokens each other's adapters."""
    from kb_nano_amd import LoraAdd
    with pytest.raises(ValueError, match="adapter_ids"):
        LoraAdd()(*lora_inputs(*lead), torch.zeros(ids, dtype=torch.int32), None, inplace)


@pytest.mark.parametrize("lead,ids", [((2, 3), (2, 3)), ((2, 3), (6,)), ((6,), (2, 3)), ((2, 1, 3), (2, 3)), ((4, 1), (4,)), ((4,), (4, 1)),
                                      ((4,), (1, 4)), ((), (1,)), ((), ())])
def test_ids_in_the_rows_order_are_taken(no_launch, lead, ids):
    """As x's leading dimensions, flat, or beside flat rows."""
    from kb_nano_amd import LoraAdd
    with pytest.raises(AssertionError, match="launched"):
        LoraAdd()(*lora_inputs(*lead), torch.zeros(ids, dtype=torch.int32))
