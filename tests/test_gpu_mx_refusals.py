"""What a refused few-token call tells the caller to use instead."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("fmt", ["fp8", "mxfp4"])
def test_more_tokens_name_a_layer_that_takes_the_weights(gpu_device, fmt):
    """The sorted-token and contiguous layers take FP8 weights only."""
    from tests.test_gpu_few_token_experts import call, make
    d = make(65, 8, 256, 128, 2, fmt, torch.bfloat16, 1, gpu_device)
    with pytest.raises(ValueError, match="65 tokens, at most 64") as e:
        call(d)
    assert ("FusedExperts" in str(e.value)) == (fmt == "fp8")
    assert ("in parts" in str(e.value)) == (fmt == "mxfp4")
    parts = [call({**d, "x": d["x"][i:i + 64], "ids": d["ids"][i:i + 64], "tw": d["tw"][i:i + 64]}) for i in (0, 64)]
    assert [p.shape[0] for p in parts] == [64, 1]
