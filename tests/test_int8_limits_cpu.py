"""What 8-bit products, norms around a block and log probabilities refuse at the ends of their ranges, and results over what is read."""
import pytest
import torch

from onnx_genai_b200 import ops
from onnx_genai_b200.ops import int8


def _rand(*s, seed=0):
    return torch.randn(*s, generator=torch.Generator().manual_seed(seed))


@pytest.mark.parametrize("rows", [2**28, 2**29, 2**30])
def test_more_rows_than_a_grid_counts_are_refused_by_name(rows):
    assert ops.MAX_LOGPROB_ROWS * 8 < 2**31 <= (ops.MAX_LOGPROB_ROWS + 1) * 8
    # (tensors without memory: nothing is computed whether the call is refused or not)
    with pytest.raises(ValueError, match="rows"):
        ops.token_logprobs(torch.empty(rows, 4, device="meta"), torch.empty(rows, dtype=torch.int32, device="meta"))
