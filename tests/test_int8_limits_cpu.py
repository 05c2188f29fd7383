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


def test_products_over_their_factors_or_bias_are_refused():
    m, n, k = 4, 16, 32
    buf = torch.zeros(m, 64)
    w = int8.quantize_weight(_rand(n, k))
    rows = int8.quantize_rows(_rand(m, k, seed=1))
    out = buf[:, 8:8 + n]
    for at in (0, 8, 15, 23, 64 + 10, 3 * 64):                     # the last reaches the last row from its start
        over = torch.as_strided(buf, (n,), (1,), at)
        for kw in (dict(w_scale=over), dict(bias=over)):
            with pytest.raises(ValueError):
                int8.gemm_int8(**{"a": rows, "w": w.q, "w_scale": w.scale, "out": out, **kw})
    with pytest.raises(ValueError):
        int8.gemm_int8(int8.Int8Rows(rows.q, torch.as_strided(buf, (m,), (1,), 2 * 64 + 8)), w.q, w.scale, out=out)
    beside = buf[2, 40:40 + n]                                     # between the rows of the result
    beside.copy_(_rand(n, seed=2))
    want = int8.gemm_int8(rows, w.q, w.scale, bias=beside.clone(), out_dtype=torch.float32)
    assert torch.equal(int8.gemm_int8(rows, w.q, w.scale, bias=beside, out=out), want)
    behind = torch.as_strided(buf, (n,), (1,), 3 * 64 + 8 + n)
    assert torch.equal(int8.gemm_int8(rows, w.q, w.scale, bias=behind, out=out), int8.gemm_int8(rows, w.q, w.scale, out_dtype=torch.float32))
