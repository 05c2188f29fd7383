"""8-bit products, their rows and the norms around a block: the statements that CPU tensors run, and what the entry points refuse."""
import math

import pytest
import torch

from onnx_genai_b200 import ops
from onnx_genai_b200.ops import int8


def _rand(*s, seed=0):
    return torch.randn(*s, generator=torch.Generator().manual_seed(seed))


def test_rows_are_within_half_a_step_and_ties_go_to_even():
    x = _rand(9, 37)
    r = int8.quantize_rows(x)
    assert r.q.stride(0) % 16 == 0 and r.q.dtype == torch.int8
    assert torch.equal(r.scale, x.abs().amax(1) / 127.0)
    # half a step, and the roundings of the factor (2^-24 of 127 steps) and of the check itself
    assert float(((r.float() - x).abs() / r.scale[:, None]).max()) <= 0.5 + 127 * 2.0 ** -22
    tie = torch.tensor([[254.0, 127.0, 3.0, -1.0, 1.0, 5.0]])      # factor 2: 127, 63.5, 1.5, -0.5, 0.5, 2.5
    assert int8.quantize_rows(tie).q.tolist() == [[127, 64, 2, 0, 0, 2]]


def test_rows_without_a_size():
    x = torch.tensor([[0.0, 0.0], [1.0, math.inf], [math.nan, 1.0], [1e-42, -1e-42], [3e38, -1e38]])
    r = int8.quantize_rows(x)
    assert r.q.tolist() == [[0, 0], [0, 0], [0, 0], [127, -127], [127, -42]]
    assert float(r.scale[0]) == 0.0 and bool(torch.isnan(r.scale[1:3]).all()) and bool(torch.isfinite(r.scale[3:]).all())
    w = int8.quantize_weight(_rand(5, 2))
    y = int8.gemm_int8(r, w.q, w.scale, out_dtype=torch.float32)
    assert bool((y[0] == 0).all()) and bool(torch.isnan(y[1:3]).all()) and bool(torch.isfinite(y[3]).all())
    assert not bool(torch.isnan(y[4]).any())          # 3e38 times a weight above 1.13 is past the type's range: plus or minus infinity


def test_product_against_dense():
    x, w, bias, res = _rand(7, 50), int8.quantize_weight(_rand(20, 50, seed=1)), _rand(20, seed=2), _rand(7, 20, seed=3)
    want = int8.quantize_rows(x).float().double() @ w.float().double().t() + bias.double() + res.double()
    got = int8.gemm_int8(x, w.q, w.scale, bias=bias, residual=res)
    assert got.dtype == torch.float32
    torch.testing.assert_close(got.double(), want, rtol=2.0 ** -20, atol=2.0 ** -18)
    out = torch.empty(7, 20, dtype=torch.float16)
    assert int8.gemm_int8(int8.quantize_rows(x), w.q, w.scale, out=out) is out


def test_gated_weight_is_padded_with_nothing():
    gate, up, x = _rand(130, 40), _rand(130, 40, seed=1), _rand(3, 40, seed=2)
    w = int8.quantize_gate_up(gate, up)
    assert w.q.shape == (512, 40)
    y = int8.gemm_int8(x, w.q, w.scale, epilogue="swiglu")
    g, u = int8.gemm_int8(x, *int8.quantize_weight(gate)), int8.gemm_int8(x, *int8.quantize_weight(up))
    torch.testing.assert_close(y[:, :130], torch.nn.functional.silu(g) * u, rtol=2.0 ** -20, atol=2.0 ** -18)
    assert y.shape == (3, 256) and bool((y[:, 130:] == 0).all())


@pytest.mark.parametrize("gate", [None, "channel", "token"])
def test_block_norm_is_the_formula(gate):
    x, y, post, pre = _rand(4, 30), _rand(4, 30, seed=1), _rand(30, seed=2), _rand(30, seed=3)
    g = None if gate is None else _rand(30, seed=4) if gate == "channel" else _rand(4, 30, seed=4)
    rms = lambda v, w: v / (v.pow(2).mean(1, keepdim=True) + 1e-5).sqrt() * w.double()     # noqa: E731
    want = 0.5 * x.double() + 2.0 * rms(y.double(), post) * (1.0 if g is None else torch.sigmoid(g.double()))
    stream = x.clone()
    h = int8.block_norm(stream, y, post=post, gate=g, pre=pre, eps=1e-5, x_scale=0.5, y_scale=2.0, gate_sigmoid=True)
    torch.testing.assert_close(stream.double(), want, rtol=2.0 ** -18, atol=2.0 ** -18)
    torch.testing.assert_close(h.double(), rms(want, pre), rtol=2.0 ** -18, atol=2.0 ** -18)
    rows = int8.block_norm(x, y, post=post, gate=g, pre=pre, eps=1e-5, x_scale=0.5, y_scale=2.0, gate_sigmoid=True, x_out=torch.empty_like(x), int8=True)
    assert torch.equal(rows.q, int8.quantize_rows(h).q)


def test_block_norm_without_a_block_leaves_the_stream():
    x = _rand(3, 8)
    keep = x.clone()
    h = int8.block_norm(x, pre=torch.ones(8))
    assert torch.equal(x, keep) and h.shape == x.shape
    assert torch.equal(int8.block_norm(x, x_scale=2.0), 2.0 * keep) and torch.equal(x, 2.0 * keep)


def test_what_products_refuse():
    x, w = _rand(2, 32), int8.quantize_weight(_rand(256, 32))
    bad = [dict(w=w.q[:, :16]), dict(w=w.q.float()), dict(w_scale=w.scale[:5]), dict(w_scale=w.scale.double()), dict(w_scale=None), dict(bias=_rand(3)),
           dict(epilogue="gelu"), dict(epilogue="residual"), dict(epilogue="swiglu", residual=_rand(2, 128)), dict(residual=_rand(2, 255)),
           dict(out=torch.empty(2, 256, dtype=torch.float64)), dict(out=torch.empty(256, 2).t()), dict(out_dtype=torch.int32),
           dict(residual=_rand(2, 256).bfloat16(), out_dtype=torch.float32), dict(a=x.double()), dict(a=x[0])]
    for b in bad:
        with pytest.raises(ValueError):
            int8.gemm_int8(**{"a": x, "w": w.q, "w_scale": w.scale, **b})
    with pytest.raises(ValueError):
        int8.gemm_int8(x, w.q[:255], w.scale[:255], epilogue="swiglu")
    with pytest.raises(ValueError):
        int8.gemm_int8(torch.zeros(1, int8.MAX_K + 1), torch.zeros(1, int8.MAX_K + 1, dtype=torch.int8), torch.ones(1))
    with pytest.raises(ValueError):
        int8.quantize_rows(torch.zeros(3, 0))
    with pytest.raises(ValueError):
        int8.quantize_weight(torch.tensor([[1.0, math.inf]]))


def test_what_block_norm_refuses():
    x = _rand(2, 8)
    bad = [dict(y=_rand(2, 7)), dict(y=_rand(3, 8)), dict(post=torch.ones(8)), dict(gate=torch.ones(8)), dict(pre=torch.ones(7)), dict(y=x.double()),
           dict(y=x, post=torch.ones(8), pre=torch.ones(8).bfloat16()), dict(x_out=x.bfloat16()), dict(int8=True, out=torch.empty(2, 8)),
           dict(out=torch.empty(2, 8), out_dtype=torch.bfloat16), dict(y=_rand(8, 2).t()), dict(y=x, gate=_rand(3, 8))]
    for b in bad:
        with pytest.raises(ValueError):
            int8.block_norm(x, **b)
    with pytest.raises(ValueError):
        int8.block_norm(_rand(4, 4).t()[:, :3], pre=torch.ones(3))


def test_log_probabilities_are_the_formula():
    x = 3.0 * _rand(6, 50)
    x[1, 10:] = -math.inf
    x[2] = -math.inf
    x[3, 4] = math.nan
    x[4, :] = 1.0
    tokens = torch.tensor([3, 20, 0, 7, 49, -1])
    r = ops.token_logprobs(x, tokens, top=5, entropy=True)
    lp = torch.log_softmax(x.double(), 1)
    assert abs(float(r.logprob[0]) - float(lp[0, 3])) < 1e-6 and int(r.rank[0]) == int((x[0] > x[0, 3]).sum())
    assert float(r.logprob[1]) == -math.inf and int(r.rank[1]) == 10
    assert math.isnan(r.logprob[2]) and math.isnan(r.entropy[2]) and r.top_ids[2].tolist() == [0, 1, 2, 3, 4]
    assert math.isnan(r.logprob[3]) and math.isnan(r.entropy[3]) and 4 not in r.top_ids[3].tolist()
    assert r.top_ids[4].tolist() == [0, 1, 2, 3, 4] and abs(float(r.entropy[4]) - math.log(50)) < 1e-6
    assert float(r.logprob[5]) == 0.0 and int(r.rank[5]) == -1
    assert torch.equal(r.top_ids[0].long(), torch.topk(x[0], 5).indices)
    plain = ops.token_logprobs(x, tokens.int())
    assert plain.entropy is None and plain.top_ids is None and torch.equal(plain.rank, r.rank)


def test_what_log_probabilities_refuse():
    x = _rand(2, 40)
    for args in (dict(logits=x[0], tokens=torch.zeros(2).int()), dict(logits=x.double(), tokens=torch.zeros(2).int()), dict(logits=x, tokens=torch.zeros(3).int()),
                 dict(logits=x, tokens=torch.zeros(2)), dict(logits=x, tokens=torch.zeros(2).int(), top=33), dict(logits=x[:, :4], tokens=torch.zeros(2).int(), top=5),
                 dict(logits=x, tokens=torch.zeros(2).int(), top=-1), dict(logits=x[:, :0], tokens=torch.zeros(2).int())):
        with pytest.raises(ValueError):
            ops.token_logprobs(**args)


def test_results_that_share_memory_are_refused():
    buf = torch.zeros(4, 64)
    x, w = buf[:2, :32], int8.quantize_weight(_rand(32, 32))
    for out in (x, buf[1:3, :32], buf[:2, 16:48]):
        with pytest.raises(ValueError):
            int8.gemm_int8(x, w.q, w.scale, out=out)
    with pytest.raises(ValueError):
        int8.gemm_int8(_rand(2, 32), w.q, w.scale, residual=buf[:2, :32], out=buf[:2, 8:40])
    assert int8.gemm_int8(_rand(2, 32), w.q, w.scale, residual=x, out=x) is x
    beside = buf[:2, 32:]                                            # columns of one buffer, side by side
    assert torch.equal(int8.gemm_int8(x, w.q, w.scale, out=beside), int8.gemm_int8(x, w.q, w.scale))
    assert int8.block_norm(x, _rand(2, 32), out=beside) is beside
    y = _rand(2, 32)
    for kw in (dict(out=buf[1:3, :32]), dict(x_out=buf[:2, 8:40]), dict(x_out=y, out=y), dict(x_out=torch.empty(3, 32)[:2], out=x, y=y[:, :0])):
        with pytest.raises(ValueError):
            int8.block_norm(x, **{"y": y, **kw})
    keep = x.clone()
    want = int8.block_norm(keep, y.clone(), pre=torch.ones(32))
    assert torch.equal(int8.block_norm(x, y, pre=torch.ones(32), out=y), want) and torch.equal(x, keep)      # h in the place of y


def test_more_rows_than_the_kernels_count_are_refused():
    many = torch.zeros(1, 16).expand(2**31, 16)
    w = int8.quantize_weight(_rand(16, 16))
    for call in (lambda: int8.quantize_rows(many), lambda: int8.gemm_int8(many, w.q, w.scale), lambda: int8.block_norm(many, x_scale=1.0),
                 lambda: int8.gemm_int8(_rand(1, 16), torch.zeros(1, 16, dtype=torch.int8).expand(2**31, 16), torch.zeros(1).expand(2**31)),
                 lambda: ops.token_logprobs(many, torch.zeros(1, dtype=torch.int32).expand(2**31))):
        with pytest.raises(ValueError):
            call()
