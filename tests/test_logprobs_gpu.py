"""Log probabilities of given tokens on the GPU, against the formulas in 64 bits."""
import math

import pytest
import torch

from onnx_genai_b200 import ops
from onnx_genai_b200.ops import reference

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def _case(rows, vocab, dtype, seed, pad=0, masked=False):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = (3.0 * torch.randn(rows, vocab + pad, generator=g, device="cuda")).to(dtype)[:, :vocab]
    tokens = torch.randint(0, vocab, (rows,), generator=g, device="cuda")
    if masked:
        x.masked_fill_(torch.rand(rows, vocab, generator=g, device="cuda") < 0.9, -math.inf)
    return x, tokens


def _check(x, tokens, top, entropy=True):
    got = ops.token_logprobs(x, tokens, top=top, entropy=entropy)
    rows, vocab = x.shape
    lp, rank, ent, ids, lps = reference.token_logprobs(x.cpu(), tokens.cpu(), top, entropy)
    assert torch.equal(got.rank.cpu(), rank)
    finite = x.double().masked_fill(~torch.isfinite(x), 0.0)
    m = torch.where(torch.isfinite(x), x, -math.inf).double().amax(1).clamp_min(-1e30).cpu()
    # A thread adds at most vocab / 256 values in a row, the joins add 11 more; the approximate exponential is off by 2^-22, and by the rounding of its
    # argument, which weighs |d| exp(-|d|) < 0.4 of 2^-23: relative errors of s.  The differences x - m and - log s round by 2^-24 of their sizes.
    s_off = (vocab / 256 + 11) * 2.0 ** -24 + 2.0 ** -21
    size = finite.abs().amax(1).cpu() + math.log(vocab + 1) + m.abs().clamp_max(1e4)
    off = s_off + 3 * 2.0 ** -24 * size

    def close(a, b, bound):
        a, b, bound = a.double().cpu(), b.double(), torch.as_tensor(bound, dtype=torch.float64)
        assert torch.equal(torch.isnan(a), torch.isnan(b)) and torch.equal(torch.isinf(a), torch.isinf(b))
        ok = torch.isfinite(b)
        assert bool((((a - b).abs() <= bound.expand_as(b)) | ~ok).all()), float(((a - b).abs() - bound.expand_as(b))[ok].max())
    close(got.logprob, lp, off)
    if entropy:
        # t / s: both sums' errors, weighed by the mean of |x - m|, which is below the entropy and 1 together
        close(got.entropy, ent, (2 * s_off + 2.0 ** -22) * (2.0 + math.log(vocab)))
    else:
        assert got.entropy is None
    if top:
        assert torch.equal(got.top_ids.cpu(), ids)
        close(got.top_logprobs, lps, off[:, None])
    else:
        assert got.top_ids is None and got.top_logprobs is None


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("rows,vocab,top,pad", [(1, 1, 1, 0), (2, 5, 5, 3), (3, 100, 32, 0), (1, 4097, 20, 0), (7, 32000, 8, 0), (200, 5003, 20, 5), (1, 151936, 5, 0),
                                                (20, 50257, 32, 0), (75, 50257, 1, 7), (400, 1000, 3, 0)])
def test_sizes_types_and_strides(rows, vocab, top, pad, dtype):
    x, tokens = _case(rows, vocab, dtype, rows + vocab, pad)
    _check(x, tokens, top)
    _check(x, tokens.int(), 0, entropy=False)
    _check(x[:, 1:], (tokens - 1).clamp_min(0), min(top, vocab - 1), entropy=False) if vocab > 1 else None
    ops.check_status()


@pytest.mark.parametrize("rows,vocab", [(300, 152064), (148, 32000), (16, 200000)])
def test_many_rows_of_a_vocabulary(rows, vocab):
    x, tokens = _case(rows, vocab, BF16, rows)
    _check(x, tokens, 20)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_masks(dtype):
    x, tokens = _case(9, 20011, dtype, 3, masked=True)
    x[1] = -math.inf                                           # nothing is left
    x[2] = -math.inf
    x[2, 777] = 1.5                                            # one token is
    x[3] = torch.finfo(dtype).min                              # everything at the type's lowest value
    x[4, 100:] = torch.finfo(dtype).min
    x[5, 3] = math.nan
    x[6] = math.nan
    x[7, 9] = math.inf
    x[8, :] = 0.25                                             # every value alike
    tokens[2], tokens[4] = 777, 20000
    _check(x, tokens, 20)
    ops.check_status()


@pytest.mark.parametrize("rows", [1, 200])
def test_orders_that_are_hard_on_the_list_of_the_likeliest(rows):
    vocab = 70001
    up = torch.linspace(-5.0, 5.0, vocab, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(4)
    tokens = torch.randint(0, vocab, (rows,), generator=g, device="cuda")
    for row in (up, up.flip(0), torch.zeros_like(up), (torch.arange(vocab, device="cuda") % 7).float(), -up.abs(), torch.where(up > 4.999, up, -up)):
        for dtype in (F32, BF16):
            _check(row.to(dtype).repeat(rows, 1), tokens, 32)


def test_zeros_of_either_sign_are_alike():
    x = torch.zeros(2, 3000, device="cuda")
    x[0, ::2] = -0.0
    x[1, 1::2] = -0.0
    r = ops.token_logprobs(x, torch.zeros(2, device="cuda", dtype=torch.int32), top=4)
    assert r.top_ids.tolist() == [[0, 1, 2, 3]] * 2 and r.rank.tolist() == [0, 0]


def test_tokens_that_ask_for_nothing_or_do_not_exist():
    x, tokens = _case(5, 3000, BF16, 8)
    tokens[1], tokens[3] = -1, -100
    _check(x, tokens, 3)
    ops.check_status()
    tokens[2] = 3000
    tokens[4] = 2 ** 40
    _check(x, tokens, 3)
    with pytest.raises(ops._native.KernelError):
        ops.check_status()
    assert ops.token_logprobs(x[:0], tokens[:0], top=3, entropy=True).top_ids.shape == (0, 3)


def test_long_rows_past_32_bits():
    """Rows 2^27 values apart: the last begins past 2^31 bytes and values."""
    wide = torch.zeros(17, 2 ** 27, device="cuda", dtype=BF16)
    x = wide[:, :5000]
    x.copy_(_case(17, 5000, BF16, 9)[0])
    _check(x, torch.arange(17, device="cuda"), 4)


def test_replayed_graph_and_streams():
    xs = [_case(6, 40000, BF16, s)[0] for s in range(3)]
    tokens = torch.arange(6, device="cuda", dtype=torch.int32)
    want = [ops.token_logprobs(x, tokens, top=6, entropy=True) for x in xs]
    x = xs[0].clone()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        r = ops.token_logprobs(x, tokens, top=6, entropy=True)
    for i in (1, 2, 0):
        x.copy_(xs[i])
        graph.replay()
        for a, b in zip(r, want[i]):
            assert torch.equal(a, b)
    streams = [torch.cuda.Stream() for _ in xs]
    torch.cuda.synchronize()
    got = []
    for s, v in zip(streams, xs):
        with torch.cuda.stream(s):
            got.append([ops.token_logprobs(v, tokens, top=6, entropy=True) for _ in range(5)])
    torch.cuda.synchronize()
    for many, right in zip(got, want):
        for one in many:
            for a, b in zip(one, right):
                assert torch.equal(a, b)
