"""8-bit products, their rows and the norms around a block on the GPU, against the formulas in 64 bits."""
import math

import pytest
import torch

from onnx_genai_b200 import ops
from onnx_genai_b200.ops import int8, reference

pytestmark = pytest.mark.gpu

HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}     # half a step, relative
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _rand(g, *s):
    return torch.randn(*s, generator=g, device="cuda")


def _rows(g, m, k, dtype, pad=0):
    """Rows inside a wider matrix, one of them zero and one of a single value where there are enough."""
    x = _rand(g, m, k + pad).to(dtype)[:, :k]
    if m > 3:
        x[1] = 0.0
        x[2] = 0.0
        x[2, k // 2] = -2.0
    return x


def _weight(g, n, k):
    q = torch.randint(-127, 128, (n, (k + 15) // 16 * 16), generator=g, device="cuda", dtype=torch.int8)[:, :k]
    return q, (0.5 + torch.rand(n, generator=g, device="cuda")) * 0.01


@pytest.mark.parametrize("m,k,dtype,pad", [(1, 1, F32, 0), (3, 7, BF16, 0), (5, 8, F16, 3), (1, 3584, BF16, 0), (700, 896, BF16, 8), (33, 1001, F16, 0),
                                           (1, 18944, BF16, 0), (2, 70000, F32, 1), (600, 4864, F32, 0), (400, 20001, BF16, 0), (3000, 897, BF16, 0), (500, 3583, F16, 0),
                                           (700, 1001, F32, 0), (300, 16383, BF16, 0), (310, 32761, F16, 0), (309, 32767, BF16, 0), (2000, 50, F32, 1), (1, 8191, BF16, 0)])
def test_rows_are_the_formula_bit_by_bit(m, k, dtype, pad):
    x = _rows(_gen(m + k), m, k, dtype, pad)
    r = int8.quantize_rows(x)
    q, s = reference.quantize_rows(x)
    assert torch.equal(r.scale, s) and torch.equal(r.q, q)


def test_rows_at_ties_and_at_the_ends_of_the_range():
    half = torch.arange(-127, 128, device="cuda").float() / 2.0
    x = torch.stack([half * 2.0 ** e for e in (-140, -126, -100, -60, 0, 60, 100, 119)])
    x[:, 0] = x[:, 0] * 2.0                                                        # the peak: 127 halves and the steps are one apart
    x = torch.cat([x, torch.tensor([math.inf, math.nan, 3.4e38], device="cuda")[:, None] * torch.ones(3, 255, device="cuda")])
    for dtype in (F32, BF16):
        t = x.to(dtype)
        r = int8.quantize_rows(t)
        q, s = reference.quantize_rows(t)
        assert torch.equal(r.q, q)
        assert torch.equal(torch.nan_to_num(r.scale, nan=-1.0), torch.nan_to_num(s, nan=-1.0))


def _check_product(g, m, n, k, dtype, bias, residual, gated, as_rows=False, out_dtype=None):
    x = _rows(g, m, k, dtype)
    w, c = _weight(g, n, k)
    n_out = n // 2 if gated else n
    b = _rand(g, n) if bias else None
    out_dtype = out_dtype or (BF16 if as_rows else dtype)
    res = _rand(g, m, n_out).to(out_dtype) if residual else None
    a = int8.quantize_rows(x) if as_rows else x
    got = int8.gemm_int8(a, w, c, bias=b, residual=res, epilogue="swiglu" if gated else "none", out_dtype=out_dtype)
    q, s = reference.quantize_rows(x)
    plain = (q.double() @ w.double().t()) * s.double()[:, None] * c.double()
    if b is not None:
        plain = plain + b.double()
    # the sum as a float, two factors (the second fused with the bias): three roundings, of the product or of product and bias
    off = 3 * 2.0 ** -24 * (plain.abs() + (b.double().abs() if b is not None else 0.0))
    want = plain
    if gated:
        v = plain.view(m, -1, 2, 128)
        gate, up = v[:, :, 0].reshape(m, -1), v[:, :, 1].reshape(m, -1)
        o = off.view(m, -1, 2, 128)
        want = torch.nn.functional.silu(gate) * up
        # silu's slope is at most 1.1; its exponential and division are off by 2^-21 + |gate| 2^-23 and a few 2^-23
        off = 1.1 * o[:, :, 0].reshape(m, -1) * up.abs() + o[:, :, 1].reshape(m, -1) * gate.abs() + want.abs() * (2.0 ** -20 + gate.abs() * 2.0 ** -23)
    if res is not None:
        want = want + res.double()
        off = off + 2.0 ** -24 * want.abs()
    tiny = torch.finfo(out_dtype).smallest_normal * torch.finfo(out_dtype).eps         # steps of subnormal results
    assert got.shape == (m, n_out) and got.dtype == out_dtype
    far = (got.double() - want).abs() - (off + HALF[out_dtype] * (want.abs() + off) + tiny)
    assert float(far.max()) <= 0.0, float(far.max())


@pytest.mark.parametrize("m", [1, 2, 15, 16, 17, 48, 77, 129, 256])
@pytest.mark.parametrize("n,k", [(1, 1), (33, 16), (128, 128), (1001, 2039), (4608, 3584)])
def test_few_rows(m, n, k):
    _check_product(_gen(m * n + k), m, n, k, BF16, True, True, False)


@pytest.mark.parametrize("m,n,k,dtype,bias,residual", [
    (257, 129, 65, F16, True, False), (300, 20000, 896, BF16, False, True), (513, 4608, 3584, BF16, True, False), (1024, 896, 4864, F32, False, True),
    (2000, 2560, 2048, BF16, True, True), (4096, 3584, 1000, F16, False, False), (64, 151936, 896, BF16, False, False), (1, 152064, 3584, BF16, False, False),
    (3, 40000, 130, F32, True, False), (7, 512, 131072, BF16, False, False), (4001, 1111, 333, BF16, True, True)])
def test_all_divisions_of_the_work(m, n, k, dtype, bias, residual):
    _check_product(_gen(m + n + k), m, n, k, dtype, bias, residual, False)


@pytest.mark.parametrize("m,n,k,dtype", [(1, 256, 64, BF16), (5, 9728, 896, BF16), (77, 37888, 3584, BF16), (128, 1024, 777, F16), (300, 9728, 896, F32),
                                         (1000, 11008 * 2, 512, BF16), (1, 37888, 3584, BF16), (2049, 768, 300, F16), (17, 256 * 300, 200, BF16)])
def test_gated(m, n, k, dtype):
    _check_product(_gen(m + n), m, n, k, dtype, False, False, True)
    _check_product(_gen(m + n + 1), m, n, k, dtype, True, False, True, as_rows=True)


@pytest.mark.parametrize("m,n,k", [(1, 4608, 3584), (300, 20000, 896), (2000, 2560, 2048)])
@pytest.mark.parametrize("out_dtype", [BF16, F16, F32])
def test_rows_made_beforehand(m, n, k, out_dtype):
    _check_product(_gen(m), m, n, k, BF16, True, True, False, as_rows=True, out_dtype=out_dtype)


def test_every_code_and_the_largest_sums():
    """128 * 127 * 131072 has 31 bits: every sum is exact, whatever its size."""
    k = int8.MAX_K
    x = torch.full((2, k), 1.0, device="cuda")
    x[1] = -1.0
    w = torch.full((130, k), -128, device="cuda", dtype=torch.int8)
    w[1] = 127
    c = torch.ones(130, device="cuda")
    y = int8.gemm_int8(x, w, c)
    q, s = reference.quantize_rows(x)
    want = (q.double() @ w.double().t()) * s.double()[:, None]
    assert float(((y.double() - want).abs() - 3 * 2.0 ** -24 * want.abs()).max()) <= 0.0


def test_strides_and_results_in_place():
    g = _gen(5)
    w, c = _weight(g, 500, 300)
    wide = _rand(g, 40, 700).bfloat16()
    x, res = wide[:, 100:400], wide[:, 150:650]
    want = int8.gemm_int8(x.contiguous(), w, c, residual=res.contiguous())
    out = torch.full((40, 640), 7.0, device="cuda", dtype=BF16)
    got = int8.gemm_int8(x, w, c, residual=res, out=out[:, 33:533])
    assert torch.equal(got, want) and bool((out[:, :33] == 7.0).all()) and bool((out[:, 533:] == 7.0).all())
    stream = res.contiguous()
    assert torch.equal(int8.gemm_int8(x, w, c, residual=stream, out=stream), want)
    assert torch.equal(int8.gemm_int8(x.t().contiguous().t(), w, c, residual=res), want)
    rows = int8.quantize_rows(x)
    deep = torch.zeros(40, 512, device="cuda", dtype=torch.int8)
    deep[:, 16:316] = rows.q
    assert torch.equal(int8.gemm_int8(int8.Int8Rows(deep[:, 16:316], rows.scale), w, c, residual=res), want)


def test_rows_that_are_not_numbers_stay_their_own():
    g = _gen(6)
    w, c = _weight(g, 200, 256)
    x = _rand(g, 20, 256)
    x[3, 5], x[7, 0], x[9] = math.inf, math.nan, 0.0
    y = int8.gemm_int8(x, w, c)
    bad = torch.isnan(y).all(1)
    assert bad.nonzero()[:, 0].tolist() == [3, 7] and bool((y[9] == 0).all()) and bool(torch.isfinite(y[~bad]).all())


def test_what_is_refused():
    g = _gen(7)
    w, c = _weight(g, 64, 40)
    x = _rand(g, 3, 40)
    with pytest.raises(ValueError):
        int8.gemm_int8(x, w.contiguous()[:, :40], c)                 # rows at 40 bytes
    with pytest.raises(ValueError):
        int8.gemm_int8(x, w, c.cpu())
    with pytest.raises(ValueError):
        int8.gemm_int8(x, w.cpu(), c)
    with pytest.raises(ValueError):
        int8.gemm_int8(int8.Int8Rows(int8.quantize_rows(x).q.contiguous(), c[:3]), w, c)
    with pytest.raises(ValueError):
        int8.block_norm(torch.zeros(1, int8.MAX_HIDDEN + 1, device="cuda"))
    assert int8.gemm_int8(x[:0], w, c).shape == (0, 64)
    assert int8.quantize_rows(x[:0]).q.shape == (0, 40) and int8.block_norm(x[:0], pre=torch.ones(40, device="cuda")).shape == (0, 40)


# ---- norms ----
def _norm_case(g, m, n, stream, dtype, post, gate, wtype, pad=0):
    x = (4.0 * _rand(g, m, n + pad)).to(stream)[:, :n]
    y = _rand(g, m, n + 2 * pad).to(dtype)[:, pad:pad + n]
    kw = {"post": _rand(g, n).to(wtype) if post else None, "pre": _rand(g, n).to(wtype),
          "gate": None if gate == "none" else _rand(g, n).to(dtype) if gate == "channel" else _rand(g, m, n).to(dtype)}
    return x, y, kw


def _norm_want(x, y, kw, eps, xs, ys, sigmoid):
    """(x', its bound, h, its bound) before they are rounded to their types.  A sum of n squares over threads with at most 32 each and a tree is off by
    (32 + 14) 2^-24 at most, its root by half of that, rsqrt and a handful of products by 2^-24 or 2^-23 each: below 2^-18 in all."""
    part = y.double()
    if kw["post"] is not None:
        part = part / (part.pow(2).mean(1, keepdim=True) + eps).sqrt() * kw["post"].double()
    if kw["gate"] is not None:
        part = part * (torch.sigmoid(kw["gate"].double()) if sigmoid else kw["gate"].double())
    new = xs * x.double() + ys * part
    off = 2.0 ** -18 * (abs(xs) * x.double().abs() + abs(ys) * part.abs())
    root = (new.pow(2).mean(1, keepdim=True) + eps).sqrt()
    h = new / root * kw["pre"].double()
    # an error of the stream reaches h by itself and through the root of its mean square
    through = off.pow(2).mean(1, keepdim=True).sqrt() / root
    return new, off, h, off / root * kw["pre"].double().abs() + h.abs() * (2.0 ** -18 + through)


@pytest.mark.parametrize("m,n,pad", [(1, 1, 0), (1, 3584, 0), (3, 33, 0), (600, 64, 8), (700, 896, 0), (5, 1001, 0), (400, 3584, 0), (310, 8192, 8), (2, 16384, 0),
                                     (350, 16383, 0), (2000, 897, 0), (700, 3583, 0), (320, 8191, 0), (1500, 203, 0), (310, 10003, 0), (400, 130, 4), (900, 1024, 0)])
@pytest.mark.parametrize("stream,dtype,post,gate,wtype", [(BF16, BF16, True, "channel", F32), (F32, BF16, True, "token", F32), (F32, F16, False, "none", F16),
                                                          (F16, F32, True, "token", BF16), (F32, F32, True, "token", F32), (BF16, F16, True, "channel", BF16),
                                                          (BF16, F32, False, "none", F32)])
def test_block_norm(m, n, pad, stream, dtype, post, gate, wtype):
    g = _gen(m * 31 + n)
    x, y, kw = _norm_case(g, m, n, stream, dtype, post, gate, wtype, pad)
    sigmoid = gate == "token"
    new, off, h, h_off = _norm_want(x, y, kw, 1e-5, 0.9, 1.7, sigmoid)
    keep = x.clone()
    args = dict(kw, eps=1e-5, x_scale=0.9, y_scale=1.7, gate_sigmoid=sigmoid)
    out = int8.block_norm(x, y, x_out=torch.empty_like(x), out_dtype=dtype, **args)
    assert torch.equal(x, keep) and out.dtype == dtype
    far = (out.double() - h).abs() - (h_off + HALF[dtype] * (h.abs() + h_off) + 1e-30 + (2.0 ** -24 if dtype == F16 else 0.0))
    assert float(far.max()) <= 0.0, float(far.max())
    rows = int8.block_norm(x, y, int8=True, **args)                       # in place
    far = (x.double() - new).abs() - (off + HALF[stream] * (new.abs() + off) + (2.0 ** -24 if stream == F16 else 0.0))
    assert float(far.max()) <= 0.0, float(far.max())
    # codes are within half a step of h / factor, and h's own error
    s = rows.scale.double()[:, None]
    assert float(((rows.q.double() * s - h).abs() - (0.5 * s + h_off + 2.0 ** -20 * h.abs())).max()) <= 0.0
    peak = h.abs().amax(1)
    assert float(((rows.scale.double() * 127.0 - peak).abs() - (h_off.amax(1) + 2.0 ** -22 * peak)).max()) <= 0.0


def test_block_norm_parts_that_are_left_out():
    g = _gen(11)
    x = _rand(g, 9, 896)
    keep = x.clone()
    w = _rand(g, 896)
    h = int8.block_norm(x, pre=w)
    assert torch.equal(x, keep)
    torch.testing.assert_close(h, reference.rms(x, w, 1e-6), rtol=2.0 ** -18, atol=0.0)
    assert torch.equal(int8.block_norm(x, keep, y_scale=-1.0), torch.zeros_like(x)) and bool((x == 0).all())
    z = int8.block_norm(x, pre=w, int8=True)
    assert bool((z.q == 0).all()) and bool((z.scale == 0).all())          # a stream of zeros


# ---- as they are used ----
def test_an_8_bit_block_and_its_score():
    """norm -> gated product -> product -> norm -> LM head -> log probabilities, one call after the other on one stream; against the same formulas in
    64 bits on the 8-bit rows that the calls made."""
    g = _gen(21)
    t, hidden, inter, vocab = 37, 896, 4864, 5003
    x = _rand(g, t, hidden).bfloat16()
    gate_up, down, head = (int8.quantize_weight(0.05 * _rand(g, n, k)) for n, k in ((2 * inter, hidden), (hidden, inter), (vocab, hidden)))
    n1, n2 = _rand(g, hidden), _rand(g, hidden)
    tokens = torch.randint(0, vocab, (t,), generator=g, device="cuda")
    rows = int8.block_norm(x, pre=n1, int8=True)
    act = int8.gemm_int8(rows, gate_up.q, gate_up.scale, epilogue="swiglu")
    y = int8.gemm_int8(act, down.q, down.scale)
    last = int8.block_norm(x, y, pre=n2, int8=True)
    logits = int8.gemm_int8(last, head.q, head.scale, out_dtype=F32)
    r = ops.token_logprobs(logits, tokens, top=3, entropy=True)
    ops.check_status()
    v = (rows.float().double() @ gate_up.float().double().t()).view(t, -1, 2, 128)
    want_act = (torch.nn.functional.silu(v[:, :, 0]) * v[:, :, 1]).reshape(t, -1)
    torch.testing.assert_close(act.double(), want_act, rtol=2.0 ** -8, atol=1e-4)
    torch.testing.assert_close(y.double(), int8.quantize_rows(act).float().double() @ down.float().double().t(), rtol=2.0 ** -8, atol=1e-4)
    lp = torch.log_softmax(last.float().double() @ head.float().double().t(), 1)
    torch.testing.assert_close(r.logprob.double(), lp.gather(1, tokens[:, None])[:, 0], rtol=1e-5, atol=1e-4)
    torch.testing.assert_close(r.top_logprobs.double(), lp.topk(3).values, rtol=1e-5, atol=1e-4)


def test_replayed_graphs_streams_and_two_calls_at_once():
    g = _gen(22)
    cases = [(1, 4608, 3584), (20, 20000, 512), (300, 20000, 896)]        # a cluster, ranges, whole tiles and ranges
    for m, n, k in cases:
        w, c = _weight(g, n, k)
        xs = [_rand(g, m, k).bfloat16() for _ in range(3)]
        want = [int8.gemm_int8(x, w, c) for x in xs]
        x = xs[0].clone()
        int8.gemm_int8(x, w, c)
        torch.cuda.synchronize()
        graphs = []
        for _ in range(2):
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                y = int8.gemm_int8(x, w, c)
                z = int8.gemm_int8(int8.quantize_rows(x), w, c)
            graphs.append((graph, y, z))
        for i in (1, 2, 0, 1):
            x.copy_(xs[i])
            for graph, y, z in graphs:
                graph.replay()
            for graph, y, z in graphs:
                assert torch.equal(y, want[i]) and torch.equal(z, want[i])
        streams = [torch.cuda.Stream() for _ in range(3)]
        torch.cuda.synchronize()
        got = []
        for s, v in zip(streams, xs):
            with torch.cuda.stream(s):
                got.append([int8.gemm_int8(v, w, c) for _ in range(4)])
        torch.cuda.synchronize()
        for many, right in zip(got, want):
            for one in many:
                assert torch.equal(one, right)
    ops.check_status()


def test_products_inside_a_step_whose_kernels_start_early():
    g = _gen(23)
    w, c = _weight(g, 2048, 2048)
    x = _rand(g, 8, 2048).bfloat16()
    n = torch.ones(2048, device="cuda")

    def step(v):
        v = v.clone()
        for _ in range(3):
            rows = int8.block_norm(v, pre=n, int8=True)
            y = int8.gemm_int8(rows, w, c)
            y = int8.gemm_int8(y, w, c)
            int8.block_norm(v, y, y_scale=0.1)
        return v
    want = step(x)
    with ops.launch_scope(ops.rows_workspace(16, x.device), True):
        torch.cuda.synchronize()
        got = step(x)
    assert torch.equal(got, want)
    ops.check_status()


@pytest.mark.parametrize("m,n", [(700, 897), (300, 3584), (5, 64), (900, 50)])
def test_norms_in_the_place_of_what_they_read(m, n):
    g = _gen(m)
    x, y, kw = _norm_case(g, m, n, BF16, BF16, True, "token", F32)
    new = torch.empty_like(x)
    h = int8.block_norm(x, y, x_out=new, gate_sigmoid=True, **kw)
    a, b = x.clone(), y.clone()
    assert int8.block_norm(a, b, out=b, gate_sigmoid=True, **kw) is b
    assert torch.equal(a, new) and torch.equal(b, h)
    a, b = x.clone(), y.clone()
    rows = int8.block_norm(a, b, x_out=b, gate_sigmoid=True, int8=True, **kw)
    assert torch.equal(a, x) and torch.equal(b, new) and torch.equal(rows.q, int8.block_norm(x, y, x_out=new, gate_sigmoid=True, int8=True, **kw).q)


@pytest.mark.parametrize("m,n,k,gated,cut", [(20, 19072, 11000, False, True), (100, 20000, 15000, False, True), (40, 38400, 13000, True, True),
                                             (3000, 5000, 14000, False, False), (8192, 3584, 18944, False, True)])
def test_long_k_and_tiles_that_are_cut_into_ranges(m, n, k, gated, cut):
    # cut where a few tiles more than fill the SMs: workspace beyond that for the rows
    assert (int8._workspace(m, n, k, gated, False) > 0) is cut
    _check_product(_gen(m + n), m, n, k, BF16, True, not gated, gated)
    _check_product(_gen(m + k), m, n, k, F16, True, False, gated, as_rows=True)


@pytest.mark.parametrize("m,n,k,dtype,bias,residual", [(4100, 4001, 4096, F32, False, True), (300, 29000, 3100, BF16, True, False), (1025, 11008, 4097, F16, True, True)])
def test_long_products_of_many_tiles(m, n, k, dtype, bias, residual):
    g = _gen(m)
    _check_product(g, m, n, k, dtype, bias, residual, False)
    x, (w, c) = _rows(g, m, k, dtype), _weight(g, n, k)
    res = _rand(g, m, n).to(dtype) if residual else None
    whole = int8.gemm_int8(x, w, c, residual=res)
    parts = [int8.gemm_int8(x[i:i + 160], w, c, residual=None if res is None else res[i:i + 160]) for i in range(0, m, 160)]
    assert torch.equal(whole, torch.cat(parts))            # divided in another way: whole numbers add up to the same
    buf = torch.full((m + 1, n + 8), 7.0, device="cuda", dtype=dtype)
    int8.gemm_int8(x, w, c, residual=res, out=buf[:m, :n])
    assert torch.equal(buf[:m, :n], whole) and bool((buf[m] == 7.0).all()) and bool((buf[:, n:] == 7.0).all())


def test_long_products_on_two_streams_and_replayed():
    g = _gen(5)
    x, (w, c) = _rows(g, 700, 3200, BF16), _weight(g, 19200, 3200)
    want = int8.gemm_int8(x, w, c)
    streams, got = [torch.cuda.Stream() for _ in range(2)], []
    torch.cuda.synchronize()
    for _ in range(3):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(int8.gemm_int8(x, w, c))
    torch.cuda.synchronize()
    assert all(torch.equal(want, t) for t in got)
    graph, y = torch.cuda.CUDAGraph(), torch.empty_like(want)
    with torch.cuda.graph(graph):
        int8.gemm_int8(x, w, c, out=y)
    for i in range(2):
        x.mul_(-1.0)
        y.zero_()
        graph.replay()
        assert torch.equal(y, -want if i == 0 else want)
    ops.check_status()
