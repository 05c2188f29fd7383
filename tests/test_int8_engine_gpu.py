"""8-bit operators inside the engine on the GPU: the pool of pages, texts that share a prefix, log probabilities against 64 bits, and the divisions of
the work under replay and on several streams."""
import math
import subprocess
import sys

import numpy as np
import pytest
import torch

from onnx_genai_b200 import ops
from onnx_genai_b200.engine.api import Engine, GenerateOptions
from onnx_genai_b200.engine.llm_engine import EngineConfig, LLMEngine
from onnx_genai_b200.engine.processors import LogitProcessor
from onnx_genai_b200.models.config import DecoderConfig
from onnx_genai_b200.models.decoder import random_weights
from onnx_genai_b200.ops import hybrid, int8

pytestmark = pytest.mark.gpu

GIB = 1 << 30


PAGES = """
import torch
from onnx_genai_b200.engine.llm_engine import EngineConfig, LLMEngine
from onnx_genai_b200.models.config import DecoderConfig
from onnx_genai_b200.models.decoder import random_weights

cfg = DecoderConfig(name="wide", num_layers=8, hidden=2048, num_heads=16, num_kv_heads=4, head_dim=128, intermediate=8192, vocab=1024, rope_theta=1e6,
                    tie_embeddings=False, qkv_bias=True, max_position=4096)
weights = random_weights(cfg, "cuda", seed=1)
matrices = sum(t.numel() for l in weights.layers for t in (l.qkv_w, l.o_w, l.gate_up_w, l.down_w))
torch.cuda.empty_cache()
free, total = torch.cuda.mem_get_info()
# a share of the device that leaves pages one GiB with the weights as they are
eng = LLMEngine(EngineConfig(model=cfg, max_seqs=64, max_seq_len=4096, max_tokens_per_step=512, weight_dtype="int8",
                             gpu_memory_utilization=1.0 - (free - 2 ** 30) / total), weights=weights, device="cuda")
print(eng.num_pages, cfg.num_layers * 2 * cfg.num_kv_heads * cfg.head_dim * 16 * 2, matrices)
"""


def test_pages_get_the_memory_that_8_bit_weights_give_back():
    """In a process of its own: what other tests still hold inside the allocator's blocks decides which of these can go back to the device."""
    r = subprocess.run([sys.executable, "-c", PAGES], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr
    pages, page, matrices = (int(v) for v in r.stdout.split()[-3:])
    # half of the matrices' bytes come back; an eighth of that for the step's buffers and what the allocator's blocks leave between them
    assert pages < 64 * 256 + 64 and pages * page > GIB + matrices * 7 // 8


CFG = DecoderConfig(name="g", num_layers=3, hidden=256, num_heads=8, num_kv_heads=2, head_dim=64, intermediate=480, vocab=1024, rope_theta=1e6,
                    tie_embeddings=False, qkv_bias=True, max_position=1024)


def _llm(**kw):
    return LLMEngine(EngineConfig(model=CFG, num_pages=256, max_seqs=8, max_tokens_per_step=512, max_seq_len=512, **kw), device="cuda")


def _tokens(n, seed=0):
    return np.random.default_rng(seed).integers(0, CFG.vocab, size=n).tolist()


@pytest.mark.parametrize("rows", [8, 256])
def test_scores_of_texts_that_share_a_prefix(rows):
    shared = _tokens(70, 1)
    texts = [shared + _tokens(n, 2 + n) for n in (5, 100, 1)] + [shared]
    llm, fresh = _llm(max_logit_rows=rows), _llm(max_logit_rows=rows, enable_prefix_cache=False)
    for again in range(2):
        for got, text in zip(llm.score(texts, top=3, entropy=True), texts):
            want, = fresh.score([text], top=3, entropy=True)
            assert torch.equal(got.logprob, want.logprob) and torch.equal(got.top_ids, want.top_ids) and torch.equal(got.entropy, want.entropy)
    ops.check_status()


def test_forced_rows_behind_cached_pages():
    tokens = _tokens(200, 3)

    def row(llm):
        sid = llm.open_forced(tokens, [199])
        ran, got = 0, []
        while llm.forced_pending(sid) > 0:
            out = llm.step()
            ran += out.num_tokens
            got += out.forced_logits.get(sid, [])
        llm.close_forced(sid)
        assert [p for p, _ in got] == [199]
        return got[0][1].double(), ran
    llm = _llm()
    first, ran = row(llm)
    second, rest = row(llm)
    assert ran == 200 and rest == 200 - 192
    # the last 8 tokens by themselves: bf16 activations of sums in another order
    assert float((first - second).norm() / first.norm()) < 3e-2


class _Watch(LogitProcessor):
    """Leaves logits as they are and keeps the largest; a processor of unknown effect sends a request over the host."""

    def __init__(self):
        self.peak = []

    def process(self, token_ids, logits):
        self.peak.append(float(np.abs(logits).max()))
        return logits


def test_log_probabilities_of_greedy_answers_against_the_softmax_in_64_bits():
    """On the device they are sums in 32 bits of approximate exponentials; the host's way takes the same rows in 64."""
    eng = Engine(_llm(enable_prefix_cache=False))
    opt = GenerateOptions(max_new_tokens=24, greedy=True, ignore_eos=True, logprobs=20)
    for n in (5, 130):
        before = ops.launch_counts["token_logprobs"]
        a = eng.generate(_tokens(n, n), opt)
        on_device = ops.launch_counts["token_logprobs"] - before
        watch = _Watch()
        b = eng.generate(_tokens(n, n), opt, processors=(watch,))
        assert on_device == 24 and ops.launch_counts["token_logprobs"] == before + 24 and len(watch.peak) == 24 and a.token_ids == b.token_ids
        for (lp, top), (lp64, top64), peak in zip(a.logprobs, b.logprobs, watch.peak):
            # s: a thread adds at most vocab / 256 values in a row, joins add 11, the exponential is off by 2^-21 with its argument's rounding; then
            # x - m and - log s round by 2^-24 of their sizes, at most 2 peak and 2 peak + log vocab
            bound = (CFG.vocab / 256 + 11) * 2.0 ** -24 + 2.0 ** -21 + 2.0 ** -24 * (4.0 * peak + 2.0 * math.log(CFG.vocab))
            assert bound < 1e-4 and abs(lp - lp64) <= bound
            assert len(top) == len(top64) == 20 and all(abs(v - w) <= bound for (_, v), (_, w) in zip(top, top64))


@pytest.mark.parametrize("m,n,k,gated,cut", [
    (20, 4608, 3584, False, False),        # 36 tiles: a cluster each
    (20, 19072, 11000, False, True),       # 149 tiles, one more than SMs: it is cut into ranges
    (40, 38400, 13000, True, True),        # gated, 150 tiles
    (300, 20000, 896, False, False),       # whole tiles
    (8192, 3584, 18944, False, True),      # pairs of CTAs, 448 tiles on 74 pairs: four are cut
])
@pytest.mark.parametrize("as_rows", [False, True])
def test_every_division_of_the_work_replayed_and_on_several_streams(m, n, k, gated, cut, as_rows):
    """Counters (zeroed by the rows' kernel, or where rows come beforehand by a memset) and partial sums are a call's own: two graphs, three streams."""
    assert (int8._workspace(m, n, k, gated, False) > 0) is cut
    g = torch.Generator(device="cuda").manual_seed(m + n)
    w = torch.randint(-127, 128, (n, (k + 15) // 16 * 16), generator=g, device="cuda", dtype=torch.int8)[:, :k]
    c = (0.5 + torch.rand(n, generator=g, device="cuda")) * 0.01
    xs = [torch.randn(m, k, generator=g, device="cuda").bfloat16() for _ in range(3)]
    kw = {"epilogue": "swiglu"} if gated else {}
    made = [int8.quantize_rows(x) for x in xs]
    run = lambda a: int8.gemm_int8(a, w, c, **kw)                   # noqa: E731
    want = [run(r if as_rows else x) for r, x in zip(made, xs)]
    # the other way, divided alike, and a part of the rows, divided in another way: whole numbers add up to the same
    assert torch.equal(run(xs[0] if as_rows else made[0]), want[0])
    part = int8.Int8Rows(made[0].q[:3], made[0].scale[:3])
    assert torch.equal(run(part), want[0][:3])
    x, r = xs[0].clone(), int8.quantize_rows(xs[0])
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = run(r if as_rows else x)
        graphs.append((graph, y))
    for i in (1, 2, 0, 0, 1):
        x.copy_(xs[i])
        r.q.copy_(made[i].q)
        r.scale.copy_(made[i].scale)
        for graph, y in graphs:
            y.fill_(7.0)
            graph.replay()
            graph.replay()
        for graph, y in graphs:
            assert torch.equal(y, want[i])
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    got = []
    for _ in range(3):
        for s, a in zip(streams, made if as_rows else xs):
            with torch.cuda.stream(s):
                got.append(run(a))
    torch.cuda.synchronize()
    for i, y in enumerate(got):
        assert torch.equal(y, want[i % 3])
    ops.check_status()


@pytest.mark.parametrize("t,w", [(1, 896), (37, 2048), (700, 1001 // 8 * 8)])
@pytest.mark.parametrize("post", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_block_norm_and_norm_step_are_one_step(t, w, post, dtype):
    """The step between two sublayers of the hybrid decoders, x += post(y), h = norm(x), is a case of block_norm: both are within 2^-18 of the formula
    (tests/test_int8_gpu.py), and so within 2^-17 of each other before they round."""
    g = torch.Generator(device="cuda").manual_seed(t + w)
    x, y = torch.randn(t, w, generator=g, device="cuda"), torch.randn(t, w, generator=g, device="cuda").to(dtype)
    pw, nw = (1.0 + 0.2 * torch.randn(w, generator=g, device="cuda") for _ in range(2))
    a, h = x.clone(), torch.empty(t, w, device="cuda", dtype=dtype)
    hybrid.norm_step(a, y, hybrid.RmsNorm(pw, 1e-6) if post else None, hybrid.RmsNorm(nw, 1e-6), h)
    b = x.clone()
    got = int8.block_norm(b, y, post=pw if post else None, pre=nw, eps=1e-6, out_dtype=dtype)
    part = (b - x).abs()
    off = 2.0 ** -17 * (x.abs() + part) + 2.0 ** -23 * b.abs()
    assert bool(((a - b).abs() <= off).all())
    size = b.pow(2).mean(1, keepdim=True).sqrt()
    through = off.pow(2).mean(1, keepdim=True).sqrt() / size
    half = 2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -24
    bound = off / size * nw.abs() + got.abs().float() * (2.0 ** -17 + through + 2.0 * half)
    assert bool(((h.float() - got.float()).abs() <= bound).all())
