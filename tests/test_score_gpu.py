"""Scoring, log probabilities of answers and decoders with 8-bit weights on the GPU engine."""
import numpy as np
import pytest
import torch

from onnx_genai_b200 import ops
from onnx_genai_b200.engine.api import Engine, GenerateOptions
from onnx_genai_b200.engine.llm_engine import EngineConfig, LLMEngine
from onnx_genai_b200.models.config import DecoderConfig
from onnx_genai_b200.models.decoder import quantize_int8, random_weights

pytestmark = pytest.mark.gpu

CFG = DecoderConfig(name="g", num_layers=3, hidden=256, num_heads=8, num_kv_heads=2, head_dim=64, intermediate=480, vocab=1024, rope_theta=1e6,
                    tie_embeddings=False, qkv_bias=True, max_position=1024)


def _llm(device="cuda", weights=None, cfg=CFG, **kw):
    return LLMEngine(EngineConfig(model=cfg, num_pages=256, max_seqs=8, max_tokens_per_step=512, max_seq_len=512, max_logit_rows=256, **kw), weights=weights, device=device)


def _tokens(n, seed=0):
    return np.random.default_rng(seed).integers(0, CFG.vocab, size=n).tolist()


def _rows(llm, tokens):
    sid = llm.open_forced(tokens, range(len(tokens)))
    rows = []
    while llm.forced_pending(sid) > 0:
        rows += llm.step().forced_logits.get(sid, [])
    llm.close_forced(sid)
    return torch.stack([r for _, r in rows]).double()


def test_scores_are_the_log_softmax_of_the_rows():
    llm = _llm()
    before = ops.launch_counts["token_logprobs"]
    tokens = _tokens(200)
    r, = llm.score([tokens], top=5, entropy=True)
    assert ops.launch_counts["token_logprobs"] > before
    lp = torch.log_softmax(_rows(llm, tokens), 1)[:-1].cpu()
    torch.testing.assert_close(r.logprob.double(), lp.gather(1, torch.tensor(tokens[1:])[:, None])[:, 0], rtol=0, atol=1e-4)
    torch.testing.assert_close(r.top_logprobs.double(), lp.topk(5).values, rtol=0, atol=1e-4)
    torch.testing.assert_close(r.entropy.double(), -(lp.exp() * lp).sum(1), rtol=0, atol=1e-4)


@pytest.mark.parametrize("cuda_graphs", [False, True])
def test_greedy_answers_with_log_probabilities_stay_on_the_device(cuda_graphs):
    eng = Engine(_llm(cuda_graphs=cuda_graphs))
    prompts = [_tokens(n, n) for n in (5, 40, 17)]
    base = eng.generate_batch(prompts, GenerateOptions(max_new_tokens=12, greedy=True, ignore_eos=True))
    d2h = eng.llm.d2h_bytes
    got = eng.generate_batch(prompts, GenerateOptions(max_new_tokens=12, greedy=True, ignore_eos=True, logprobs=4))
    assert eng.llm.d2h_bytes - d2h < 3 * 12 * CFG.vocab and not eng.llm.device_logprobs
    for p, a, b in zip(prompts, base, got):
        assert a.token_ids == b.token_ids and len(b.logprobs) == 12
        r, = eng.llm.score([p + b.token_ids])
        want = r.logprob[len(p) - 1:].tolist()
        for (lp, top), tok, w in zip(b.logprobs, b.token_ids, want):
            # scored as a prompt, decoded row by row: bf16 activations of two orders of sums
            assert top[0][0] == tok and top[0][1] == lp and len(top) == 4 and abs(lp - w) < 0.1
    sampled = eng.generate(prompts[0], GenerateOptions(max_new_tokens=3, temperature=0.8, seed=3, ignore_eos=True, logprobs=2))
    assert len(sampled.logprobs) == 3                      # drawn tokens still go over the host


def test_a_decoder_with_8_bit_weights_against_the_cpu_engine():
    wg, wc = random_weights(CFG, "cuda", seed=11, std=0.05), random_weights(CFG, "cpu", seed=11, std=0.05, dtype=torch.float32)
    for lg, lc in zip(wg.layers, wc.layers):
        for name in ("qkv_w", "qkv_b", "o_w", "gate_up_w", "down_w"):
            getattr(lc, name).copy_(getattr(lg, name).float().cpu())
    wc.embed.copy_(wg.embed.float().cpu())
    wc.lm_head.copy_(wg.lm_head.float().cpu())
    gpu, cpu = _llm(weights=wg, weight_dtype="int8"), _llm("cpu", weights=wc, weight_dtype="int8")
    for a, b in zip(gpu.weights.layers, cpu.weights.layers):
        for name in ("qkv", "o", "gate_up", "down"):
            assert torch.equal(a.int8[name].q.cpu(), b.int8[name].q) and torch.equal(a.int8[name].scale.cpu(), b.int8[name].scale)
    tokens = _tokens(150, 4)
    before = dict(ops.launch_counts)
    got = _rows(gpu, tokens).cpu()
    want = _rows(cpu, tokens)
    # the bound of the same comparison with dense weights: bf16 against 32 bits
    assert float((got - want).norm() / want.norm()) < 3e-2
    assert ops.launch_counts["gemm_int8"] - before.get("gemm_int8", 0) == 4 * CFG.num_layers
    assert ops.launch_counts["block_norm"] - before.get("block_norm", 0) == 2 * CFG.num_layers
    ops.check_status()


@pytest.mark.parametrize("kv_dtype,cuda_graphs", [("bf16", False), ("bf16", True), ("fp8", False)])
def test_8_bit_weights_in_continuous_batching(kv_dtype, cuda_graphs):
    """The same requests twice.  (Without the prefix cache: with it the second run decodes the last token of a 65-token prompt where the first ran it in a
    chunk, and attention sums in another order.)"""
    cfg = CFG.replace(num_heads=4, head_dim=128) if kv_dtype == "fp8" else CFG          # one-byte pages are built for heads of 128
    w = quantize_int8(random_weights(cfg, "cuda", seed=2, std=0.08))
    llm = _llm(weights=w, cfg=cfg, weight_dtype="int8", kv_dtype=kv_dtype, cuda_graphs=cuda_graphs, enable_prefix_cache=False)
    prompts = [np.asarray(_tokens(n, n), dtype=np.int32) for n in (3, 64, 65, 200, 1)]
    outs = llm.generate(prompts, max_new_tokens=20)
    assert all(len(o) == 20 for o in outs)
    again = llm.generate(prompts, max_new_tokens=20)
    assert [list(a) for a in outs] == [list(a) for a in again]
    ops.check_status()
