"""Scoring beside what an engine does otherwise: after requests, over cached prefixes, and weights that are turned into 8 bits."""
import numpy as np
import pytest
import torch

from onnx_genai_b200.engine.llm_engine import EngineConfig, LLMEngine
from onnx_genai_b200.models.config import DecoderConfig
from onnx_genai_b200.models.decoder import random_weights

CFG = DecoderConfig(name="t", num_layers=2, hidden=64, num_heads=4, num_kv_heads=2, head_dim=16, intermediate=96, vocab=300,
                    rope_theta=1e4, tie_embeddings=True, qkv_bias=True, max_position=512)


def _weights():
    return random_weights(CFG, "cpu", seed=5, std=0.3, dtype=torch.float32)


def _engine(weights=None, **kw):
    return LLMEngine(EngineConfig(model=CFG, num_pages=128, max_seqs=4, max_tokens_per_step=64, max_seq_len=256, **kw), weights=weights or _weights(), device="cpu")


def _tokens(n, seed=0):
    return np.random.default_rng(seed).integers(0, CFG.vocab, size=n).tolist()


def test_an_engine_scores_after_it_has_generated():
    tokens = _tokens(20)
    want, = _engine().score([tokens])
    eng = _engine()
    eng.generate([[1, 2, 3]], 4)
    got, = eng.score([tokens])
    assert torch.equal(got.logprob, want.logprob)
    sid = eng.add_request([1, 2, 3], 2)
    while eng.has_work:
        eng.step()
    eng.core.release(sid)
    again, = eng.score([tokens])
    assert torch.equal(again.logprob, want.logprob)
    eng.add_request([1, 2, 3], 2)
    with pytest.raises(RuntimeError):
        eng.score([tokens])
