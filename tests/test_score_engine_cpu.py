"""Scoring beside what an engine does otherwise: after requests, over cached prefixes, and weights that are turned into 8 bits."""
import numpy as np
import pytest
import torch

from onnx_genai_b200.engine.llm_engine import EngineConfig, LLMEngine
from onnx_genai_b200.models.config import DecoderConfig
from onnx_genai_b200.models.decoder import quantize_int8, random_weights

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


def _forced(eng, tokens, want):
    """Rows of the wanted places, and how many tokens the engine computed for them."""
    sid = eng.open_forced(tokens, want)
    rows, computed = [], 0
    while eng.forced_pending(sid) > 0:
        out = eng.step()
        rows += out.forced_logits.get(sid, [])
        computed += out.num_tokens
    eng.close_forced(sid)
    assert [p for p, _ in rows] == list(want)
    return torch.stack([r for _, r in rows]), computed


@pytest.mark.parametrize("first,cached", [(0, 0), (15, 0), (16, 16), (47, 32), (48, 48), (63, 48), (89, 80)])
def test_forced_rows_take_from_the_prefix_cache_what_lies_ahead_of_them(first, cached):
    tokens = _tokens(90, 3)
    want = list(range(first, 90, 17)) + ([89] if (89 - first) % 17 else [])
    fresh, all_of_it = _forced(_engine(max_logit_rows=90, enable_prefix_cache=False), tokens, want)
    eng = _engine(max_logit_rows=90)
    _, computed = _forced(eng, tokens, [89])
    assert computed == all_of_it == 90
    rows, computed = _forced(eng, tokens, want)
    assert computed == 90 - cached
    torch.testing.assert_close(rows, fresh, rtol=0, atol=1e-4)


def test_scores_of_texts_that_share_a_prefix():
    shared = _tokens(50, 4)
    texts = [shared + _tokens(n, 5 + n) for n in (3, 30, 1)] + [shared]
    eng = _engine()
    for text, r in zip(texts, eng.score(texts, top=2, entropy=True)):
        want, = _engine(enable_prefix_cache=False).score([text], top=2, entropy=True)
        torch.testing.assert_close(r.logprob, want.logprob, rtol=0, atol=1e-5)
        assert torch.equal(r.top_ids, want.top_ids)


@pytest.mark.parametrize("bad", ["int4", "experts", "infinite"])
def test_weights_that_cannot_be_held_in_8_bits_stay_as_they_are(bad):
    w = _weights()
    last = w.layers[1]
    if bad == "int4":
        last.quant = {"o": None}
    elif bad == "experts":
        last.router_w = torch.zeros(4, CFG.hidden)
    else:
        last.down_w[3, 5] = float("inf")
    keep = [(l.qkv_w, l.qkv_b, l.o_w, l.gate_up_w, l.down_w) for l in w.layers]
    with pytest.raises(ValueError, match="layer 1"):
        quantize_int8(w)
    for l, was in zip(w.layers, keep):
        assert not l.int8 and all(a is b for a, b in zip((l.qkv_w, l.qkv_b, l.o_w, l.gate_up_w, l.down_w), was))
