"""Scoring given texts, and decoders with 8-bit weights, on the CPU engine."""
import json
import math
import subprocess
import sys

import numpy as np
import pytest
import torch

from onnx_genai_b200.engine.api import Engine, GenerateOptions
from onnx_genai_b200.engine.llm_engine import EngineConfig, LLMEngine
from onnx_genai_b200.models.config import DecoderConfig
from onnx_genai_b200.models.decoder import quantize_int8, random_weights
from onnx_genai_b200.ops import reference as ref
from onnx_genai_b200.package.export import export_package

CFG = DecoderConfig(name="t", num_layers=2, hidden=64, num_heads=4, num_kv_heads=2, head_dim=16, intermediate=96, vocab=300,
                    rope_theta=1e4, tie_embeddings=True, qkv_bias=True, max_position=512)


def _weights():
    return random_weights(CFG, "cpu", seed=5, std=0.3, dtype=torch.float32)


def _engine(weights=None, **kw):
    return LLMEngine(EngineConfig(model=CFG, num_pages=128, max_seqs=4, max_tokens_per_step=64, max_seq_len=256, **kw), weights=weights or _weights(), device="cpu")


def _logits(eng, tokens):
    """Rows of all positions, by the forced sequences' own way."""
    eng.cfg.enable_prefix_cache = False
    rows, at, sid = [], 0, None
    while at < len(tokens):
        piece = tokens[at:at + eng.logit_row_limit]
        if sid is None:
            sid = eng.open_forced(piece, range(len(piece)))
        else:
            eng.extend_forced(sid, piece, range(len(piece)))
        at += len(piece)
        while eng.forced_pending(sid) > 0:
            rows += eng.step().forced_logits.get(sid, [])
    eng.close_forced(sid)
    assert [p for p, _ in rows] == list(range(len(tokens)))
    return torch.stack([r for _, r in rows]).double()


@pytest.mark.parametrize("n", [1, 2, 4, 17, 130])
def test_scores_are_the_log_softmax_of_the_rows(n):
    tokens = np.random.default_rng(n).integers(0, CFG.vocab, size=n).tolist()
    lp = torch.log_softmax(_logits(_engine(enable_prefix_cache=False), tokens), 1)[:-1]
    eng = _engine()
    for again in range(2):                      # the second time its pages are in the prefix cache
        r, = eng.score([tokens], top=3, entropy=True)
        assert r.logprob.shape == (n - 1,) and r.top_ids.shape == (n - 1, 3)
        if n > 1:
            torch.testing.assert_close(r.logprob.double(), lp.gather(1, torch.tensor(tokens[1:])[:, None])[:, 0], rtol=0, atol=1e-5)
            torch.testing.assert_close(r.entropy.double(), -(lp.exp() * lp).sum(1), rtol=0, atol=1e-5)
            assert torch.equal(r.top_ids.long(), lp.topk(3).indices)
    assert not eng.has_work and not eng.forced


def test_pieces_of_any_size_give_the_same_scores():
    tokens = np.random.default_rng(3).integers(0, CFG.vocab, size=90).tolist()
    a, = _engine().score([tokens])
    b, c = _engine(max_logit_rows=200).score([tokens, tokens[:40]])
    torch.testing.assert_close(a.logprob, b.logprob, rtol=0, atol=1e-5)
    torch.testing.assert_close(c.logprob, b.logprob[:39], rtol=0, atol=1e-5)


def test_what_score_refuses():
    eng = _engine()
    for bad in ([[]], [[CFG.vocab]], [[-1, 3]]):
        with pytest.raises(ValueError):
            eng.score(bad)
    with pytest.raises(ValueError):
        eng.score([[1] * 300])
    for top in (-1, 33):
        with pytest.raises(ValueError):
            eng.score([[1, 2, 3]], top=top)
    assert not eng.forced and not eng.scoring
    eng.add_request([1, 2, 3], 2)
    with pytest.raises(RuntimeError):
        eng.score([[1, 2]])


def _oracle_int8(w, tokens):
    """A decoder whose products take 8-bit rows, in 64 bits, over all tokens at once."""
    rms = lambda v, g: v / (v.pow(2).mean(-1, keepdim=True) + CFG.rms_eps).sqrt() * g.double()      # noqa: E731

    def product(v, m, bias=None):
        q, s = ref.quantize_rows(v.float())
        y = (q.double() * s.double()[:, None]) @ (m.q.double() * m.scale.double()[:, None]).t()
        return y if bias is None else y + bias.double()
    t, d = len(tokens), CFG.head_dim
    x = w.embed[torch.tensor(tokens)].double()
    cs = ref.rope_table(CFG.max_position, d, CFG.rope_theta)
    for l in w.layers:
        qkv = product(rms(x, l.ln1), l.int8["qkv"], l.int8["qkv_b"])
        q, k, v = qkv.split([CFG.num_heads * d, CFG.num_kv_heads * d, CFG.num_kv_heads * d], 1)
        turn = lambda z: ref.apply_rope(z.float().view(t, -1, d), torch.arange(t), cs, d).double()    # noqa: E731
        q, k, v = turn(q), turn(k), v.view(t, -1, d)
        heads = []
        for h in range(CFG.num_heads):
            kv = h // (CFG.num_heads // CFG.num_kv_heads)
            a = q[:, h] @ k[:, kv].t() / math.sqrt(d)
            heads.append(torch.softmax(a.masked_fill(torch.ones(t, t).triu(1).bool(), -math.inf), 1) @ v[:, kv])
        x = x + product(torch.cat(heads, 1), l.int8["o"])
        g = product(rms(x, l.ln2), l.int8["gate_up"]).view(t, -1, 2, 128)
        x = x + product((torch.nn.functional.silu(g[:, :, 0]) * g[:, :, 1]).reshape(t, -1), l.int8["down"])
    return rms(x, w.final_norm) @ w.lm_head.double().t()


def test_a_decoder_with_8_bit_weights_is_its_formula():
    tokens = np.random.default_rng(9).integers(0, CFG.vocab, size=40).tolist()
    eng = _engine(weight_dtype="int8", enable_prefix_cache=False)
    got = _logits(eng, tokens)
    want = _oracle_int8(eng.weights, tokens)
    # 32 against 64 bits decide a few codes that lie next to a half differently: one step in 127 of one of a row's 64 values or more
    assert float((got - want).norm() / want.norm()) < 1e-2
    assert eng.weights.layers[0].qkv_w is None and eng.weights.layers[0].int8["down"].q.shape == (64, 128)
    dense = _logits(_engine(enable_prefix_cache=False), tokens)
    # weights and rows in 8 bits: half a step each of 1/127 of a maximum some three times the root mean square, in two layers of four products
    assert 1e-4 < float((got - dense).norm() / dense.norm()) < 0.1


def test_what_8_bit_weights_refuse():
    w = quantize_int8(_weights())
    assert quantize_int8(w) is w                          # nothing is done twice
    with pytest.raises(ValueError):
        _engine(weight_dtype="int4")
    with pytest.raises(ValueError):
        _engine(weight_dtype="int8", weight_offload_layers=1)
    w = _weights()
    w.layers[1].quant = {"o": None}
    with pytest.raises(ValueError):
        quantize_int8(w)


@pytest.fixture(scope="module")
def model_dir(tmp_path_factory):
    return export_package(CFG, _weights(), str(tmp_path_factory.mktemp("pkg")))


def test_engine_and_command(model_dir):
    eng = Engine.from_dir(model_dir, device="cpu", num_pages=128, max_seqs=4, max_tokens_per_step=64)
    a, b = eng.score(["hello world", [5, 6, 7]], top=2)
    assert a["token_ids"] == eng.tokenize("hello world") and len(a["logprobs"]) == len(a["token_ids"]) - 1 == len(a["top"])
    assert abs(math.log(b["perplexity"]) + sum(b["logprobs"]) / 2) < 1e-9 and all(len(t) == 2 for t in b["top"])
    assert eng.score([[5]])[0]["perplexity"] is None
    r = subprocess.run([sys.executable, "-m", "onnx_genai_b200", "score", model_dir, "--ids", "--text", "5 6 7", "--device", "cpu", "--weight-dtype", "int8"],
                       capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    doc = json.loads(r.stdout)
    assert doc["token_ids"] == [5, 6, 7] and "perplexity" in r.stderr
    eight = Engine.from_dir(model_dir, device="cpu", num_pages=128, max_seqs=4, max_tokens_per_step=64, weight_dtype="int8")
    assert doc["logprobs"] == eight.score([[5, 6, 7]])[0]["logprobs"]
    assert len(eight.generate([5, 6, 7], GenerateOptions(max_new_tokens=4, ignore_eos=True)).token_ids) == 4
