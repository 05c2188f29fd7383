"""The score command over models that find a text next to impossible."""
import json
import math

import torch

from onnx_genai_b200.cli import main
from onnx_genai_b200.engine.api import Engine, perplexity
from onnx_genai_b200.models.config import DecoderConfig
from onnx_genai_b200.models.decoder import random_weights
from onnx_genai_b200.package.export import export_package

CFG = DecoderConfig(name="t", num_layers=1, hidden=64, num_heads=4, num_kv_heads=2, head_dim=16, intermediate=96, vocab=300,
                    rope_theta=1e4, tie_embeddings=False, qkv_bias=False, max_position=128)


def _model(tmp_path, **change):
    w = random_weights(CFG, "cpu", seed=5, std=0.3, dtype=torch.float32)
    for name, factor in change.items():
        getattr(w, name).mul_(factor)
    return export_package(CFG, w, str(tmp_path / "pkg"))


def test_perplexity():
    assert perplexity(-math.log(8.0)) == math.exp(math.log(8.0)) and perplexity(0.0) == 1.0
    assert perplexity(-800.0) == math.inf and perplexity(-math.inf) == math.inf and math.isnan(perplexity(math.nan))


def _strict(name):
    raise AssertionError(f"{name} is not JSON")


def test_a_perplexity_past_the_range_is_said_and_written_as_null(tmp_path, capsys):
    model = _model(tmp_path, lm_head=1e4)
    doc, = Engine.from_dir(model, device="cpu", num_pages=32, max_seqs=2).score([[5, 6, 7, 8]])
    assert min(doc["logprobs"]) < -710.0 and doc["perplexity"] == math.inf
    assert main(["score", model, "--ids", "--text", "5 6 7 8", "--device", "cpu", "--logit-rows", "8"]) == 0
    out, err = capsys.readouterr()
    line = json.loads(out.strip().splitlines()[-1], parse_constant=_strict)
    assert line["perplexity"] is None and len(line["logprobs"]) == 3 and min(line["logprobs"]) < -710.0 and "perplexity inf" in err
