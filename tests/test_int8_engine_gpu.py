"""8-bit operators inside the engine on the GPU: the pool of pages, texts that share a prefix, log probabilities against 64 bits, and the divisions of
the work under replay and on several streams."""
import torch
import pytest

from onnx_genai_b200.engine.llm_engine import EngineConfig, LLMEngine
from onnx_genai_b200.models.config import DecoderConfig
from onnx_genai_b200.models.decoder import random_weights

pytestmark = pytest.mark.gpu

GIB = 1 << 30


def test_pages_get_the_memory_that_8_bit_weights_give_back():
    cfg = DecoderConfig(name="wide", num_layers=8, hidden=2048, num_heads=16, num_kv_heads=4, head_dim=128, intermediate=8192, vocab=1024, rope_theta=1e6,
                        tie_embeddings=False, qkv_bias=True, max_position=4096)
    weights = random_weights(cfg, "cuda", seed=1)
    matrices = sum(t.numel() for l in weights.layers for t in (l.qkv_w, l.o_w, l.gate_up_w, l.down_w))
    torch.cuda.empty_cache()
    free, total = torch.cuda.mem_get_info()
    # a share of the device that leaves pages one GiB with the weights as they are
    eng = LLMEngine(EngineConfig(model=cfg, max_seqs=64, max_seq_len=4096, max_tokens_per_step=512, weight_dtype="int8",
                                 gpu_memory_utilization=1.0 - (free - GIB) / total), weights=weights, device="cuda")
    page = cfg.num_layers * 2 * cfg.num_kv_heads * cfg.head_dim * 16 * 2
    # half of the matrices' bytes come back; an eighth of that for the step's buffers and what the allocator's blocks leave between them
    assert eng.num_pages < 64 * 256 + 64 and eng.num_pages * page > GIB + matrices * 7 // 8
