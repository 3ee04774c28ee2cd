"""What the 8-bit forms leave of the device's memory: room that 8-bit weights give back, scratch of prompt portions."""
import gc

import pytest
import torch

pytestmark = pytest.mark.gpu


def test_room_that_8_bit_weights_give_back():
    """The pool is sized from the device's free memory: what the bfloat16 matrices took has to be given back to the device, not kept by
    torch's allocator.  A fifth of it may stay in blocks that 8-bit matrices share with others."""
    from tiny_llm_infer_b200.cache import CacheManager
    from tiny_llm_infer_b200.config import Qwen3Config
    from tiny_llm_infer_b200.engine import random_model
    from tiny_llm_infer_b200.engine.llm_engine import estimate_num_kv_blocks
    layers, hidden, inter = 4, 2048, 6144
    cfg = Qwen3Config(hidden_size=hidden, intermediate_size=inter, num_hidden_layers=layers, num_attention_heads=16, num_key_value_heads=8,
                      tie_word_embeddings=True, head_dim=128, vocab_size=4096, max_position_embeddings=4096, rms_norm_eps=1e-6, rope_theta=1e6,
                      layer_types=("full_attention",) * layers)
    gc.collect()
    torch.cuda.empty_cache()
    model = random_model(cfg, seed=1, dtype=torch.bfloat16, device="cuda:0", std=0.02)
    torch.cuda.synchronize()
    torch.cuda.empty_cache()

    def room():
        return estimate_num_kv_blocks(model, 16, torch.bfloat16, 256, 0.9, "cuda:0")
    before = room()
    numbers = layers * (hidden * (16 + 8 + 8) * 128 + 16 * 128 * hidden + 3 * hidden * inter)
    model.use_fp8_weights()
    gained = (room() - before) * sum(CacheManager.bytes_per_page(model.cache_needs(), 16, torch.bfloat16).values())
    assert gained >= 0.8 * numbers, (gained, numbers)
