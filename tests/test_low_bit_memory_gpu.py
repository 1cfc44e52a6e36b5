"""What a model with 4-bit weights leaves free on the device."""

import pytest
import torch

pytestmark = pytest.mark.gpu

RAW = dict(architectures=["Qwen2ForCausalLM"], hidden_size=2048, intermediate_size=8192, num_hidden_layers=6, num_attention_heads=16, num_key_value_heads=4,
           head_dim=128, vocab_size=2000, rope_theta=1e6, rms_norm_eps=1e-6, tie_word_embeddings=False, max_position_embeddings=4096)


def test_the_original_weights_go_back_to_the_device():
    """Each layer's projections are 120 MB in bfloat16 and 31 MB in 4 bits: what is reserved beyond the tensors is at most one layer's originals and its
    stacked copy of gates and ups (the allocator may keep a segment that a small tensor lies in), not all layers' originals."""
    from pyre_b200 import Engine
    from pyre_b200.config import config_from_dict
    cfg = config_from_dict(RAW)
    layer = 2 * 2048 * (2048 + 2 * 512 + 2048 + 3 * 8192)
    over, pages = {}, {}
    for bits in (None, 4):
        torch.cuda.empty_cache()
        before = torch.cuda.memory_reserved() - torch.cuda.memory_allocated()
        eng = Engine(config=cfg, seed=0, weight_bits=bits, max_cache_tokens=4096)
        over[bits] = torch.cuda.memory_reserved() - torch.cuda.memory_allocated() - before
        del eng
        torch.cuda.empty_cache()
        eng = Engine(config=cfg, seed=0, weight_bits=bits, cache_memory_fraction=0.05)
        pages[bits] = eng.cache.num_pages
        del eng
    assert over[4] <= layer + 2 * 2048 * 2 * 8192, over
    saved = 6 * (layer - layer // 4 - layer // 128)      # a byte half, and two bytes of scale per 128 elements
    page_bytes = 6 * 2 * 4 * 128 * 2 * 16
    assert pages[4] - pages[None] >= 0.05 * 0.5 * saved / page_bytes, pages
