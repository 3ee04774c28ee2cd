"""A model's 8-bit forms are taken whole or not at all; no GPU needed."""
import pytest
import torch

from tiny_llm_infer_b200 import ops
from tiny_llm_infer_b200.config.base import describe_model
from tiny_llm_infer_b200.models.model import Model
from tiny import TINIES


def qwen():
    model = Model(describe_model(TINIES["D"]["cfg"]), torch.bfloat16, "cpu")
    model.loaded = True
    assert len(model.blocks) > 1
    return model


def test_a_cache_that_one_mixer_cannot_keep_changes_none():
    model = qwen()
    model.blocks[-1].mixer.dtype = torch.float32
    needs = model.cache_needs()
    with pytest.raises(ValueError, match="8-bit cache"):
        model.use_fp8_cache(16)
    assert not model.fp8_cache and not any(m.cache_fp8 for b in model.blocks for m in b.mixers())
    assert model.cache_needs() == needs


@pytest.mark.parametrize("part", ["ffn", "mixer", "norm2"])
def test_weights_that_one_part_cannot_keep_change_none(part, monkeypatch):
    made = []
    monkeypatch.setattr(ops, "quantize_weight_fp8", lambda w, gated=False: made.append(w))
    model = qwen()
    for block in model.blocks:                                  # 344 is no multiple of 16
        block.ffn.inter = 352
    last = model.blocks[-1]
    if part == "norm2":
        last.norm2.width = 32784                                # more than a row's kernel takes
    else:
        setattr(getattr(last, part), "hidden", 1032)
    with pytest.raises(ValueError):
        model.use_fp8_weights()
    assert not made and not model.fp8_weights and not any(b.norm1.rows_fp8 or b.norm2.rows_fp8 for b in model.blocks)


def test_a_model_of_parts_with_the_form_is_taken(monkeypatch):
    made = []
    monkeypatch.setattr(ops, "quantize_weight_fp8", lambda w, gated=False: made.append(gated))
    model = qwen()
    for block in model.blocks:
        block.ffn.inter = 352
    model.use_fp8_weights()
    model.use_fp8_cache(16)
    assert made == [False, False, True, False] * len(model.blocks) and model.fp8_weights and model.fp8_cache
    assert all(b.norm1.rows_fp8 and b.norm2.rows_fp8 and b.mixer.cache_fp8 for b in model.blocks)


def test_other_weights_are_not_loaded_over_8_bit_ones(monkeypatch):
    """The norms already hand on 8-bit rows, which a bfloat16 matrix does not take."""
    monkeypatch.setattr(ops, "quantize_weight_fp8", lambda w, gated=False: None)
    model = qwen()
    for block in model.blocks:
        block.ffn.inter = 352
    model.use_fp8_weights()
    with pytest.raises(ValueError, match="8 bits"):
        model.load({})


def test_pages_beside_which_one_layers_pages_fit_in_bfloat16():
    """The pool of an 8-bit cache leaves room for the scratch of a step's portions: one layer's pages as bfloat16."""
    from tiny_llm_infer_b200.cache import CacheManager
    from tiny_llm_infer_b200.engine.llm_engine import estimate_num_kv_blocks
    model = qwen()
    model.use_fp8_cache(16)
    needs, gib = model.cache_needs(), 1 << 30
    eight = sum(CacheManager.bytes_per_page(needs, 16, torch.uint8).values())
    mixer = model.blocks[0].mixer
    layer = 2 * mixer.kv_heads * 16 * mixer.head_dim * 2
    free, total = 40 * gib, 64 * gib
    pages = estimate_num_kv_blocks(model, 16, torch.uint8, 256, 0.9, "cuda:0", memory=(free, total))
    budget = int(total * 0.9) - (total - free) - total // 20
    assert pages * (eight + layer) <= budget < (pages + 2) * (eight + layer + layer // 8)


@pytest.mark.parametrize("form", ["weights", "cache"])
def test_a_runner_is_of_the_form_that_its_model_had(form, monkeypatch):
    """Its graphs hold the places of the matrices and pages that they were captured with."""
    from tiny_llm_infer_b200.cache import CacheManager
    from tiny_llm_infer_b200.engine import ModelRunner, StepEntry
    from tiny_llm_infer_b200.engine.runner import StepError
    monkeypatch.setattr(ops, "quantize_weight_fp8", lambda w, gated=False: None)
    model = qwen()
    for block in model.blocks:
        block.ffn.inter = 352
    cache = CacheManager(model.cache_needs(), 16, 8, max_slots=2, max_seq_len=64, dtype=torch.bfloat16, device="cpu")
    runner = ModelRunner(model, cache, max_batch_tokens=64)
    prepared = runner.prepare([StepEntry("a", [1, 2, 3], [2])])
    monkeypatch.setattr(model, "forward", lambda *a: pytest.fail("the step was run"))
    model.use_fp8_weights() if form == "weights" else model.use_fp8_cache(16)
    with pytest.raises(StepError, match="form"):
        runner.run(prepared)
    with pytest.raises(StepError, match="form"):
        runner.step([StepEntry("a", [1, 2, 3], [2])])
