"""Captured prompt steps over the 8-bit cache: what a replay gives for other prompts, pages and positions, beside the same kernels launched
one by one."""
import pytest
import torch

from tiny import TINIES, make_folder, prompt

pytestmark = pytest.mark.gpu


def runner_of(folder, page):
    from tiny_llm_infer_b200.cache import CacheManager
    from tiny_llm_infer_b200.engine import ModelRunner, load_model
    model, _ = load_model(folder, torch.bfloat16, "cuda:0", "fp8")
    model.use_fp8_cache(page)
    cache = CacheManager(model.cache_needs(), page, 120, max_slots=6, max_seq_len=640, dtype=torch.uint8, device="cuda:0")
    return ModelRunner(model, cache, max_batch_tokens=512, prompt_graphs=True)


@pytest.mark.parametrize("full", [True, False])
def test_replayed_prompt_steps(full, tmp_path):
    """Portions of 192 tokens, alone, two together and beside a decoding request; six rounds of other prompts.  The other runner forgets
    every layout before it comes again, so it launches the same kernels one by one."""
    from dataclasses import replace
    from tiny_llm_infer_b200.engine import StepEntry
    tiny = TINIES["E"]
    cfg = replace(tiny["cfg"], intermediate_size=336)
    if full:
        cfg = replace(cfg, sliding_window=None, layer_types=("full_attention",) * 2)
    folder, vocab = make_folder(dict(tiny, cfg=cfg), tmp_path / "m"), cfg.vocab_size
    page = 16 if full else tiny["page_size"]
    runners = [runner_of(folder, page) for _ in range(2)]
    replayed = 0

    def both(*entries):
        nonlocal replayed
        rows = []
        for runner in runners:
            if runner is runners[1]:
                runner._prompt_seen.clear()
            held = dict(runner._prompt_graphs)
            take = runner._step_prompt_graph
            used = []
            runner._step_prompt_graph = lambda signature, ctx, take=take: (used.append(signature), take(signature, ctx))[1]
            rows.append(runner.step([StepEntry(r, list(tokens), list(want)) for r, tokens, want in entries]).clone())
            del runner._step_prompt_graph
            if runner is runners[0]:
                replayed += any(signature in held for signature in used)
        assert torch.equal(rows[0], rows[1])

    for turn in range(6):
        a, b, c = (prompt(100 * turn + i, n, vocab) for i, n in enumerate((392, 384, 260 + 10 * turn)))
        both(("c", c, [len(c) - 1]))
        both(("a", a[:192], []), ("b", b[:192], [191]))
        both(("a", a[192:384], [100, 191]))
        both(("b", b[192:], [191]), ("c", [turn], [0]))
        for i in range(384, 392):
            both(("a", a[i:i + 1], [0]))
        for runner in runners:
            for request in ("a", "b", "c") if turn % 2 else ("b", "a", "c"):
                runner.release(request)
            runner.check_kernels()
            runner.cache.audit()
    assert replayed >= 3 * 3 and not runners[1]._prompt_graphs
