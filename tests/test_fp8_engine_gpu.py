"""8-bit weights and an 8-bit cache through the engine: the step function in four ways of cutting against the plain implementation with
the weights' 8-bit values, generation with preemption and a shared prefix, the command line, refusals.

Tolerance.  A number rounded to e4m3 is off by 2^-4 of itself at most, 2^-4 / sqrt 3 = 3.6% in the mean square at worst.  An
attention's output meets three such roundings on its values (norm's rows, cache, heads' outputs: 6.3%) and three on its scores of
order one (6.3% of the weights): 9%; a feed-forward's two on gate and up, one on their product: 6.3%.  Two layers of both, errors
independent: sqrt(2 * 9^2 + 2 * 6.3^2) = 15.5% of the sub-layers' outputs, so of the logits' spread at most, and bfloat16's own 6%
(``test_real_sizes_gpu.py``) beside it: 17%.  A row is one draw of it, whose hundreds of entries share what attention errs in: half as
much again, 25%, is allowed."""
import os
import subprocess
import sys

import pytest
import torch

import plain_qwen3 as plain
from tiny import TINIES, make_folder, prompt

pytestmark = pytest.mark.gpu
RMS = 0.25


def values_of(model, w):
    """The plain implementation's weights, with the matrices that the model keeps in 8 bits as the values they stand for."""
    w = dict(w)
    for i, block in enumerate(model.blocks):
        p, mixer, ffn = f"model.layers.{i}.", block.mixer, block.ffn
        q, kv = mixer.q_heads * mixer.head_dim, mixer.kv_heads * mixer.head_dim
        parts = mixer.w_qkv.values().cpu().double().split([q, kv, kv])
        for name, t in zip("qkv", parts):
            w[f"{p}self_attn.{name}_proj.weight"] = t
        w[p + "self_attn.o_proj.weight"] = mixer.w_o.values().cpu().double()
        both = ffn.w_gate_up.values().cpu().double().view(ffn.inter // 8, 2, 8, ffn.hidden)
        w[p + "mlp.gate_proj.weight"] = both[:, 0].reshape(ffn.inter, ffn.hidden)
        w[p + "mlp.up_proj.weight"] = both[:, 1].reshape(ffn.inter, ffn.hidden)
        w[p + "mlp.down_proj.weight"] = ffn.w_down.values().cpu().double()
    return w


def runner_for(folder, tiny, weights, cache8, requests):
    from tiny_llm_infer_b200.cache import CacheManager
    from tiny_llm_infer_b200.engine import ModelRunner, load_model, selfcheck
    model, _ = load_model(folder, torch.bfloat16, "cuda:0", "fp8" if weights else None)
    if cache8:
        model.use_fp8_cache(tiny["page_size"])
    cache = CacheManager(model.cache_needs(), tiny["page_size"], selfcheck.pages_for(requests, tiny["page_size"]), max_slots=4, max_seq_len=320,
                         dtype=torch.uint8 if cache8 else torch.bfloat16, device="cuda:0")
    return model, ModelRunner(model, cache, max_batch_tokens=512)


@pytest.fixture(scope="module")
def folders(tmp_path_factory):
    made = {}
    for name in ("D", "E"):
        cfg = TINIES[name]["cfg"]
        tiny = TINIES[name]
        # feed-forward widths of 344 and 328 are no multiples of 16: 8-bit weights want 352 and 336
        from dataclasses import replace
        tiny = dict(tiny, cfg=replace(cfg, intermediate_size=cfg.intermediate_size + 8))
        made[name] = (make_folder(tiny, tmp_path_factory.mktemp(f"fp8_{name}")), tiny)
    return made


@pytest.mark.parametrize("name", ["D", "E"])
@pytest.mark.parametrize("weights,cache8", [(True, False), (False, True), (True, True)])
def test_four_ways_of_cutting(folders, name, weights, cache8):
    from tiny_llm_infer_b200.engine import selfcheck
    folder, tiny = folders[name]
    vocab = tiny["cfg"].vocab_size
    requests = {str(i): prompt(i, n, vocab) for i, n in enumerate((70, 300, 130, 41))}
    wanted = {k: selfcheck.wanted_positions(len(v), tail=12) for k, v in requests.items()}
    model, runner = runner_for(folder, tiny, weights, cache8, requests)
    cut = selfcheck.CutRunner(runner, requests, wanted)
    rows = cut.all_ways(seed=3)
    runner.check_kernels()
    runner.cache.audit()
    cfg, w = plain.read_model(folder)
    if weights:
        w = values_of(model, w)
    for request, tokens in requests.items():
        want = plain.logits_of(cfg, w, tokens).float()
        for (way, r, pos), row in rows.items():
            if r == request:
                off = float((row.cpu() - want[pos]).square().mean().sqrt() / want[pos].std())
                assert off <= RMS, (way, r, pos, off)


def test_generation_with_a_small_pool_and_a_shared_prefix(folders):
    """Greedy tokens are, within a quarter of the logits' spread, the argmax of the same engine's logits of the whole sequence."""
    from tiny_llm_infer_b200 import LLM, SamplingParams
    from tiny_llm_infer_b200.engine import StepEntry
    folder, tiny = folders["E"]
    from dataclasses import replace
    start = prompt(50, 64, 640)
    prompts = [start + prompt(i, n, 640) for i, n in enumerate((3, 20, 50))] + [prompt(9, 130, 640)]
    llm = LLM(str(folder), max_model_len=256, num_kv_blocks=12, block_size=32, max_num_batched_tokens=96, max_num_seqs=4, quantization="fp8",
              kv_cache_dtype="fp8")
    outs = llm.generate(prompts, SamplingParams(max_tokens=24, ignore_eos=True))
    llm.cache.audit()
    roomy = LLM(str(folder), max_model_len=256, num_kv_blocks=40, block_size=32, max_num_batched_tokens=256, max_num_seqs=4, quantization="fp8",
                kv_cache_dtype="fp8", use_cuda_graphs=False, overlap_scheduling=False)
    for p, o in zip(prompts, outs):
        ids = p + o.token_ids
        logits = roomy.runner.step([StepEntry("check", ids[:-1], list(range(len(p) - 1, len(ids) - 1)))]).clone()
        roomy.runner.release("check")
        for row, token in zip(logits, o.token_ids):
            assert float(row.max() - row[token]) <= 0.25 * float(row.std())
    # what a page costs, and that the pool is sized for it
    from tiny_llm_infer_b200.cache import CacheManager
    heads, dim, page = 1, 128, 32
    assert sum(CacheManager.bytes_per_page(llm.model.cache_needs(), page, torch.uint8).values()) == 2 * heads * page * (2 * dim + 8)
    assert replace(tiny["cfg"]).num_hidden_layers == 2


def test_preemption(folders):
    """Four requests of one page each that all grow a second one, on six pages: some are put back and computed again."""
    from tiny_llm_infer_b200 import LLM, SamplingParams
    from tiny_llm_infer_b200.engine import StepEntry
    folder, _ = folders["E"]
    prompts = [prompt(60 + i, 31, 640) for i in range(4)]
    llm = LLM(str(folder), max_model_len=128, num_kv_blocks=6, block_size=32, max_num_batched_tokens=128, max_num_seqs=4, quantization="fp8",
              kv_cache_dtype="fp8")
    outs = llm.generate(prompts, SamplingParams(max_tokens=20, ignore_eos=True))
    assert llm.engine.counters.preemptions > 0
    llm.cache.audit()
    for p, o in zip(prompts, outs):
        ids = p + o.token_ids
        logits = llm.runner.step([StepEntry("check", ids[:-1], list(range(len(p) - 1, len(ids) - 1)))]).clone()
        llm.runner.release("check")
        for row, token in zip(logits, o.token_ids):
            assert float(row.max() - row[token]) <= 0.25 * float(row.std())


def test_a_shared_prefix_and_prompt_graphs(folders, tmp_path):
    """Full attention only (the prefix cache is off with windows): the same prompts again, their pages shared; prompt steps replayed."""
    from dataclasses import replace
    from tiny_llm_infer_b200 import LLM, SamplingParams
    tiny = TINIES["E"]
    cfg = replace(tiny["cfg"], intermediate_size=336, sliding_window=None, layer_types=("full_attention",) * 2)
    folder = make_folder(dict(tiny, cfg=cfg), tmp_path / "m")
    llm = LLM(str(folder), max_model_len=512, num_kv_blocks=64, block_size=16, max_num_batched_tokens=192, max_num_seqs=2, quantization="fp8",
              kv_cache_dtype="fp8", prompt_graphs=True)
    params = SamplingParams(max_tokens=6, ignore_eos=True)
    p = prompt(3, 192 * 2, 640)
    first = llm.generate([p], params)[0].token_ids
    again = [llm.generate([q], params)[0].token_ids for q in (prompt(4, 192 * 2, 640), prompt(5, 192 * 2, 640), p)]
    assert llm.engine.counters.prefix_cached_tokens > 0
    assert len(first) == 6 and len(again[2]) == 6
    llm.cache.audit()


@pytest.mark.parametrize("weights,cache8", [(True, False), (True, True)])
def test_real_widths_beside_bfloat16(weights, cache8):
    """Two layers of Qwen3-8B widths, a request of 2,200 tokens and three short ones: 8 bits beside bfloat16, the same weights.  The
    weights' own rounding is one more of every product's: sqrt(2) of the tolerance's 15.5%, 22%, and half as much again."""
    from tiny_llm_infer_b200.cache import CacheManager
    from tiny_llm_infer_b200.config import Qwen3Config
    from tiny_llm_infer_b200.engine import ModelRunner, random_model, selfcheck
    cfg = Qwen3Config(hidden_size=4096, intermediate_size=12288, num_hidden_layers=2, num_attention_heads=32, num_key_value_heads=8,
                      tie_word_embeddings=False, head_dim=128, vocab_size=32768, max_position_embeddings=40960, rms_norm_eps=1e-6, rope_theta=1e6,
                      layer_types=("full_attention",) * 2)
    gen = torch.Generator().manual_seed(7)
    requests = {str(i): torch.randint(0, cfg.vocab_size, (n,), generator=gen).tolist() for i, n in enumerate((2200, 300, 150, 90))}
    wanted = {k: selfcheck.wanted_positions(len(v)) for k, v in requests.items()}
    rows = []
    for eight in (False, True):
        model = random_model(cfg, seed=11, dtype=torch.bfloat16, device="cuda:0", std=0.02)
        if eight and weights:
            model.use_fp8_weights()
        if eight and cache8:
            model.use_fp8_cache(16)
        cache = CacheManager(model.cache_needs(), 16, selfcheck.pages_for(requests, 16), max_slots=4, max_seq_len=2240,
                             dtype=torch.uint8 if eight and cache8 else torch.bfloat16, device="cuda:0")
        runner = ModelRunner(model, cache, max_batch_tokens=2240)
        rows.append(selfcheck.CutRunner(runner, requests, wanted).all_ways(seed=3))
        runner.check_kernels()
    result = selfcheck.compare(rows[1], rows[0], 0.3)
    print({k: round(v, 4) for k, v in result.items()})
    for way in ("whole", "tail", "portions", "mixed"):
        assert result[way + ":rms"] <= 0.33, result


def test_command_line(folders):
    from tiny_llm_infer_b200 import LLM, SamplingParams
    folder, _ = folders["D"]
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    got = subprocess.run([sys.executable, os.path.join(root, "bin", "model_main"), "--infer", "--model", str(folder), "--prompt-ids", "5,6,7,8,9", "--max-seq-len",
                          "64", "--max-new-tokens", "5", "--num-kv-blocks", "8", "--quantization", "fp8", "--kv-cache-dtype", "fp8"],
                         capture_output=True, text=True, timeout=300)
    assert got.returncode == 0, got.stderr
    llm = LLM(str(folder), max_model_len=64, num_kv_blocks=8, max_num_seqs=1, quantization="fp8", kv_cache_dtype="fp8")
    want = llm.generate([[5, 6, 7, 8, 9]], SamplingParams(max_tokens=5))[0].token_ids
    assert got.stdout.strip().splitlines()[-1] == ",".join(map(str, want))


def test_refusals(folders, tmp_path):
    from tiny_llm_infer_b200 import LLM
    folder, _ = folders["D"]
    odd = make_folder(TINIES["F"], tmp_path / "odd")
    for kw in (dict(dtype="float32", quantization="fp8"), dict(dtype="float32", kv_cache_dtype="fp8"), dict(kv_cache_dtype="fp8", block_size=8),
               dict(quantization="int4"), dict(kv_cache_dtype="int8")):
        with pytest.raises(ValueError):
            LLM(str(folder), max_model_len=64, num_kv_blocks=8, **kw)
    for kw in (dict(quantization="fp8"), dict(kv_cache_dtype="fp8")):
        with pytest.raises(ValueError):
            LLM(str(odd), max_model_len=64, num_kv_blocks=8, **kw)


def test_a_loaded_model_keeps_its_form(folders):
    from tiny_llm_infer_b200 import LLM, SamplingParams
    from tiny_llm_infer_b200.engine import load_model
    folder, _ = folders["E"]
    loaded = load_model(str(folder), torch.bfloat16, "cuda:0", "fp8")
    with pytest.raises(ValueError, match="already"):
        loaded[0].use_fp8_weights()
    first = LLM("", loaded=loaded, max_model_len=64, num_kv_blocks=8, kv_cache_dtype="fp8")
    with pytest.raises(ValueError, match="keeps its cache"):
        LLM("", loaded=loaded, max_model_len=64, num_kv_blocks=8)
    second = LLM("", loaded=loaded, max_model_len=64, num_kv_blocks=8, kv_cache_dtype="fp8")
    params = SamplingParams(max_tokens=4, ignore_eos=True)
    assert first.generate([[1, 2, 3]], params)[0].token_ids == second.generate([[1, 2, 3]], params)[0].token_ids
