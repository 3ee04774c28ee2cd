"""What of the 8-bit operators needs no GPU: the checks of weights and rows, how a product is cut."""
import pytest
import torch

from tiny_llm_infer_b200 import ops
from tiny_llm_infer_b200.ops import fp8


def e4m3(*shape):
    return torch.zeros(shape, dtype=torch.float8_e4m3fn)


def test_weights_say_what_they_want():
    ops.Fp8Weight(e4m3(200, 144), torch.ones(2, 2))
    ops.Fp8Weight(e4m3(272, 128), torch.ones(4, 1), gated=True)
    for q, scales, gated in ((e4m3(200, 144), torch.ones(2, 1), False), (e4m3(200, 144), torch.ones(1, 2), False), (e4m3(272, 128), torch.ones(3, 1), True),
                             (e4m3(264, 128), torch.ones(4, 1), True), (e4m3(16, 24), torch.ones(1, 1), False), (e4m3(0, 16), torch.ones(0, 1), False),
                             (torch.zeros(16, 16), torch.ones(1, 1), False), (e4m3(16, 16), torch.ones(1, 1, dtype=torch.float64), False),
                             (e4m3(32, 32).t()[:16], torch.ones(1, 1), False)):
        with pytest.raises(ops.KernelError):
            ops.Fp8Weight(q, scales, gated)


def test_rows_say_what_they_want():
    assert tuple(ops.Fp8Rows(e4m3(3, 144), torch.ones(3, 2)).shape) == (3, 144)
    for q, scales in ((e4m3(3, 144), torch.ones(3, 1)), (e4m3(3, 144), torch.ones(2, 2)), (e4m3(3, 24), torch.ones(3, 1)), (torch.zeros(3, 16), torch.ones(3, 1))):
        with pytest.raises(ops.KernelError):
            ops.Fp8Rows(q, scales)


def test_values_follow_the_layout_of_the_scales():
    q = torch.ones(272, 144).to(torch.float8_e4m3fn)
    plain = ops.Fp8Weight(q, torch.arange(6.0).view(3, 2)).values()
    assert plain[127, 127] == 0 and plain[127, 128] == 1 and plain[128, 0] == 2 and plain[271, 143] == 5
    gated = ops.Fp8Weight(q, torch.arange(8.0).view(4, 2), gated=True).values()
    # row 16 j + i is gate row 8 j + i, eight further its up row; gate row 128 is row 256
    assert gated[0, 0] == 0 and gated[8, 0] == 2 and gated[247, 0] == 0 and gated[255, 143] == 3 and gated[256, 0] == 4 and gated[264, 0] == 6


@pytest.mark.parametrize("rows", [9, 16, 17, 33, 64, 128, 129, 500, 2048, 100000])
@pytest.mark.parametrize("n,k", [(8, 16), (1024, 128), (4096, 4096), (24576, 4096), (130, 12288), (48, 2064)])
@pytest.mark.parametrize("gated,to_float", [(False, False), (True, False), (False, True)])
def test_shares_cover_all_blocks_and_none_is_empty(rows, n, k, gated, to_float):
    route, splits, each = fp8._plan(rows, n, k, 148, gated, to_float)
    kb = -(-k // 128)
    assert (splits == 1 or route == fp8.TILES) and (splits - 1) * each < kb <= splits * each
    assert route != fp8.SKINNY or rows <= 16
    assert route != fp8.PAIRS or not to_float


def test_scratch_holds_what_a_product_leaves_in_it():
    # rows in 8 bits, their scales rounded up to 16 bytes, sums
    kind, route, splits, each, size, kernels = fp8._call(61, 4096, 4096, 1, False, False, 148)
    assert (kind, route) == (1, fp8.TILES) and size == 61 * 4096 + 61 * 32 * 4 + 4 * splits * 61 * 4096 and kernels == 3
    assert fp8._call(8, 4096, 4096, 1, False, False, 148)[0::4] == (fp8.INSIDE, 0)
    kind, route, splits, each, size, kernels = fp8._call(3, 512, 144, 0, True, False, 148)
    assert (kind, route, kernels) == (0, fp8.SKINNY, 3) and size == 3 * 144 + 32 + 4 * 3 * 256
    assert fp8._call(2048, 24576, 4096, fp8.ROWS8, True, False, 148)[1:5:3] == (fp8.PAIRS, 0)


def test_tensors_of_the_host_are_refused():
    with pytest.raises(ops.KernelError):
        ops.quantize_rows_fp8(torch.zeros(2, 16))
    with pytest.raises(ops.KernelError):
        ops.quantize_weight_fp8(torch.zeros(16, 16))
    with pytest.raises(ops.KernelError):
        ops.linear(torch.zeros(2, 16), ops.Fp8Weight(e4m3(16, 16), torch.ones(1, 1)))


def test_only_models_with_the_form_are_taken(tmp_path):
    """Parts without an 8-bit form, models that are not bfloat16 or not loaded, unknown words: refused in words, on any machine."""
    from tiny_llm_infer_b200 import LLM
    from tiny_llm_infer_b200.config.base import describe_model
    from tiny_llm_infer_b200.engine import load_model
    from tiny_llm_infer_b200.models.model import Model
    from tiny import TINIES
    import tiny_panolorn
    qwen = Model(describe_model(TINIES["D"]["cfg"]), torch.bfloat16, "cpu")
    with pytest.raises(ValueError, match="after they are loaded"):
        qwen.use_fp8_weights()
    other = Model(describe_model(tiny_panolorn.P1["cfg"]), torch.bfloat16, "cpu")
    other.loaded = True
    with pytest.raises(ValueError, match="no 8-bit"):
        other.use_fp8_weights()
    with pytest.raises(ValueError, match="no 8-bit cache"):
        other.use_fp8_cache(16)
    full = Model(describe_model(TINIES["D"]["cfg"]), torch.float32, "cpu")
    full.loaded = True
    with pytest.raises(ValueError):
        full.use_fp8_weights()
    with pytest.raises(ValueError):
        full.use_fp8_cache(16)
    with pytest.raises(ValueError):
        qwen.use_fp8_cache(24)
    with pytest.raises(ValueError, match="int4"):
        load_model(tmp_path, torch.bfloat16, "cpu", "int4")
    with pytest.raises(ValueError, match="kv_cache_dtype"):
        LLM(str(tmp_path), device="cpu", kv_cache_dtype="int8")
    with pytest.raises(ValueError, match="quantization"):
        LLM(str(tmp_path), device="cpu", loaded=(qwen, None), quantization="fp8")


def test_a_page_of_the_cache_in_bytes():
    from tiny_llm_infer_b200.cache import CacheManager
    from tiny_llm_infer_b200.config.base import describe_model
    from tiny_llm_infer_b200.models.model import Model
    from tiny import TINIES
    model = Model(describe_model(TINIES["D"]["cfg"]), torch.bfloat16, "cpu")
    model.use_fp8_cache(16)
    sizes = CacheManager.bytes_per_page(model.cache_needs(), 16, torch.uint8)
    assert sizes == {None: 16 * 2 * (64 + 64 + 8), 80: 16 * 2 * (64 + 64 + 8)}
    cache = CacheManager(model.cache_needs(), 16, 4, max_slots=2, max_seq_len=64, dtype=torch.uint8, device="cpu")
    keys, values, scales = cache.view(0).planes
    assert keys.shape == values.shape == (4, 2, 16, 64) and scales.shape == (4, 2, 16, 8) and keys.stride(0) == scales.stride(0) == 16 * 2 * 136
    assert (values.data_ptr() - keys.data_ptr(), scales.data_ptr() - keys.data_ptr()) == (2048, 4096)


def test_pages_of_portions():
    from types import SimpleNamespace

    def seg(pos0, length):
        return SimpleNamespace(pos0=pos0, length=length)
    ctx = SimpleNamespace(segments=[seg(500, 1), seg(0, 16), seg(15, 2), seg(100, 33)])
    assert fp8.portion_pages(ctx, 16, None, 40) == (9, 1 + 2 + 9)
    assert fp8.portion_pages(ctx, 16, 20, 40) == (4, 1 + 2 + 4)      # from the page of 81 to that of 132
    assert fp8.portion_pages(SimpleNamespace(segments=[seg(5, 1)]), 16, None, 40) == (1, 1)
    assert fp8.portion_pages(ctx, 16, 20, 40, capturing=True) == (40, 120)


def test_how_one_token_attention_is_cut():
    """A block each where that is soon over or there are rows enough, a cluster each for a few longer rows, shares for a few of the longest."""
    cut = fp8.attention_cut
    assert cut(1, 8, 4, 64, 148) == cut(16, 8, 2, 600, 148) == cut(24, 8, 2, 1000, 148) == cut(64, 8, 4, 4096, 148) == cut(0, 8, 4, 9999, 148) == (0, 1)
    assert cut(1, 8, 4, 4095, 148) == cut(1, 8, 4, 1000, 148) == (0, 8) and cut(8, 8, 4, 2000, 148) == (0, 4)
    assert cut(2, 8, 4, 131072, 148) == (444, 1) and cut(2, 1, 16, 100000, 148) == (296, 1)
    assert cut(513, 8, 4, 100000, 148) == (0, 1)
    for rows in (1, 3, 17, 100, 512, 700):
        for reach in (1, 129, 5000, 200000):
            blocks, cluster = cut(rows, 8, 4, reach, 148)
            assert cluster in (1, 2, 4, 8) and blocks in (0, 444) and (cluster == 1 or (blocks == 0 and rows * 8 * cluster <= 2.6 * 148))
            assert blocks == 0 or rows <= 512


def test_a_weight_keeps_its_tensors():
    """Its products know the tensors by their place: others make another weight."""
    weight = ops.Fp8Weight(torch.zeros((16, 32), dtype=torch.float8_e4m3fn), torch.ones((1, 1)))
    assert weight.q.shape == weight.shape and weight.scales.shape == (1, 1) and weight.dtype == torch.float8_e4m3fn
    for name in ("q", "scales"):
        with pytest.raises(AttributeError):
            setattr(weight, name, getattr(weight, name).clone())
