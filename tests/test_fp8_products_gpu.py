"""Rows, weights and products in 8 bits (``ops/fp8.py``) against their definitions in 64 bits."""
import pytest
import torch

import fp8_reference as ref

pytestmark = pytest.mark.gpu

# rows x columns x K: one row, one past and short of tiles of 16, 128 and 256, sums of one block and less, K short of a block, sizes
# of the models, each kernel (up to 8, 16, 32 rows; tiles of 128 and 256; shares of K)
SIZES = [(1, 16, 16), (1, 1024, 2048), (3, 24, 144), (8, 6144, 4096), (9, 1000, 272), (16, 256, 1024), (17, 130, 528), (32, 4096, 512),
         (33, 264, 1040), (61, 4096, 4096), (128, 128, 128), (129, 257, 1296), (300, 1608, 2192), (500, 8192, 640), (2048, 6144, 256)]


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def rows_of(g, t, k, dtype):
    spread = torch.exp(torch.randn((t, 1), generator=g, device="cuda") * 3) * torch.exp(torch.randn((1, k), generator=g, device="cuda"))
    return (torch.randn((t, k), generator=g, device="cuda") * spread).to(dtype)


def check_rows(got, x):
    """Scales to the bit, values within half a step, and no larger than the largest."""
    scales = ref.row_scales(x)
    assert torch.equal(got.scales, scales)
    per = scales[:, ref.block_of(x.shape[1], x.device)]
    assert ((got.values().double() - x.double()).abs() <= ref.half_step(x, per)).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("t,k", [(1, 16), (2, 128), (3, 144), (17, 4096), (501, 1552), (0, 256), (1500, 8208)])
def test_rows(t, k, dtype):
    from tiny_llm_infer_b200 import ops
    x = rows_of(gen(t + k), t, k, dtype)
    if t > 1:
        x[t // 2] = 0.0                                       # a row of zeros, and one far below the floor
        x[0] = x[0] * 1e-36
    check_rows(ops.quantize_rows_fp8(x), x)


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("n,k,dtype", [(16, 16, torch.float32), (128, 128, torch.bfloat16), (272, 400, torch.bfloat16), (1040, 2048, torch.float32)])
def test_weights(n, k, dtype, gated):
    from tiny_llm_infer_b200 import ops
    w = rows_of(gen(n), n, k, dtype)
    q = ops.quantize_weight_fp8(w, gated)
    scales = (ref.gated_weight_scales if gated else ref.weight_scales)(w)
    assert torch.equal(q.scales, scales)
    rows = torch.arange(n, device="cuda")
    rows = 2 * (rows // 16 * 8 // 128) + rows // 8 % 2 if gated else rows // 128
    per = scales[rows][:, ref.block_of(k, "cuda")]
    assert ((q.values().double() - w.double()).abs() <= ref.half_step(w, per)).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("t,n,k", SIZES)
def test_products(t, n, k, dtype):
    from tiny_llm_infer_b200 import ops
    g = gen(t + n)
    x, w = rows_of(g, t, k, dtype), rows_of(g, n, k, torch.float32) * 0.02
    weight = ops.quantize_weight_fp8(w)
    rows = ops.quantize_rows_fp8(x)
    y = ops.linear(x, weight)
    again = ops.linear(rows, weight, out_dtype=dtype)
    ops.check_error_word("cuda")
    assert y.dtype == dtype and tuple(y.shape) == (t, n)
    # rounded inside the product or before it: the same 8-bit rows; the sums may run in another order
    exact, off = ref.product_bound(rows.values().double(), weight.values().double(), dtype)
    assert ((y.double() - exact).abs() <= off).all()
    assert ((again.double() - exact).abs() <= off).all()
    assert torch.equal(again, ops.linear(rows, weight, out_dtype=dtype))


@pytest.mark.parametrize("act", ["silu", "gelu_tanh", "relu", "clamped_swish"])
@pytest.mark.parametrize("t,inter,k", [(1, 16, 16), (1, 1536, 1024), (8, 12288, 512), (13, 144, 400), (31, 784, 640), (61, 1024, 1024), (200, 272, 656),
                                       (129, 12288, 256), (700, 4112, 384)])
def test_gated(t, inter, k, act):
    from tiny_llm_infer_b200 import ops
    g = gen(t + inter)
    x = (torch.randn((t, k), generator=g, device="cuda") * 2).to(torch.bfloat16)
    gate, up = (torch.randn((inter, k), generator=g, device="cuda") * 0.05 for _ in range(2))
    weight = ops.quantize_weight_fp8(ops.interleave_gate_up(gate, up), gated=True)
    rows = ops.quantize_rows_fp8(x)
    consts = (7.0, 1.7) if act == "clamped_swish" else None
    values = weight.values().double().view(inter // 8, 2, 8, k)
    (zg, dg), (zu, du) = (ref.product_bound(rows.values().double(), values[:, i].reshape(inter, k), torch.float32) for i in (0, 1))
    if act == "silu":
        a, u = zg * torch.sigmoid(zg), zu
    elif act == "relu":
        a, u = zg.clamp_min(0), zu
    elif act == "gelu_tanh":
        a, u = 0.5 * zg * (1 + torch.tanh(0.7978845608028654 * (zg + 0.044715 * zg ** 3))), zu
    else:
        a, u = zg.clamp_max(7.0) * torch.sigmoid(1.7 * zg.clamp_max(7.0)), zu.clamp(-7.0, 7.0) + 1
    exact = a * u
    # the activations' slopes are at most 1.2 (clamped swish 1.1); float32 functions off by a few 2^-23 of the gate (2^-19 bounds
    # the cancellation in 1 + tanh too)
    off = 1.2 * dg * u.abs() + du * a.abs() + 1.2 * dg * du + 2.0 ** -19 * zg.abs() * u.abs()
    for got in (ops.linear_swiglu(x, weight, act=act, consts=consts), ops.linear_swiglu(rows, weight, act=act, consts=consts)):
        assert tuple(got.shape) == (t, inter)
        # the scale follows the largest of a block, the value is the nearest to a number within `off`
        scales = ref.row_scales(exact.float())
        reach = ref.row_scales((exact.abs() + off).float()) * (1 + 2.0 ** -20)
        least = ref.row_scales((exact.abs() - off).clamp_min(0).float()) * (1 - 2.0 ** -20)
        assert (got.scales <= reach).all() and (got.scales >= least).all() and scales.shape == got.scales.shape
        per = got.scales[:, ref.block_of(inter, "cuda")]
        assert ((got.values().double() - exact).abs() <= off + ref.half_step(exact.abs() + off, per)).all()
    ops.check_error_word("cuda")


@pytest.mark.parametrize("gain_dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("delta_dtype", [None, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("t,width", [(1, 16), (3, 144), (8, 4096), (129, 1552), (2, 4112), (5, 8192), (2, 32768)])
def test_norm(t, width, delta_dtype, gain_dtype):
    from tiny_llm_infer_b200 import ops
    g = gen(t + width)
    h = rows_of(g, t, width, torch.float32)
    if t > 2:
        h[1] = 0.0
    delta = None if delta_dtype is None else rows_of(g, t, width, delta_dtype)
    gain = (torch.rand(width, generator=g, device="cuda") + 0.5).to(gain_dtype)
    total = h.clone() if delta is None else h + delta.float()
    v = total.double()
    exact = gain.double() * v / torch.sqrt((v * v).mean(dim=1, keepdim=True) + 1e-6)
    got = ops.add_rmsnorm_fp8(h, delta, gain, 1e-6)
    assert torch.equal(h, total)
    # float32: squares and a sum of `width` terms, half of that after the root, a handful of roundings
    off = exact.abs() * (width / 2 + 8) * 2.0 ** -24
    scales = ref.row_scales(exact.float())
    assert ((got.scales - scales).abs() <= scales * ((width / 2 + 10) * 2.0 ** -24)).all()
    per = got.scales[:, ref.block_of(width, "cuda")]
    assert ((got.values().double() - exact).abs() <= off + ref.half_step(exact.abs() + off, per)).all()


@pytest.mark.parametrize("t", [2, 20, 70, 300])
def test_not_a_number_stays_in_its_row_and_columns(t):
    from tiny_llm_infer_b200 import ops
    g = gen(t)
    n, k = 520, 400
    x, w = rows_of(g, t, k, torch.bfloat16), rows_of(g, n, k, torch.float32)
    before = ops.linear(x, ops.quantize_weight_fp8(w))
    x2, w2 = x.clone(), w.clone()
    x2[0, 130] = float("nan")
    x2[1, 399] = float("inf")
    after = ops.linear(x2, ops.quantize_weight_fp8(w))
    assert torch.isnan(after[:2]).all() and torch.equal(after[2:], before[2:])
    w2[200, 3] = float("nan")                              # one weight: its row
    after = ops.linear(x, ops.quantize_weight_fp8(w2))
    others = torch.arange(n, device="cuda") != 200
    assert torch.isnan(after[:, 200]).all() and torch.equal(after[:, others], before[:, others])


@pytest.mark.parametrize("t", [1, 8, 40, 400])
def test_captured_and_replayed(t):
    """Norm, gated product and product as one graph, replayed on other numbers; a second stream."""
    from tiny_llm_infer_b200 import ops
    g = gen(t)
    width, inter = 512, 1040
    weight_in = ops.quantize_weight_fp8(ops.interleave_gate_up(torch.randn((inter, width), generator=g, device="cuda"),
                                                               torch.randn((inter, width), generator=g, device="cuda")), gated=True)
    weight_out = ops.quantize_weight_fp8(torch.randn((width, inter), generator=g, device="cuda"))
    gain = torch.ones(width, device="cuda")
    h = torch.randn((t, width), generator=g, device="cuda")

    def unit():
        return ops.linear(ops.linear_swiglu(ops.add_rmsnorm_fp8(h, None, gain, 1e-6), weight_in), weight_out)
    first = unit()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert torch.equal(unit(), first)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = unit()
    for _ in range(2):
        h.copy_(torch.randn((t, width), generator=g, device="cuda"))
        graph.replay()
        assert torch.equal(out, unit())
    ops.check_error_word("cuda")


def test_refusals():
    from tiny_llm_infer_b200 import ops
    weight = ops.quantize_weight_fp8(torch.randn(64, 64, device="cuda"))
    gated = ops.quantize_weight_fp8(torch.randn(64, 64, device="cuda"), gated=True)
    x = torch.randn(4, 64, device="cuda")
    for call in (lambda: ops.linear(x[:, :48].contiguous(), weight), lambda: ops.linear(x.half(), weight), lambda: ops.linear(x.t(), weight),
                 lambda: ops.linear(x, weight, out_dtype=torch.float16), lambda: ops.linear(x, gated), lambda: ops.linear_swiglu(x, weight),
                 lambda: ops.linear(x, weight, bias=torch.zeros(64, device="cuda")), lambda: ops.linear_swiglu(x, gated, torch.bfloat16),
                 lambda: ops.linear(torch.randn(4 * 64 + 1, device="cuda")[1:].view(4, 64), weight), lambda: ops.linear(x.cpu(), weight),
                 lambda: ops.quantize_rows_fp8(torch.randn(4, 40, device="cuda")), lambda: ops.quantize_weight_fp8(torch.randn(64, 40, device="cuda")),
                 lambda: ops.quantize_weight_fp8(torch.randn(40, 64, device="cuda"), gated=True),
                 lambda: ops.add_rmsnorm_fp8(x, None, torch.ones(48, device="cuda"), 1e-6), lambda: ops.add_rmsnorm_fp8(x, None, torch.ones(64, device="cuda"), 0.0),
                 lambda: ops.add_rmsnorm_fp8(x, x[:2], torch.ones(64, device="cuda"), 1e-6),
                 lambda: ops.add_rmsnorm_fp8(torch.zeros((1, 32784), device="cuda"), None, torch.ones(32784, device="cuda"), 1e-6)):
        with pytest.raises(ops.KernelError):
            call()
