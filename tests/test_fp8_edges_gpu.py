"""The 8-bit operators at the edges of what they take: scales of zero, missing pages, numbers that are none, long rings and many pieces,
against 64 bits."""
import math

import pytest
import torch

from test_fp8_attention_gpu import exact_row, fill, gen, planes_of, tables

pytestmark = pytest.mark.gpu


def a_request(g, n, page, kv_heads, dim, spread=(0.3, 0.5)):
    """One request of n keys in a cache of its own: planes, its table, (keys, values) float64, and where each token lies."""
    pages = -(-n // page) + 2
    planes = planes_of(pages, kv_heads, page, dim)
    table = tables(g, [n], page, pages, pages)
    kept = fill(g, planes, table, [n], page, spread)[0]
    token = torch.arange(n, device="cuda")
    return planes, table, kept, table[0].long()[token // page], token % page


WAYS = [dict(), dict(cluster=1), dict(cluster=2), dict(cluster=8), dict(blocks=3), dict(blocks=64)]


def attend(q, planes, n, table, page, q_heads, kv_heads, dim, window=None, **how):
    from tiny_llm_infer_b200 import ops
    out = torch.full_like(q, 7.0)
    position, slot = (torch.tensor([i], dtype=torch.int32, device="cuda") for i in (n - 1, 0))
    ops.paged_attention_decode_fp8(q, planes, position, slot, None, 1, table, page, q_heads, kv_heads, dim, window, 1 / math.sqrt(dim), out, n, **how)
    return out


@pytest.mark.parametrize("how", WAYS)
@pytest.mark.parametrize("smallest", [0.0, 1e-40])
@pytest.mark.parametrize("n,window,dim", [(1, None, 128), (5, None, 128), (37, None, 64), (64, None, 128), (200, None, 128), (333, 70, 64), (333, 70, 128)])
def test_values_with_a_scale_of_zero_count(n, window, dim, smallest, how):
    """A value whose scale is zero (or below the normal numbers) adds nothing to the sum, and its key's weight counts, wherever in the
    row it lies: every third token, and the row's first and last."""
    g = gen(n + dim)
    page, kv_heads, q_heads = 16, 2, 8
    planes, table, (keys, values), at, place = a_request(g, n, page, kv_heads, dim)
    scales = planes[2].view(torch.float32)
    none = torch.arange(n, device="cuda") % 3 == 0
    none[n - 1] = True
    if window:
        none[n - window] = True
    scales[at[none], :, place[none], 1] = smallest
    values = values.clone()
    values[:, none] = 0.0
    q = torch.randn((1, q_heads * dim), generator=g, device="cuda").to(torch.bfloat16)
    out = attend(q, planes, n, table, page, q_heads, kv_heads, dim, window, **how)
    want, off = exact_row(q[0].double().view(q_heads, dim), keys, values, n - 1, window, 1 / math.sqrt(dim))
    # what a scale of 1e-40 leaves out: 448 scales at most, weights that add up to one at most
    assert ((out[0].double() - want).abs() <= off + 448 * smallest).all()


@pytest.mark.parametrize("how", WAYS)
@pytest.mark.parametrize("n,gone", [(40, (1,)), (100, (0, 3)), (300, (0, 1, 2, 7, 18)), (33, (2,))])
def test_keys_of_missing_pages_do_not_count(n, gone, how):
    """Pages of the table that name none, beside values with a scale of zero, which do count."""
    g = gen(n)
    page, kv_heads, q_heads, dim = 16, 2, 8, 128
    planes, table, (keys, values), at, place = a_request(g, n, page, kv_heads, dim)
    token = torch.arange(n, device="cuda")
    none = token % 5 == 2
    planes[2].view(torch.float32)[at[none], :, place[none], 1] = 0.0
    values = values.clone()
    values[:, none] = 0.0
    there = torch.ones(n, dtype=torch.bool, device="cuda")
    for p in gone:
        table[0, p] = -1
        there[p * page:(p + 1) * page] = False
    q = torch.randn((1, q_heads * dim), generator=g, device="cuda").to(torch.bfloat16)
    out = attend(q, planes, n, table, page, q_heads, kv_heads, dim, **how)
    left = int(there.sum())
    want, off = exact_row(q[0].double().view(q_heads, dim), keys[:, there], values[:, there], left - 1, None, 1 / math.sqrt(dim))
    assert ((out[0].double() - want).abs() <= off).all()


def dev(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def step_of(portions):
    """A step of portions (slot, tokens, position of the first), as the runner lays them out: its context, positions and slots."""
    from types import SimpleNamespace
    seg, pos, slots, dec, tiles, row = [], [], [], [], [], 0
    for s, (slot, n, first) in enumerate(portions):
        seg.append((slot, row, n, first))
        pos += range(first, first + n)
        slots += [slot] * n
        if n == 1:
            dec.append(row)
        else:
            tiles += [(s, o) for o in range(0, n, 64)]
        row += n
    tiles.sort(key=lambda t: (t[1] % 256 != 0, t[1] % 128 != 0))
    ctx = SimpleNamespace(tokens=row, segments=[SimpleNamespace(length=n, pos0=p) for _, n, p in portions], seg_info=dev(seg), dec_rows=dev(dec), n_dec=len(dec),
                          pf_tiles=dev(tiles), n_tiles=len(tiles), n_tiles128=sum(t[1] % 128 == 0 for t in tiles), n_tiles256=sum(t[1] % 256 == 0 for t in tiles),
                          max_context=max(first + n for _, n, first in portions))
    return ctx, dev(pos), dev(slots)


def check_portions(out, q, ctx, pos, slots, kept, q_heads, dim, window=None):
    """Rows of portions: keys, values and the prompt kernels' weights pass through bfloat16 (2^-8 each) beside what a single token's do."""
    single, scale = set(ctx.dec_rows.tolist()), 1 / math.sqrt(dim)
    for i in range(ctx.tokens):
        keys, values = kept[int(slots[i])]
        p = int(pos[i])
        want, off = exact_row(q[i].double().view(q_heads, dim), keys, values, p, window, scale)
        if i not in single:
            first = max(0, p + 1 - window) if window else 0
            k, v = keys[:, first:p + 1], values[:, first:p + 1]
            query = q[i].double().view(keys.shape[0], -1, dim)
            e = (query.abs() @ k.abs().transpose(1, 2)).amax(-1, keepdim=True) * scale * 2.0 ** -8
            mass = torch.softmax(query @ k.transpose(1, 2) * scale, dim=-1) @ v.abs()
            off = off + (mass * (torch.expm1(2 * e) + 2 * 2.0 ** -8) * 1.02).reshape(-1)
        assert ((out[i].double() - want).abs() <= off).all(), i


def shared_prefix(g, requests, prefix, own, page, kv_heads, dim):
    """Requests whose first ``prefix`` pages are the same ones, ``own`` further pages each, in a pool with room for one more."""
    pages = prefix + requests * own + 1
    planes = planes_of(pages, kv_heads, page, dim)
    table = torch.empty((requests, prefix + own), dtype=torch.int32, device="cuda")
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    table[:, :prefix] = order[:prefix]
    table[:, prefix:] = order[prefix:prefix + requests * own].view(requests, own)
    return planes, table


def test_portions_that_share_a_prefix_take_no_more_than_the_pool():
    """Five portions of 20 tokens behind 20 shared pages: scratch for the pool's 31 pages, not for the 110 that they list."""
    from tiny_llm_infer_b200 import ops
    g = gen(31)
    q_heads, kv_heads, dim, page = 8, 8, 64, 64
    planes, table = shared_prefix(g, 5, 20, 2, page, kv_heads, dim)
    lengths = [20 * page + 20 + 12 * r for r in range(5)]
    assert max(lengths) <= table.shape[1] * page
    for r, n in enumerate(lengths):                             # the prefix is written once: the first request's
        fill(g, planes, table[r:r + 1], [n], page, (0.3, 0.3))
    ctx, pos, slots = step_of([(r, 20, n - 20) for r, n in enumerate(lengths)])
    q = torch.randn((100, q_heads * dim), generator=g, device="cuda").to(torch.bfloat16)
    out = torch.empty_like(q)

    def call():
        ops.paged_attention_fp8(q, planes, pos, slots, table, page, q_heads, kv_heads, dim, None, 1 / math.sqrt(dim), out, ctx)
    call()
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    held = torch.cuda.memory_allocated()
    call()
    torch.cuda.synchronize()
    assert torch.cuda.max_memory_allocated() - held <= planes[0].shape[0] * 2 * kv_heads * page * dim * 2 + (1 << 20)


@pytest.mark.parametrize("dim,page,window", [(64, 32, None), (128, 16, None), (128, 48, 200)])
def test_portions_that_share_pages(dim, page, window):
    """Long shared prefixes, a single token beside them, and two portions whose tables are the same: one ends inside a page in which the
    other goes on."""
    from test_fp8_attention_gpu import stored
    from tiny_llm_infer_b200 import ops
    g = gen(dim + page)
    q_heads, kv_heads, prefix = 8, 2, 9
    planes, table = shared_prefix(g, 5, prefix, 3, page, kv_heads, dim)
    table[4] = table[3]
    start = prefix * page
    new = [(0, 70, start - 40), (1, 33, start), (2, 1, start + 7), (3, 5, start + 1), (4, page, start + 6)]
    lengths = [first + n for _, n, first in new]
    assert max(lengths) <= table.shape[1] * page
    for r in (0, 1, 2, 4):                                      # the fifth's table is the fourth's, and its tokens are more
        fill(g, planes, table[r:r + 1], [lengths[r]], page, (0.3, 0.3))
    ctx, pos, slots = step_of(new)
    q = torch.randn((ctx.tokens, q_heads * dim), generator=g, device="cuda").to(torch.bfloat16)
    out = torch.empty_like(q)
    args = (planes, pos, slots, table, page, q_heads, kv_heads, dim, window, 1 / math.sqrt(dim))
    ops.paged_attention_fp8(q, *args, out, ctx)
    ops.check_error_word("cuda")
    kept = [stored(planes, table, r, n, page) for r, n in enumerate(lengths)]
    check_portions(out, q, ctx, pos, slots, kept, q_heads, dim, window)
    # captured and replayed, for other portions of as many tokens
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.paged_attention_fp8(q, *args, out, ctx)
    for back in (0, 3, 11):
        other, p2, s2 = step_of([(r, n, first - back) for r, n, first in new])
        other.max_context = ctx.max_context
        ctx.seg_info.copy_(other.seg_info)
        pos.copy_(p2)
        out.fill_(7.0)
        graph.replay()
        want = torch.empty_like(q)
        ops.paged_attention_fp8(q, planes, p2, s2, table, page, q_heads, kv_heads, dim, window, 1 / math.sqrt(dim), want, other)
        assert torch.equal(out, want)
    ops.check_error_word("cuda")


def test_a_weight_made_of_rows_that_the_kernel_ahead_still_writes():
    """The weight-streaming product fetches weights before the kernel ahead of it has ended.  Rows that have just been brought to 8 bits,
    taken as a weight of one output, are there all the same."""
    import fp8_reference as ref
    from tiny_llm_infer_b200 import ops
    g = gen(41)
    k = 4096
    x = torch.randn((4, k), generator=g, device="cuda").to(torch.bfloat16)
    meet = ops.quantize_rows_fp8(x).values().double()
    busy = torch.randn((4096, 4096), generator=g, device="cuda")
    vectors = torch.randn((40, 1, k), generator=g, device="cuda").to(torch.bfloat16)
    torch.cuda.synchronize()
    kept = []
    for v in vectors:
        busy @ busy                                            # the host gets ahead: the kernels behind it start back to back
        rows = ops.quantize_rows_fp8(v)
        weight = ops.Fp8Weight(rows.q, rows.scales)
        kept.append((rows, ops.linear(x, weight)))
    for rows, y in kept:
        exact, off = ref.product_bound(meet, rows.values().double(), torch.bfloat16)
        assert ((y.double() - exact).abs() <= off).all()


@pytest.mark.parametrize("kv_heads,others,blocks", [(1, 0, 444), (8, 0, 444), (1, 59, 444), (1, 59, 100), (2, 29, 100)])
def test_more_than_thirty_two_pieces(kv_heads, others, blocks):
    """One long row in many pieces, alone (the warps of a block add them together) and beside short ones (a warp for a head), cut into
    chunks and into equal shares."""
    from tiny_llm_infer_b200 import ops
    g = gen(kv_heads + others + blocks)
    group, dim, page = 4, 128, 16
    q_heads = kv_heads * group
    lengths = [30001] + [1 + 7 * i % 90 for i in range(others)]
    pages = sum(-(-n // page) for n in lengths) + 1
    planes = planes_of(pages, kv_heads, page, dim)
    table = tables(g, lengths, page, pages, -(-lengths[0] // page))
    kept = fill(g, planes, table, lengths, page, (0.5, 1.0))
    n = len(lengths)
    q = (torch.randn((n, q_heads * dim), generator=g, device="cuda") * 2).to(torch.bfloat16)
    pos, slots = dev([length - 1 for length in lengths]), dev(list(range(n)))
    side, first = torch.cuda.Stream(), torch.full_like(q, 7.0)

    def call(out):
        return ops.paged_attention_decode_fp8(q, planes, pos, slots, None, n, table, page, q_heads, kv_heads, dim, None, 1 / math.sqrt(dim), out, lengths[0],
                                              blocks=blocks)
    call(first)
    for r in range(n):
        want, off = exact_row(q[r].double().view(q_heads, dim), *kept[r], lengths[r] - 1, None, 1 / math.sqrt(dim))
        assert ((first[r].double() - want).abs() <= off).all()
    # on another stream, and captured and replayed for other lengths
    out = torch.full_like(q, 7.0)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call(out)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(out, first)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(out)
    for back in (0, 1, 9000, 29990):
        pos[0] = lengths[0] - 1 - back
        graph.replay()
        assert torch.equal(out, call(torch.full_like(q, 7.0)))
        want, off = exact_row(q[0].double().view(q_heads, dim), *kept[0], lengths[0] - 1 - back, None, 1 / math.sqrt(dim))
        assert ((out[0].double() - want).abs() <= off).all()


@pytest.mark.parametrize("what", ["query nan", "query inf", "key nan", "value nan", "key scale nan", "key scale inf", "value scale nan", "value scale inf"])
@pytest.mark.parametrize("how", WAYS)
def test_numbers_that_are_none(what, how):
    """They reach what the formula gives them to and nothing else: the other heads, the other dims of a value."""
    g = gen(len(what))
    page, kv_heads, q_heads, dim, n, key = 16, 2, 8, 128, 300, 217
    planes, table, (keys, values), at, place = a_request(g, n, page, kv_heads, dim)
    scales = planes[2].view(torch.float32)
    q = torch.randn((1, q_heads * dim), generator=g, device="cuda").to(torch.bfloat16)
    keys, values = keys.clone(), values.clone()
    odd = float("nan") if what.endswith("nan") else float("inf")
    if what.startswith("query"):
        q[0, dim + 5] = odd                                    # head 1
    elif what == "key nan":
        planes[0][at[key], 1, place[key], 9] = 0x7F
        keys[1, key, 9] = odd
    elif what == "value nan":
        planes[1][at[key], 1, place[key], 9] = 0x7F
        values[1, key, 9] = odd
    else:
        which = 0 if what.startswith("key") else 1
        old = scales[at[key], 1, place[key], which].double()
        scales[at[key], 1, place[key], which] = odd
        if which:
            values[1, key] = values[1, key] / old * odd
    out = attend(q, planes, n, table, page, q_heads, kv_heads, dim, **how)[0].double()
    query = q[0].double().view(kv_heads, -1, dim)
    s = query @ keys.transpose(1, 2) / math.sqrt(dim)
    if what.startswith("key scale"):                           # a score is its product times the scale
        s[1, :, key] = s[1, :, key] * odd
    p = torch.softmax(s, dim=-1)
    want = (p @ values).reshape(-1)
    finite = torch.isfinite(want)
    # where the formula has no number there is none; an infinite scale of a value is one of all its dims
    assert not torch.isfinite(out[~finite]).any() and (~finite).any() and finite.any()
    assert torch.isfinite(out[finite]).all()
    clean = torch.nan_to_num(keys, 0.0, 0.0, 0.0), torch.nan_to_num(values, 0.0, 0.0, 0.0)
    if what != "key scale inf":                                # there the other keys of a head share its weight
        _, off = exact_row(torch.nan_to_num(query, 0.0, 0.0, 0.0).reshape(q_heads, dim), *clean, n - 1, None, 1 / math.sqrt(dim))
        assert ((out - want).abs() <= off)[finite].all()


@pytest.mark.parametrize("t,n,k", [(2048, 6144, 4096), (1000, 10240, 2064), (1500, 4112, 12288)])
def test_products_by_pairs_that_turn_their_rings(t, n, k):
    """Tens of blocks of K a tile and several tiles a pair of SMs: every stage is used many times over."""
    import fp8_reference as ref
    from test_fp8_products_gpu import rows_of
    from tiny_llm_infer_b200 import ops
    assert ops.fp8._plan(t, n, k, 148)[0] == ops.fp8.PAIRS
    g = gen(t + n)
    x, w = rows_of(g, t, k, torch.bfloat16), rows_of(g, n, k, torch.float32) * 0.02
    weight, rows = ops.quantize_weight_fp8(w), ops.quantize_rows_fp8(x)
    y = ops.linear(x, weight)
    ops.check_error_word("cuda")
    exact, off = ref.product_bound(rows.values().double(), weight.values().double(), torch.bfloat16)
    assert ((y.double() - exact).abs() <= off).all()
    assert torch.equal(y, ops.linear(rows, weight))


@pytest.mark.parametrize("t,inter,k", [(600, 12288, 4096), (2048, 2064, 2064)])
def test_gated_products_by_pairs_that_turn_their_rings(t, inter, k):
    import fp8_reference as ref
    from tiny_llm_infer_b200 import ops
    assert ops.fp8._plan(t, 2 * inter, k, 148, gated=True)[0] == ops.fp8.PAIRS
    g = gen(t + inter)
    x = (torch.randn((t, k), generator=g, device="cuda") * 2).to(torch.bfloat16)
    gate, up = (torch.randn((inter, k), generator=g, device="cuda") * 0.02 for _ in range(2))
    weight, rows = ops.quantize_weight_fp8(ops.interleave_gate_up(gate, up), gated=True), ops.quantize_rows_fp8(x)
    got = ops.linear_swiglu(x, weight)
    ops.check_error_word("cuda")
    values = weight.values().double().view(inter // 8, 2, 8, k)
    (zg, dg), (zu, du) = (ref.product_bound(rows.values().double(), values[:, i].reshape(inter, k), torch.float32) for i in (0, 1))
    a = zg * torch.sigmoid(zg)
    exact = a * zu
    off = 1.2 * dg * zu.abs() + du * a.abs() + 1.2 * dg * du + 2.0 ** -19 * zg.abs() * zu.abs()      # the slope of silu is at most 1.1
    per = got.scales[:, ref.block_of(inter, "cuda")]
    assert ((got.values().double() - exact).abs() <= off + ref.half_step(exact.abs() + off, per)).all()
    assert (got.scales <= ref.row_scales((exact.abs() + off).float()) * (1 + 2.0 ** -20)).all()
    assert (got.scales >= ref.row_scales((exact.abs() - off).clamp_min(0).float()) * (1 - 2.0 ** -20)).all()


def test_calls_of_no_rows():
    """A step's part without rows is an empty result, as with the bfloat16 operators, not an error."""
    from tiny_llm_infer_b200 import ops
    width, inter, q_heads, kv_heads, dim, page = 64, 32, 4, 2, 64, 16
    weight = ops.quantize_weight_fp8(torch.randn((48, width), device="cuda"))
    gated = ops.quantize_weight_fp8(torch.randn((2 * inter, width), device="cuda"), gated=True)
    h = torch.zeros((0, width), device="cuda")
    rows = ops.add_rmsnorm_fp8(h, None, torch.ones(width, device="cuda"), 1e-6)
    for x in (h, h.to(torch.bfloat16), rows, ops.quantize_rows_fp8(h)):
        assert tuple(ops.linear(x, weight).shape) == (0, 48)
        got = ops.linear_swiglu(x, gated)
        assert tuple(got.shape) == tuple(got.q.shape) == (0, inter) and tuple(got.scales.shape) == (0, 1) and tuple(got.values().shape) == (0, inter)
    planes = planes_of(3, kv_heads, page, dim)
    before = [p.clone() for p in planes]
    table, none = torch.zeros((1, 3), dtype=torch.int32, device="cuda"), dev([])
    q = torch.zeros((0, q_heads * dim), dtype=torch.bfloat16, device="cuda")
    qkv = torch.zeros((0, (q_heads + 2 * kv_heads) * dim), dtype=torch.bfloat16, device="cuda")
    ops.qk_norm_rope_store_fp8(qkv, None, None, 1.0, None, 0, none, none, table, planes, page, torch.empty_like(q), q_heads, kv_heads, dim,
                               ops.QK_STORE | ops.QK_QOUT)
    assert all(torch.equal(a, b) for a, b in zip(planes, before))
    ops.paged_attention_decode_fp8(q, planes, none, none, None, 0, table, page, q_heads, kv_heads, dim, None, 0.1, torch.empty_like(q), 48)
    ops.paged_attention_fp8(q, planes, none, none, table, page, q_heads, kv_heads, dim, None, 0.1, torch.empty_like(q))
    # rows there, none of them asked for
    q, one = torch.zeros((2, q_heads * dim), dtype=torch.bfloat16, device="cuda"), dev([0, 0])
    out = torch.full_like(q, 7.0)
    ops.paged_attention_decode_fp8(q, planes, one, one, none, 0, table, page, q_heads, kv_heads, dim, None, 0.1, out, 48)
    assert (out == 7).all()


@pytest.mark.parametrize("t,n,k", [(70001, 264, 144), (65536, 136, 272)])
def test_products_of_very_many_rows(t, n, k):
    import fp8_reference as ref
    from tiny_llm_infer_b200 import ops
    g = gen(t)
    x = torch.randn((t, k), generator=g, device="cuda").to(torch.bfloat16)
    w = torch.randn((n // 16 * 16, k), generator=g, device="cuda") * 0.1
    weight, gated, rows = ops.quantize_weight_fp8(w), ops.quantize_weight_fp8(w[:128].contiguous(), gated=True), ops.quantize_rows_fp8(x)
    exact, off = ref.product_bound(rows.values().double(), weight.values().double(), torch.bfloat16)
    assert ((ops.linear(x, weight).double() - exact).abs() <= off).all()
    few = ops.linear_swiglu(ops.Fp8Rows(rows.q[-7:].contiguous(), rows.scales[-7:].contiguous()), gated)
    many = ops.linear_swiglu(x, gated)
    ops.check_error_word("cuda")
    # the last rows by another kernel: within the rounding to 8 bits of each
    a, b, scale = few.values(), many.values()[-7:], torch.maximum(few.scales, many.scales[-7:])
    assert ((a - b).abs() <= torch.maximum(a.abs(), b.abs()) * 2.0 ** -3 * 1.01 + scale * 2.0 ** -9).all()
