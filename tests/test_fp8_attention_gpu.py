"""The 8-bit paged cache (``ops/fp8.py``): what is stored, one-token attention over it, pages back in bfloat16, against 64 bits."""
import math
from types import SimpleNamespace

import pytest
import torch

import fp8_reference as ref

pytestmark = pytest.mark.gpu


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def planes_of(pages, kv_heads, page, dim):
    """A cache of 8-bit pages as the cache manager lays it out, every byte 0x7f: keys and values NaN, scales NaN."""
    plane = kv_heads * page * dim
    flat = torch.full((pages, 2 * plane + kv_heads * page * 8), 0x7F, dtype=torch.uint8, device="cuda")
    flat[:, 2 * plane:].view(torch.float32).fill_(float("nan"))
    return (flat[:, :plane].unflatten(1, (kv_heads, page, dim)), flat[:, plane:2 * plane].unflatten(1, (kv_heads, page, dim)),
            flat[:, 2 * plane:].unflatten(1, (kv_heads, page, 8)))


def fill(g, planes, table, lengths, page, spread):
    """Keys and values of every request's tokens, pages as the table says; (keys, values) [request][kv_heads, length, dim] float64."""
    kv_heads, dim = planes[0].shape[1], planes[0].shape[3]
    kept = []
    for r, n in enumerate(lengths):
        both = []
        token = torch.arange(n, device="cuda")
        at = table[r].long()[token // page]
        for which in range(2):
            x = torch.randn((n, kv_heads, dim), generator=g, device="cuda")
            x = x * torch.exp(spread[which] * torch.randn((n, kv_heads, 1), generator=g, device="cuda"))
            if n > 3:
                x[n // 2, 0] = 0.0
            scale = ref.row_scales(x.reshape(n * kv_heads, dim)).view(n, kv_heads)
            q = (x / scale[..., None]).to(torch.float8_e4m3fn)
            planes[which][at, :, token % page] = q.view(torch.uint8)
            planes[2].view(torch.float32)[at, :, token % page, which] = scale
            both.append((q.double() * scale.double()[..., None]).transpose(0, 1))
        kept.append(both)
    return kept


def tables(g, lengths, page, pages, width):
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    table = torch.full((len(lengths), width), -1, dtype=torch.int32, device="cuda")
    at = 0
    for r, n in enumerate(lengths):
        held = -(-n // page)
        table[r, :held] = order[at:at + held]
        at += held
    return table


def exact_row(query, keys, values, pos, window, scale):
    """(output, how far off) of one row: query [q_heads, dim] float64, keys and values [kv_heads, length, dim]."""
    kv_heads, _, dim = keys.shape
    group = query.shape[0] // kv_heads
    first = max(0, pos + 1 - window) if window else 0
    k, v = keys[:, first:pos + 1], values[:, first:pos + 1]
    q = query.view(kv_heads, group, dim)
    s = (q @ k.transpose(1, 2)) * scale
    p = torch.softmax(s, dim=-1)
    out = p @ v
    # a score: dim products and their sum in float32, a rounding each, three more for the factors, and what float16 leaves of the
    # smallest queries (2^-28 of the largest); base 2 and its exponential: 2^-22 of the score and of the result
    sums = (q.abs() @ k.abs().transpose(1, 2)) * scale
    rest = q.abs().amax(-1, keepdim=True) * 2.0 ** -28 * k.abs().sum(-1)[:, None, :] * scale
    e = (sums * ((dim + 8) * 2.0 ** -23) + rest + s.abs() * 2.0 ** -22).amax(-1, keepdim=True)
    # weights: float16 with 11 bits (2^-11), or 2^-40 of the heaviest term's weight times the largest e4m3; sums in float32
    mass = p @ v.abs()
    heaviest = (p[..., None] * v.abs().amax(-1)[:, None, :, None]).amax(2)
    off = mass * (torch.expm1(2 * e) + 2.0 ** -11 + (p.shape[-1] + 64) * 2.0 ** -23) + heaviest * p.shape[-1] * 2.0 ** -39
    return out.reshape(-1), (off + (out.abs() + off) * 2.0 ** -8).reshape(-1)


CASES = [  # q_heads, kv_heads, dim, page, window, positions
    (1, 1, 64, 16, 0, [0]), (1, 1, 128, 16, 0, [0, 1, 14, 15, 16, 17]), (32, 8, 128, 16, 0, [4094, 63, 700]), (16, 8, 64, 32, 0, [31, 32, 33, 1500]),
    (40, 8, 128, 16, 0, [129, 1000]), (16, 1, 128, 64, 0, [2047, 5]), (24, 2, 64, 16, 0, [640, 641]), (8, 8, 128, 32, 1, [0, 40, 333]),
    (32, 8, 128, 16, 17, [3, 16, 40, 800]), (16, 8, 64, 16, 1000, [999, 1000, 1001, 3000]), (12, 4, 128, 48, 33, [200, 47, 48]), (64, 4, 128, 16, 0, [9000])]


@pytest.mark.parametrize("splits", [None, 1, 2, 7, 64])
@pytest.mark.parametrize("q_heads,kv_heads,dim,page,window,positions", CASES)
def test_one_token_rows(q_heads, kv_heads, dim, page, window, positions, splits):
    one_token_rows(q_heads, kv_heads, dim, page, window, positions, blocks=splits)


@pytest.mark.parametrize("cluster", [1, 2, 4, 8])
@pytest.mark.parametrize("q_heads,kv_heads,dim,page,window,positions", CASES)
def test_one_token_rows_by_clusters(q_heads, kv_heads, dim, page, window, positions, cluster):
    one_token_rows(q_heads, kv_heads, dim, page, window, positions, cluster=cluster)


def one_token_rows(q_heads, kv_heads, dim, page, window, positions, **how):
    """Rows in another order than their slots, one of no request between them, rows not asked for left alone; what pages hold behind
    a request's last token, and pages of nobody, is NaN."""
    from tiny_llm_infer_b200 import ops
    g = gen(q_heads * dim + window + len(positions))
    lengths = [p + 1 for p in positions]
    pages = sum(-(-n // page) for n in lengths) + 3
    planes = planes_of(pages, kv_heads, page, dim)
    table = tables(g, lengths, page, pages, -(-max(lengths) // page) + 2)
    kept = fill(g, planes, table, lengths, page, (0.3, 1.5))
    n = len(positions)
    total = n + 2
    # row 0 belongs to nobody, the last is not asked for
    slots = torch.tensor([-1] + list(range(n - 1, -1, -1)) + [0], dtype=torch.int32, device="cuda")
    pos = torch.tensor([0] + positions[::-1] + [0], dtype=torch.int32, device="cuda")
    rows = torch.arange(n + 1, dtype=torch.int32, device="cuda")
    q = (torch.randn((total, q_heads * dim), generator=g, device="cuda") * 3).to(torch.bfloat16)
    out = torch.full_like(q, 7.0)
    scale = 1 / math.sqrt(dim)
    ops.paged_attention_decode_fp8(q, planes, pos, slots, rows, n + 1, table, page, q_heads, kv_heads, dim, window or None, scale, out, max(lengths), **how)
    assert (out[0] == 0).all() and (out[-1] == 7).all()
    for i in range(n):
        r = n - 1 - i
        want, off = exact_row(q[1 + i].double().view(q_heads, dim), *kept[r], positions[r], window, scale)
        assert ((out[1 + i].double() - want).abs() <= off).all()
    again = torch.full_like(q, 7.0)
    ops.paged_attention_decode_fp8(q, planes, pos, slots, rows, n + 1, table, page, q_heads, kv_heads, dim, window or None, scale, again, max(lengths), **how)
    assert torch.equal(out, again)


def test_values_of_very_different_sizes():
    """A value a million times the others at a key of no weight, a heavy key of tiny value: the weights keep to the heaviest term."""
    from tiny_llm_infer_b200 import ops
    g = gen(5)
    kv_heads, group, dim, page, n = 2, 4, 128, 16, 600
    planes = planes_of(n // page + 1, kv_heads, page, dim)
    table = tables(g, [n], page, n // page + 1, n // page + 1)
    keep = fill(g, planes, table, [n], page, (0.0, 0.0))[0]
    token = torch.arange(n, device="cuda")
    at = table[0].long()[token // page]
    q = torch.randn((1, kv_heads * group * dim), generator=g, device="cuda").to(torch.bfloat16)
    scales = planes[2].view(torch.float32)
    for key, factor in ((77, 2.0 ** 20), (300, 2.0 ** -20)):
        scales[at[key], :, key % page, 1] *= factor
        keep[1][:, key] *= factor
    # key 77 far below the others, 300 far above, for every query of its head
    mean = q.double().view(kv_heads, group, dim).mean(1)
    for key, size in ((77, -8.0), (300, 4.0)):
        k = (mean * size).float()
        s = ref.row_scales(k)
        k8 = (k / s).to(torch.float8_e4m3fn)
        planes[0][at[key], :, key % page] = k8.view(torch.uint8)
        scales[at[key], :, key % page, 0] = s[:, 0]
        keep[0][:, key] = k8.double() * s.double()
    for splits in (1, 5):
        out = torch.empty_like(q)
        ops.paged_attention_decode_fp8(q, planes, torch.tensor([n - 1], dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda"), None, 1,
                                       table, page, kv_heads * group, kv_heads, dim, None, 0.1, out, n, splits)
        want, off = exact_row(q[0].double().view(-1, dim), *keep, n - 1, 0, 0.1)
        assert ((out[0].double() - want).abs() <= off).all()


def test_queries_of_any_size():
    """Zeros, the smallest and the largest bfloat16 numbers as queries: scores of zero weigh all keys alike, scores far apart one alone."""
    from tiny_llm_infer_b200 import ops
    g = gen(6)
    dim, page, n = 64, 16, 40
    planes = planes_of(3, 1, page, dim)
    table = tables(g, [n], page, 3, 3)
    keys, values = fill(g, planes, table, [n], page, (0.0, 0.0))[0]
    q = torch.randn((4, dim), generator=g, device="cuda")
    q = torch.stack([q[0] * 0, q[1] * 1e-39, q[2] * 1e30, q[3]]).to(torch.bfloat16).reshape(1, 4 * dim)
    out = torch.empty_like(q)
    ops.paged_attention_decode_fp8(q, planes, torch.tensor([n - 1], dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda"), None, 1,
                                   table, page, 4, 1, dim, None, 0.125, out, n, 2)
    got = out.double().view(4, dim)
    mean = values[0].mean(0)
    bound = values[0].abs().mean(0) * 2.0 ** -10 + mean.abs() * 2.0 ** -8 * (1 + 2.0 ** -8)
    assert ((got[0] - mean).abs() <= bound).all() and ((got[1] - mean).abs() <= bound).all()
    top = values[0][int((q.double().view(4, dim)[2] @ keys[0].t()).argmax())]
    assert ((got[2] - top).abs() <= top.abs() * (2.0 ** -8 + 2.0 ** -11 * 1.01)).all()


def test_pages_past_four_gigabytes():
    from tiny_llm_infer_b200 import ops
    g = gen(7)
    kv_heads, dim, page, n = 8, 128, 16, 100
    plane = kv_heads * page * dim
    pages = (5 << 30) // (2 * plane + kv_heads * page * 8)
    flat = torch.empty((pages, 2 * plane + kv_heads * page * 8), dtype=torch.uint8, device="cuda")
    planes = (flat[:, :plane].unflatten(1, (kv_heads, page, dim)), flat[:, plane:2 * plane].unflatten(1, (kv_heads, page, dim)),
              flat[:, 2 * plane:].unflatten(1, (kv_heads, page, 8)))
    table = (pages - 1 - torch.arange(7, device="cuda")).to(torch.int32)[None].contiguous()
    keys, values = fill(g, planes, table, [n], page, (0.3, 0.3))[0]
    q = torch.randn((1, 32 * dim), generator=g, device="cuda").to(torch.bfloat16)
    out = torch.empty_like(q)
    ops.paged_attention_decode_fp8(q, planes, torch.tensor([n - 1], dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda"), None, 1,
                                   table, page, 32, kv_heads, dim, None, 0.09, out, n)
    want, off = exact_row(q[0].double().view(32, dim), keys, values, n - 1, 0, 0.09)
    assert ((out[0].double() - want).abs() <= off).all()


def stored(planes, table, r, n, page):
    """(keys, values) [kv_heads, n, dim] float64 of a request's tokens as the cache holds them."""
    token = torch.arange(n, device="cuda")
    at = table[r].long()[token // page]
    scales = planes[2].view(torch.float32)[at, :, token % page].double()
    return [(planes[i][at, :, token % page].view(torch.float8_e4m3fn).double() * scales[..., i:i + 1]).transpose(0, 1) for i in (0, 1)]


@pytest.mark.parametrize("tokens", [3, 70])
@pytest.mark.parametrize("dim,page", [(64, 32), (128, 16)])
@pytest.mark.parametrize("norm,rope,use_table", [(True, True, True), (True, True, False), (False, False, False)])
def test_store(tokens, dim, page, norm, rope, use_table):
    from tiny_llm_infer_b200 import ops
    g = gen(tokens + dim)
    q_heads, kv_heads = 6, 3
    pages = -(-tokens // page) + 4
    planes = planes_of(pages, kv_heads, page, dim)
    before = [p.clone() for p in planes]
    table = tables(g, [tokens + 40], page, pages, pages)
    first = 9
    pos = torch.arange(first, first + tokens, dtype=torch.int32, device="cuda")
    slots = torch.zeros(tokens, dtype=torch.int32, device="cuda")
    slots[1] = -1
    qkv = (torch.randn((tokens, (q_heads + 2 * kv_heads) * dim), generator=g, device="cuda") * 2).to(torch.bfloat16)
    qkv[0, -dim:] = 0                                           # a value of zeros
    gains = [(torch.rand(dim, generator=g, device="cuda") + 0.5) for _ in range(2)] if norm else [None, None]
    inv = (1e4 ** (-torch.arange(0, dim, 2, device="cuda").float() / dim)) if rope else None
    angles = ops.rope_table(pos, inv) if rope else None
    q_out = torch.full((tokens, q_heads * dim), 7.0, dtype=torch.bfloat16, device="cuda")
    flags = (ops.QK_NORM if norm else 0) | (ops.QK_ROPE if rope else 0) | ops.QK_STORE | ops.QK_QOUT
    ops.qk_norm_rope_store_fp8(qkv, gains[0], gains[1], 1e-6, inv, dim if rope else 0, pos, slots, table, planes, page, q_out, q_heads, kv_heads, dim, flags,
                               angles if use_table else None)
    x = qkv.double().view(tokens, q_heads + 2 * kv_heads, dim).clone()
    slack = torch.zeros_like(x)
    for lo, hi, gain in ((0, q_heads, gains[0]), (q_heads, q_heads + kv_heads, gains[1])):
        part = x[:, lo:hi]
        if norm:
            part = gain.double() * part / torch.sqrt((part * part).mean(-1, keepdim=True) + 1e-6)
        if rope:
            cos, sin = angles.double()[:, 0, None], angles.double()[:, 1, None]
            a, b = part[..., :dim // 2], part[..., dim // 2:]
            size = torch.cat([a.abs() + b.abs()] * 2, dim=-1)
            part = torch.cat([a * cos - b * sin, a * sin + b * cos], dim=-1)
        else:
            size = part.abs()
        x[:, lo:hi], slack[:, lo:hi] = part, size * 2.0 ** -18          # a sum of `dim` squares and a dozen float32 operations
    live = torch.arange(tokens, device="cuda") != 1
    q_want = x[:, :q_heads].reshape(tokens, -1)
    q_slack = slack[:, :q_heads].reshape(tokens, -1)
    assert ((q_out.double() - q_want).abs() <= q_slack + (q_want.abs() + q_slack) * 2.0 ** -8)[live].all() and (q_out[1] == 7).all()
    at = table[0].long()[pos.long() // page]
    where = pos.long() % page
    for i in range(2):
        want = x[:, q_heads + i * kv_heads:q_heads + (i + 1) * kv_heads]
        lax = slack[:, q_heads + i * kv_heads:q_heads + (i + 1) * kv_heads]
        scale = planes[2].view(torch.float32)[at, :, where, i][live].double()
        largest = (want.abs().amax(-1).clamp_min(2.0 ** -100) / 448)[live]
        assert ((scale - largest).abs() <= largest * 2.0 ** -17).all()
        got = planes[i][at, :, where].view(torch.float8_e4m3fn).double()[live] * scale[..., None]
        assert ((got - want[live]).abs() <= lax[live] + ref.half_step((want.abs() + lax)[live], scale[..., None])).all()
    # nothing else was written: neither the skipped row's place nor other tokens' or pages'
    for i, (new, old) in enumerate(zip(planes, before)):
        new = new.clone()
        new[at[live], :, where[live]] = old[at[live], :, where[live]]
        assert torch.equal(new, old)


@pytest.mark.parametrize("q_heads,kv_heads,dim,page", [(32, 8, 128, 16), (16, 8, 64, 32), (6, 2, 128, 48)])
@pytest.mark.parametrize("window", [0, 100])
def test_a_step_of_portions_and_single_tokens(q_heads, kv_heads, dim, page, window):
    """Two portions behind keys of earlier steps and two single tokens, as the runner lays them out."""
    from tiny_llm_infer_b200 import ops
    g = gen(dim + window)
    earlier, new = [37, 0, 300, 20], [1, 150, 67, 1]
    lengths = [a + b for a, b in zip(earlier, new)]
    pages = sum(-(-n // page) for n in lengths) + 2
    planes = planes_of(pages, kv_heads, page, dim)
    table = tables(g, lengths, page, pages, 12 + 500 // page)
    kept = fill(g, planes, table, lengths, page, (0.3, 0.3))
    total = sum(new)
    q = torch.randn((total, q_heads * dim), generator=g, device="cuda").to(torch.bfloat16)
    seg, pos, slots, dec, tiles, row = [], [], [], [], [], 0
    for r, n in enumerate(new):
        seg.append((r, row, n, earlier[r]))
        pos += range(earlier[r], earlier[r] + n)
        slots += [r] * n
        if n == 1:
            dec.append(row)
        else:
            tiles += [(r, o) for o in range(0, n, 64)]
        row += n
    tiles.sort(key=lambda t: (t[1] % 256 != 0, t[1] % 128 != 0))

    def dev(x):
        return torch.tensor(x, dtype=torch.int32, device="cuda")
    segments = [SimpleNamespace(length=n, pos0=p) for _, _, n, p in seg]
    ctx = SimpleNamespace(tokens=total, segments=segments, seg_info=dev(seg), dec_rows=dev(dec), n_dec=2, pf_tiles=dev(tiles), n_tiles=len(tiles),
                          n_tiles128=sum(t[1] % 128 == 0 for t in tiles), n_tiles256=sum(t[1] % 256 == 0 for t in tiles), max_context=max(lengths))
    out = torch.empty_like(q)
    scale = 1 / math.sqrt(dim)
    ops.paged_attention_fp8(q, planes, dev(pos), dev(slots), table, page, q_heads, kv_heads, dim, window or None, scale, out, ctx)
    ops.check_error_word("cuda")
    for i in range(total):
        r = slots[i]
        keys, values = kept[r]
        want, off = exact_row(q[i].double().view(q_heads, dim), keys, values, pos[i], window, scale)
        if i not in dec:
            # keys and values pass through bfloat16 on their way (2^-8 each), and so do the weights of the prompt kernels
            qa, first = q[i].double().abs().view(kv_heads, -1, dim), max(0, pos[i] + 1 - window) if window else 0
            k, v = keys[:, first:pos[i] + 1].abs(), values[:, first:pos[i] + 1]
            qk = (q[i].double().view(kv_heads, -1, dim) @ keys[:, first:pos[i] + 1].transpose(1, 2)) * scale
            e = (qa @ k.transpose(1, 2)).amax(-1, keepdim=True) * scale * 2.0 ** -8
            mass = torch.softmax(qk, dim=-1) @ v.abs()
            off = off + (mass * (torch.expm1(2 * e) + 2 * 2.0 ** -8) * 1.02).reshape(-1)
        assert ((out[i].double() - want).abs() <= off).all()


def test_store_and_read_together_in_a_graph():
    """A token stored and read in one captured step, replayed token by token, against the same calls one by one."""
    from tiny_llm_infer_b200 import ops
    g = gen(11)
    q_heads, kv_heads, dim, page, steps = 8, 2, 128, 16, 40
    planes, others = planes_of(4, kv_heads, page, dim), planes_of(4, kv_heads, page, dim)
    table = tables(g, [64], page, 4, 4)
    pos, slot = torch.zeros(1, dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
    qkv = torch.zeros((1, (q_heads + 2 * kv_heads) * dim), dtype=torch.bfloat16, device="cuda")

    def step(cache):
        q, out = (torch.empty((1, q_heads * dim), dtype=torch.bfloat16, device="cuda") for _ in range(2))
        ops.qk_norm_rope_store_fp8(qkv, None, None, 1.0, None, 0, pos, slot, table, cache, page, q, q_heads, kv_heads, dim, ops.QK_STORE | ops.QK_QOUT)
        return ops.paged_attention_decode_fp8(q, cache, pos, slot, None, 1, table, page, q_heads, kv_heads, dim, None, 0.088, out, 64)
    step(planes)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(planes)
    for i in range(steps):
        qkv.copy_(torch.randn(qkv.shape, generator=g, device="cuda").to(torch.bfloat16))
        pos.fill_(i)
        graph.replay()
        assert torch.equal(out, step(others))
        keys, values = stored(planes, table, 0, i + 1, page)
        want, off = exact_row(qkv[0, :q_heads * dim].double().view(q_heads, dim), keys, values, i, 0, 0.088)
        assert ((out[0].double() - want).abs() <= off).all()


def test_refusals():
    from tiny_llm_infer_b200 import ops
    planes = planes_of(3, 2, 16, 64)
    q = torch.zeros((2, 4 * 64), dtype=torch.bfloat16, device="cuda")
    one = torch.zeros(2, dtype=torch.int32, device="cuda")
    table = torch.zeros((1, 3), dtype=torch.int32, device="cuda")

    def call(q=q, planes=planes, pos=one, slots=one, rows=None, n=2, table=table, page=16, qh=4, kvh=2, dim=64, out=None):
        return ops.paged_attention_decode_fp8(q, planes, pos, slots, rows, n, table, page, qh, kvh, dim, None, 0.1, torch.empty_like(q) if out is None else out, 48)
    call()
    for kw in (dict(q=q.float()), dict(planes=planes[:2]), dict(planes=(planes[0], planes[1], planes[1])), dict(pos=one.long()), dict(n=3), dict(page=8),
               dict(qh=2, dim=128), dict(table=table.long()), dict(pos=one[:1]), dict(out=q[:1]), dict(q=q.cpu()),
               dict(planes=tuple(p.transpose(1, 2).contiguous().transpose(1, 2) for p in planes)), dict(kvh=1)):
        with pytest.raises(ops.KernelError):
            call(**kw)
    big = planes_of(1, 2, 8, 64)
    with pytest.raises(ops.KernelError):
        call(planes=big, page=8)
    with pytest.raises(ops.KernelError):
        call(q=torch.zeros((2, 2 * 17 * 64), dtype=torch.bfloat16, device="cuda"), qh=34)
    qkv = torch.zeros((2, 8 * 64), dtype=torch.bfloat16, device="cuda")
    inv = torch.ones(16, device="cuda")
    for kw in (dict(rot=32, inv=inv, flags=ops.QK_ROPE), dict(flags=ops.QK_NORM), dict(qkv=qkv.float()), dict(qkv=qkv[:, :7 * 64].contiguous())):
        with pytest.raises(ops.KernelError):
            ops.qk_norm_rope_store_fp8(kw.get("qkv", qkv), None, None, 1.0, kw.get("inv"), kw.get("rot", 0), one, one, table, planes, 16, q.clone(), 4, 2, 64,
                                       kw.get("flags", 0) | ops.QK_STORE | ops.QK_QOUT)


@pytest.mark.parametrize("blocks", [0, 30])
def test_a_position_past_the_block_table_reads_no_other_memory(blocks):
    """The last key that the table has room for is as far as a row sees."""
    from tiny_llm_infer_b200 import ops
    g = gen(13)
    planes = planes_of(4, 2, 16, 64)
    table = tables(g, [64], 16, 4, 4)
    fill(g, planes, table, [64], 16, (0.3, 0.3))
    q = torch.randn((1, 4 * 64), generator=g, device="cuda").to(torch.bfloat16)
    outs = []
    for pos in (63, 64, 100000):
        outs.append(torch.empty_like(q))
        ops.paged_attention_decode_fp8(q, planes, torch.tensor([pos], dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda"),
                                       None, 1, table, 16, 4, 2, 64, None, 0.125, outs[-1], 64, blocks)
    assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])


def test_many_rows_of_a_step():
    """More rows than share blocks, and as many as do: every row as if it were alone, rows of no request between them."""
    from tiny_llm_infer_b200 import ops
    g = gen(17)
    q_heads, kv_heads, dim, page = 4, 2, 64, 16
    lengths = [1 + (37 * i) % 700 for i in range(40)]
    pages = sum(-(-n // page) for n in lengths)
    planes = planes_of(pages, kv_heads, page, dim)
    table = tables(g, lengths, page, pages, 44)
    fill(g, planes, table, lengths, page, (0.3, 0.3))
    for total, blocks in ((512, 444), (512, 1), (700, 0), (700, None), (240, 0), (256, None), (129, 512)):
        slots = torch.tensor([-1 if i % 7 == 3 else (i * 11) % 40 for i in range(total)], dtype=torch.int32, device="cuda")
        pos = torch.tensor([lengths[(i * 11) % 40] - 1 for i in range(total)], dtype=torch.int32, device="cuda")
        q = torch.randn((total, q_heads * dim), generator=g, device="cuda").to(torch.bfloat16)
        out = torch.empty_like(q)
        ops.paged_attention_decode_fp8(q, planes, pos, slots, None, total, table, page, q_heads, kv_heads, dim, None, 0.125, out, 700, blocks)
        assert (out[slots < 0] == 0).all()
        for i in (0, 1, 5, total // 2, total - 1):
            if i % 7 == 3:
                continue
            r = (i * 11) % 40
            keys, values = stored(planes, table, r, lengths[r], page)
            want, off = exact_row(q[i].double().view(q_heads, dim), keys, values, lengths[r] - 1, 0, 0.125)
            assert ((out[i].double() - want).abs() <= off).all()
    with pytest.raises(ops.KernelError):
        ops.paged_attention_decode_fp8(q, planes, pos, slots, None, 129, table, page, q_heads, kv_heads, dim, None, 0.125, out, 700, 513)


@pytest.mark.parametrize("how", [dict(blocks=0), dict(blocks=30), dict(cluster=4), dict(cluster=8)])
@pytest.mark.parametrize("dim", [64, 128])
def test_what_no_page_holds_does_not_count(dim, how):
    """Entries of the table without a page, or with one the cache does not have: their keys are left out, in the middle, at either end and
    everywhere; slots and positions of no request give zeros."""
    from tiny_llm_infer_b200 import ops
    g = gen(19)
    q_heads, kv_heads, page, length = 8, 2, 16, 400
    planes = planes_of(25, kv_heads, page, dim)
    table = tables(g, [length] * 1, page, 25, 25)
    fill(g, planes, table, [length], page, (0.3, 0.3))
    keys, values = stored(planes, table, 0, length, page)
    gone = [[], [3, 4, 11], [0], [24], [0, 1, 2, 22, 23, 24], list(range(25)), [24], []]
    tabs = table.repeat(len(gone), 1)
    for r, pages in enumerate(gone):
        tabs[r, pages] = torch.tensor([-1 if i % 2 else 25 + 1000 * r for i in range(len(pages))], dtype=torch.int32, device="cuda")
    n = len(gone)
    pos = torch.tensor([length - 1] * (n - 2) + [385, -5], dtype=torch.int32, device="cuda")
    slots = torch.tensor(list(range(n - 1)) + [n - 1], dtype=torch.int32, device="cuda")
    q = torch.randn((n + 1, q_heads * dim), generator=g, device="cuda").to(torch.bfloat16)
    pos, slots = torch.cat([pos, pos[:1]]), torch.cat([slots, slots[-1:] + 1])          # and a slot behind the table
    out = torch.empty_like(q)
    ops.paged_attention_decode_fp8(q, planes, pos, slots, None, n + 1, tabs, page, q_heads, kv_heads, dim, None, 0.125, out, length, **how)
    for r in range(n + 1):
        left = [j for j in range(pos[r] + 1) if r < n - 1 and j // page not in gone[r]]
        if not left:
            assert (out[r] == 0).all()
            continue
        want, off = exact_row(q[r].double().view(q_heads, dim), keys[:, left], values[:, left], len(left) - 1, 0, 0.125)
        assert ((out[r].double() - want).abs() <= off).all()


def test_a_store_outside_the_cache_is_left_out():
    """Positions behind the table's room, slots it does not have and pages the cache does not have: nothing is written for them."""
    from tiny_llm_infer_b200 import ops
    q_heads, kv_heads, dim, page = 4, 2, 64, 16
    planes = planes_of(3, kv_heads, page, dim)
    for plane in planes:
        plane.fill_(7)
    table = torch.tensor([[0, 3], [-1, 1 << 20]], dtype=torch.int32, device="cuda")
    pos = torch.tensor([16, 32, 1 << 30, -1, 0, 16, 0, 5], dtype=torch.int32, device="cuda")
    slots = torch.tensor([0, 0, 1, 1, 1, 1, 2, 0], dtype=torch.int32, device="cuda")
    qkv = torch.randn((8, (q_heads + 2 * kv_heads) * dim), generator=gen(23), device="cuda").to(torch.bfloat16)
    q_out = torch.empty((8, q_heads * dim), dtype=torch.bfloat16, device="cuda")
    ops.qk_norm_rope_store_fp8(qkv, None, None, 1.0, None, 0, pos, slots, table, planes, page, q_out, q_heads, kv_heads, dim, ops.QK_STORE | ops.QK_QOUT)
    assert torch.equal(q_out, qkv[:, :q_heads * dim])
    held = planes[2].view(torch.float32)[0, :, 5].clone()
    assert (held > 0).all() and (held < 1).all()
    for plane in planes:
        plane[0, :, 5] = 7                                        # the one row with a place
        assert (plane == 7).all()
