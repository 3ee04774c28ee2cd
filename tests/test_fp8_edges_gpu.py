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
