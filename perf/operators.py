"""Serving in 8 bits: the operators of this engine that read 8-bit weights and an 8-bit cache, as cases that can be timed and
compared.

Three kinds:

  linear        rows in bfloat16 times a weight kept as e4m3 values with a float32 scale per block of 128 x 128: every 128 numbers
                of a row are scaled and rounded to e4m3 too, products are summed in float32
  feed_forward  RMSNorm of the float32 residual stream, gate and up products, silu(gate) * up, down product; the normed rows
                and the gated unit's outputs reach the products as e4m3 rows with a scale per 128 columns
  attention     one new token per request over a paged cache of e4m3 keys and values with one float32 scale per token and head for
                the key and one for the value

Sizes are those of ``bench.py`` (Qwen3-8B and Qwen3-0.6B) and odd ones around them.  Where ``own`` is false, ``run`` computes the
operators from elementary torch operations in float32.
"""
from __future__ import annotations

import math

import torch

own = False

DEV = "cuda:0"
BLOCK = 128
EPS = 1e-6
E4M3_MAX = 448.0
SMALLEST = 2.0 ** -100          # what a block's largest magnitude is taken to be at least


# --------------------------------------------------------------------------- the cases
def listed():
    return [
        # the smallest call: the output projection of the smallest model for one chat request
        dict(name="linear_one_row", kind="linear", rows=1, k=2048, n=1024),
        # eight requests decode: the fused q|k|v projection of the 8B model
        dict(name="linear_eight_rows", kind="linear", rows=8, k=4096, n=6144),
        # a short portion of a prompt beside decoding requests
        dict(name="linear_odd_portion", kind="linear", rows=61, k=4096, n=4096),
        # a ragged portion with sizes that end inside blocks of 128
        dict(name="linear_ragged", kind="linear", rows=509, k=2192, n=1608),
        # a prompt of 2048 tokens: the fused q|k|v projection of the 8B model
        dict(name="linear_prompt", kind="linear", rows=2048, k=4096, n=6144),
        # one request decodes through the feed-forward of the 8B model
        dict(name="feed_forward_one_row", kind="feed_forward", rows=1, width=4096, inter=12288),
        # eight requests decode through it
        dict(name="feed_forward_eight_rows", kind="feed_forward", rows=8, width=4096, inter=12288),
        # a prompt of 2048 tokens through it
        dict(name="feed_forward_prompt", kind="feed_forward", rows=2048, width=4096, inter=12288),
        # one request at a context of 4095 tokens, heads of the 8B model
        dict(name="attention_one_request", kind="attention", requests=1, context=4095, q_heads=32, kv_heads=8, dim=128, page=16, window=0),
        # sixty-four requests with contexts between 1000 and 4096
        dict(name="attention_sixty_four", kind="attention", requests=64, context=4096, q_heads=32, kv_heads=8, dim=128, page=16, window=0),
        # two requests with very long contexts
        dict(name="attention_long", kind="attention", requests=2, context=131072, q_heads=32, kv_heads=8, dim=128, page=64, window=0),
        # narrow heads with a sliding window, larger pages
        dict(name="attention_window", kind="attention", requests=24, context=3333, q_heads=16, kv_heads=8, dim=64, page=32, window=1000),
    ]


def _between(rng, lo, hi):
    """A whole number whose logarithm is spread evenly."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    kind = rng.choice(["linear", "linear", "feed_forward", "attention", "attention"])
    if kind == "linear":
        return dict(kind=kind, rows=_between(rng, 1, 2048), k=16 * _between(rng, 32, 256), n=8 * _between(rng, 64, 768))
    if kind == "feed_forward":
        return dict(kind=kind, rows=_between(rng, 1, 2048), width=16 * _between(rng, 64, 256), inter=16 * _between(rng, 96, 768))
    kv_heads = rng.choice([1, 2, 4, 8])
    context = _between(rng, 16, 65536)
    requests = min(_between(rng, 1, 64), max(1, 262144 // context))
    window = rng.choice([0, 0, 0, _between(rng, 8, 4096)])
    return dict(kind=kind, requests=requests, context=context, q_heads=kv_heads * rng.choice([1, 2, 4, 5, 8, 16]), kv_heads=kv_heads,
                dim=rng.choice([64, 128, 128]), page=rng.choice([16, 16, 32, 64]), window=window)


# --------------------------------------------------------------------------- inputs
def _weight(gen, n, k):
    """An [n, k] matrix as e4m3 values and float32 scales per block of 128 x 128, as a checkpoint of 8-bit weights holds them."""
    w = torch.randn((n, k), generator=gen, device=DEV) * (0.02 * torch.exp(0.3 * torch.randn((n, 1), generator=gen, device=DEV)))
    nb, kb = -(-n // BLOCK), -(-k // BLOCK)
    padded = torch.zeros((nb * BLOCK, kb * BLOCK), device=DEV)
    padded[:n, :k] = w
    blocks = padded.view(nb, BLOCK, kb, BLOCK)
    scales = blocks.abs().amax(dim=(1, 3)).clamp_min(SMALLEST) / E4M3_MAX
    q = (blocks / scales[:, None, :, None]).to(torch.float8_e4m3fn).view(nb * BLOCK, kb * BLOCK)
    return q[:n, :k].contiguous(), scales.contiguous()


def _activations(gen, rows, width):
    """Rows as a network makes them: of order one, a few columns much larger than the others."""
    column = torch.exp(0.5 * torch.randn(width, generator=gen, device=DEV))
    column = torch.where(torch.rand(width, generator=gen, device=DEV) < 0.01, column * 8, column)
    return torch.randn((rows, width), generator=gen, device=DEV) * column


def _interleaved(a, b):
    """Rows of two matrices in turn, eight of the one and eight of the other: how the engine lays gate and up out."""
    n, k = a.shape
    return torch.stack([a.view(n // 8, 8, k), b.view(n // 8, 8, k)], dim=1).reshape(2 * n, k).contiguous()


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    s = dict(case)
    if case["kind"] == "linear":
        s["x"] = _activations(gen, case["rows"], case["k"]).to(torch.bfloat16)
        s["w"], s["w_scales"] = _weight(gen, case["n"], case["k"])
        if own:
            from tiny_llm_infer_b200 import ops
            s["weight"] = ops.Fp8Weight(s["w"], s["w_scales"])
    elif case["kind"] == "feed_forward":
        width, inter = case["width"], case["inter"]
        s["h"] = _activations(gen, case["rows"], width)
        s["gain"] = 0.8 + 0.4 * torch.rand(width, generator=gen, device=DEV)
        (gate, gate_scales), (up, up_scales) = _weight(gen, inter, width), _weight(gen, inter, width)
        # gate and up as one matrix, eight rows of each in turn; their scales in turn, block by block
        as_bytes = _interleaved(gate.view(torch.uint8), up.view(torch.uint8))
        s["gate_up"] = as_bytes.view(torch.float8_e4m3fn)
        s["gate_up_scales"] = torch.stack([gate_scales, up_scales], dim=1).reshape(-1, gate_scales.shape[1]).contiguous()
        s["down"], s["down_scales"] = _weight(gen, width, inter)
        if own:
            from tiny_llm_infer_b200 import ops
            s["w_gate_up"] = ops.Fp8Weight(s["gate_up"], s["gate_up_scales"], gated=True)
            s["w_down"] = ops.Fp8Weight(s["down"], s["down_scales"])
    else:
        requests, context, page = case["requests"], case["context"], case["page"]
        kv_heads, dim = case["kv_heads"], case["dim"]
        lengths = torch.randint(max(1, context // 4), context + 1, (requests,), generator=gen, device=DEV)
        lengths[0] = context
        per = -(-context // page)
        held = -(-lengths // page)
        total = int(held.sum())
        order = torch.randperm(total, generator=gen, device=DEV).to(torch.int32)       # pages as they come in a long run
        table = torch.full((requests, per), -1, dtype=torch.int32, device=DEV)
        inside = torch.arange(per, device=DEV)[None, :] < held[:, None]
        table[inside] = order
        # a page: its keys [kv_heads, page, dim], its values, then [kv_heads, page] pairs of scales (key, value)
        plane = kv_heads * page * dim
        pages = torch.zeros((total, 2 * plane + kv_heads * page * 8), dtype=torch.uint8, device=DEV)
        column = torch.exp(0.5 * torch.randn((kv_heads, 1, dim), generator=gen, device=DEV))
        for at, spread in ((0, 0.1), (1, 0.5)):
            for first in range(0, total, 2048):
                n = min(2048, total - first)
                x = torch.randn((n, kv_heads, page, dim), generator=gen, device=DEV) * column
                x = x * torch.exp(spread * torch.randn((n, kv_heads, page, 1), generator=gen, device=DEV))
                scale = x.abs().amax(dim=-1).clamp_min(SMALLEST) / E4M3_MAX
                q = (x / scale[..., None]).to(torch.float8_e4m3fn).view(torch.uint8)
                pages[first:first + n, at * plane:(at + 1) * plane] = q.reshape(n, plane)
                pages[first:first + n, 2 * plane:].view(torch.float32).view(n, kv_heads, page, 2)[..., at] = scale
        s["pages"] = pages
        s["planes"] = (pages[:, :plane].unflatten(1, (kv_heads, page, dim)), pages[:, plane:2 * plane].unflatten(1, (kv_heads, page, dim)),
                       pages[:, 2 * plane:].unflatten(1, (kv_heads, page, 8)))
        s["table"], s["positions"] = table, (lengths - 1).to(torch.int32)
        s["slots"] = torch.arange(requests, dtype=torch.int32, device=DEV)
        s["q"] = (2.0 * torch.randn((requests, case["q_heads"] * dim), generator=gen, device=DEV)).to(torch.bfloat16)
        s["out"] = torch.empty_like(s["q"])
    return s


# --------------------------------------------------------------------------- one pass
def _rounded_rows(x):
    """Rows as the e4m3 values with scales stand for them: float32 in, float32 out."""
    rows, k = x.shape
    kb = -(-k // BLOCK)
    blocks = torch.nn.functional.pad(x, (0, kb * BLOCK - k)).view(rows, kb, BLOCK)
    scales = (blocks.abs().amax(dim=-1, keepdim=True).clamp_min(SMALLEST)) / E4M3_MAX
    q = (blocks * (1.0 / scales)).to(torch.float8_e4m3fn)
    return (q.to(torch.float32) * scales).view(rows, kb * BLOCK)[:, :k]


def _values(q, scales):
    """A weight's float32 values."""
    n, k = q.shape
    return q.to(torch.float32) * scales.repeat_interleave(BLOCK, 0)[:n].repeat_interleave(BLOCK, 1)[:, :k]


def _plain_attention(s):
    requests, page, dim, kv_heads = s["requests"], s["page"], s["dim"], s["kv_heads"]
    group = s["q_heads"] // kv_heads
    at = s["table"].clamp_min(0).long()                              # [requests, pages of a request]
    keys, values, scales = s["planes"]

    def gathered(plane, which):
        q = plane[at].view(torch.float8_e4m3fn).to(torch.float32)    # [requests, pages, kv_heads, page, dim]
        scale = scales[at].view(torch.float32)[..., which:which + 1]
        return (q * scale).transpose(1, 2).reshape(requests, kv_heads, -1, dim)

    query = s["q"].to(torch.float32).view(requests, kv_heads, group, dim)
    score = torch.matmul(query, gathered(keys, 0).transpose(2, 3)) / math.sqrt(dim)
    token = torch.arange(score.shape[-1], device=DEV)
    pos = s["positions"][:, None]
    seen = token[None, :] <= pos
    if s["window"]:
        seen = seen & (token[None, :] > pos - s["window"])
    score = score.masked_fill(~seen[:, None, None, :], -math.inf)
    weight = torch.exp(score - score.amax(dim=-1, keepdim=True))
    weight = weight / weight.sum(dim=-1, keepdim=True)
    return torch.matmul(weight, gathered(values, 1)).reshape(requests, -1).to(torch.bfloat16)


def run(s):
    if s["kind"] == "linear":
        if own:
            from tiny_llm_infer_b200 import ops
            return ops.linear(s["x"], s["weight"])
        return torch.matmul(_rounded_rows(s["x"].to(torch.float32)), _values(s["w"], s["w_scales"]).t()).to(torch.bfloat16)
    if s["kind"] == "feed_forward":
        if own:
            from tiny_llm_infer_b200 import ops
            x = ops.add_rmsnorm_fp8(s["h"], None, s["gain"], EPS)
            return ops.linear(ops.linear_swiglu(x, s["w_gate_up"]), s["w_down"])
        h = s["h"]
        x = _rounded_rows(s["gain"] * h / torch.sqrt(h.square().mean(dim=-1, keepdim=True) + EPS))
        inter, width = s["inter"], s["width"]
        both = s["gate_up"].view(inter // 8, 2, 8, width)
        halves = s["gate_up_scales"].view(-1, 2, s["gate_up_scales"].shape[1])
        gate = torch.matmul(x, _values(both[:, 0].reshape(inter, width), halves[:, 0]).t())
        up = torch.matmul(x, _values(both[:, 1].reshape(inter, width), halves[:, 1]).t())
        act = _rounded_rows(gate / (1.0 + torch.exp(-gate)) * up)
        return torch.matmul(act, _values(s["down"], s["down_scales"]).t()).to(torch.bfloat16)
    if own:
        from tiny_llm_infer_b200 import ops
        return ops.paged_attention_decode_fp8(s["q"], s["planes"], s["positions"], s["slots"], None, s["requests"], s["table"], s["page"],
                                              s["q_heads"], s["kv_heads"], s["dim"], s["window"] or None, 1.0 / math.sqrt(s["dim"]),
                                              s["out"], s["context"])
    return _plain_attention(s)


# --------------------------------------------------------------------------- what a pass cannot do without
def _keys(case):
    """Keys that all requests together read, for the mean length of a request."""
    first, others = case["context"], (max(1, case["context"] // 4) + case["context"]) / 2
    if case["window"]:
        first, others = min(first, case["window"]), min(others, case["window"])
    return first + (case["requests"] - 1) * others


def work(case):
    if case["kind"] == "linear":
        t, k, n = case["rows"], case["k"], case["n"]
        return {"bytes": 2 * t * k + n * k + 4 * -(-n // BLOCK) * -(-k // BLOCK) + 2 * t * n, "flops": 2.0 * t * n * k}
    if case["kind"] == "feed_forward":
        t, w, i = case["rows"], case["width"], case["inter"]
        return {"bytes": 4 * t * w + 4 * w + 3 * w * i + 3 * 4 * -(-w // BLOCK) * -(-i // BLOCK) + 2 * t * w, "flops": 6.0 * t * w * i}
    keys = _keys(case)
    return {"bytes": keys * case["kv_heads"] * (2 * case["dim"] + 8) + 4 * case["requests"] * case["q_heads"] * case["dim"],
            "flops": 4.0 * keys * case["q_heads"] * case["dim"]}


# --------------------------------------------------------------------------- the definition in 64 bits
def _nearest_e4m3(v):
    """The e4m3 value nearest to v, ties to the even one, held within the largest: three bits behind the leading one, exponents from
    -6 up."""
    _, exponent = torch.frexp(v)
    step = torch.ldexp(torch.ones_like(v), (exponent - 1).clamp_min(-6) - 3)
    return (torch.round(v / step) * step).clamp(-E4M3_MAX, E4M3_MAX)


def _rounded_rows64(x):
    out = torch.empty_like(x)
    for k0 in range(0, x.shape[1], BLOCK):
        part = x[:, k0:k0 + BLOCK]
        top = part.abs().max(dim=1, keepdim=True).values
        scale = (torch.maximum(top, torch.full_like(top, SMALLEST)) / E4M3_MAX).to(torch.float32).to(torch.float64)
        out[:, k0:k0 + BLOCK] = _nearest_e4m3(part / scale) * scale
    return out


def _product64(x, q, scales):
    """Block by block of the weight's rows."""
    n, k = q.shape
    out = torch.empty((x.shape[0], n), dtype=torch.float64, device=x.device)
    column = torch.arange(k, device=x.device) // BLOCK
    for n0 in range(0, n, BLOCK):
        w = q[n0:n0 + BLOCK].to(torch.float64) * scales[n0 // BLOCK].to(torch.float64)[column]
        out[:, n0:n0 + BLOCK] = x @ w.t()
    return out


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "linear":
        return _product64(_rounded_rows64(s["x"].to(torch.float64)), s["w"], s["w_scales"])
    if case["kind"] == "feed_forward":
        h = s["h"].to(torch.float64)
        x = _rounded_rows64(s["gain"].to(torch.float64) * h * torch.rsqrt((h * h).sum(dim=1, keepdim=True) / h.shape[1] + EPS))
        rows = torch.arange(2 * case["inter"], device=DEV)
        is_up = (rows // 8) % 2 == 1
        both = s["gate_up"].view(torch.uint8)
        gate = _product64(x, both[~is_up].view(torch.float8_e4m3fn), s["gate_up_scales"][0::2])
        up = _product64(x, both[is_up].view(torch.float8_e4m3fn), s["gate_up_scales"][1::2])
        return _product64(_rounded_rows64(gate * torch.sigmoid(gate) * up), s["down"], s["down_scales"])
    group, dim, page = case["q_heads"] // case["kv_heads"], case["dim"], case["page"]
    out = torch.empty((case["requests"], case["q_heads"], dim), dtype=torch.float64, device=DEV)
    for r, pos in enumerate(s["positions"].tolist()):
        first = max(0, pos + 1 - case["window"]) if case["window"] else 0
        token = torch.arange(first, pos + 1, device=DEV)
        where = s["table"][r].long()[token // page]
        for head in range(case["kv_heads"]):
            key, value = (s["planes"][i][where, head, token % page].view(torch.float8_e4m3fn).to(torch.float64) for i in (0, 1))
            scale = s["planes"][2][where, head, token % page].view(torch.float32).to(torch.float64)
            query = s["q"][r].view(-1, dim)[head * group:(head + 1) * group].to(torch.float64)
            p = torch.softmax(query @ (key * scale[:, :1]).t() / math.sqrt(dim), dim=1)
            out[r, head * group:(head + 1) * group] = p @ (value * scale[:, 1:])
    return out.view(case["requests"], -1)
