"""The definitions of the 8-bit operators in 64 bits, for the tests: what a block's scale is, how far a rounding may be off, products
of values."""
import torch

BLOCK = 128


def block_of(n, device=None):
    return torch.arange(n, device=device) // BLOCK


def row_scales(x):
    """[T, ceil(K / 128)] float32: the largest magnitude of 128 columns, at least 2^-100, over 448."""
    t, k = x.shape
    kb = -(-k // BLOCK)
    padded = torch.zeros((t, kb * BLOCK), dtype=torch.float32, device=x.device)
    padded[:, :k] = x.float()
    largest = padded.view(t, kb, BLOCK).abs().amax(dim=2).clamp_min(2.0 ** -100)
    return largest / torch.full_like(largest, 448.0)        # the quotient (torch multiplies by a number's reciprocal instead)


def weight_scales(w):
    n, k = w.shape
    nb = -(-n // BLOCK)
    padded = torch.zeros((nb * BLOCK, k), dtype=torch.float32, device=w.device)
    padded[:n] = w.float()
    largest = padded.view(nb, BLOCK, k).abs().amax(dim=1)
    return row_scales(largest)


def gated_weight_scales(w):
    n, k = w.shape
    pairs = w.view(n // 16, 2, 8, k)
    gate, up = (weight_scales(pairs[:, i].reshape(n // 2, k)) for i in (0, 1))
    return torch.stack([gate, up], dim=1).reshape(-1, gate.shape[1])


def half_step(x, scale):
    """How far the e4m3 value nearest to x / scale may be from x: half a step is 2^-4 of the number, or 2^-10 scales below the smallest
    normal value 2^-6; the product with the reciprocal scale, in float32, is off by up to 2^-22 of itself before that."""
    x, scale = x.double(), scale.double()
    return torch.maximum(x.abs() * 2.0 ** -4, scale * 2.0 ** -10) * (1 + 2.0 ** -20)


def product_bound(x, w, out_dtype):
    """(exact, how far off) of x . w^T for float64 values x, w: float32 sums of K terms, a rounding a term at the most, each of 2^-23 of
    what the magnitudes add up to, the scales' product and its use (3 roundings), and the rounding of the result."""
    exact, total = x @ w.t(), x.abs() @ w.abs().t()
    sums = total * ((x.shape[1] + 8) * 2.0 ** -23)
    rounding = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}[out_dtype]
    return exact, sums + rounding * (exact.abs() + sums)
