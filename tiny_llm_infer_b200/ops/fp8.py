"""Weights, rows and caches in 8 bits: e4m3 values with float32 scales, and the kernels that read them (``csrc/fp8*.cu``).

A block of numbers with largest magnitude A is kept as e4m3(x (1 / s)) and s = max(A, 2^-100) / 448, in float32.  A weight has a scale per
block of 128 x 128, a row that meets it one per 128 columns, a key or value of the cache one per head.  A product sums the 128 terms of
a block in float32, multiplies by both scales and adds the blocks in float32:

    y[t, n] = sum_b sx[t, b] sw[n / 128, b] sum_{k in b} qx[t, k] qw[n, k]

``ops.linear`` and ``ops.linear_swiglu`` take an ``Fp8Weight`` in the place of a weight, and rows in bfloat16, float32 or as ``Fp8Rows``.
Which kernel runs goes by the number of rows, the last bits of a row with it; what is rounded to 8 bits does not depend on it.
Infinities and NaN in a row of x reach the outputs of that row alone (as NaN), in a weight those of its block's columns.
"""
from __future__ import annotations

import ctypes
import functools
from typing import Optional

import torch

BLOCK = 128
E4M3 = torch.float8_e4m3fn
SMALLEST = 2.0 ** -100
LARGEST = 448.0
NORM_WIDTH = 32768       # columns that add_rmsnorm_fp8 takes


_package = None


def _ops():
    """The package of the kernels (imported late: it imports this module)."""
    global _package
    if _package is None:
        from .. import ops
        _package = ops
    return _package


def declare(h) -> None:
    """Signatures of the C entry points."""
    vp, i32, f32, i64 = ctypes.c_void_p, ctypes.c_int, ctypes.c_float, ctypes.c_longlong
    sigs = {
        "tllm_fp8_rows": [vp, i32, vp, vp, i32, i32, vp],
        "tllm_fp8_linear": [vp, vp, i32, vp, vp, vp, i32, i32, i32, i32, i32, i32, i32, vp, vp, vp],
        "tllm_fp8_gated": [vp, vp, i32, vp, vp, vp, vp, i32, i32, i32, i32, i32, i32, i32, f32, f32, vp, vp, vp],
        "tllm_add_rmsnorm_fp8": [vp, vp, i32, vp, i32, f32, vp, vp, i32, i32, vp],
        "tllm_fp8_weight": [vp, i32, vp, vp, i32, i32, i32, vp],
        "tllm_fp8_settle": [vp],
        "tllm_qk_norm_rope_store_fp8": [vp, vp, vp, i32, f32, vp, i32, vp, vp, vp, i32, i32, vp, vp, vp, i64, i32, i32, vp, i32, i32, i32, i32,
                                        i32, vp, vp],
        "tllm_attention_fp8_decode": [vp, vp, vp, vp, i64, i32, vp, vp, vp, i32, vp, i32, i32, i32, i32, i32, i32, i32, f32, i32, i32, vp, vp, vp],
        "tllm_attention_fp8_unpack": [vp, vp, vp, i64, i32, vp, i32, vp, i32, i32, i32, i32, i32, i32, i32, i32, vp, vp, vp],
    }
    for name, args in sigs.items():
        fn = getattr(h, name)
        fn.argtypes = args
        fn.restype = i32


def _blocks(n: int) -> int:
    return -(-n // BLOCK)


def _refuse(text: str):
    raise _ops().KernelError(text)


def _here(*tensors) -> None:
    """Contiguous CUDA tensors of the current device (the kernels go to its current stream)."""
    current = -2
    for t in tensors:
        if t is None:
            continue
        if not t.is_cuda or not t.is_contiguous():
            _refuse("kernels take contiguous CUDA tensors")
        if current == -2:
            current = _ops()._raw_device()
        if t.get_device() != current:
            _refuse(f"a tensor of {t.device}, the current device is cuda:{current}")


class Fp8Weight:
    """A weight [N, K] as e4m3 values ``q`` and float32 ``scales`` [ceil(N / 128), ceil(K / 128)].  ``gated``: the rows are N / 2 gate
    and N / 2 up rows interleaved by eight (``ops.interleave_gate_up``), and the scales [2 ceil(N / 2 / 128), ceil(K / 128)] are those
    of 128 gate rows, of the up rows that belong to them, and so on.  K is a multiple of 16.  Made on the stream that its tensors were
    written on; a kernel of this package that writes them later is followed by some other work before the next product."""
    __slots__ = ("_q", "_scales", "gated", "shape", "device", "index", "_at")

    def __init__(self, q: torch.Tensor, scales: torch.Tensor, gated: bool = False):
        if q.dtype != E4M3 or q.dim() != 2 or scales.dtype != torch.float32:
            _refuse(f"an 8-bit weight is a matrix of float8_e4m3fn with float32 scales, got {q.dtype} {tuple(q.shape)} and {scales.dtype}")
        n, k = q.shape
        if n == 0 or k == 0 or k % 16:
            _refuse(f"an 8-bit weight's columns are a multiple of 16, got {n} x {k}")
        if gated and n % 16:
            _refuse(f"interleaved gate and up rows come in sixteens, got {n}")
        want = (2 * _blocks(n // 2) if gated else _blocks(n), _blocks(k))
        if tuple(scales.shape) != want:
            _refuse(f"an 8-bit weight of {n} x {k} has scales {list(want)}, got {list(scales.shape)}")
        if q.device != scales.device or not q.is_contiguous() or not scales.is_contiguous() or q.data_ptr() % 16:
            _refuse("an 8-bit weight and its scales are contiguous on one device, the weight 16-byte aligned")
        self._q, self._scales, self.gated = q, scales, bool(gated)
        # what every product asks for, of the tensors as they have been checked
        self.shape, self.device, self.index = q.shape, q.device, q.get_device()
        self._at = (q.data_ptr(), scales.data_ptr())
        if q.is_cuda:                            # products fetch weights before the kernel ahead of them has ended: what wrote these has
            ops = _ops()
            with torch.cuda.device(q.device):
                ops._check(ops.lib().tllm_fp8_settle(ops._stream()), "fp8_settle")

    def __reduce__(self):                        # a copy has places of its own
        return Fp8Weight, (self._q, self._scales, self.gated)

    @property
    def pointers(self):
        """Where values and scales lie."""
        at = (self._q.data_ptr(), self._scales.data_ptr())
        if at != self._at:
            _refuse("the tensors of an 8-bit weight have been moved: make another weight of them")
        return at

    @property
    def q(self) -> torch.Tensor:
        return self._q

    @property
    def scales(self) -> torch.Tensor:
        return self._scales

    @property
    def dtype(self):
        return E4M3

    def values(self) -> torch.Tensor:
        """The float32 numbers that the weight stands for (for tests and comparisons)."""
        n, k = self.q.shape
        rows = torch.arange(n, device=self.q.device)
        if self.gated:
            rows = 2 * ((rows // 16 * 8) // BLOCK) + rows // 8 % 2
        else:
            rows = rows // BLOCK
        columns = torch.arange(k, device=self.q.device) // BLOCK
        return self.q.to(torch.float32) * self.scales[rows][:, columns]


class Fp8Rows:
    """Rows [T, K] as e4m3 values ``q`` and float32 ``scales`` [T, ceil(K / 128)]: what the products take.  Rows that a kernel makes
    lie in one buffer, the values first; ``q`` and ``scales`` are views of it."""
    __slots__ = ("shape", "index", "_q", "_scales", "_buffer", "_at")

    def __init__(self, q: torch.Tensor, scales: torch.Tensor):
        if q.dtype != E4M3 or q.dim() != 2 or scales.dtype != torch.float32 or tuple(scales.shape) != (q.shape[0], _blocks(q.shape[1])):
            _refuse(f"8-bit rows are a matrix of float8_e4m3fn with float32 scales [rows, columns / 128], got {q.dtype} {tuple(q.shape)}, "
                    f"{scales.dtype} {tuple(scales.shape)}")
        if q.shape[1] == 0 or q.shape[1] % 16:
            _refuse(f"8-bit rows have a multiple of 16 columns, got {q.shape[1]}")
        if q.device != scales.device or not q.is_contiguous() or not scales.is_contiguous() or q.data_ptr() % 16:
            _refuse("8-bit rows and their scales are contiguous on one device, the rows 16-byte aligned")
        self.shape, self._q, self._scales, self._buffer = q.shape, q, scales, None
        self._at, self.index = (q.data_ptr(), scales.data_ptr()), q.get_device()

    def __reduce__(self):                        # a copy has places of its own
        return Fp8Rows, (self.q, self.scales)

    @property
    def pointers(self):
        """Where values and scales lie."""
        if self._buffer is None and (self._q.data_ptr(), self._scales.data_ptr()) != self._at:
            _refuse("the tensors of 8-bit rows have been moved: make other rows of them")
        return self._at

    @property
    def q(self) -> torch.Tensor:
        if self._q is None:
            rows, k = self.shape
            self._q = self._buffer[:rows * k].view(E4M3).view(rows, k)
        return self._q

    @property
    def scales(self) -> torch.Tensor:
        if self._scales is None:
            rows, k = self.shape
            self._scales = self._buffer[rows * k:rows * k + 4 * rows * _blocks(k)].view(torch.float32).view(rows, _blocks(k))
        return self._scales

    @property
    def dtype(self):
        return E4M3

    @property
    def device(self):
        return (self._q if self._buffer is None else self._buffer).device

    def values(self) -> torch.Tensor:
        """The float32 numbers that the rows stand for (for tests and comparisons)."""
        columns = torch.arange(self.shape[1], device=self.device) // BLOCK
        return self.q.to(torch.float32) * self.scales[:, columns]


def _empty_rows(rows: int, k: int, device) -> Fp8Rows:
    made = Fp8Rows.__new__(Fp8Rows)              # right by construction
    made._buffer = buffer = torch.empty(rows * k + 4 * rows * -(-k // BLOCK), dtype=torch.uint8, device=device)
    at = buffer.data_ptr()
    made.shape, made._at, made.index, made._q, made._scales = (rows, k), (at, at + rows * k), buffer.get_device(), None, None
    return made


def _columns(k: int) -> None:
    if k == 0 or k % 16:
        _refuse(f"8-bit rows have a multiple of 16 columns, got {k}")


def quantize_weight_fp8(weight: torch.Tensor, gated: bool = False) -> Fp8Weight:
    """A bfloat16 or float32 weight [N, K] in 8 bits (K a multiple of 16); ``gated``: its rows are interleaved gate and up rows."""
    ops = _ops()
    _here(weight)
    if weight.dim() != 2 or weight.numel() == 0:
        _refuse(f"a weight is a matrix, got {tuple(weight.shape)}")
    n, k = weight.shape
    _columns(k)
    if gated and n % 16:
        _refuse(f"interleaved gate and up rows come in sixteens, got {n}")
    q = torch.empty((n, k), dtype=E4M3, device=weight.device)
    scales = torch.empty((2 * _blocks(n // 2) if gated else _blocks(n), _blocks(k)), dtype=torch.float32, device=weight.device)
    ops._check(ops.lib().tllm_fp8_weight(ops._p(weight), ops._dt(weight), ops._p(q), ops._p(scales), n, k, int(gated), ops._stream()), "fp8_weight")
    return Fp8Weight(q, scales, gated)


def quantize_rows_fp8(x: torch.Tensor) -> Fp8Rows:
    """Rows [T, K] (bfloat16 or float32, K a multiple of 16) in 8 bits."""
    ops = _ops()
    _here(x)
    if x.dim() != 2:
        _refuse(f"rows are a matrix, got {tuple(x.shape)}")
    _columns(x.shape[1])
    out = _empty_rows(x.shape[0], x.shape[1], x.device)
    ops._check(ops.lib().tllm_fp8_rows(ops._p(x), ops._dt(x), *out.pointers, x.shape[0], x.shape[1], ops._stream()), "fp8_rows")
    return out


def add_rmsnorm_fp8(h: torch.Tensor, delta: Optional[torch.Tensor], gain: torch.Tensor, eps: float) -> Fp8Rows:
    """``add_rmsnorm`` whose output rows come out in 8 bits, rounded from float32: h += delta (float32, written back), then
    gain * h / sqrt(mean(h^2) + eps).  Widths that are multiples of 16 up to 32768."""
    ops = _ops()
    _here(h, delta, gain)
    if h.dtype != torch.float32 or h.dim() != 2 or gain.numel() != h.shape[1] or (delta is not None and delta.shape != h.shape):
        _refuse(f"add_rmsnorm_fp8: stream {h.dtype} {tuple(h.shape)}, delta {None if delta is None else tuple(delta.shape)}, gain {tuple(gain.shape)}")
    _columns(h.shape[1])
    out = _empty_rows(h.shape[0], h.shape[1], h.device)
    ops._check(ops.lib().tllm_add_rmsnorm_fp8(ops._p(h), ops._p(delta), ops.BF16 if delta is None else ops._dt(delta), ops._p(gain), ops._dt(gain),
                                              float(eps), *out.pointers, h.shape[0], h.shape[1], ops._stream()),
               "add_rmsnorm_fp8")
    return out


SKINNY_ROWS = 8          # up to this many rows always the weight-streaming kernel,
SKINNY_WIDE_ROWS = 16    # and up to this many where it is ahead of the tensor cores' kernels
SKINNY_INSIDE_K = 4096   # up to this many columns it rounds eight bfloat16 rows itself
SKINNY, TILES, PAIRS = 0, 1, 2           # routes of csrc/fp8_product.cu
ROWS8, INSIDE = 2, 3                     # kinds of rows there, beside float32 and bfloat16


def _plan(rows: int, n: int, k: int, sms: int, gated: bool = False, to_float: bool = False):
    """(route, shares of K, blocks per share) of a product with ``n`` weight rows, by what the kernels take, in us.  Tiles of 128 x 128:
    4 and, for every round of tiles, 0.7 and 0.37 a block of K; more than one share, and gated products, leave float32 sums for another kernel:
    1 and their bytes twice at 8 TB/s.  Tiles of 256 x 256 by pairs of SMs: 3 and, a round, 1 and 0.47 a block.  Nine to sixteen rows by the
    weight-streaming kernel: 2.5 and the weight's bytes at 3 TB/s.  (Measured and by this rule, rows x columns x K: 61 x 4096 x 4096 in 4 shares 9.5
    and 9.7, in one 14.5 and 16.5, in 5 (two rounds) 12.3 and 12.8; 128 in 4 10.4 and 10.8, 17 in 4 9.2 and 8.9; 61 x 4096 x 12288 in 4 16.2 and
    15.6; 61 x 24576 x 4096 in one share 29 both; 300 x 4096 x 4096 tiles 14.9 and 16.5, pairs 18.0 and 19.0; 1200 x 4096 x 4096 pairs 33 and 35,
    tiles 40 and 42; 16 x 24576 x 4096 streaming 37 and 36, 16 x 4096 x 4096 8.0 both.)"""
    kb = _blocks(k)
    tiles = _blocks(rows) * _blocks(n)
    best = None
    for splits in range(1, max(1, min(16, kb // 2)) + 1):
        each = -(-kb // splits)
        used = -(-kb // each)
        us = 4 + -(-tiles * used // sms) * (0.7 + 0.37 * each)
        if used > 1 or gated or to_float:
            us += 1 + 8 * used * rows * n / 8e6
        if best is None or us < best[0]:
            best = (us, TILES, used, each)
    if not to_float:                             # pairs write bfloat16 or, gated, 8 bits
        us = 3 + -(-(-(-rows // 256) * -(-n // 256)) // (sms // 2)) * (1 + 0.47 * kb)
        if us < best[0]:
            best = (us, PAIRS, 1, kb)
    if rows <= SKINNY_WIDE_ROWS and 2.5 + n * k / 3e6 < best[0]:
        best = (0, SKINNY, 1, kb)
    return best[1:]


@functools.lru_cache(maxsize=8192)
def _call(rows: int, n: int, k: int, kind: int, gated: bool, to_float: bool, sms: int):
    """(kind of rows, route, shares, blocks per share, bytes of scratch, kernels) of a product."""
    if rows <= SKINNY_ROWS:
        route, splits, each = SKINNY, 1, _blocks(k)
        if kind == 1 and rows <= 8 and k <= SKINNY_INSIDE_K:
            kind = INSIDE
    else:
        route, splits, each = _plan(rows, n, k, sms, gated, to_float)
    scratch = 0 if kind in (ROWS8, INSIDE) else rows * k + -(-4 * rows * _blocks(k) // 16) * 16
    kernels = 1 + (kind not in (ROWS8, INSIDE))
    if gated:
        if route != PAIRS:
            scratch += 4 * rows * (n // 2 if route == SKINNY else splits * n)
            kernels += 1
    elif route == TILES and (splits > 1 or to_float):
        scratch += 4 * splits * rows * n
        kernels += 1
    return kind, route, splits, each, scratch, kernels


def _rows_and_weight(x, weight: Fp8Weight):
    """(rows, columns, kind, values, scales) of rows that may meet the weight."""
    ops = _ops()
    if type(x) is Fp8Rows:
        kind, (values, scales), index = ROWS8, x.pointers, x.index
    else:
        if not x.is_cuda or not x.is_contiguous():
            _refuse("kernels take contiguous CUDA tensors")
        kind = ops._DT.get(x.dtype)
        if kind is None or x.dim() != 2:
            _refuse(f"a product with an 8-bit weight takes rows in bfloat16, float32 or 8 bits, got {x.dtype} {tuple(x.shape)}")
        values, scales, index = x.data_ptr(), None, x.get_device()
        if values % 16:
            _refuse("rows must be 16-byte aligned")
    current = ops._raw_device()
    if index != current or weight.index != current:
        _refuse(f"rows of cuda:{index}, a weight of {weight.device}, the current device is cuda:{current}")
    rows, k = x.shape
    if k != weight.shape[1]:
        _refuse(f"rows of {k} columns, a weight of {weight.shape[1]}")
    return rows, k, kind, values, scales


def linear_fp8(x, weight: Fp8Weight, out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """y[T, N] = x . weight^T: ``x`` bfloat16, float32 (both rounded to 8 bits per 128 columns) or ``Fp8Rows``; bfloat16 or float32 out
    (default: x's type, bfloat16 for 8-bit rows)."""
    ops = _ops()
    rows, k, kind, values, scales = _rows_and_weight(x, weight)
    if weight.gated:
        _refuse("a gated weight belongs to linear_swiglu")
    want = out_dtype or (torch.bfloat16 if kind == ROWS8 else x.dtype)
    code = ops._DT.get(want)
    if code is None:
        _refuse(f"unsupported dtype {want}")
    n, device = weight.shape[0], weight.device
    y = torch.empty((rows, n), dtype=want, device=device)
    if rows == 0:
        return y
    kind, route, splits, each, size, kernels = _call(rows, n, k, kind, False, code == 0, ops.SM_COUNT)
    scratch = torch.empty(size, dtype=torch.uint8, device=device) if size else None
    word = None
    if route != SKINNY:
        word = ops.error_word(device).data_ptr()
        ops.tcgen05_calls += 1
    ops._check(ops.lib().tllm_fp8_linear(values, scales, kind, *weight.pointers, y.data_ptr(), code, rows, n, k, route, splits, each,
                                         scratch.data_ptr() if size else None, word, ops._stream()), "fp8_linear", kernels)
    return y


def linear_swiglu_fp8(x, weight: Fp8Weight, act: str = "silu", consts=None) -> Fp8Rows:
    """act(x . Wg^T) * (x . Wu^T) for a gated 8-bit weight, as 8-bit rows for the product that follows, rounded from float32."""
    ops = _ops()
    rows, k, kind, values, scales = _rows_and_weight(x, weight)
    if not weight.gated:
        _refuse("linear_swiglu takes a gated 8-bit weight (gate and up rows interleaved by eight)")
    n, device = weight.shape[0], weight.device
    inter = n // 2
    _columns(inter)
    limit, slope = ops._consts(act, consts)
    out = _empty_rows(rows, inter, device)
    if rows == 0:
        return out
    kind, route, splits, each, size, kernels = _call(rows, n, k, kind, True, False, ops.SM_COUNT)
    scratch = torch.empty(size, dtype=torch.uint8, device=device) if size else None
    word = None
    if route != SKINNY:
        word = ops.error_word(device).data_ptr()
        ops.tcgen05_calls += 1
    ops._check(ops.lib().tllm_fp8_gated(values, scales, kind, *weight.pointers, *out.pointers, rows, inter, k, route, splits, each, ops.ACTIVATIONS[act],
                                        limit, slope, scratch.data_ptr() if size else None, word, ops._stream()), "fp8_gated", kernels)
    return out


# --------------------------------------------------------------------------- the cache
SCALE_BYTES = 8          # per token and head: the key's float32 scale, the value's


def cache_planes(kv_heads: int, head_dim: int):
    """The planes (heads, bytes) of an 8-bit cache of keys and values: e4m3 keys, e4m3 values, pairs of float32 scales."""
    return ((kv_heads, head_dim), (kv_heads, head_dim), (kv_heads, SCALE_BYTES))


def cache_takes(page_size: int, q_heads: int, kv_heads: int, head_dim: int) -> bool:
    """Whether the kernels of the 8-bit cache take these sizes."""
    return head_dim in (64, 128) and page_size % 16 == 0 and q_heads % kv_heads == 0 and q_heads // kv_heads <= 16


def _planes(planes, page_size: int, kv_heads: int, head_dim: int):
    """(keys, values, scales, bytes from page to page, pages) of an 8-bit cache's planes, checked."""
    if len(planes) != 3:
        _refuse(f"an 8-bit cache has planes of keys, values and scales, got {len(planes)}")
    k, v, s = planes
    apart, pages, current = k.stride(0), k.shape[0], _ops()._raw_device()
    for plane, width in ((k, head_dim), (v, head_dim), (s, SCALE_BYTES)):
        if not plane.is_cuda or plane.dtype is not torch.uint8 or plane.shape != (pages, kv_heads, page_size, width):
            _refuse(f"an 8-bit cache's plane is uint8 [pages, {kv_heads}, {page_size}, {width}], got {plane.dtype} {tuple(plane.shape)}")
        if plane.stride() != (apart, page_size * width, width, 1):
            _refuse("an 8-bit cache's planes are dense within a page and equally far apart")
        if plane.get_device() != current:
            _refuse(f"a tensor of {plane.device}, the current device is cuda:{current}")
    return k.data_ptr(), v.data_ptr(), s.data_ptr(), apart, pages


def _int32(what: str, *tensors) -> None:
    for t in tensors:
        if t is not None and t.dtype != torch.int32:
            _refuse(f"{what}: positions, slots, rows and block tables are int32, got {t.dtype}")


def qk_norm_rope_store_fp8(qkv: torch.Tensor, q_gain, k_gain, eps: float, inv_freq, rotary_dim: int, positions: torch.Tensor,
                           token_slot: torch.Tensor, block_table, planes, page_size: int, q_out, q_heads: int, kv_heads: int, head_dim: int,
                           flags: int, table: Optional[torch.Tensor] = None) -> None:
    """``qk_norm_rope_store`` into an 8-bit cache: ``planes`` = (keys, values, scales), ``cache_planes``.  bfloat16 rows, head widths 64 and
    128, the whole head rotated or nothing.  What belongs to no slot, position or page that the table and the cache have is not stored."""
    ops = _ops()
    _here(qkv, q_gain, k_gain, inv_freq, positions, token_slot, block_table, q_out, table)
    _int32("qk_norm_rope_store_fp8", positions, token_slot, block_table)
    tokens = qkv.shape[0]
    if qkv.dtype != torch.bfloat16 or qkv.dim() != 2 or qkv.shape[1] != (q_heads + 2 * kv_heads) * head_dim:
        _refuse(f"qk_norm_rope_store_fp8: rows of {(q_heads + 2 * kv_heads) * head_dim} bfloat16 numbers, got {qkv.dtype} {tuple(qkv.shape)}")
    if positions.numel() < tokens or token_slot.numel() < tokens:
        _refuse("qk_norm_rope_store_fp8: a position and a slot for every row")
    if table is not None and (table.dtype != torch.float32 or tuple(table.shape) != (tokens, 2, rotary_dim // 2)):
        _refuse(f"qk_norm_rope_store_fp8: rotary table {table.dtype} {tuple(table.shape)}")
    if inv_freq is not None and (inv_freq.dtype != torch.float32 or inv_freq.numel() != rotary_dim // 2):
        _refuse("qk_norm_rope_store_fp8: a float32 frequency per rotated pair")
    for gain in (q_gain, k_gain):
        if gain is not None and gain.numel() != head_dim:
            _refuse(f"qk_norm_rope_store_fp8: gains of {head_dim} numbers, got {gain.numel()}")
    if q_gain is not None and k_gain is not None and q_gain.dtype != k_gain.dtype:
        _refuse("qk_norm_rope_store_fp8: gains of one type")
    if q_out is not None and (q_out.dtype != torch.bfloat16 or tuple(q_out.shape) != (tokens, q_heads * head_dim)):
        _refuse(f"qk_norm_rope_store_fp8: queries go to bfloat16 [{tokens}, {q_heads * head_dim}], got {q_out.dtype} {tuple(q_out.shape)}")
    k, v, s, stride, held = _planes(planes, page_size, kv_heads, head_dim) if planes is not None else (None, None, None, 0, 0)
    if tokens == 0:
        return
    ops._check(ops.lib().tllm_qk_norm_rope_store_fp8(
        ops._p(qkv), ops._p(q_gain), ops._p(k_gain), ops._dt(q_gain) if q_gain is not None else ops.F32, float(eps), ops._p(inv_freq), rotary_dim,
        ops._p(positions), ops._p(token_slot), ops._p(block_table),
        *(block_table.shape if block_table is not None else (0, 0)), k, v, s, stride, held, page_size, ops._p(q_out), tokens, q_heads, kv_heads, head_dim, flags, ops._p(table), ops._stream()), "qk_norm_rope_store_fp8")


def _attention_operands(what, q, out, positions, token_slot, rows, n_rows, block_table, q_heads, kv_heads, head_dim) -> None:
    _here(q, out, positions, token_slot, rows, block_table)
    if not positions.dtype is token_slot.dtype is block_table.dtype is torch.int32 or (rows is not None and rows.dtype is not torch.int32):
        _refuse(f"{what}: positions, slots, rows and block tables are int32")
    shape = q.shape
    if q.dtype is not torch.bfloat16 or out.dtype is not torch.bfloat16 or len(shape) != 2 or shape[1] != q_heads * head_dim or out.shape != shape:
        _refuse(f"{what}: queries and outputs are bfloat16 [rows, {q_heads * head_dim}], got {q.dtype} {tuple(shape)} and {out.dtype} {tuple(out.shape)}")
    if n_rows > (shape[0] if rows is None else rows.numel()) or positions.numel() < shape[0] or token_slot.numel() < shape[0]:
        _refuse(f"{what}: {n_rows} rows of {shape[0]}, a position and a slot for each")


SHARED_ROWS = 512        # rows that may share blocks


@functools.lru_cache(maxsize=8192)
def attention_cut(rows: int, kv_heads: int, group: int, reach: int, sms: int):
    """(blocks that share all rows' keys, blocks of a cluster) for ``paged_attention_decode_fp8``: (0, 1) for one block per (row, key/value head),
    (0, 2 to 8) for a cluster of them, (as many as are resident, 1) for shares and a second kernel that adds them; whichever should take least,
    in us, for rows of at most ``reach`` keys.  The lengths are on the device: rows are taken to hold 0.65 of the longest on average, and heads to be 128 wide.
    A block of its own: 4.1, and 0.9 for every 128 keys, up to 1.4 times that where
    SMs have several, or what HBM takes for all keys.  A cluster: 5.4, 1 for every 100 blocks, and 0.95 to 1.3 for every 128 keys of a block.  Shares: 12, and 2.4
    for every 32 keys that a warp gets.
    Measured, us, own block, best cluster, shares, rows x heads of 128, rows between a quarter of the longest and all of it: 1 x 8, 1000 11.3, 6.7, 10.1;
    1 x 8, 4095 34, 10.7, 13.1; 1 x 8, 16384 117, 21.6, 18.6; 8 x 8, 1000 12.9, 10.4, 14.5; 8 x 8, 4095 34, 17.4, 19.8; 16 x 8, 4095 34, 26.7, 26.8; 24 x 8, 4096 43,
    35, 35; 37 x 8, 4096 47, -, 49; 64 x 8, 4096 62, -, 72; 128 x 8, 4096 122, -, 125; 64 x 8 of 64, 4096 40, -, 48.
    Rows all of one length, for which the rule is not always right: 8 x 8, 4095 34, 18.4, 23; 16 x 8, 4095 35, 29, 34 (it takes shares);
    24 x 8, 4096 45, 41, 46; 37 x 8, 4096 53, -, 61; 64 x 8, 4096 119, -, 99 (a block each, in two waves); 128 x 8, 4096 187, -, 182; 64 x 8 of 64, 4096 68, -, 58."""
    if rows == 0:
        return 0, 1
    pairs, mean = rows * kv_heads, 0.65 + 0.35 / rows
    resident = (3 if group <= 8 else 2) * sms
    best = (4.1 + max(0.9 * -(-reach // 128) * min(1.4, 1 + pairs / 1000), 2.93e-5 * pairs * reach), 0, 1)
    for size in (2, 4, 8):
        if pairs * size <= 2.6 * sms:
            best = min(best, (5.4 + pairs * size / 100 + 0.95 * -(-reach // (128 * size)) * (1 + pairs * size / 1000), 0, size))
    if rows <= SHARED_ROWS:
        best = min(best, (12 + 2.4 * max(1.0, mean * pairs * reach / 32 / (4 * resident)), resident, 1))
    return best[1:]


def paged_attention_decode_fp8(q, planes, positions, token_slot, rows, n_rows, block_table, page_size, q_heads, kv_heads, head_dim, window, scale,
                               out, max_context, blocks=None, cluster=None):
    """Attention of one-token rows (``rows``: their indices, None for the first ``n_rows``) over an 8-bit paged cache, ``planes`` =
    (keys, values, scales): positions max(0, pos - window + 1) .. pos of the row's own request.  One block of threads takes a
    (row, key/value head), with ``cluster`` = 2, 4 or 8 that many together; with ``blocks`` (at most 512, for at most 512 rows) so many
    share all rows' keys, and a second kernel adds the pieces of a row in their order (neither given: ``attention_cut``).  Rows of no
    request (a negative slot, or none of the table's; a negative position) become zeros, and so do rows without a key; what no page of
    the cache holds does not count, and a position behind the table's room is held within it.  Scales are zero or more; a value whose scale
    is zero counts with its key's weight.  Rows of ``out`` that are not asked for
    stay as they are.  ``max_context``: no row's position is at or behind it (what is taken goes by it)."""
    ops = _ops()
    _attention_operands("paged_attention_decode_fp8", q, out, positions, token_slot, rows, n_rows, block_table, q_heads, kv_heads, head_dim)
    k, v, s, stride, held = _planes(planes, page_size, kv_heads, head_dim)
    max_pages = block_table.shape[1]
    if n_rows == 0:
        return out
    if blocks is None and cluster is None:
        reach = min(max_context, max_pages * page_size)
        blocks, cluster = attention_cut(n_rows, kv_heads, q_heads // kv_heads, min(reach, window) if window else reach, ops.SM_COUNT)
    blocks, cluster = blocks or 0, cluster or 1
    scratch = None
    if blocks:
        scratch = q.new_empty((n_rows * kv_heads + blocks) * (q_heads // kv_heads) * (head_dim + 3) + n_rows + 2, dtype=torch.float32)
    ops._check(ops.lib().tllm_attention_fp8_decode(
        q.data_ptr(), k, v, s, stride, held, positions.data_ptr(), token_slot.data_ptr(), None if rows is None else rows.data_ptr(), n_rows,
        block_table.data_ptr(), block_table.shape[0], max_pages, page_size, q_heads, kv_heads, head_dim, window or 0, scale, blocks, cluster,
        None if scratch is None else scratch.data_ptr(), out.data_ptr(), ops._stream()), "paged_attention_decode_fp8", 2 if blocks else 1)
    return out


def portion_pages(ctx, page_size: int, window: Optional[int], most: int, capturing: bool = False):
    """(pages of the portion that has most, pages of all portions) that a step's portions may read, none more than ``most``.  A step that
    is being captured is replayed with other portions of as many tokens: room for the most."""
    counts = [1]
    for s in ctx.segments:
        if s.length > 1:
            first = max(0, s.pos0 - window + 1) if window else 0
            counts.append((s.pos0 + s.length - 1) // page_size - first // page_size + 1)
    if capturing:
        return most, most * max(1, len(counts) - 1)
    return max(counts), max(1, sum(counts) - 1)


def paged_attention_fp8(q, planes, positions, token_slot, block_table, page_size, q_heads, kv_heads, head_dim, window, scale, out, ctx=None):
    """``paged_attention`` over an 8-bit paged cache: one-token rows on ``paged_attention_decode_fp8``; the pages of longer segments are
    brought back to bfloat16 in scratch, at most as many as the cache has, which the prompt kernels read: there a key or value is rounded once more,
    after its scale.  Every page that a portion sees is held, as ``paged_attention`` has it: the prompt kernels read a missing one as zeros, where one-token
    rows leave its keys out.  Without a context every row is a one-token row."""
    ops = _ops()
    tokens = q.shape[0]
    if ctx is None or ctx.pf_tiles is None or ctx.tokens != tokens:
        return paged_attention_decode_fp8(q, planes, positions, token_slot, None, tokens, block_table, page_size, q_heads, kv_heads, head_dim, window, scale,
                                          out, block_table.shape[1] * page_size)
    if ctx.n_dec:
        paged_attention_decode_fp8(q, planes, positions, token_slot, ctx.dec_rows, ctx.n_dec, block_table, page_size, q_heads, kv_heads, head_dim,
                                   window, scale, out, ctx.max_context)
    if ctx.n_tiles:
        _attention_operands("paged_attention_fp8", q, out, positions, token_slot, None, tokens, block_table, q_heads, kv_heads, head_dim)
        k, v, s, stride, held = _planes(planes, page_size, kv_heads, head_dim)
        segments, most = ctx.seg_info.shape[0], min(-(-ctx.max_context // page_size), block_table.shape[1])
        per, capacity = portion_pages(ctx, page_size, window, most, torch.cuda.is_current_stream_capturing())
        by_page = capacity > held                # portions that share pages: the places of the cache's own
        capacity = min(capacity, held)
        pages = torch.empty((capacity, 2, kv_heads, page_size, head_dim), dtype=torch.bfloat16, device=q.device)
        table = torch.empty_like(block_table)
        ops._check(ops.lib().tllm_attention_fp8_unpack(k, v, s, stride, held, ops._p(ctx.seg_info), segments, ops._p(block_table), block_table.shape[1], page_size,
                                                       kv_heads, head_dim, int(window or 0), per, capacity, int(by_page), ops._p(pages), ops._p(table), ops._stream()),
                   "attention_fp8_unpack", 2 if by_page else 1)
        ops._attention_tiles(q, pages, table, page_size, q_heads, kv_heads, head_dim, window, scale, out, ctx)
    return out
