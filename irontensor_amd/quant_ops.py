"""Serving in 8 and 4 bits, on the MI355X C ABI: a quantised key/value cache, the attention that reads it,
and the linear layer on an 8-bit weight. No counterpart in the reference, whose inference
(src/inference) recomputes the whole prompt for every token.

A decoding step: project (linear_i8), rotate (rope), kv_cache_write the new token, cached_attention,
project. Every op launches hand-written HIP through libirontensor_hip.so; there is no fallback. With `out`
tensors and positions that are on the device (upload_positions) no call synchronises or allocates, so a step
can be captured into a graph after it has run once.
"""
from __future__ import annotations

import ctypes as C
import math
from typing import Optional, Sequence, Tuple, Union

import numpy as np

from . import _lib
from .errors import InnerDimensionMismatch, InvalidValue, Panic, PrecisionMismatch, ShapeMismatch, UnsupportedDimensions, check
from .tensor import Context, Precision, Tensor, _Buffer

_P = Precision


class Positions:
    """int32 words on the device, one for each sequence (upload_positions); `write` replaces them, stream-ordered,
    at the same address, so a captured step reads the new ones at its next replay."""

    __slots__ = ("_buf", "size")

    def __init__(self, values, ctx: Optional[Context] = None):
        v = _host_i32(values, "positions")
        self.size = v.size
        self._buf = _Buffer(ctx or Context.global_(), 4 * v.size)
        self.write(v)

    @property
    def ptr(self) -> int:
        return self._buf.ptr

    @property
    def ctx(self) -> Context:
        return self._buf.ctx

    def write(self, values) -> None:
        v = _host_i32(values, "positions")
        if v.size != self.size:
            raise ShapeMismatch("positions", str([self.size]), str([v.size]))
        if v.size:
            check(self.ctx.lib.it_memcpy_h2d(self.ctx.handle, C.c_void_p(self.ptr), v.ctypes.data_as(C.c_void_p),
                                             v.nbytes), "positions")

    def numpy(self) -> np.ndarray:
        v = np.empty(self.size, np.int32)
        if v.size:
            check(self.ctx.lib.it_memcpy_d2h(self.ctx.handle, v.ctypes.data_as(C.c_void_p), C.c_void_p(self.ptr),
                                             v.nbytes), "positions")
        return v


def _host_i32(values, what: str) -> np.ndarray:
    v = np.asarray(values)
    if v.size and v.dtype.kind not in "iu":
        raise InvalidValue(what, f"expected integers, got {v.dtype}")
    v = v.astype(np.int64).ravel()
    if v.size and (v.min() < -2 ** 31 or v.max() >= 2 ** 31):
        raise InvalidValue(what, "a value does not fit 32 bits")
    return np.ascontiguousarray(v, dtype=np.int32)


def upload_positions(values, ctx: Optional[Context] = None) -> Positions:
    """Device copy of one int32 per sequence: the `start` (or `count`) of the cache operations."""
    return Positions(values, ctx)


class KvCache:
    """Keys and values of up to `capacity` tokens of `batch` sequences with `kv_heads` heads of 64, 128 or 256
    channels, in 4 or 8 bits (it_kv_cache). Starts as zeros. `bytes` is its size on the device."""

    def __init__(self, batch: int, kv_heads: int, capacity: int, head_dim: int, bits: int = 4,
                 ctx: Optional[Context] = None):
        size = C.c_size_t()
        check(_lib.load().it_kv_cache_bytes(int(bits), int(batch), int(kv_heads), int(capacity), int(head_dim),
                                            C.byref(size)), "kv_cache")
        self.batch, self.kv_heads, self.capacity = int(batch), int(kv_heads), int(capacity)
        self.head_dim, self.bits, self.bytes = int(head_dim), int(bits), int(size.value)
        self.ctx = ctx or Context.global_()
        self._buf = _Buffer(self.ctx, self.bytes)
        self._desc = _lib.KvCacheDesc(self.bits, self.batch, self.kv_heads, self.capacity, self.head_dim, self._buf.ptr)
        self._ref = C.byref(self._desc)
        self.clear()

    def clear(self) -> None:
        """Every position reads as zeros again."""
        if self.bytes:
            check(self.ctx.lib.it_zero(self.ctx.handle, C.c_void_p(self._buf.ptr), self.bytes), "kv_cache")


def _bshd(t: Tensor, what: str, op: str) -> list:
    s = t.shape()
    if len(s) != 4:
        raise UnsupportedDimensions(op, f"4D {what} [batch, seq, heads, dim]", s)
    if t.precision() not in (_P.FP32, _P.BF16):
        raise PrecisionMismatch(op, "FP32 or BF16", t.precision().name)
    return s


def _same_ctx(op: str, ctx: Context, *things) -> None:
    for t in things:
        if t is not None and t.ctx is not ctx:
            raise InvalidValue(op, "a tensor belongs to another context")


def _checked(op: str, what: str, cache: KvCache, v, low: int, high: int):
    """Positions as they are; host integers as an int32 array within [low, high]."""
    if v is None:
        return None
    if not isinstance(v, Positions):
        v = _host_i32(v, op)
        if v.size and (v.min() < low or v.max() > high):
            raise InvalidValue(op, f"{what} must be in [{low}, {high}], got {v.tolist()}")
    if v.size != cache.batch:
        raise ShapeMismatch(op, f"{what} of {cache.batch} sequences", f"{v.size}")
    return v


def _start_count(op: str, cache: KvCache, n: int, start, count) -> Tuple[Positions, Optional[Positions]]:
    """Both on the device. A host start has to leave room for the tokens: n, or the host's counts (what device
    Positions hold is the kernel's to check)."""
    count = _checked(op, "count", cache, count, 0, n)
    start = _checked(op, "start", cache, start, 0, cache.capacity if count is not None else cache.capacity - n)
    if isinstance(start, np.ndarray) and isinstance(count, np.ndarray):
        if start.size and int((start.astype(np.int64) + count).max()) > cache.capacity:
            raise InvalidValue(op, f"start + count passes the capacity {cache.capacity}")
    up = lambda v: Positions(v, cache.ctx) if isinstance(v, np.ndarray) else v  # noqa: E731
    return up(start), up(count)


def _ptr(t) -> Optional[int]:
    return t.ptr if t is not None else None


def kv_cache_write(cache: KvCache, k: Tensor, v: Tensor, start: Union[Positions, Sequence[int]],
                   count: Union[Positions, Sequence[int], None] = None) -> None:
    """Quantises k and v [batch, n, kv_heads, head_dim] (FP32 or BF16) into positions start[b] .. of the cache;
    of sequence b the first count[b] tokens (default all n). Host integers are checked against the
    capacity; with device Positions a token outside it is not written."""
    op = "kv_cache_write"
    ks = _bshd(k, "K", op)
    if v.shape() != ks:
        raise ShapeMismatch(op, str(ks), str(v.shape()))
    if v.precision() is not k.precision():
        raise PrecisionMismatch(op, k.precision().name, v.precision().name)
    b, n, h, d = ks
    if (b, h, d) != (cache.batch, cache.kv_heads, cache.head_dim):
        raise ShapeMismatch(op, f"[{cache.batch}, n, {cache.kv_heads}, {cache.head_dim}]", str(ks))
    start, count = _start_count(op, cache, n, start, count)
    _same_ctx(op, cache.ctx, k, v, start, count)
    lay = _lib.AttnLayout(h, n * h * d, d, h * d)
    check(cache.ctx.lib.it_kv_cache_write(cache.ctx.handle, int(k.precision()), cache._ref, n, C.byref(lay), k.ptr, v.ptr,
                                          start.ptr, _ptr(count)), op)


def kv_cache_read(cache: KvCache, begin: int, n: int, precision: Precision = _P.FP32, *,
                  out: Optional[Sequence[Tensor]] = None) -> Tuple[Tensor, Tensor]:
    """(K, V) [batch, n, kv_heads, head_dim]: what positions begin .. begin + n - 1 of every sequence stand for, in
    `precision`, or into the pair `out` in theirs."""
    op = "kv_cache_read"
    shape = [cache.batch, n, cache.kv_heads, cache.head_dim]
    if out is None:
        if n < 0:
            raise InvalidValue(op, "negative size")
        out = (Tensor.empty(shape, precision, cache.ctx), Tensor.empty(shape, precision, cache.ctx))
    k, v = out
    for t in (k, v):
        _bshd(t, "output", op)
        if t.shape() != shape:
            raise ShapeMismatch(op, str(shape), str(t.shape()))
    if v.precision() is not k.precision():
        raise PrecisionMismatch(op, k.precision().name, v.precision().name)
    _same_ctx(op, cache.ctx, k, v)
    h, d = cache.kv_heads, cache.head_dim
    lay = _lib.AttnLayout(max(h, 1), n * h * d, d, max(h * d, d))
    check(cache.ctx.lib.it_kv_cache_read(cache.ctx.handle, int(k.precision()), cache._ref, begin, n, C.byref(lay), k.ptr,
                                         v.ptr), op)
    return k, v


def cached_attention(q: Tensor, cache: KvCache, start: Union[Positions, Sequence[int]],
                     count: Union[Positions, Sequence[int], None] = None, scale: Optional[float] = None, *,
                     out: Optional[Tensor] = None) -> Tensor:
    """softmax(scale Q.K^T).V of q [batch, n, heads, head_dim] (FP32 or BF16) over the cache: query i of sequence b
    stands at position start[b] + i and sees the positions up to its own, whose tokens kv_cache_write has put
    there. heads is a multiple of the cache's heads. Queries at count[b] and beyond give zeros. scale: default
    1 / sqrt(head_dim). `out` may be q itself."""
    op = "cached_attention"
    qs = _bshd(q, "Q", op)
    b, n, h, d = qs
    if b != cache.batch or d != cache.head_dim:
        raise ShapeMismatch(op, f"[{cache.batch}, n, heads, {cache.head_dim}]", str(qs))
    if out is None:
        out = Tensor.empty(qs, q.precision(), q.ctx)
    elif out.shape() != qs:
        raise ShapeMismatch(op, str(qs), str(out.shape()))
    elif out.precision() is not q.precision():
        raise PrecisionMismatch(op, q.precision().name, out.precision().name)
    start, count = _start_count(op, cache, n, start, count)
    _same_ctx(op, cache.ctx, q, out, start, count)
    lay = _lib.AttnLayout(max(h, 1), n * h * d, d, max(h * d, d))
    check(cache.ctx.lib.it_cached_attention(cache.ctx.handle, int(q.precision()), cache._ref, h, n,
                                            1.0 / math.sqrt(d) if scale is None else float(scale), C.byref(lay), None,
                                            q.ptr, start.ptr, _ptr(count), out.ptr), op)
    return out


class Int8Matrix:
    """A matrix [rows, cols] in 8-bit codes with an FP32 step for each row (quantize_i8): a weight with a step per
    output channel, or activations with one per token. Rows are padded with zeros to a multiple of 128."""

    def __init__(self, rows: int, cols: int, ctx: Context):
        self.rows, self.cols, self.ld = int(rows), int(cols), (int(cols) + 127) // 128 * 128
        self.ctx = ctx
        self._codes = _Buffer(ctx, self.rows * self.ld)
        self.steps = Tensor.empty([self.rows], _P.FP32, ctx)

    @property
    def ptr(self) -> int:
        return self._codes.ptr

    def shape(self) -> list:
        return [self.rows, self.cols]

    def codes(self) -> np.ndarray:
        """Host copy of the codes, int8 [rows, cols]."""
        c = np.empty([self.rows, self.ld], np.int8)
        if c.size:
            check(self.ctx.lib.it_memcpy_d2h(self.ctx.handle, c.ctypes.data_as(C.c_void_p), C.c_void_p(self.ptr),
                                             c.nbytes), "codes")
        return c[:, :self.cols]


def quantize_i8(x: Tensor) -> Int8Matrix:
    """x [rows, cols] (FP32 or BF16) as 8-bit codes with a step per row, max|row| * (1 / 127)."""
    op = "quantize_i8"
    if len(x.shape()) != 2:
        raise UnsupportedDimensions(op, "a 2D tensor", x.shape())
    if x.precision() not in (_P.FP32, _P.BF16):
        raise PrecisionMismatch(op, "FP32 or BF16", x.precision().name)
    m = Int8Matrix(*x.shape(), x.ctx)
    check(x.ctx.lib.it_quantize_i8(x.ctx.handle, int(x.precision()), m.rows, m.cols, x.ptr, m.cols, m.ptr, m.ld,
                                   m.steps.ptr), op)
    return m


def _check_bias(op: str, bias: Optional[Tensor], n: int) -> None:
    if bias is None:
        return
    if bias.precision() is not _P.FP32:
        raise PrecisionMismatch(op, "FP32 bias", bias.precision().name)
    if bias.numel() != n:
        raise ShapeMismatch(op, f"bias of {n} elements", str(bias.shape()))


def _check_out(op: str, out: Optional[Tensor], shape: list, precision: Precision, ctx: Context) -> Tensor:
    if out is None:
        return Tensor.empty(shape, precision, ctx)
    if out.shape() != shape:
        raise ShapeMismatch(op, str(shape), str(out.shape()))
    if out.precision() is not precision:
        raise PrecisionMismatch(op, precision.name, out.precision().name)
    return out


def matmul_i8(a: Int8Matrix, b: Int8Matrix, bias: Optional[Tensor] = None, out_precision: Precision = _P.FP32, *,
              out: Optional[Tensor] = None) -> Tensor:
    """a.b^T of the values the two stand for, a [M, K] and b [N, K], plus an FP32 bias [N]: exact 32-bit sums of the
    codes' products, times the row's and the column's step."""
    op = "matmul_i8"
    if a.cols != b.cols:
        raise InnerDimensionMismatch(op, a.shape(), b.shape())
    _check_bias(op, bias, b.rows)
    out = _check_out(op, out, [a.rows, b.rows], out_precision if out is None else out.precision(), a.ctx)
    _same_ctx(op, a.ctx, b, bias, out)
    check(a.ctx.lib.it_gemm_i8(a.ctx.handle, int(out.precision()), a.rows, b.rows, a.ld, a.ptr, a.ld, a.steps.ptr, b.ptr,
                               b.ld, b.steps.ptr, _ptr(bias), out.ptr, b.rows), op)
    return out


def linear_i8(x: Tensor, weight: Int8Matrix, bias: Optional[Tensor] = None, *, out: Optional[Tensor] = None) -> Tensor:
    """linear (src/nn/linear.rs:87-145) on an 8-bit weight: x [.., in] (FP32 or BF16) quantised per token, times
    weight^T, plus an FP32 bias, in x's precision. `out` may be x itself."""
    op = "linear_i8"
    shape = x.shape()
    if not shape:
        raise Panic("Input must have at least one dimension")
    if shape[-1] != weight.cols:
        raise InnerDimensionMismatch(op, shape, weight.shape())
    if x.precision() not in (_P.FP32, _P.BF16):
        raise PrecisionMismatch(op, "FP32 or BF16", x.precision().name)
    _check_bias(op, bias, weight.rows)
    out = _check_out(op, out, shape[:-1] + [weight.rows], x.precision(), x.ctx)
    _same_ctx(op, x.ctx, weight, bias, out)
    rows = math.prod(shape[:-1])
    check(x.ctx.lib.it_linear_i8(x.ctx.handle, int(x.precision()), rows, weight.rows, weight.cols, x.ptr, weight.cols,
                                 weight.ptr, weight.ld, weight.steps.ptr, _ptr(bias), out.ptr, weight.rows), op)
    return out


class LinearI8:
    """Linear (src/nn/linear.rs:20-86) with its weight quantised once, for inference."""

    def __init__(self, weight: Int8Matrix, bias: Optional[Tensor] = None):
        _check_bias("linear_i8", bias, weight.rows)
        self.weight, self.bias = weight, bias
        self.out_features, self.in_features = weight.shape()

    @staticmethod
    def from_weight(weight: Tensor, bias: Optional[Tensor] = None) -> "LinearI8":
        """From a [out, in] FP32 or BF16 weight."""
        return LinearI8(quantize_i8(weight), bias)

    def forward(self, input: Tensor, *, out: Optional[Tensor] = None) -> Tensor:
        return linear_i8(input, self.weight, self.bias, out=out)
