"""What the quantised serving operators refuse, on the CPU: through the C ABI before the context is used, and in the
Python mirror before anything reaches the library."""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

from irontensor_amd import _lib
from irontensor_amd.tensor import Precision, Tensor

CTX = C.c_void_p(C.addressof(C.create_string_buffer(4096)))  # never read: every call here is refused first


def _desc(bits=4, batch=2, kv_heads=2, capacity=10, head_dim=64, data=256):
    return _lib.KvCacheDesc(bits, batch, kv_heads, capacity, head_dim, data)


def _write(desc=None, ctx=CTX, dtype=0, n=3, lay=None, k=256, v=256, start=256):
    return _lib.load().it_kv_cache_write(ctx, dtype, C.byref(desc or _desc()), n, C.byref(lay) if lay else None, k, v, start,
                                         None)


def _read(desc=None, ctx=CTX, dtype=0, begin=0, n=3, lay=None, k=256, v=256):
    return _lib.load().it_kv_cache_read(ctx, dtype, C.byref(desc or _desc()), begin, n, C.byref(lay) if lay else None, k, v)


def _attend(desc=None, ctx=CTX, dtype=0, heads=4, n=3, scale=1.0, ql=None, ol=None, q=256, start=256, o=256):
    return _lib.load().it_cached_attention(ctx, dtype, C.byref(desc or _desc()), heads, n, scale, C.byref(ql) if ql else None,
                                           C.byref(ol) if ol else None, q, start, None, o)


@pytest.mark.parametrize("call", [_write, _read, _attend])
def test_cache_arguments(call):
    assert call(ctx=None) == _lib.IT_ERR_NULL and "ctx" in _lib.last_error()
    for dtype in (1, 3, -1):
        assert call(dtype=dtype) == _lib.IT_ERR_PRECISION
    for bits in (0, 2, 5, 16, -4):
        assert call(_desc(bits=bits)) == _lib.IT_ERR_INVALID and "bits" in _lib.last_error()
    for d in (0, 32, 63, 96, 512, -64):
        assert call(_desc(head_dim=d)) == _lib.IT_ERR_DIMS and "head_dim" in _lib.last_error()
    for kw in ({"batch": -1}, {"kv_heads": -1}, {"capacity": -1}):
        assert call(_desc(**kw)) == _lib.IT_ERR_INVALID
    for kw in ({"batch": 2 ** 40}, {"kv_heads": 2 ** 62}, {"capacity": 2 ** 62}, {"batch": 2 ** 20, "kv_heads": 2 ** 20}):
        assert call(_desc(**kw)) == _lib.IT_ERR_DIMS
    assert call(_desc(data=None)) == _lib.IT_ERR_NULL
    assert call(_desc(data=264)) == _lib.IT_ERR_INVALID and "aligned" in _lib.last_error()
    assert call(n=-1) == _lib.IT_ERR_INVALID
    lib = _lib.load()
    assert lib.it_kv_cache_write(CTX, 0, None, 1, None, 256, 256, 256, None) == _lib.IT_ERR_NULL


def test_a_head_stays_below_two_gib():
    lib, size = _lib.load(), C.c_size_t()
    assert lib.it_kv_cache_bytes(4, 1, 1, 14_000_000, 128, C.byref(size)) == 0
    assert size.value == 14_000_000 * (128 + 2 * 4 + 2) < 2 ** 31
    assert lib.it_kv_cache_bytes(4, 1, 1, 16_000_000, 128, C.byref(size)) == _lib.IT_ERR_DIMS
    assert lib.it_kv_cache_bytes(8, 64, 64, 65, 64, C.byref(size)) == 0
    assert size.value == 64 * 64 * 128 * (2 * 64 + 2 * 2 + 2)
    assert lib.it_kv_cache_bytes(8, 64, 0, 65, 64, C.byref(size)) == 0 and size.value == 0
    assert lib.it_kv_cache_bytes(8, 1, 1, 1, 64, None) == _lib.IT_ERR_NULL


@pytest.mark.parametrize("call,names", [(_write, ("k", "v", "start")), (_read, ("k", "v")), (_attend, ("q", "o", "start"))])
def test_null_buffers(call, names):
    for name in names:
        assert call(**{name: None}) == _lib.IT_ERR_NULL, name


def test_layouts():
    lay = lambda h=2, bs=640, hs=64, rs=128: _lib.AttnLayout(h, bs, hs, rs)  # noqa: E731
    for call, name, h in ((_write, "lay", 2), (_read, "lay", 2), (_attend, "ql", 4), (_attend, "ol", 4)):
        for bad in (lay(h, rs=63), lay(h, bs=-1), lay(h, hs=-1), lay(0), lay(h, rs=2 ** 62)):
            assert call(**{name: bad}) == _lib.IT_ERR_INVALID
        assert call(**{name: lay(3)}) == _lib.IT_ERR_SHAPE


def test_read_range():
    assert _read(begin=-1) == _lib.IT_ERR_INVALID
    for begin, n in ((8, 3), (11, 0), (0, 11), (5, 2 ** 62), (2 ** 62, 1)):
        assert _read(begin=begin, n=n) == _lib.IT_ERR_SHAPE, (begin, n)


def test_attention_arguments():
    for scale in (0.0, -1.0, float("nan"), float("inf")):
        assert _attend(scale=scale) == _lib.IT_ERR_INVALID and "scale" in _lib.last_error()
    assert _attend(heads=3) == _lib.IT_ERR_SHAPE
    assert _attend(heads=-2) == _lib.IT_ERR_INVALID
    assert _attend(_desc(kv_heads=0), heads=2) == _lib.IT_ERR_SHAPE
    assert _attend(heads=2 ** 20, n=2 ** 20) == _lib.IT_ERR_DIMS
    assert _write(n=2 ** 60) == _lib.IT_ERR_DIMS


def test_gemm_arguments():
    lib = _lib.load()

    def gemm(ctx=CTX, dtype=0, m=4, n=5, k=32, a=256, lda=32, sa=256, b=256, ldb=32, sb=256, c=256, ldc=5):
        return lib.it_gemm_i8(ctx, dtype, m, n, k, a, lda, sa, b, ldb, sb, None, c, ldc)

    assert gemm(ctx=None) == _lib.IT_ERR_NULL
    assert gemm(dtype=1) == _lib.IT_ERR_PRECISION
    for kw in ({"m": -1}, {"n": -1}, {"lda": 16}, {"ldb": 40}, {"lda": 33}, {"ldc": 4}, {"a": 264}, {"b": 257}, {"k": -16}):
        assert gemm(**kw) == _lib.IT_ERR_INVALID, kw
    for kw in ({"k": 33, "lda": 48, "ldb": 48}, {"k": 131072, "lda": 131072, "ldb": 131072}, {"lda": 2 ** 23},
               {"m": 2 ** 35, "n": 2 ** 35, "ldc": 2 ** 35}):
        assert gemm(**kw) == _lib.IT_ERR_DIMS, kw
    for name in ("a", "b", "sa", "sb", "c"):
        assert gemm(**{name: None}) == _lib.IT_ERR_NULL, name

    def linear(ctx=CTX, dtype=0, m=4, n=5, k=30, x=256, ldx=30, w=256, ldw=32, sw=256, y=256, ldy=5):
        return lib.it_linear_i8(ctx, dtype, m, n, k, x, ldx, w, ldw, sw, None, y, ldy)

    assert linear(ctx=None) == _lib.IT_ERR_NULL
    assert linear(dtype=1) == _lib.IT_ERR_PRECISION
    for kw in ({"k": -1}, {"ldx": 29}, {"ldw": 16}, {"ldy": 4}, {"w": 260}, {"m": -1}):
        assert linear(**kw) == _lib.IT_ERR_INVALID, kw
    assert linear(k=130945, ldx=131057, ldw=131072) == _lib.IT_ERR_DIMS
    for name in ("x", "w", "sw", "y"):
        assert linear(**{name: None}) == _lib.IT_ERR_NULL, name

    def quantize(ctx=CTX, dtype=0, rows=3, cols=20, x=256, ldx=20, codes=256, ldc=32, steps=256):
        return lib.it_quantize_i8(ctx, dtype, rows, cols, x, ldx, codes, ldc, steps)

    assert quantize(ctx=None) == _lib.IT_ERR_NULL
    assert quantize(dtype=2 ** 30) == _lib.IT_ERR_PRECISION
    for kw in ({"rows": -1}, {"ldx": 19}, {"ldc": 20}, {"ldc": 16}, {"codes": 264}):
        assert quantize(**kw) == _lib.IT_ERR_INVALID, kw
    assert quantize(rows=2 ** 32) == _lib.IT_ERR_DIMS
    for name in ("x", "codes", "steps"):
        assert quantize(**{name: None}) == _lib.IT_ERR_NULL, name


# ------------------------------------------------------------------ the Python mirror

class _NoDevice:
    ptr = 256
    ctx = None


def _t(shape, prec=Precision.FP32):
    return Tensor(_NoDevice(), shape, prec)


class _Cache:
    batch, kv_heads, capacity, head_dim, bits, ctx = 2, 2, 10, 64, 4, None


def test_mirror_cache_errors():
    import irontensor_amd as it
    k = _t([2, 3, 2, 64])
    with pytest.raises(it.UnsupportedDimensions):
        it.kv_cache_write(_Cache, _t([2, 3, 128]), k, [0, 0])
    with pytest.raises(it.ShapeMismatch):
        it.kv_cache_write(_Cache, k, _t([2, 4, 2, 64]), [0, 0])
    with pytest.raises(it.ShapeMismatch):
        it.kv_cache_write(_Cache, _t([2, 3, 4, 64]), _t([2, 3, 4, 64]), [0, 0])
    with pytest.raises(it.PrecisionMismatch):
        it.kv_cache_write(_Cache, k, _t([2, 3, 2, 64], Precision.BF16), [0, 0])
    with pytest.raises(it.PrecisionMismatch):
        it.kv_cache_write(_Cache, _t([2, 3, 2, 64], Precision.FP16), _t([2, 3, 2, 64], Precision.FP16), [0, 0])
    for start, count in (([0, 8], None), ([-1, 0], None), ([0, 9], [3, 2]), ([0, 2 ** 40], None), ([0.5, 1], None),
                         ([0, 0], [0, 4]), ([0, 0], [-1, 0])):
        with pytest.raises(it.InvalidValue):
            it.kv_cache_write(_Cache, k, k, start, count)
    for start, count in (([0], None), ([0, 0, 0], None), ([0, 0], [1])):
        with pytest.raises(it.ShapeMismatch):
            it.kv_cache_write(_Cache, k, k, start, count)
    with pytest.raises(it.ShapeMismatch):
        it.cached_attention(_t([2, 1, 4, 128]), _Cache, [0, 0])
    with pytest.raises(it.ShapeMismatch):
        it.cached_attention(_t([2, 1, 4, 64]), _Cache, [0, 0], out=_t([2, 1, 2, 64]))
    with pytest.raises(it.PrecisionMismatch):
        it.cached_attention(_t([2, 1, 4, 64]), _Cache, [0, 0], out=_t([2, 1, 4, 64], Precision.BF16))
    with pytest.raises(it.ShapeMismatch):
        it.kv_cache_read(_Cache, 0, 3, out=(k, _t([2, 4, 2, 64])))
    with pytest.raises(it.PrecisionMismatch):
        it.kv_cache_read(_Cache, 0, 3, out=(k, _t([2, 3, 2, 64], Precision.BF16)))
    with pytest.raises(it.InvalidValue):
        it.kv_cache_read(_Cache, 0, -1)
    with pytest.raises(it.InvalidValue, match="bits"):
        it.KvCache(1, 1, 8, 64, 3)


class _Matrix:
    def __init__(self, rows, cols):
        self.rows, self.cols, self.ctx = rows, cols, None

    def shape(self):
        return [self.rows, self.cols]


def test_mirror_linear_errors():
    import irontensor_amd as it
    with pytest.raises(it.UnsupportedDimensions):
        it.quantize_i8(_t([2, 3, 4]))
    with pytest.raises(it.PrecisionMismatch):
        it.quantize_i8(_t([2, 3], Precision.FP16))
    w = _Matrix(5, 7)
    with pytest.raises(it.InnerDimensionMismatch):
        it.linear_i8(_t([2, 8]), w)
    with pytest.raises(it.Panic):
        it.linear_i8(_t([]), w)
    with pytest.raises(it.PrecisionMismatch):
        it.linear_i8(_t([2, 7], Precision.FP16), w)
    with pytest.raises(it.ShapeMismatch):
        it.linear_i8(_t([2, 7]), w, _t([7]))
    with pytest.raises(it.PrecisionMismatch):
        it.linear_i8(_t([2, 7]), w, _t([5], Precision.BF16))
    with pytest.raises(it.ShapeMismatch):
        it.linear_i8(_t([2, 7]), w, out=_t([2, 7]))
    with pytest.raises(it.PrecisionMismatch):
        it.linear_i8(_t([2, 7]), w, out=_t([2, 5], Precision.BF16))
    with pytest.raises(it.InnerDimensionMismatch):
        it.matmul_i8(w, _Matrix(5, 8))
    with pytest.raises(it.ShapeMismatch):
        it.matmul_i8(w, _Matrix(3, 7), out=_t([5, 5]))
    assert np.asarray(it.Positions.__slots__).size == 2
