"""8-bit products on the GPU: the quantiser bit for bit, the integer sums exactly, and the linear layer."""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

import quantref as ref
from irontensor_amd import _lib

pytestmark = pytest.mark.gpu


def _tensor(it, x, prec):
    if prec == "bf16":
        return it.Tensor.from_f32_as_bf16(x, x.shape)
    return it.Tensor.from_f32_slice(x, x.shape)


def _round(x, prec):
    return ref.rne_bf16(x) if prec == "bf16" else np.asarray(x, np.float32)


@pytest.mark.parametrize("prec", ["f32", "bf16"])
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 15), (2, 16), (5, 17), (7, 255), (4, 256), (3, 1237), (2, 4096),
                                       (3, 20001), (300, 64)])
def test_quantize_rows(it, prec, rows, cols):
    rng = np.random.default_rng(cols)
    x = _round(rng.standard_normal((rows, cols)) * 10.0 ** rng.uniform(-6, 6, (rows, 1)), prec)
    m = it.quantize_i8(_tensor(it, x, prec))
    s = ref.steps(x, cols, 127, bf16=False)
    assert np.array_equal(m.steps.numpy(), s[:, 0])
    assert np.array_equal(m.codes(), ref.codes(x, s, cols, 127))


def test_quantize_borders(it):
    """Halves and their neighbours at a step of one, zeros, tiny rows, the largest numbers, NaN and infinity."""
    x = np.zeros((9, 33), np.float32)
    x[0] = np.arange(33) - 16.5
    x[0, 0] = 127
    x[1] = np.nextafter(x[0], np.float32(1000))
    x[2] = np.nextafter(x[0], np.float32(-1000))
    x[1, 0] = x[2, 0] = 127
    x[4] = 1e-41
    x[5] = np.linspace(-3.4e38, 3.4e38, 33)
    x[6] = x[7] = x[8] = 1
    x[6, 32], x[7, 0], x[8, 5] = np.nan, np.inf, -np.inf
    m = it.quantize_i8(it.Tensor.from_f32_slice(x, x.shape))
    s = ref.steps(x, 33, 127, bf16=False)
    got = m.steps.numpy()
    assert np.array_equal(got[:6], s[:6, 0]) and np.isnan(got[6:]).all()
    assert np.array_equal(m.codes(), ref.codes(x, s, 33, 127))


def _product(it, a, b, sa, sb, bias=None, prec="f32", lda=None, ldb=None, ldc=None):
    """it_gemm_i8 on codes as they are; columns past K hold other codes, rows of C past N stay."""
    (m, k), n = a.shape, b.shape[0]
    ctx = it.Context.global_()
    lda, ldb, ldc = lda or k, ldb or k, ldc or n
    rng = np.random.default_rng(0)

    def put(x, ld):
        w = rng.integers(-128, 128, (x.shape[0], ld)).astype(np.int8)
        w[:, :k] = x
        pad = np.zeros((w.size + 3) // 4 * 4, np.int8)
        pad[:w.size] = w.ravel()
        return it.Tensor.from_f32_slice(pad.view(np.float32), [pad.size // 4])

    ta, tb = put(a, lda), put(b, ldb)
    tsa, tsb = (it.Tensor.from_f32_slice(s, [len(s)]) for s in (sa, sb))
    tbias = None if bias is None else it.Tensor.from_f32_slice(bias, [n])
    c = _tensor(it, np.full((m, ldc), 7, np.float32), prec)
    st = ctx.lib.it_gemm_i8(ctx.handle, _lib.IT_BF16 if prec == "bf16" else _lib.IT_F32, m, n, k, ta.ptr, lda, tsa.ptr,
                            tb.ptr, ldb, tsb.ptr, None if bias is None else tbias.ptr, c.ptr, ldc)
    assert st == 0, _lib.last_error()
    out = c.numpy()
    assert (out[:, n:] == 7).all()
    return out[:, :n]


SIZES = [(1, 1, 16), (1, 16, 16), (2, 100, 48), (3, 17, 128), (4, 768, 256), (8, 33, 2048), (15, 129, 144), (16, 64, 4096),
         (17, 100, 112), (32, 255, 512), (33, 48, 1040), (64, 64, 64), (65, 130, 272), (100, 500, 1248), (128, 128, 128),
         (129, 257, 384), (250, 300, 4112), (257, 129, 2064), (300, 1000, 96), (513, 700, 640)]


@pytest.mark.parametrize("m,n,k", SIZES)
def test_sums_are_exact(it, m, n, k):
    """Steps of one: an FP32 result is the rounded integer sum. Codes over all of -128 .. 127."""
    rng = np.random.default_rng(m + n + k)
    a, b = (rng.integers(-128, 128, s).astype(np.int8) for s in ((m, k), (n, k)))
    got = _product(it, a, b, np.ones(m), np.ones(n))
    want = (a.astype(np.int64) @ b.astype(np.int64).T).astype(np.float32)
    assert np.array_equal(got, want)


@pytest.mark.parametrize("prec", ["f32", "bf16"])
@pytest.mark.parametrize("m,n,k", [(1, 300, 320), (5, 301, 272), (16, 77, 1040), (40, 129, 144), (140, 203, 528),
                                   (300, 513, 1040)])
def test_steps_bias_and_strides(it, prec, m, n, k):
    """Roundings: the sum to FP32, two products and the bias, 2^-24 each, and BF16's 2^-8."""
    rng = np.random.default_rng(n)
    a, b = (rng.integers(-127, 128, s).astype(np.int8) for s in ((m, k), (n, k)))
    sa, sb = (rng.uniform(0.5, 2, x).astype(np.float32) / 127 for x in (m, n))
    bias = rng.standard_normal(n).astype(np.float32)
    got = _product(it, a, b, sa, sb, bias, prec, k + 48, k + 16, n + 5)
    y = (a.astype(np.int64) @ b.astype(np.int64).T) * sa.astype(np.float64)[:, None] * sb.astype(np.float64)
    want = y + bias
    bound = 2.0 ** -24 * (4 * np.abs(y) + 2 * np.abs(want))
    if prec == "bf16":
        bound = bound * (1 + 2.0 ** -8) + 2.0 ** -8 * np.abs(want)
    assert (np.abs(got - want) <= bound).all()


@pytest.mark.parametrize("m", [1, 20, 130])
def test_longest_sums(it, m):
    """K at its limit with every product at its largest: sums up to 128 * 128 * 131056 = 2147221504 < 2^31."""
    k, n = 131056, 3
    a, b = np.full((m, k), -128, np.int8), np.full((n, k), -128, np.int8)
    b[1] = 127
    got = _product(it, a, b, np.ones(m), np.ones(n))
    assert np.array_equal(got, np.tile(np.float32([128 * 128 * k, -128 * 127 * k, 128 * 128 * k]), (m, 1)))


def test_empty_products(it):
    z = np.zeros
    assert _product(it, z((3, 16), np.int8), z((5, 16), np.int8), np.ones(3), np.ones(5), np.arange(5.0)).tolist() == [[0, 1, 2, 3, 4]] * 3
    ctx = it.Context.global_()
    c, s, bias = (it.Tensor.from_f32_slice(np.full(n, 3.0), [n]) for n in (6, 8, 3))
    assert ctx.lib.it_gemm_i8(ctx.handle, 0, 2, 3, 0, None, 0, s.ptr, None, 0, s.ptr, bias.ptr, c.ptr, 3) == 0
    assert c.numpy().tolist() == [3.0] * 6  # K = 0: the bias
    assert ctx.lib.it_gemm_i8(ctx.handle, 0, 0, 3, 16, None, 16, None, None, 16, None, None, None, 3) == 0
    w = it.quantize_i8(it.Tensor.from_f32_slice(np.ones(5 * 7), [5, 7]))
    assert it.linear_i8(it.Tensor.empty([0, 7]), w).shape() == [0, 5]


@pytest.mark.parametrize("prec", ["f32", "bf16"])
@pytest.mark.parametrize("m,n,k,bias", [(1, 768, 256, False), (1, 5, 1, True), (4, 688, 300, True), (16, 256, 1237, False),
                                        (31, 100, 77, True), (129, 513, 301, False), (1000, 701, 300, True),
                                        (2, 33, 700, False), (3, 17, 129, True), (7, 50, 4096, True), (8, 19, 4096, False),
                                        (9, 64, 3640, True), (16, 100, 2048, True), (1, 40, 20001, False)])
def test_linear(it, prec, m, n, k, bias):
    rng = np.random.default_rng(k)
    x, w = _round(rng.standard_normal((m, k)), prec), (rng.standard_normal((n, k)) * 0.02).astype(np.float32)
    bi = rng.standard_normal(n).astype(np.float32) if bias else None
    tb = None if bi is None else it.Tensor.from_f32_slice(bi, [n])
    layer = it.LinearI8.from_weight(it.Tensor.from_f32_slice(w, w.shape), tb)
    got = layer.forward(_tensor(it, x, prec)).numpy()
    # the sums in whole numbers: in float64 the values' own products leave 1e-17 where a sum is 0
    sx, sw = (ref.steps(v, k, 127, bf16=False) for v in (x, w))
    y = (ref.codes(x, sx, k, 127) @ ref.codes(w, sw, k, 127).T) * sx.astype(np.float64) * sw[:, 0].astype(np.float64)
    want = y if bi is None else y + bi
    bound = 2.0 ** -24 * (4 * np.abs(y) + 2 * np.abs(want))
    if prec == "bf16":
        bound = bound * (1 + 2.0 ** -8) + 2.0 ** -8 * np.abs(want)
    assert (np.abs(got - want) <= bound).all()
    both = it.matmul_i8(it.quantize_i8(_tensor(it, x, prec)), layer.weight, tb, it.Precision.BF16 if prec == "bf16" else it.Precision.FP32)
    assert np.array_equal(both.numpy(), got)


@pytest.mark.parametrize("prec", ["f32", "bf16"])
@pytest.mark.parametrize("m,n", [(1, 256), (8, 512), (3, 1440), (70, 144)])
def test_output_over_the_input(it, prec, m, n):
    """Y in X's place, also where one launch would read X and write Y."""
    rng = np.random.default_rng(n)
    x = _round(rng.standard_normal((m, n)), prec)
    layer = it.LinearI8.from_weight(it.Tensor.from_f32_slice(rng.standard_normal((n, n)), [n, n]))
    want = layer.forward(_tensor(it, x, prec)).numpy()
    over = _tensor(it, x, prec)
    assert np.array_equal(layer.forward(over, out=over).numpy(), want)


def test_rows_do_not_touch_each_other(it):
    """A NaN or infinite token makes its own row NaN, the others the same bits; 3D inputs keep their shape."""
    rng = np.random.default_rng(0)
    x = rng.standard_normal((2, 9, 130)).astype(np.float32)
    layer = it.LinearI8.from_weight(it.Tensor.from_f32_slice(rng.standard_normal((50, 130)), [50, 130]))
    clean = layer.forward(it.Tensor.from_f32_slice(x, x.shape)).numpy()
    x[1, 3, 7], x[0, 0, 129] = np.nan, np.inf
    got = layer.forward(it.Tensor.from_f32_slice(x, x.shape)).numpy()
    assert got.shape == (2, 9, 50) and np.isnan(got[1, 3]).all() and np.isnan(got[0, 0]).all()
    keep = np.ones((2, 9), bool)
    keep[1, 3] = keep[0, 0] = False
    assert np.array_equal(got[keep], clean[keep])


def test_captured_layers_share_the_scratch(it):
    """Two graphs of linear_i8 with different sizes on one context, replayed in turn with eager work between."""
    rng = np.random.default_rng(1)
    ctx, sets = it.Context.global_(), []
    for m, n, k in ((3, 200, 160), (70, 90, 333)):
        layer = it.LinearI8.from_weight(it.Tensor.from_f32_slice(rng.standard_normal((n, k)), [n, k]))
        x, out = it.Tensor.from_f32_slice(rng.standard_normal((m, k)), [m, k]), it.Tensor.empty([m, n])
        want = layer.forward(x).numpy()
        assert ctx.lib.it_capture_begin(ctx.handle) == 0
        layer.forward(x, out=out)
        g = C.c_void_p()
        assert ctx.lib.it_capture_end(ctx.handle, C.byref(g)) == 0, _lib.last_error()
        sets.append((g, layer, x, out, want))
    try:
        for _ in range(4):
            for g, _, _, out, _ in sets:
                assert ctx.lib.it_zero(ctx.handle, out.ptr, out.byte_size()) == 0
                assert ctx.lib.it_graph_launch(ctx.handle, g) == 0
            for _, layer, x, out, want in sets:
                assert np.array_equal(out.numpy(), want)
                assert np.array_equal(layer.forward(x).numpy(), want)
    finally:
        for s in sets:
            ctx.lib.it_graph_destroy(s[0])
