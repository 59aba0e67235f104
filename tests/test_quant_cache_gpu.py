"""The quantised key/value cache on the GPU: what is written reads back as the definition says, bit for bit, and
nothing else changes; and attention over it against float64."""
from __future__ import annotations

import ctypes as C
import math

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


def _keys(rng, shape, prec):
    x = rng.standard_normal(shape)
    x[..., 5::37] *= 8
    return _round(x, prec)


def _same(got, want):
    """Equal bit for bit where finite, NaN where NaN."""
    want = np.asarray(want, np.float32)
    assert np.array_equal(np.isnan(got), np.isnan(want))
    fine = ~np.isnan(want)
    bad = np.nonzero(got[fine] != want[fine])[0]
    assert not bad.size, (bad.size, got[fine][bad[:4]], want[fine][bad[:4]])


# ------------------------------------------------------------------ write and read

@pytest.mark.parametrize("prec", ["f32", "bf16"])
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_write_then_read(it, prec, bits, d):
    """Ragged starts (off the four-token blocks) and counts over a cache that holds other tokens."""
    b, h, cap = 5, 3, 70
    rng = np.random.default_rng(100 * d + bits)
    old = [_keys(rng, (b, cap, h, d), prec) for _ in range(2)]
    cache = it.KvCache(b, h, cap, d, bits)
    it.kv_cache_write(cache, *(_tensor(it, x, prec) for x in old), [0] * b)
    want = [w.copy() for w in ref.cache_values(*old, bits)]
    for n, start, count in ((1, [0, 1, 2, 3, 69], None), (3, [0, 5, 6, 7, 67], [3, 0, 1, 2, 3]),
                            (33, [0, 1, 2, 3, 37], None), (9, [60, 8, 4, 31, 61], [9, 9, 8, 1, 0])):
        new = [_keys(rng, (b, n, h, d), prec) for _ in range(2)]
        it.kv_cache_write(cache, *(_tensor(it, x, prec) for x in new), start, count)
        for w, x in zip(want, ref.cache_values(*new, bits)):
            for bi in range(b):
                m = n if count is None else count[bi]
                w[bi, start[bi]:start[bi] + m] = x[bi, :m]
        for begin, m in ((0, cap), (3, 1), (6, 13), (69, 1), (5, 0)):
            got = it.kv_cache_read(cache, begin, m)
            for g, w in zip(got, want):
                _same(g.numpy(), w[:, begin:begin + m])
    for g, w in zip(it.kv_cache_read(cache, 0, cap, it.Precision.BF16), want):
        _same(g.numpy(), ref.rne_bf16(w.astype(np.float32)))


@pytest.mark.parametrize("bits", [4, 8])
def test_untouched_positions_read_zero(it, bits):
    cache = it.KvCache(2, 2, 9, 64, bits)
    for t in it.kv_cache_read(cache, 0, 9):
        assert not t.numpy().any() and not np.signbit(t.numpy()).any()
    x = _tensor(it, np.ones((2, 1, 2, 64), np.float32), "f32")
    it.kv_cache_write(cache, x, x, [4, 8])
    k, v = (t.numpy() for t in it.kv_cache_read(cache, 0, 9))
    assert np.count_nonzero(k) == np.count_nonzero(v) == 2 * 2 * 64
    cache.clear()
    assert not it.kv_cache_read(cache, 0, 9)[0].numpy().any()


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("prec", ["f32", "bf16"])
def test_values_at_borders(it, prec, bits):
    """Exact halves (to even), values one step of FP32 beside them, zeros, groups too small for a step, the largest
    numbers, and groups that hold a NaN or an infinity."""
    d, levels = 64, 7 if bits == 4 else 127
    rng = np.random.default_rng(3)
    x = np.zeros((1, 24, 1, d), np.float32)
    for t in range(8):  # the step is 2^e exactly; codes n + 1/2 and their neighbours
        step = np.float32(2.0 ** (3 * t - 12))
        n = rng.integers(-levels, levels, d).astype(np.float32) + np.float32(0.5)
        x[0, t, 0] = n * step
        x[0, t, 0, 1::3] = np.nextafter(x[0, t, 0, 1::3], np.float32(np.inf))
        x[0, t, 0, 2::3] = np.nextafter(x[0, t, 0, 2::3], np.float32(-np.inf))
        x[0, t, 0, ::32] = levels * step
    x[0, 9] = 1e-40
    x[0, 10] = rng.standard_normal(d) * 2.0 ** -126
    x[0, 11] = rng.standard_normal(d) * 2.0 ** -122
    x[0, 12] = rng.uniform(-1, 1, d) * 3.38e38
    x[0, 13], x[0, 14], x[0, 15] = (rng.standard_normal(d) for _ in range(3))
    x[0, 13, 0, 40], x[0, 14, 0, 3], x[0, 15, 0, 63] = np.nan, np.inf, -np.inf
    x[0, 16:] = rng.standard_normal((8, 1, d)) * 10.0 ** rng.uniform(-20, 20, (8, 1, 1))
    x = _round(x, prec)
    cache = it.KvCache(1, 1, 24, d, bits)
    t = _tensor(it, x, prec)
    it.kv_cache_write(cache, t, t, [0])
    k, v = it.kv_cache_read(cache, 0, 24)
    with np.errstate(over="ignore"):
        wk, wv = (w.astype(np.float32) for w in ref.cache_values(x, x, bits))
    _same(k.numpy(), wk)
    _same(v.numpy(), wv)
    assert np.isnan(v.numpy()[0, 13:16]).all() and np.isnan(k.numpy()[0, 13]).sum() == 32


@pytest.mark.parametrize("bits", [4, 8])
def test_positions_outside_the_cache_are_not_written(it, bits):
    """Device positions that the host has not seen: negative, across the end, past it and at the integers' ends."""
    b, n, cap, d = 8, 6, 13, 64
    rng = np.random.default_rng(5)
    old = _keys(rng, (b, cap, 1, d), "f32")
    cache = it.KvCache(b, 1, cap, d, bits)
    t = _tensor(it, old, "f32")
    it.kv_cache_write(cache, t, t, [0] * b)
    new = _keys(rng, (b, n, 1, d), "f32")
    start = [-6, -3, -1, 9, 12, 13, 2 ** 31 - 1, -2 ** 31]
    count = [6, 7, 100, 6, 6, 6, 6, -1]
    t = _tensor(it, new, "f32")
    it.kv_cache_write(cache, t, t, it.upload_positions(start), it.upload_positions(count))
    want = ref.cache_values(old, old, bits)
    for w, x in zip(want, ref.cache_values(new, new, bits)):
        for bi in range(b):
            for i in range(max(0, min(n, count[bi]))):
                if 0 <= start[bi] + i < cap:
                    w[bi, start[bi] + i] = x[bi, i]
    for g, w in zip(it.kv_cache_read(cache, 0, cap), want):
        _same(g.numpy(), w)


def _strided(it, rng, b, n, heads, d, prec, skew):
    """(buffer, pointer offset in elements, layout, values [b, n, heads, d]): rows of a wider matrix, head rows
    apart, `skew` elements off the alignment."""
    hs, rs = d + 8 + skew, heads * (d + 8 + skew) + 16 + skew
    flat = _round(rng.standard_normal(b * n * rs + 64), prec)
    idx = (skew + np.arange(b)[:, None, None, None] * n * rs + np.arange(n)[:, None, None] * rs
           + np.arange(heads)[:, None] * hs + np.arange(d))
    return flat, skew, _lib.AttnLayout(heads, n * rs, hs, rs), idx


@pytest.mark.parametrize("prec", ["f32", "bf16"])
@pytest.mark.parametrize("skew", [0, 1])
@pytest.mark.parametrize("bits", [4, 8])
def test_strided_rows(it, prec, skew, bits):
    """K, V, Q and O as parts of wider rows, aligned to 16 bytes or to an element only; what lies between stays."""
    b, n, hkv, share, d, cap = 2, 5, 2, 3, 64, 12
    rng = np.random.default_rng(11 + skew)
    lib, ctx = it.Context.global_().lib, it.Context.global_()
    e, dt = (2, _lib.IT_BF16) if prec == "bf16" else (4, _lib.IT_F32)
    kf, off, lay, idx = _strided(it, rng, b, n, hkv, d, prec, skew)
    vf, _, _, _ = _strided(it, rng, b, n, hkv, d, prec, skew)
    qf, _, qlay, qidx = _strided(it, rng, b, n, hkv * share, d, prec, skew)
    cache = it.KvCache(b, hkv, cap, d, bits)
    kt, vt, qt = (_tensor(it, x, prec) for x in (kf, vf, qf))
    start = it.upload_positions([0, 7])
    check = lambda st: (_ for _ in ()).throw(AssertionError(_lib.last_error())) if st else None  # noqa: E731
    check(lib.it_kv_cache_write(ctx.handle, dt, cache._ref, n, C.byref(lay), kt.ptr + off * e, vt.ptr + off * e, start.ptr,
                                None))
    kw, vw = ref.cache_values(kf[idx], vf[idx], bits)
    k0, v0 = (np.zeros((b, cap, hkv, d)) for _ in range(2))
    for bi, s in enumerate((0, 7)):
        k0[bi, s:s + n], v0[bi, s:s + n] = kw[bi], vw[bi]
    for g, w in zip(it.kv_cache_read(cache, 0, cap), (k0, v0)):
        _same(g.numpy(), w)
    ko, vo = (_tensor(it, np.full(kf.shape, 9, np.float32), prec) for _ in range(2))
    check(lib.it_kv_cache_read(ctx.handle, dt, cache._ref, 7, n, C.byref(lay), ko.ptr + off * e, vo.ptr + off * e))
    for t, w in ((ko, k0), (vo, v0)):
        got, want = t.numpy(), np.full(kf.shape, 9, np.float32)
        want[idx] = _round(w[:, 7:12].astype(np.float32), prec)
        _same(got, want)
    ot = _tensor(it, np.full(qf.shape, 9, np.float32), prec)
    check(lib.it_cached_attention(ctx.handle, dt, cache._ref, hkv * share, n, 0.125, C.byref(qlay), None, qt.ptr + off * e,
                                  start.ptr, None, ot.ptr + off * e))
    want = ref.attend(qf[qidx], k0, v0, [0, 7], [n, n], 0.125)
    got = ot.numpy()
    assert (np.abs(got[qidx] - want[0]) <= ref.attend_bound(want, cap, d, prec == "bf16")).all()
    got[qidx] = 9
    assert (got == 9).all()


# ------------------------------------------------------------------ attention

def _attend(it, rng, prec, bits, d, b, hkv, share, n, cap, start, count, fill=None):
    k, v = _keys(rng, (b, cap, hkv, d), prec), _round(rng.standard_normal((b, cap, hkv, d)), prec)
    q = _round(rng.standard_normal((b, n, hkv * share, d)), prec)
    if fill is not None:
        fill(k, v)
    cache = it.KvCache(b, hkv, cap, d, bits)
    if cap:
        it.kv_cache_write(cache, _tensor(it, k, prec), _tensor(it, v, prec), [0] * b)
    qt = _tensor(it, q, prec)
    o = it.cached_attention(qt, cache, it.upload_positions(start), None if count is None else it.upload_positions(count))
    kw, vw = ref.cache_values(k, v, bits)
    return qt, cache, o.numpy(), ref.attend(q, kw, vw, start, [n] * b if count is None else count, d ** -0.5)


def _near(got, want, cap, d, prec):
    o, bound = want[0], ref.attend_bound(want, cap, d, prec == "bf16")
    err = np.abs(got - o)
    assert (err <= bound).all(), float((err / np.maximum(bound, 1e-300)).max())
    if prec == "f32" and np.abs(o).max() > 0:
        assert err.max() / np.abs(o).max() <= 1e-5


@pytest.mark.parametrize("prec", ["f32", "bf16"])
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("share,n,cap", [(1, 1, 1), (1, 1, 33), (4, 1, 300), (16, 1, 129), (7, 5, 77), (1, 17, 64),
                                         (3, 40, 200)])
def test_attention(it, prec, bits, d, share, n, cap):
    rng = np.random.default_rng(d + 10 * n + share)
    b, hkv = 2, 2
    start = [cap - n, (cap - n) // 2]
    _, _, got, want = _attend(it, rng, prec, bits, d, b, hkv, share, n, cap, start, None)
    _near(got, want, cap, d, prec)


@pytest.mark.parametrize("prec", ["f32", "bf16"])
@pytest.mark.parametrize("d", [64, 128])
def test_attention_of_a_ragged_batch(it, prec, d):
    """Lengths of zero and one, counts below n, starts before the cache and past its end."""
    b, n, cap = 9, 6, 150
    start = [0, 0, 144, 149, 200, -3, -6, 60, 2 ** 31 - 2]
    count = [6, 1, 6, 6, 6, 6, 6, 0, -5]
    rng = np.random.default_rng(d)
    _, _, got, want = _attend(it, rng, prec, 4, d, b, 2, 3, n, cap, start, count)
    _near(got, want, cap, d, prec)
    assert not got[6:].any() and not got[5, :3].any() and not got[1, 1:].any()  # -6 + 5 is still before the cache
    assert got[5, 3].any() and got[4].any()


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("share,n,cap", [(3, 50, 150), (1, 128, 128), (16, 17, 333)])
def test_prompts_of_a_large_batch(it, bits, d, share, n, cap):
    """Many rows of many sequences, ragged: some sequences against float64, padded queries give zeros, and poisoned
    positions that nobody sees change no bit."""
    b, hkv, prec = 64, 2 if (n * share + 127) // 128 > 1 else 4, "bf16"
    rng = np.random.default_rng(cap + d)
    k, v = _keys(rng, (b, cap, hkv, d), prec), _round(rng.standard_normal((b, cap, hkv, d)), prec)
    q = _round(rng.standard_normal((b, n, hkv * share, d)), prec)
    start = rng.integers(0, cap - n + 1, b)
    count = np.where(np.arange(b) % 3 == 1, rng.integers(0, n + 1, b), n)
    start[0], count[0], start[1], count[1], start[4], count[4] = cap - n, n, 0, 0, -n // 2, n
    start[5] = cap + 3
    outs = []
    for bad in (0.0, np.nan):
        for bi in range(b):
            end = max(0, int(start[bi]) + int(count[bi]))
            k[bi, end:, :, 3], v[bi, end:, :, 5] = bad, bad
        cache = it.KvCache(b, hkv, cap, d, bits)
        it.kv_cache_write(cache, _tensor(it, k, prec), _tensor(it, v, prec), [0] * b)
        outs.append(it.cached_attention(_tensor(it, q, prec), cache, it.upload_positions(start), it.upload_positions(count)).numpy())
        if bad == 0.0:
            kw, vw = ref.cache_values(k, v, bits)
    assert np.array_equal(outs[0], outs[1])
    some = [0, 1, 4, 5, 7, 33, 63]
    _near(outs[0][some], ref.attend(q[some], kw[some], vw[some], start[some], count[some], d ** -0.5), cap, d, prec)
    for bi in range(b):
        assert not outs[0][bi, max(0, count[bi]):].any()


@pytest.mark.parametrize("prec", ["f32", "bf16"])
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("n", [1, 9, 70])
def test_hidden_positions_do_not_matter(it, prec, bits, n):
    """NaN, infinities and the largest numbers at positions that a query does not see: the same bits as zeros there.
    With n > 1 the poison of a later query's token is hidden from the earlier ones only."""
    cap, d, at = 300, 64, 200
    outs = []
    for bad in (0.0, np.nan, np.inf, 3e38):
        def fill(k, v):
            k[:, at:, :, 3], v[:, at:, :, 9] = bad, bad
        rng = np.random.default_rng(8)
        start = [at - n, at - n - 5, 7 - min(n, 7)]
        _, _, got, _ = _attend(it, rng, prec, bits, d, 3, 1, 4, n, cap, start, None, fill)
        outs.append(got)
    for o in outs[1:]:
        assert np.isfinite(o).all() and np.array_equal(o, outs[0])
    if n > 1:  # the last queries see one poisoned token, the others none
        def fill(k, v):
            v[:, at, :, 9] = np.nan
        _, _, got, _ = _attend(it, np.random.default_rng(8), prec, bits, d, 1, 1, 4, n, cap, [at - n + 1], None, fill)
        assert np.isnan(got[:, -1]).all() and np.isfinite(got[:, :-1]).all()


@pytest.mark.parametrize("prec", ["f32", "bf16"])
@pytest.mark.parametrize("n", [4, 70])
def test_padded_queries_do_not_matter(it, prec, n):
    """Queries at count and beyond may hold anything: zeros come out, and the others' bits stay."""
    b, hkv, share, d, cap = 2, 2, 3, 64, 90
    rng = np.random.default_rng(n)
    k, v = (_tensor(it, _keys(rng, (b, cap, hkv, d), prec), prec) for _ in range(2))
    cache = it.KvCache(b, hkv, cap, d, 4)
    it.kv_cache_write(cache, k, v, [0] * b)
    q = _round(rng.standard_normal((b, n, hkv * share, d)), prec)
    start, count = it.upload_positions([5, 0]), it.upload_positions([n - 3, 1])
    clean = it.cached_attention(_tensor(it, q, prec), cache, start, count).numpy()
    q[0, n - 3:], q[1, 1:] = np.nan, np.inf
    got = it.cached_attention(_tensor(it, q, prec), cache, start, count).numpy()
    assert np.array_equal(got, clean) and not got[0, n - 3:].any() and not got[1, 1:].any() and got[0, 0].any()


@pytest.mark.parametrize("prec", ["f32", "bf16"])
@pytest.mark.parametrize("n,cap", [(1, 3000), (1, 40), (70, 90)])
def test_output_over_the_queries(it, prec, n, cap):
    b, hkv, share, d = 2, 2, 3, 64
    rng = np.random.default_rng(n + cap)
    k, v = (_tensor(it, _keys(rng, (b, cap, hkv, d), prec), prec) for _ in range(2))
    cache = it.KvCache(b, hkv, cap, d, 4)
    it.kv_cache_write(cache, k, v, [0] * b)
    q = _round(rng.standard_normal((b, n, hkv * share, d)), prec)
    want = it.cached_attention(_tensor(it, q, prec), cache, [cap - n, 5]).numpy()
    over = _tensor(it, q, prec)
    assert np.array_equal(it.cached_attention(over, cache, [cap - n, 5], out=over).numpy(), want)


@pytest.mark.parametrize("prec", ["f32", "bf16"])
def test_visible_nan_and_infinity(it, prec):
    for which in ("k", "v"):
        def fill(k, v):
            (k if which == "k" else v)[0, 20, 0, 1] = np.inf if which == "v" else np.nan
        _, _, got, _ = _attend(it, np.random.default_rng(1), prec, 8, 64, 2, 1, 2, 1, 40, [39, 39], None, fill)
        assert np.isnan(got[0]).all() and np.isfinite(got[1]).all()


@pytest.mark.parametrize("prec", ["f32", "bf16"])
def test_large_scores(it, prec):
    """Scores in the thousands, rising and falling along the row: one key takes nearly all, and nothing overflows."""
    for order in (1, -1):
        def fill(k, v):
            t = np.arange(k.shape[1], dtype=np.float32)[::order]
            k[:] = (t / 4)[None, :, None, None] * np.sign(np.arange(64) % 2 - 0.5)
            k[:] = _round(k, prec)
        rng = np.random.default_rng(2)
        _, _, got, want = _attend(it, rng, prec, 8, 64, 1, 1, 4, 1, 700, [699], None, fill)
        # mag is in the thousands: a score's own FP32 rounding, (D + 24) 2^-24 mag, is up to 1e-2 here
        assert np.isfinite(got).all()
        assert (np.abs(got - want[0]) <= ref.attend_bound(want, 700, 64, prec == "bf16")).all()


@pytest.mark.parametrize("prec,bits,d,share,n,cap", [("f32", 4, 64, 1, 1, 5000), ("bf16", 4, 128, 4, 1, 9001),
                                                     ("bf16", 8, 64, 7, 2, 3333), ("f32", 8, 128, 16, 3, 2049)])
def test_keys_split_among_blocks(it, prec, bits, d, share, n, cap):
    """Few rows and many keys: the same bits at every call, the last block's joining included, and the arrival
    counters left as they were."""
    rng = np.random.default_rng(cap)
    start = [cap - n, 700]
    qt, cache, got, want = _attend(it, rng, prec, bits, d, 2, 1, share, n, cap, start, None)
    _near(got, want, cap, d, prec)
    pos = it.upload_positions(start)
    for _ in range(5):
        assert np.array_equal(it.cached_attention(qt, cache, pos).numpy(), got)
    pos.write([3, 255])
    short = it.cached_attention(qt, cache, pos).numpy()
    pos.write(start)
    assert np.array_equal(it.cached_attention(qt, cache, pos).numpy(), got)
    assert np.isfinite(short).all() and not np.array_equal(short, got)


def test_empty_sizes(it):
    P = it.Precision
    empty = it.KvCache(2, 1, 0, 64, 4)
    q = it.Tensor.from_f32_slice(np.ones(2 * 3 * 2 * 64), [2, 3, 2, 64])
    assert not it.cached_attention(q, empty, it.upload_positions([0, 5])).numpy().any()
    cache = it.KvCache(2, 1, 8, 64, 4)
    none = it.Tensor.empty([2, 0, 1, 64], P.FP32)
    it.kv_cache_write(cache, none, none, [0, 8])
    assert it.cached_attention(it.Tensor.empty([2, 0, 2, 64], P.FP32), cache, [0, 0]).shape() == [2, 0, 2, 64]
    assert it.kv_cache_read(cache, 8, 0)[0].shape() == [2, 0, 1, 64]
    nobody = it.KvCache(0, 1, 8, 64, 4)
    assert it.cached_attention(it.Tensor.empty([0, 1, 2, 64], P.FP32), nobody, []).shape() == [0, 1, 2, 64]


# ------------------------------------------------------------------ as a program runs them

def _graph(it, ctx, f):
    assert ctx.lib.it_capture_begin(ctx.handle) == 0, _lib.last_error()
    try:
        f()
    finally:
        g = C.c_void_p()
        st = ctx.lib.it_capture_end(ctx.handle, C.byref(g))
    assert st == 0, _lib.last_error()
    return g


@pytest.mark.parametrize("prec", ["f32", "bf16"])
def test_two_captured_steps_share_the_scratch(it, prec):
    """Two graphs of the same context, one token each, replayed in turn with eager calls and new positions between."""
    rng = np.random.default_rng(6)
    ctx, cap, d = it.Context.global_(), 3000, 64
    P = it.Precision.BF16 if prec == "bf16" else it.Precision.FP32
    sets = []
    for hkv, share in ((2, 4), (1, 3)):
        k, v = (_keys(rng, (1, cap, hkv, d), prec) for _ in range(2))
        cache, same = (it.KvCache(1, hkv, cap, d, 4) for _ in range(2))
        for c in (cache, same):
            it.kv_cache_write(c, _tensor(it, k, prec), _tensor(it, v, prec), [0])
        new = [_tensor(it, _keys(rng, (1, 1, hkv, d), prec), prec) for _ in range(2)]
        q = _tensor(it, _keys(rng, (1, 1, hkv * share, d), prec), prec)
        pos, out = it.upload_positions([5]), it.Tensor.empty(q.shape(), P)

        def step(cache=cache, new=new, q=q, pos=pos, out=out):
            it.kv_cache_write(cache, *new, pos)
            it.cached_attention(q, cache, pos, out=out)

        step()
        sets.append((_graph(it, ctx, step), cache, same, new, q, pos, out))
    try:
        for at in (0, 2999, 17, 1500, 1501):
            for g, _, _, _, _, pos, _ in sets:
                pos.write([at])
                assert ctx.lib.it_graph_launch(ctx.handle, g) == 0
            for g, cache, same, new, q, pos, out in sets:
                got = out.numpy()
                it.kv_cache_write(same, *new, pos)
                if at == 0:
                    it.kv_cache_write(same, *new, [5])  # what the step before the capture wrote
                assert np.array_equal(got, it.cached_attention(q, same, pos).numpy())
                for a, b in zip(it.kv_cache_read(cache, 0, cap), it.kv_cache_read(same, 0, cap)):
                    assert np.array_equal(a.numpy(), b.numpy())
    finally:
        for s in sets:
            ctx.lib.it_graph_destroy(s[0])


def test_second_context_and_side_stream(it):
    """The same call on another context's stream and on the side stream: the same bits."""
    rng = np.random.default_rng(9)
    k, v, q = (_keys(rng, s, "bf16") for s in ((1, 2500, 2, 128), (1, 2500, 2, 128), (1, 1, 8, 128)))
    outs = []
    other = it.Context(0)
    for ctx in (it.Context.global_(), other):
        tensors = [it.Tensor.from_f32_as_bf16(x, x.shape, ctx) for x in (k, v, q)]
        cache = it.KvCache(1, 2, 2500, 128, 4, ctx)
        it.kv_cache_write(cache, *tensors[:2], [0])
        pos = it.upload_positions([2499], ctx)
        outs.append(it.cached_attention(tensors[2], cache, pos).numpy())
        assert ctx.lib.it_side_begin(ctx.handle) == 0
        side = it.cached_attention(tensors[2], cache, pos)
        assert ctx.lib.it_side_end(ctx.handle) == 0
        main = it.cached_attention(tensors[2], cache, pos)
        assert ctx.lib.it_side_join(ctx.handle) == 0
        outs += [side.numpy(), main.numpy()]
    for o in outs[1:]:
        assert np.array_equal(o, outs[0])


@pytest.mark.parametrize("bits", [4, 8])
def test_decoding_a_small_layer(it, bits):
    """One attention layer on 8-bit weights over a prompt and then token by token: projection, rotation, cache write,
    attention and output projection give what the same tokens give in one piece. The pieces see the same
    cached values, and a row of a product depends on that row only, so the projections agree bit for bit."""
    from irontensor_amd.train_ops import rope
    rng = np.random.default_rng(4)
    b, t, heads, hkv, d, hid = 2, 24, 4, 2, 64, 96
    wqkv = it.LinearI8.from_weight(it.Tensor.from_f32_slice(rng.standard_normal(((heads + 2 * hkv) * d, hid)) * 0.1,
                                                            [(heads + 2 * hkv) * d, hid]))
    wo = it.LinearI8.from_weight(it.Tensor.from_f32_slice(rng.standard_normal((hid, heads * d)) * 0.1, [hid, heads * d]))
    x = rng.standard_normal((b, t, hid)).astype(np.float32)

    def run(cache, part, at):
        n = part.shape[1]
        y = wqkv.forward(it.Tensor.from_f32_slice(part, part.shape)).numpy().reshape(b, n, -1, d)
        q, k, v = (it.Tensor.from_f32_slice(np.ascontiguousarray(y[:, :, s]), [b, n, y[:, :, s].shape[2], d])
                   for s in (slice(0, heads), slice(heads, heads + hkv), slice(heads + hkv, None)))
        q, k = rope(q, 10000.0, at), rope(k, 10000.0, at)
        it.kv_cache_write(cache, k, v, [at] * b)
        o = it.cached_attention(q, cache, [at] * b)
        return o.numpy(), wo.forward(o.view([b, n, heads * d])).numpy()

    whole = it.KvCache(b, hkv, t, d, bits)
    o1, y1 = run(whole, x, 0)
    parts = it.KvCache(b, hkv, t, d, bits)
    got = [run(parts, x[:, :7], 0)] + [run(parts, x[:, i:i + 1], i) for i in range(7, t)]
    for a, c in zip(it.kv_cache_read(whole, 0, t), it.kv_cache_read(parts, 0, t)):
        assert np.array_equal(a.numpy(), c.numpy())
    o2 = np.concatenate([g[0] for g in got], 1)
    # the same sums in another order: FP32's accuracy, and up to a code of the output projection's input
    assert np.abs(o1 - o2).max() <= 1e-5 * np.abs(o1).max()
    y2 = np.concatenate([g[1] for g in got], 1)
    assert np.abs(y1 - y2).max() <= 2e-2 * np.abs(y1).max()
