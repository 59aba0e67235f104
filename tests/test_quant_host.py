"""The quantised serving operators' host side on the CPU, with the stand-in HIP runtime of test_host_dispatch.py:
which kernels a call launches, and what it does when scratch cannot be had."""
from __future__ import annotations

from test_host_dispatch import _run, fake  # noqa: F401  (the fixture)

CALLS = """
import numpy as np
def attend(cache, n, heads, start):
    q = it.Tensor.empty([cache.batch, n, heads, cache.head_dim], it.Precision.BF16)
    launches()
    it.cached_attention(q, cache, start, out=q)
    return launches()
def linear(m, n, k):
    w = it.quantize_i8(it.Tensor.empty([n, k]))
    x = it.Tensor.empty([m, k])
    launches()
    it.linear_i8(x, w)
    return launches()
"""


def test_launches(fake):  # noqa: F811
    """One launch each for a write, a read, attention (split or not) and a small layer; two for a larger layer."""
    _run(fake, CALLS + """
cache = it.KvCache(1, 2, 5000, 64, 4)
pos = it.upload_positions([7])
kv = it.Tensor.empty([1, 3, 2, 64])
launches()
it.kv_cache_write(cache, kv, kv, pos)
it.kv_cache_read(cache, 4, 9)
got = launches()
assert len(got) == 2 and "cache_write" in got[0] and "cache_read" in got[1], got
for n, heads in ((1, 2), (1, 32), (5, 6), (300, 4)):
    got = attend(cache, n, heads, pos)
    assert len(got) == 1 and "cached_attn" in got[0], got
assert ["gemv_i8_x" in x for x in linear(1, 40, 200)] == [True]
got = linear(16, 40, 2000)
assert len(got) == 2 and "quantize_rows" in got[0] and "gemv_i8" in got[1], got
got = linear(17, 40, 200)
assert len(got) == 2 and "quantize_rows" in got[0] and "gemm_i8_tile" in got[1], got
assert linear(0, 40, 200) == [] and attend(cache, 0, 4, pos) == []
""")


def test_output_over_the_input(fake):  # noqa: F811
    """A small layer whose output meets its input takes two launches: the first has read X when the second writes Y."""
    _run(fake, CALLS + """
w = it.quantize_i8(it.Tensor.empty([256, 256]))
x, y = it.Tensor.empty([4, 256]), it.Tensor.empty([4, 256])
launches()
it.linear_i8(x, w, out=y)
assert len(launches()) == 1
it.linear_i8(x, w, out=x)
got = launches()
assert len(got) == 2 and "quantize_rows" in got[0] and "gemv_i8" in got[1], got
""")


def test_launches_below_two_to_the_32_threads(fake):  # noqa: F811
    """More blocks than a launch holds are refused, and the most that it holds are not."""
    _run(fake, CALLS + """
from irontensor_amd import _lib
most, lib = 0xffffff, ctx.lib
quantize = lambda rows, cols: lib.it_quantize_i8(ctx.handle, 0, rows, cols, 256, cols, 256, cols, 256)
gemm = lambda m, n, k: lib.it_gemm_i8(ctx.handle, 0, m, n, k, 256, k, 256, 256, k, 256, None, 256, n)
linear = lambda m, n, k: lib.it_linear_i8(ctx.handle, 0, m, n, k, 256, k, 256, k, 256, None, 1 << 50, n)
def cache(units):
    return C.byref(_lib.KvCacheDesc(4, units, 1, 4, 256, 256))  # a write touches 2 blocks of 4 tokens, 8 a thread block
write = lambda units: lib.it_kv_cache_write(ctx.handle, 0, cache(units), 4, None, 256, 256, 256, None)
read = lambda units: lib.it_kv_cache_read(ctx.handle, 0, cache(units), 0, 4, None, 256, 256)
attend = lambda units: lib.it_cached_attention(ctx.handle, 0, cache(units), 1, 1, 1.0, None, None, 256, 256, None, 256)
launches()
for fn, args in ((quantize, (4 * most, 512)), (quantize, (most, 8192)), (gemm, (1, 16 * most, 16)), (linear, (1, 16 * most, 16)),
                 (write, (4 * most,)), (read, (8 * most,)), (attend, (most,))):
    assert fn(*args) == 0, (args, _lib.last_error())
    assert len(launches()) == 1
    over = list(args)
    over[1 if len(args) == 3 else 0] += 1
    assert fn(*over) == _lib.IT_ERR_DIMS and "one launch" in _lib.last_error(), (over, _lib.last_error())
    assert launches() == []
""")


def test_refused_scratch(fake):  # noqa: F811
    """Attention runs unsplit where its scratch is refused; a layer that needs scratch says so and launches nothing."""
    _run(fake, CALLS + """
cache = it.KvCache(1, 2, 5000, 64, 4)
pos = it.upload_positions([7])
x, w = it.Tensor.empty([40, 300]), it.quantize_i8(it.Tensor.empty([50, 300]))
y, q = it.Tensor.empty([40, 50]), it.Tensor.empty([1, 1, 2, 64])
launches()
fake.fake_hip_limit(1 << 20)
it.cached_attention(q, cache, pos, out=q)
got = launches()
assert len(got) == 1 and "cached_attn" in got[0], got
assert ctx.lib.it_mem_scratch(ctx.handle) == 0
try:
    it.linear_i8(x, w, out=y)
    raise SystemExit("not refused")
except it.DeviceError as e:
    assert "out of device memory" in str(e)
assert launches() == []
fake.fake_hip_limit((1 << 64) - 1)
it.linear_i8(x, w, out=y)
it.cached_attention(q, cache, pos, out=q)
assert len(launches()) == 3 and ctx.lib.it_mem_scratch(ctx.handle) > 0
""")


def test_capture_without_scratch(fake):  # noqa: F811
    """A capture before any eager call records attention unsplit and refuses a layer that needs scratch."""
    _run(fake, CALLS + """
cache = it.KvCache(1, 2, 5000, 64, 4)
pos = it.upload_positions([7])
x, w = it.Tensor.empty([40, 300]), it.quantize_i8(it.Tensor.empty([50, 300]))
y, q = it.Tensor.empty([40, 50]), it.Tensor.empty([1, 1, 2, 64])
launches()
assert ctx.lib.it_capture_begin(ctx.handle) == 0
it.cached_attention(q, cache, pos, out=q)
try:
    it.linear_i8(x, w, out=y)
    raise SystemExit("not refused")
except it.InvalidValue as e:
    assert "run the work once before capturing" in str(e)
g = C.c_void_p()
assert ctx.lib.it_capture_end(ctx.handle, C.byref(g)) == 0
assert len(launches()) == 1
ctx.lib.it_graph_destroy(g)
""")
