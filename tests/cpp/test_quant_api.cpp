// The quantised serving operators through the C++ host API: refusals (--cpu) and small runs on the GPU.
#include <cmath>
#include <cstdio>
#include <cstring>

#include "irontensor.hpp"

using namespace irontensor;

static int g_failed = 0, g_passed = 0;
static void expect(bool ok, const char *what) {
    ok ? ++g_passed : ++g_failed;
    if (!ok) std::printf("FAIL %s\n", what);
}
template <typename E, typename F>
static void throws(F f, const char *what) {
    try {
        f();
    } catch (const E &) {
        expect(true, what);
        return;
    } catch (...) {
    }
    expect(false, what);
}

static void cpu_tests() {
    size_t n = 0;
    expect(it_kv_cache_bytes(4, 2, 3, 65, 128, &n) == IT_OK && n == 2 * 3 * 128 * (128 + 8 + 2), "cache bytes");
    throws<InvalidValue>([] { KvCache c(1, 1, 8, 96); }, "head_dim 96");
    throws<InvalidValue>([] { KvCache c(1, 1, 8, 64, 5); }, "5 bits");
}

static void gpu_tests() {
    // Values that are whole numbers of steps read back exactly: 7 and -7 fix the step at 1.
    const size_t b = 2, n = 3, h = 2, d = 64;
    std::vector<float> k(b * n * h * d), v(k.size());
    for (size_t i = 0; i < k.size(); ++i) {
        k[i] = i % 32 == 0 ? 7.f : (float)((int)(i % 15) - 7);
        v[i] = i % 64 == 1 ? -7.f : (float)((int)(i % 13) - 6);
    }
    KvCache cache(b, h, 8, d);
    const Tensor tk = Tensor::from_f32_slice(k, {b, n, h, d}), tv = Tensor::from_f32_slice(v, {b, n, h, d});
    const Tensor start = upload_positions({1, 5});
    kv_cache_write(cache, tk, tv, start);
    const auto kv = kv_cache_read(cache, 0, 8);
    const std::vector<float> rk = kv.first.as_f32_slice(), rv = kv.second.as_f32_slice();
    bool same = true, rest = true;
    for (size_t s = 0; s < b; ++s)
        for (size_t t = 0; t < 8; ++t)
            for (size_t e = 0; e < h * d; ++e) {
                const size_t at = (s * 8 + t) * h * d + e, from = s ? 5 : 1;
                if (t >= from && t < from + n) {
                    const size_t src = (s * n + t - from) * h * d + e;
                    same = same && rk[at] == k[src] && rv[at] == v[src];
                } else {
                    rest = rest && rk[at] == 0.f && rv[at] == 0.f;
                }
            }
    expect(same, "written tokens read back");
    expect(rest, "other positions read zero");
    // One visible key: the output is its value, for both query heads of a cache head.
    KvCache one(1, 1, 4, d, 8);
    const Tensor k1 = Tensor::from_f32_slice(std::vector<float>(d, 1.f), {1, 1, 1, d});
    std::vector<float> v1(d);
    for (size_t e = 0; e < d; ++e) v1[e] = (float)e * 2.f;
    v1[0] = 127.f;
    kv_cache_write(one, k1, Tensor::from_f32_slice(v1, {1, 1, 1, d}), upload_positions({0}));
    const Tensor q = Tensor::from_f32_slice(std::vector<float>(2 * d, 0.5f), {1, 1, 2, d});
    const std::vector<float> o = cached_attention(q, one, upload_positions({0})).as_f32_slice();
    bool equal = true;
    for (size_t e = 0; e < 2 * d; ++e) equal = equal && std::fabs(o[e] - v1[e % d]) <= 1e-5f * 127.f;
    expect(equal, "attention over one key");
    throws<ShapeMismatch>([&] { cached_attention(q, cache, start); }, "batch of another cache");
    throws<ShapeMismatch>([&] { kv_cache_write(cache, tk, tv, upload_positions({0})); }, "one position for two sequences");
    // An 8-bit layer on whole numbers is exact: x in steps of 1 (127 in every row), w likewise.
    const size_t rows = 5, in = 20, out = 7;
    std::vector<float> x(rows * in), w(out * in), bias(out);
    for (size_t i = 0; i < x.size(); ++i) x[i] = i % in == 0 ? 127.f : (float)((int)(i * 7 % 31) - 15);
    for (size_t i = 0; i < w.size(); ++i) w[i] = i % in == 3 ? -127.f : (float)((int)(i * 5 % 23) - 11);
    for (size_t i = 0; i < out; ++i) bias[i] = (float)i;
    const Int8Matrix qw = quantize_i8(Tensor::from_f32_slice(w, {out, in}));
    const Tensor tb = Tensor::from_f32_slice(bias, {out}), tx = Tensor::from_f32_slice(x, {rows, in});
    const std::vector<float> y = linear_i8(tx, qw, &tb).as_f32_slice(), y2 = matmul_i8(quantize_i8(tx), qw, &tb).as_f32_slice();
    bool exact = true;
    for (size_t r = 0; r < rows; ++r)
        for (size_t c = 0; c < out; ++c) {
            double s = bias[c];
            for (size_t i = 0; i < in; ++i) s += (double)x[r * in + i] * w[c * in + i];
            exact = exact && std::fabs(y[r * out + c] - s) <= 4e-7 * std::fabs(s) + 1e-6 && y[r * out + c] == y2[r * out + c];
        }
    expect(exact, "8-bit layer");
    throws<InnerDimensionMismatch>([&] { linear_i8(Tensor::zeros({2, 21}, Precision::FP32), qw); }, "inner dimension");
}

int main(int argc, char **argv) {
    cpu_tests();
    if (!(argc > 1 && std::strcmp(argv[1], "--cpu") == 0)) {
        if (it_device_count() == 0) {
            std::printf("FAIL no HIP device visible\n");
            return 2;
        }
        gpu_tests();
    }
    std::printf("%d passed, %d failed\n", g_passed, g_failed);
    return g_failed ? 1 : 0;
}
