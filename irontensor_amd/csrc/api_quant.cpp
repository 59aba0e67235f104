// C ABI entry points of the 8- and 4-bit serving operators: argument validation, library-owned scratch and
// profiler keys. Every entry runs with the context's device current and lets no exception out.
#include <cmath>
#include <cstdint>
#include <exception>
#include <string>

#include "quant.hpp"

using it::fail;

namespace {

std::string i64(int64_t v) { return std::to_string((long long)v); }

constexpr int64_t MAX_DIM = (int64_t)1 << 40;      // sizes whose products are formed in 64 bits stay below this
constexpr int64_t MAX_REGION = (int64_t)1 << 31;   // bytes of a (sequence, head)
constexpr int64_t MAX_GRID = 0x7fffffff;
constexpr int64_t MAX_K = 131056;                  // 128^2 K < 2^31: the 32-bit sums of an 8-bit product

// The context's device, current while this lives.
struct OnDevice {
    int before = -1;
    explicit OnDevice(const it_context *ctx) {
        int d = -1;
        if (hipGetDevice(&d) != hipSuccess) d = -1;
        if (d != ctx->device) {
            before = d;
            (void)hipSetDevice(ctx->device);
        }
    }
    ~OnDevice() {
        if (before >= 0) (void)hipSetDevice(before);
    }
};

// Runs `f`, a C++ exception becoming a status.
template <typename F>
it_status guarded(const char *op, F f) {
    try {
        return f();
    } catch (const std::bad_alloc &) {
        return it::fail(IT_ERR_OOM, "out of host memory");
    } catch (const std::exception &e) {
        return fail(IT_ERR_HIP, std::string(op) + ": " + e.what());
    } catch (...) {
        return fail(IT_ERR_HIP, std::string(op) + ": unexpected exception");
    }
}

// One launch under the profiler.
template <typename K, typename F>
it_status profiled(it_context *ctx, K key, F launch) {
    if (!ctx->profiling) return launch();
    const std::string k = key();
    hipEvent_t ev = nullptr;
    it::profile_begin(ctx, k, &ev);
    const it_status st = launch();
    it::profile_end(ctx, k, ev);
    return st;
}

bool f32_or_bf16(it_dtype d) { return d == IT_F32 || d == IT_BF16; }

it_status bad_dtype(const char *op) {
    return fail(IT_ERR_PRECISION, std::string(op) + ": precision mismatch, expected FP32 or BF16");
}

// The cache's sizes; *g without data.
it_status geometry(const char *op, int bits, int64_t batch, int64_t kv_heads, int64_t capacity, int64_t head_dim,
                   it::CacheGeom *g) {
    if (bits != 4 && bits != 8) return fail(IT_ERR_INVALID, std::string(op) + ": bits must be 4 or 8, got " + i64(bits));
    if (batch < 0 || kv_heads < 0 || capacity < 0) return fail(IT_ERR_INVALID, std::string(op) + ": negative size");
    if (head_dim != 64 && head_dim != 128 && head_dim != 256)
        return fail(IT_ERR_DIMS, std::string(op) + ": unsupported dimensions, head_dim must be 64, 128 or 256, got " + i64(head_dim));
    if (batch > MAX_GRID || kv_heads > MAX_GRID || capacity > MAX_DIM || (batch > 0 && kv_heads > MAX_GRID / batch))
        return fail(IT_ERR_DIMS, std::string(op) + ": cache too large");
    const int64_t T = (capacity + it::CACHE_TILE - 1) / it::CACHE_TILE * it::CACHE_TILE;
    const int64_t row = head_dim * bits / 8;
    g->data = nullptr;
    g->v_off = T * row;
    g->ks_off = 2 * T * row;
    g->vs_off = g->ks_off + T * (head_dim / it::CACHE_GROUP) * 2;
    g->region = g->vs_off + T * 2;
    if (g->region >= MAX_REGION)
        return fail(IT_ERR_DIMS, std::string(op) + ": a head's cache must stay below 2 GiB, got " + i64(g->region) + " bytes");
    g->capacity = capacity;
    g->batch = batch;
    g->kv_heads = kv_heads;
    g->bits = bits;
    g->head_dim = (int)head_dim;
    return IT_OK;
}

it_status geometry(const char *op, const it_kv_cache *c, it::CacheGeom *g) {
    if (!c) return fail(IT_ERR_NULL, std::string(op) + ": cache is NULL");
    if (const it_status st = geometry(op, c->bits, c->batch, c->kv_heads, c->capacity, c->head_dim, g); st != IT_OK) return st;
    g->data = (char *)c->data;
    if (g->region * g->batch * g->kv_heads > 0 && !c->data) return fail(IT_ERR_NULL, std::string(op) + ": the cache's data is NULL");
    if ((uintptr_t)c->data % 16 != 0) return fail(IT_ERR_INVALID, std::string(op) + ": the cache's data must be 16-byte aligned");
    return IT_OK;
}

// `heads` heads a sequence over `rows` rows; NULL: [batch, heads, rows, head_dim] contiguous.
it_status head_layout(const char *op, const it_attn_layout *l, int64_t heads, int64_t rows, int64_t d,
                      it::HeadLayout *out) {
    if (!l) {
        *out = it::HeadLayout{heads * rows * d, rows * d, d};
        return IT_OK;
    }
    if (l->heads < 1 || l->row_stride < d || l->batch_stride < 0 || l->head_stride < 0 || l->row_stride > MAX_DIM ||
        l->batch_stride > MAX_DIM || l->head_stride > MAX_DIM)
        return fail(IT_ERR_INVALID, std::string(op) + ": bad layout strides");
    if (l->heads != heads && l->heads != 1)
        return fail(IT_ERR_SHAPE, std::string(op) + ": shape mismatch, the layout's heads must be 1 or " + i64(heads) + ", got " + i64(l->heads));
    // One head a batch stride ([batch * heads, ..]): the same address with the strides of a sequence and a head.
    *out = l->heads == heads ? it::HeadLayout{l->batch_stride, l->head_stride, l->row_stride}
                             : it::HeadLayout{heads * l->batch_stride, l->batch_stride, l->row_stride};
    return IT_OK;
}

// Whether the address ranges of two matrices meet: `rows` rows of `cols` elements of `size` bytes.
bool ranges_meet(const void *x, int64_t ldx, int64_t xcols, const void *y, int64_t ldy, int64_t ycols, int64_t rows, size_t size) {
    const uintptr_t x0 = (uintptr_t)x, x1 = x0 + (size_t)((rows - 1) * ldx + xcols) * size;
    const uintptr_t y0 = (uintptr_t)y, y1 = y0 + (size_t)((rows - 1) * ldy + ycols) * size;
    return x0 < y1 && y0 < x1;
}

}  // namespace

extern "C" {

it_status it_kv_cache_bytes(int bits, int64_t batch, int64_t kv_heads, int64_t capacity, int64_t head_dim,
                            size_t *bytes) {
    return guarded("kv_cache", [&]() -> it_status {
        if (!bytes) return fail(IT_ERR_NULL, "kv_cache: bytes is NULL");
        it::CacheGeom g;
        if (const it_status st = geometry("kv_cache", bits, batch, kv_heads, capacity, head_dim, &g); st != IT_OK) return st;
        *bytes = (size_t)g.region * (size_t)(batch * kv_heads);
        return IT_OK;
    });
}

it_status it_kv_cache_write(it_context *ctx, it_dtype dtype, const it_kv_cache *cache, int64_t n,
                            const it_attn_layout *kv_layout, const void *K, const void *V, const int32_t *start,
                            const int32_t *count) {
    const char *op = "kv_cache_write";
    return guarded(op, [&]() -> it_status {
        if (!ctx) return fail(IT_ERR_NULL, std::string(op) + ": ctx is NULL");
        if (!f32_or_bf16(dtype)) return bad_dtype(op);
        it::CacheMoveArgs a{};
        if (const it_status st = geometry(op, cache, &a.c); st != IT_OK) return st;
        if (n < 0) return fail(IT_ERR_INVALID, std::string(op) + ": negative size");
        if (const it_status st = head_layout(op, kv_layout, a.c.kv_heads, n, a.c.head_dim, &a.lay); st != IT_OK) return st;
        if (n == 0 || a.c.batch * a.c.kv_heads == 0 || a.c.capacity == 0) return IT_OK;
        if (!K || !V || !start) return fail(IT_ERR_NULL, std::string(op) + ": NULL buffer");
        a.K = K;
        a.V = V;
        a.start = start;
        a.count = count;
        a.n = n;
        a.blocks = n > MAX_DIM ? MAX_DIM : (n + 3 + 3) / 4;
        if (a.blocks > MAX_GRID || a.c.batch * a.c.kv_heads > MAX_GRID / a.blocks)
            return fail(IT_ERR_DIMS, std::string(op) + ": too many tokens");
        const OnDevice dev(ctx);
        return profiled(
            ctx, [&] { return "kv_write" + i64(a.c.bits) + "[" + i64(a.c.batch * a.c.kv_heads) + "x" + i64(n) + "x" + i64(a.c.head_dim) + "]"; },
            [&] { return it::launch_cache_write(ctx->stream, dtype == IT_BF16, a); });
    });
}

it_status it_kv_cache_read(it_context *ctx, it_dtype dtype, const it_kv_cache *cache, int64_t begin, int64_t n,
                           const it_attn_layout *kv_layout, void *K, void *V) {
    const char *op = "kv_cache_read";
    return guarded(op, [&]() -> it_status {
        if (!ctx) return fail(IT_ERR_NULL, std::string(op) + ": ctx is NULL");
        if (!f32_or_bf16(dtype)) return bad_dtype(op);
        it::CacheMoveArgs a{};
        if (const it_status st = geometry(op, cache, &a.c); st != IT_OK) return st;
        if (begin < 0 || n < 0) return fail(IT_ERR_INVALID, std::string(op) + ": negative size");
        if (begin > a.c.capacity || n > a.c.capacity - begin)
            return fail(IT_ERR_SHAPE, std::string(op) + ": tokens " + i64(begin) + " + " + i64(n) + " pass the capacity " + i64(a.c.capacity));
        if (const it_status st = head_layout(op, kv_layout, a.c.kv_heads, n, a.c.head_dim, &a.lay); st != IT_OK) return st;
        if (n == 0 || a.c.batch * a.c.kv_heads == 0) return IT_OK;
        if (!K || !V) return fail(IT_ERR_NULL, std::string(op) + ": NULL buffer");
        a.Ko = K;
        a.Vo = V;
        a.begin = begin;
        a.n = n;
        a.blocks = (begin % 4 + n + 3) / 4;
        if (a.c.batch * a.c.kv_heads > MAX_GRID / a.blocks) return fail(IT_ERR_DIMS, std::string(op) + ": too many tokens");
        const OnDevice dev(ctx);
        return profiled(
            ctx, [&] { return "kv_read" + i64(a.c.bits) + "[" + i64(a.c.batch * a.c.kv_heads) + "x" + i64(n) + "x" + i64(a.c.head_dim) + "]"; },
            [&] { return it::launch_cache_read(ctx->stream, dtype == IT_BF16, a); });
    });
}

it_status it_cached_attention(it_context *ctx, it_dtype dtype, const it_kv_cache *cache, int64_t heads, int64_t n,
                              float scale, const it_attn_layout *q_layout, const it_attn_layout *o_layout,
                              const void *Q, const int32_t *start, const int32_t *count, void *O) {
    const char *op = "cached_attention";
    return guarded(op, [&]() -> it_status {
        if (!ctx) return fail(IT_ERR_NULL, std::string(op) + ": ctx is NULL");
        if (!f32_or_bf16(dtype)) return bad_dtype(op);
        it::CachedAttnArgs a{};
        if (const it_status st = geometry(op, cache, &a.c); st != IT_OK) return st;
        if (heads < 0 || n < 0) return fail(IT_ERR_INVALID, std::string(op) + ": negative size");
        if (!(scale > 0.f) || !std::isfinite(scale)) return fail(IT_ERR_INVALID, std::string(op) + ": scale must be finite and positive");
        if (heads > 0 && (a.c.kv_heads == 0 || heads % a.c.kv_heads != 0))
            return fail(IT_ERR_SHAPE, std::string(op) + ": shape mismatch, expected heads divisible by the cache's " + i64(a.c.kv_heads) + ", got " + i64(heads));
        if (heads > MAX_GRID / 2 || (heads > 0 && n > MAX_GRID / 2 / heads)) return fail(IT_ERR_DIMS, std::string(op) + ": too many queries");
        if (const it_status st = head_layout(op, q_layout, heads, n, a.c.head_dim, &a.ql); st != IT_OK) return st;
        if (const it_status st = head_layout(op, o_layout, heads, n, a.c.head_dim, &a.ol); st != IT_OK) return st;
        if (!o_layout) a.ol = a.ql;
        if (n == 0 || heads == 0 || a.c.batch == 0) return IT_OK;
        if (!Q || !O || !start) return fail(IT_ERR_NULL, std::string(op) + ": NULL buffer");
        a.Q = Q;
        a.O = O;
        a.start = start;
        a.count = count;
        a.n = n;
        a.share = (int)(heads / a.c.kv_heads);
        a.rows = (int)(n * a.share);
        a.scale_log2 = scale * 1.4426950408889634f;
        const int64_t floats = it::plan_cached_attention(a, dtype == IT_BF16, ctx->num_cus);
        if (a.c.batch * a.c.kv_heads > MAX_GRID / a.row_blocks / a.splits) return fail(IT_ERR_DIMS, std::string(op) + ": too many queries");
        const OnDevice dev(ctx);
        if (floats > 0) {
            // Without scratch (a capture before any eager call, no memory) every row block takes all its keys.
            void *part = nullptr;
            if (it::ensure_scratch(ctx, (size_t)floats * sizeof(float), &part) == IT_OK && it::ensure_counters(ctx, &a.counters) == IT_OK) {
                a.part = (float *)part;
            } else {
                it::clear_error();
                a.splits = 1;
            }
        }
        return profiled(
            ctx, [&] { return "cached_attn" + i64(a.c.bits) + "[" + i64(a.c.batch) + "x" + i64(heads) + "/" + i64(a.c.kv_heads) + "x" + i64(n) + "x" + i64(a.c.head_dim) + ",T=" + i64(a.c.capacity) + "]"; },
            [&] { return it::launch_cached_attention(ctx->stream, dtype == IT_BF16, a); });
    });
}

it_status it_quantize_i8(it_context *ctx, it_dtype dtype, int64_t rows, int64_t cols, const void *X, int64_t ldx,
                         int8_t *codes, int64_t ldc, float *steps) {
    const char *op = "quantize_i8";
    return guarded(op, [&]() -> it_status {
        if (!ctx) return fail(IT_ERR_NULL, std::string(op) + ": ctx is NULL");
        if (!f32_or_bf16(dtype)) return bad_dtype(op);
        if (rows < 0 || cols < 0) return fail(IT_ERR_INVALID, std::string(op) + ": negative size");
        if (rows > MAX_GRID || cols > MAX_DIM || ldx > MAX_DIM || ldc > MAX_DIM) return fail(IT_ERR_DIMS, std::string(op) + ": matrix too large");
        if (ldx < cols) return fail(IT_ERR_INVALID, std::string(op) + ": ldx smaller than cols");
        if (ldc % 16 != 0 || ldc < cols) return fail(IT_ERR_INVALID, std::string(op) + ": ldc must be a multiple of 16 and at least cols");
        if (rows == 0) return IT_OK;
        if (!steps || (cols > 0 && (!X || !codes))) return fail(IT_ERR_NULL, std::string(op) + ": NULL buffer");
        if ((uintptr_t)codes % 16 != 0) return fail(IT_ERR_INVALID, std::string(op) + ": codes must be 16-byte aligned");
        const OnDevice dev(ctx);
        return profiled(
            ctx, [&] { return "quantize_i8[" + i64(rows) + "x" + i64(cols) + "]"; },
            [&] { return it::launch_quantize_i8(ctx->stream, dtype == IT_BF16, rows, cols, X, ldx, codes, ldc, steps); });
    });
}

namespace {

it_status check_gemm_i8(const char *op, int64_t M, int64_t N, int64_t K, const int8_t *A, int64_t lda, const float *sA,
                        const int8_t *B, int64_t ldb, const float *sB, const void *C, int64_t ldc) {
    if (M < 0 || N < 0 || K < 0) return fail(IT_ERR_INVALID, std::string(op) + ": negative size");
    if (K > MAX_K) return fail(IT_ERR_DIMS, std::string(op) + ": K must be at most " + i64(MAX_K) + " (32-bit sums), got " + i64(K));
    if (lda < K || ldb < K || lda % 16 != 0 || ldb % 16 != 0)
        return fail(IT_ERR_INVALID, std::string(op) + ": leading dimensions of the codes must be multiples of 16 and at least K");
    if (ldc < N) return fail(IT_ERR_INVALID, std::string(op) + ": ldc smaller than N");
    // 256 rows of an operand are addressed with 31-bit offsets.
    if (lda > (1 << 22) || ldb > (1 << 22) || ldc > MAX_DIM || M > MAX_DIM || N > MAX_DIM || (M + 15) / 16 > MAX_GRID / ((N + 15) / 16 + 1))
        return fail(IT_ERR_DIMS, std::string(op) + ": matrix too large");
    if (M == 0 || N == 0) return IT_OK;
    if (!C || !sA || !sB || (K > 0 && (!A || !B))) return fail(IT_ERR_NULL, std::string(op) + ": NULL buffer");
    if ((uintptr_t)A % 16 != 0 || (uintptr_t)B % 16 != 0) return fail(IT_ERR_INVALID, std::string(op) + ": codes must be 16-byte aligned");
    return IT_OK;
}

}  // namespace

it_status it_gemm_i8(it_context *ctx, it_dtype dtype_out, int64_t M, int64_t N, int64_t K, const int8_t *A, int64_t lda,
                     const float *steps_a, const int8_t *B, int64_t ldb, const float *steps_b, const float *bias, void *C,
                     int64_t ldc) {
    const char *op = "gemm_i8";
    return guarded(op, [&]() -> it_status {
        if (!ctx) return fail(IT_ERR_NULL, std::string(op) + ": ctx is NULL");
        if (!f32_or_bf16(dtype_out)) return bad_dtype(op);
        if (K % 16 != 0) return fail(IT_ERR_DIMS, std::string(op) + ": K must be a multiple of 16 (codes padded with zeros), got " + i64(K));
        if (const it_status st = check_gemm_i8(op, M, N, K, A, lda, steps_a, B, ldb, steps_b, C, ldc); st != IT_OK) return st;
        if (M == 0 || N == 0) return IT_OK;
        const OnDevice dev(ctx);
        const it::GemmI8Args a{A, B, steps_a, steps_b, bias, C, M, N, K, lda, ldb, ldc, dtype_out == IT_BF16, 0, 0, nullptr, 0, 0};
        return profiled(
            ctx, [&] { return "gemm_i8[" + i64(M) + "x" + i64(N) + "x" + i64(K) + "]"; },
            [&] { return it::launch_gemm_i8(ctx, a); });
    });
}

it_status it_linear_i8(it_context *ctx, it_dtype dtype, int64_t M, int64_t N, int64_t K, const void *X, int64_t ldx,
                       const int8_t *W, int64_t ldw, const float *steps_w, const float *bias, void *Y, int64_t ldy) {
    const char *op = "linear_i8";
    return guarded(op, [&]() -> it_status {
        if (!ctx) return fail(IT_ERR_NULL, std::string(op) + ": ctx is NULL");
        if (!f32_or_bf16(dtype)) return bad_dtype(op);
        const int64_t max_k = MAX_K / 128 * 128;
        if (K > max_k) return fail(IT_ERR_DIMS, std::string(op) + ": K must be at most " + i64(max_k) + " (32-bit sums), got " + i64(K));
        if (K < 0) return check_gemm_i8(op, M, N, K, nullptr, 0, nullptr, nullptr, 0, nullptr, nullptr, 0);
        // Whole k-tiles of 128 where the weight's rows have them (it_quantize_i8 pads rows that far).
        const int64_t k128 = (K + 127) / 128 * 128, kp = ldw >= k128 ? k128 : (K + 15) / 16 * 16;
        // The activations' codes go to scratch: 16 is any non-NULL aligned address for the check.
        if (const it_status st = check_gemm_i8(op, M, N, kp, (const int8_t *)16, kp, (const float *)16, W, ldw, steps_w, Y, ldy); st != IT_OK) return st;
        if (ldx < K || ldx > MAX_DIM) return fail(IT_ERR_INVALID, std::string(op) + ": ldx smaller than K");
        if (M == 0 || N == 0) return IT_OK;
        if (K > 0 && !X) return fail(IT_ERR_NULL, std::string(op) + ": NULL buffer");
        if (M > MAX_GRID) return fail(IT_ERR_DIMS, std::string(op) + ": matrix too large");
        const OnDevice dev(ctx);
        // In one launch, blocks still read X when others write Y: over X only where the codes come from scratch.
        if (it::gemv_i8_x_applicable(M, kp) && !ranges_meet(X, ldx, K, Y, ldy, N, M, dtype == IT_BF16 ? 2 : 4)) {
            const it::GemmI8Args a{nullptr, W, nullptr, steps_w, bias, Y, M, N, kp, kp, ldw, ldy, dtype == IT_BF16, 0, 0, X, ldx, (int)K};
            return profiled(
                ctx, [&] { return "linear_i8[" + i64(M) + "x" + i64(N) + "x" + i64(K) + "]"; },
                [&] { return it::launch_gemv_i8_x(ctx->stream, dtype == IT_BF16, a); });
        }
        const size_t steps_at = ((size_t)(M * kp) + 255) / 256 * 256;
        void *ws = nullptr;
        if (const it_status st = it::ensure_scratch(ctx, steps_at + (size_t)M * sizeof(float), &ws); st != IT_OK) return st;
        int8_t *codes = (int8_t *)ws;
        float *steps = (float *)((char *)ws + steps_at);
        const it_status qs = profiled(
            ctx, [&] { return "quantize_i8[" + i64(M) + "x" + i64(K) + "]"; },
            [&] { return it::launch_quantize_i8(ctx->stream, dtype == IT_BF16, M, K, X, ldx, codes, kp, steps); });
        if (qs != IT_OK) return qs;
        const it::GemmI8Args a{codes, W, steps, steps_w, bias, Y, M, N, kp, kp, ldw, ldy, dtype == IT_BF16, 0, 0, nullptr, 0, 0};
        return profiled(
            ctx, [&] { return "gemm_i8[" + i64(M) + "x" + i64(N) + "x" + i64(K) + "]"; },
            [&] { return it::launch_gemm_i8(ctx, a); });
    });
}

}  // extern "C"
