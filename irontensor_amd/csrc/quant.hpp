// What the 8- and 4-bit operators share: the quantiser, the layout of the key/value cache, and the
// arguments of their launches.
#pragma once

#include "internal.hpp"
#include "mfma.hpp"

namespace it {

// ------------------------------------------------------------------ the quantiser

// A group of values shares the step s = max|x| * (1 / L) (L: the largest code; FP32, 1 / L rounded) and keeps
// n = rne(x / s) of the step as it is stored. A step
// below the smallest normal number is stored as 0 (the group reads as zeros); a group that holds a NaN or
// an infinity gets s = NaN and codes 0, so that all of it reads as NaN.
constexpr float QUANT_TINY = 1.17549435e-38f;  // 2^-126

// The step from the largest |x|, given as its bits (compared as integers they order NaN above infinity
// above every number, so one integer maximum finds non-finite values too). BF16: the cache's steps are
// rounded to BF16, whose 8 significand bits cost nothing: codes are chosen for the step as stored. L times
// its rounding error stays below half a step for L = 7; for L = 127 a quotient up to 127.5 is clamped.
template <bool BF16>
__device__ __forceinline__ float quant_step(uint32_t maxbits, float levels) {
    if (maxbits >= 0x7f800000u) return __uint_as_float(0x7fc00000u);
    float s = __uint_as_float(maxbits) * (1.f / levels);
    if constexpr (BF16) s = bf16_to_f32(f32_to_bf16_rne(s));
    return s < QUANT_TINY ? 0.f : s;
}

// 1 / s, or 0 where every code is 0.
__device__ __forceinline__ float quant_inverse(float s) { return s > 0.f ? 1.f / s : 0.f; }

// Codes of eight values: the low byte of u[e] is rne(x[e] / s) + BIAS of the real quotient (BIAS even).
// x * inv + 3 2^22 rounds to the nearest whole number n in one FMA, off by at most one and only where the
// quotient is next to a half. The rest x - n s is exact in one FMA (its bits lie between ulp(x) and s), and so
// is its comparison with s / 2: above it the code is the next one, at it the even one. That repair is a
// branch that FP32 values hardly ever take and BF16 ones, which hit halves exactly, in every third pair of a
// wave. A quotient never passes the largest code L by a half: s is within 2^-8 (BF16) of max|x| / L, and
// 127 / (1 - 2^-8) (1 + 2^-22) < 127.5.
template <int BIAS>
__device__ __forceinline__ void quant_codes(const float (&x)[8], float s, float inv, uint32_t (&u)[8]) {
    constexpr float MAGIC = 12582912.f + BIAS;  // 3 2^22 + BIAS
    const bool live = inv > 0.f;
    const float h = live ? 0.5f * s : INFINITY;
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
        float t[2], r[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            t[i] = fmaf(x[e + i], inv, MAGIC);
            r[i] = fmaf(MAGIC - t[i], s, x[e + i]);
        }
        if (__any(fmaxf(fabsf(r[0]), fabsf(r[1])) >= h)) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const float a = fabsf(r[i]);
                if (a > h || (a == h && (__float_as_uint(t[i]) & 1u))) t[i] += copysignf(1.f, r[i]);
            }
        }
        u[e] = __float_as_uint(t[0]);
        u[e + 1] = __float_as_uint(t[1]);
    }
    if (__any(!live)) {  // a group without a step: infinities times 0 must not leave codes
#pragma unroll
        for (int e = 0; e < 8; ++e) u[e] = live ? u[e] : (uint32_t)BIAS;
    }
}

// The low bytes of a, b, c, d, first to last.
__device__ __forceinline__ uint32_t bytes4(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    const uint32_t ab = __builtin_amdgcn_perm(b, a, 0x0c0c0400u), cd = __builtin_amdgcn_perm(d, c, 0x04000c0cu);
    return ab | cd;
}

__device__ __forceinline__ uint32_t abs_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }

// ------------------------------------------------------------------ the cache

// One region for each (sequence, head): key codes, value codes, key steps, value steps, all BF16 steps.
// T = capacity rounded up to CACHE_TILE tokens, R = head_dim * bits / 8 bytes of codes a token:
//   key codes    [T][R]: a token's row holds, for lane group g = 0..3 of an MFMA operand, channels
//                32 s + 8 g .. + 7 of s = 0, 1, ..: a lane's operands of every 32-channel step are
//                consecutive bytes. In 4 bits the eight codes of an octet are one word, even channel e at
//                nibble e / 2 and odd e at nibble e / 2 + 4, so that a shift and a mask give pairs.
//   value codes  [T / 4][head_dim / 4][4 tokens][4 codes] in 4 bits, [T / 4][head_dim][4 tokens] in 8: the
//                four tokens that a lane's operand needs of a channel are together, and a token's codes are
//                whole bytes of their own (2, or 1), so appending one rewrites nobody else's.
//   key steps    [T][head_dim / 32], value steps [T].
// Codes are stored biased by 8 (128): an all-zero region reads as zeros, its steps being zero.
constexpr int64_t CACHE_TILE = 64;
constexpr int CACHE_GROUP = 32;

struct CacheGeom {
    char *data;
    int64_t region;                   // bytes of one (sequence, head)
    int64_t v_off, ks_off, vs_off;    // value codes, key steps and value steps within it
    int64_t capacity;
    int64_t batch, kv_heads;
    int bits, head_dim;
};

// Element (sequence b, head h, row, d) of a 16- or 32-bit operand: b * bs + h * hs + row * rs + d.
struct HeadLayout {
    int64_t bs, hs, rs;
    __host__ __device__ int64_t at(int64_t b, int64_t h) const { return b * bs + h * hs; }
};

struct CacheMoveArgs {
    CacheGeom c;
    const void *K, *V;      // written from
    void *Ko, *Vo;          // read into
    HeadLayout lay;
    const int32_t *start, *count;
    int64_t begin, n;
    int64_t blocks;         // 4-token blocks of a (sequence, head) that the call may touch
    int64_t units;          // blocks of all of them
};
it_status launch_cache_write(hipStream_t s, bool bf16, const CacheMoveArgs &a);
it_status launch_cache_read(hipStream_t s, bool bf16, const CacheMoveArgs &a);

struct CachedAttnArgs {
    CacheGeom c;
    const void *Q;
    void *O;
    HeadLayout ql, ol;
    const int32_t *start, *count;
    int64_t n;              // queries of a sequence
    int share;              // query heads of one cache head
    int rows;               // n * share
    int row_tiles;          // 16-row tiles of a block
    int row_blocks, splits;
    float per_key;          // keys of a block for each key of the batch, to spread them evenly
    float scale_log2;       // scale * log2 e
    float *part;            // splits > 1: partial results, and
    int *counters;          // one arrival counter for each (sequence, head, row block)
};
// Fills in row_tiles, row_blocks, splits and per_key; the floats of `part` that the launch then needs (0: none).
int64_t plan_cached_attention(CachedAttnArgs &a, bool bf16, int num_cus);
it_status launch_cached_attention(hipStream_t s, bool bf16, const CachedAttnArgs &a);

// ------------------------------------------------------------------ 8-bit products

struct GemmI8Args {
    const int8_t *A, *B;            // [M, K], [N, K]
    const float *sA, *sB, *bias;    // [M], [N], [N] or NULL
    void *C;
    int64_t M, N, K, lda, ldb, ldc;
    int out_bf16;
    int tiles_m, tiles_n;
    const void *X;                  // launch_gemv_i8_x: the activations [M, xcols] in place of A and sA
    int64_t ldx;
    int xcols;
};
it_status launch_quantize_i8(hipStream_t s, bool bf16, int64_t rows, int64_t cols, const void *X, int64_t ldx,
                             int8_t *codes, int64_t ldc, float *steps);
it_status launch_gemm_i8(it_context *ctx, GemmI8Args a);
// Quantising and product in one launch, for few and short rows (K: the padded one).
bool gemv_i8_x_applicable(int64_t M, int64_t K);
it_status launch_gemv_i8_x(hipStream_t s, bool bf16, const GemmI8Args &a);

}  // namespace it
