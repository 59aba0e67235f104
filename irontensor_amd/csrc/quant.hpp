// What the 8- and 4-bit operators' host code and kernels share: the layout of the key/value cache and the
// arguments of the launches.
#pragma once

#include <string>

#include "internal.hpp"

namespace it {

// A launch holds fewer than 2^32 threads: at most this many blocks of 256.
constexpr int64_t MAX_BLOCKS = 0xffffff;
inline it_status check_blocks(const char *op, int64_t blocks) {
    if (blocks <= MAX_BLOCKS) return IT_OK;
    return fail(IT_ERR_DIMS, std::string(op) + ": too large for one launch, " + std::to_string((long long)blocks) + " blocks");
}

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
    constexpr int64_t at(int64_t b, int64_t h) const { return b * bs + h * hs; }
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
