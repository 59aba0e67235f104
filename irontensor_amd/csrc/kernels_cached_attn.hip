// Attention of n new queries a sequence over the quantised key/value cache: n = 1 is a decoding step. No
// counterpart in the reference, whose decoding has no cache.
//
//   s_ij = scale q_i . k_j for keys j <= start + i,  o_i = sum_j softmax_j(s_ij) v_j
//
// in one pass over the cache (running maximum m and sum l of every row). The `share` query heads of a cache
// head and the n queries are the rows of one matrix, row = query * share + head, so that a cached token is
// read once for 16 rows at a time.
//
//   * Scores: S^T = K Q^T by v_mfma_f32_16x16x32_bf16, one for each 32-channel group of 16 tokens. The codes
//     are whole numbers below 2^8, exact in BF16, so a product's only roundings are FP32 sums; the group's
//     step multiplies the FP32 result, S += step * C.
//   * A lane of C holds one row (query) and four tokens, so the row statistics need two lane exchanges, and
//     its probabilities of two 16-token halves are the operand of the next product without moving:
//     O^T = V^T P^T, the value's step multiplied into p before p is rounded.
//   * BF16 queries: 4-bit codes become BF16 by one shift and one and-or a pair: 0x4180 | code << 3 is
//     16 + code. The offset (16 + 8) leaves with the queries' sums, C starting from -24 sum(q), and for the
//     values with the sum of the rounded probabilities (a product with ones). 8-bit codes are converted,
//     128 too large. P is rounded to BF16 before its product: 2^-9 a term, below the output's rounding.
//   * FP32 queries: every operand that is not a code is the sum of three BF16 terms (24 bits, three
//     products), and codes are converted with their sign: an offset would cost digits by cancellation.
//   * Keys of a row are split among the four waves of a block, and for few rows among blocks; the partial
//     (m, l, O) are joined by the waves through LDS and by the row block's last block to arrive.
#include <algorithm>
#include <cmath>

#include "quant.hpp"

namespace it {
namespace {

constexpr int CA_THREADS = 256;
constexpr int CA_TT = 32;              // tokens a wave takes at a time
constexpr float CA_RESCALE = 8.f;      // rows are rescaled when their maximum grew by more (log2 units)
constexpr int CA_DEVICE_SCOPE = 16;    // cache-policy bit sc1 of the buffer intrinsics: device scope
constexpr int64_t CA_MIN_CHUNK = 256;  // keys of a split, at least

__device__ __forceinline__ f32x4 mfma_bf16(const u32x4 &a, const u32x4 &b, const f32x4 &c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0,
                                                   0);
}

// Three BF16 terms of a pair of FP32 values, x = t0 + t1 + t2: each is the rounding of what is left.
__device__ __forceinline__ void split3(float a, float b, uint32_t (&t)[3]) {
#pragma unroll
    for (int p = 0; p < 3; ++p) {
        t[p] = pack_bf16x2(a, b);
        a -= __uint_as_float(t[p] << 16);
        b -= __uint_as_float(t[p] & 0xffff0000u);
    }
}

// Pairs of 4-bit codes as BF16 operands: nibbles k and k + 4 of w.
template <bool F32>
__device__ __forceinline__ uint32_t nibbles(uint32_t w, int k) {
    if constexpr (F32) {
        // signed 4-bit numbers / 16 (v_cvt_off_f32_i4), exact; the 16 is in the step
        const uint32_t v = w ^ 0x88888888u;
        return pack_bf16x2(__builtin_amdgcn_cvt_off_f32_i4((int)(v >> (4 * k))),
                           __builtin_amdgcn_cvt_off_f32_i4((int)(v >> (4 * k + 16))));
    } else {
        const uint32_t v = k == 0 ? w << 3 : w >> (4 * k - 3);
        return (v & 0x00780078u) | 0x41804180u;
    }
}

// Bytes 2 k and 2 k + 1 of w.
template <bool F32>
__device__ __forceinline__ uint32_t byte_pair(uint32_t w, int k) {
    const float o = F32 ? 128.f : 0.f;
    return pack_bf16x2((float)((w >> (16 * k)) & 255u) - o, (float)((w >> (16 * k + 8)) & 255u) - o);
}

template <bool F32, int BITS, int D, int RT>
struct CachedAttn {
    static constexpr int G = D / 32;        // 32-channel steps of a key
    static constexpr int OT = D / 16;       // 16-channel tiles of the output
    static constexpr int NT = F32 ? 3 : 1;  // BF16 terms of an operand
    static constexpr int ROW = D * BITS / 8;
    static constexpr int LB = D * BITS / 32;  // bytes of a lane's codes of 16 tokens (keys, or values)
    static constexpr int W = LB / 4;
    static constexpr int SW = D / 16;         // words of the key steps of four tokens
    static constexpr float OFF = F32 ? 0.f : BITS == 4 ? 24.f : 128.f;
    static constexpr float CODE = F32 && BITS == 4 ? 16.f : 1.f;  // what a code's operand was divided by

    // Codes and steps of 32 tokens, as loaded.
    struct Tile {
        uint32_t k[2][W], v[2][W], ks[2][SW], vs[2][2];
    };

    template <int N>
    __device__ __forceinline__ static void words(const char *p, uint32_t (&w)[N]) {
        if constexpr (N % 4 == 0) {
#pragma unroll
            for (int i = 0; i < N; i += 4) {
                const u32x4 v = *(const u32x4 *)(p + 4 * i);
                w[i] = v[0], w[i + 1] = v[1], w[i + 2] = v[2], w[i + 3] = v[3];
            }
        } else {
#pragma unroll
            for (int i = 0; i < N; i += 2) {
                const u32x2 v = *(const u32x2 *)(p + 4 * i);
                w[i] = v[0], w[i + 1] = v[1];
            }
        }
    }

    // t: a multiple of 32 below the padded capacity.
    __device__ __forceinline__ static void load(const CacheGeom &c, const char *region, int64_t t, int col, int g,
                                                Tile &x) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int64_t th = t + 16 * h;
            words(region + (th + col) * ROW + g * LB, x.k[h]);
            words(region + c.v_off + (th / 4 + g) * (4 * ROW) + col * LB, x.v[h]);
            words(region + c.ks_off + (th + 4 * g) * (2 * G), x.ks[h]);
            words(region + c.vs_off + (th + 4 * g) * 2, x.vs[h]);
        }
    }

    __device__ __forceinline__ static u32x4 key_operand(const uint32_t (&w)[W], int s) {
        if constexpr (BITS == 4)
            return u32x4{nibbles<F32>(w[s], 0), nibbles<F32>(w[s], 1), nibbles<F32>(w[s], 2), nibbles<F32>(w[s], 3)};
        else
            return u32x4{byte_pair<F32>(w[2 * s], 0), byte_pair<F32>(w[2 * s], 1), byte_pair<F32>(w[2 * s + 1], 0),
                         byte_pair<F32>(w[2 * s + 1], 1)};
    }

    // Channel R i + j of row i = lane % 16, tokens 4 g .. + 3 of both halves.
    __device__ __forceinline__ static u32x4 value_operand(const Tile &x, int j) {
        if constexpr (BITS == 4) {
            const int q = 2 * (j / 4), k = j % 4;
            return u32x4{nibbles<F32>(x.v[0][q], k), nibbles<F32>(x.v[0][q + 1], k), nibbles<F32>(x.v[1][q], k),
                         nibbles<F32>(x.v[1][q + 1], k)};
        } else {
            return u32x4{byte_pair<F32>(x.v[0][j], 0), byte_pair<F32>(x.v[0][j], 1), byte_pair<F32>(x.v[1][j], 0),
                         byte_pair<F32>(x.v[1][j], 1)};
        }
    }

    __device__ __forceinline__ static float half_of(uint32_t w, int i) {
        return __uint_as_float(i ? w & 0xffff0000u : w << 16);
    }
};

template <bool F32, int BITS, int D, int RT>
__global__ __launch_bounds__(CA_THREADS) void cached_attn(const CachedAttnArgs p) {
    using X = CachedAttn<F32, BITS, D, RT>;
    using T = std::conditional_t<F32, float, uint16_t>;
    constexpr int G = X::G, OT = X::OT, NT = X::NT, ROWS = 16 * RT;
    constexpr int PITCH = D + 4;  // floats of a row of the joined output in LDS
    __shared__ __attribute__((aligned(16))) float so[ROWS * PITCH];
    __shared__ float sm[4][ROWS], sl[4][ROWS];
    __shared__ int last;
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int col = lane & 15, g = lane >> 4;

    // The block's place: row block fastest, so that blocks that share keys are near each other, and a
    // contiguous range of places on every XCD (workgroup w runs on XCD w % 8).
    int64_t pid = blockIdx.x;
    const int64_t grid = gridDim.x;
    if (grid % 8 == 0) pid = (pid % 8) * (grid / 8) + pid / 8;
    const int rb = (int)(pid % p.row_blocks);
    const int split = (int)(pid / p.row_blocks % p.splits);
    const int64_t unit = pid / p.row_blocks / p.splits;  // sequence * kv_heads + cache head
    const int64_t b = unit / p.c.kv_heads, kvh = unit % p.c.kv_heads;
    const char *region = p.c.data + unit * p.c.region;
    const int row0 = rb * ROWS;

    // Keys that a query sees: limit(i) = start + i + 1 within the cache, 0 for i >= count.
    const int64_t start = p.start[b];
    int64_t cnt = p.n;
    if (p.count) cnt = min(cnt, max((int64_t)p.count[b], (int64_t)0));
    auto limit = [&](int64_t i) -> int64_t {
        return i < cnt ? min(max(start + i + 1, (int64_t)0), p.c.capacity) : 0;
    };
    const int64_t i_first = row0 / p.share, i_last = min((int64_t)(row0 + ROWS - 1) / p.share, cnt - 1);
    const int64_t total = i_last >= i_first ? limit(i_last) : 0;
    const int64_t unmasked = limit(i_first);  // every live row sees the keys below this
    // The splits' shares of the keys, whole steps of the block; as many splits as that fills.
    constexpr int64_t STEP = 4 * CA_TT;
    int64_t share = (total + p.splits - 1) / p.splits;
    share = max((share + STEP - 1) / STEP * STEP, CA_MIN_CHUNK);
    const int active = total > 0 ? (int)((total + share - 1) / share) : 1;
    if (split >= active) return;
    const int64_t t0 = split * share, t1 = min(total, t0 + share);

    // This lane's query row of each row tile, as the B operand: channels 32 s + 8 g .. + 7 of step s.
    u32x4 q[RT][G][NT];
    f32x4 init[RT][G];
    int64_t lim[RT];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        const int row = row0 + 16 * rt + col;
        const int64_t i = row / p.share;
        lim[rt] = row < p.rows ? limit(i) : 0;
        const T *src = (const T *)p.Q + p.ql.at(b * p.heads + kvh * p.share + row % p.share) + i * p.ql.rs + 8 * g;
#pragma unroll
        for (int s = 0; s < G; ++s) {
            float sum = 0.f;
            if constexpr (F32) {
                float x[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) x[e] = 0.f;
                if (lim[rt] > 0) {
                    if (p.q_vec) {
                        const f32x4 lo = *(const f32x4 *)(src + 32 * s), hi = *(const f32x4 *)(src + 32 * s + 4);
#pragma unroll
                        for (int e = 0; e < 4; ++e) x[e] = lo[e], x[4 + e] = hi[e];
                    } else {
#pragma unroll
                        for (int e = 0; e < 8; ++e) x[e] = src[32 * s + e];
                    }
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    uint32_t t[3];
                    split3(x[2 * e], x[2 * e + 1], t);
#pragma unroll
                    for (int m = 0; m < 3; ++m) q[rt][s][m][e] = t[m];
                }
            } else {
                u32x4 x = {0u, 0u, 0u, 0u};
                if (lim[rt] > 0) {
                    if (p.q_vec) {
                        x = *(const u32x4 *)(src + 32 * s);
                    } else {
#pragma unroll
                        for (int e = 0; e < 8; ++e) x[e >> 1] |= (uint32_t)src[32 * s + e] << (16 * (e & 1));
                    }
                }
                q[rt][s][0] = x;
#pragma unroll
                for (int e = 0; e < 4; ++e) sum += __uint_as_float(x[e] << 16) + __uint_as_float(x[e] & 0xffff0000u);
                sum += __shfl_xor(sum, 16, 64);
                sum += __shfl_xor(sum, 32, 64);
            }
            const float z = -X::OFF * sum;
            init[rt][s] = f32x4{z, z, z, z};
        }
    }

    f32x4 o[RT][OT], osum[RT];
    float m[RT], l[RT];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        m[rt] = -INFINITY;
        l[rt] = 0.f;
        osum[rt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int j = 0; j < OT; ++j) o[rt][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    const u32x4 ones = {0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u};

    typename X::Tile cur, nxt;
    const int64_t tw = t0 + wave * CA_TT;
    if (tw < t1) X::load(p.c, region, tw, col, g, cur);
    for (int64_t t = tw; t < t1; t += STEP) {
        X::load(p.c, region, t + STEP < t1 ? t + STEP : t, col, g, nxt);
        f32x4 sc[RT][2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) sc[rt][h] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int s = 0; s < G; ++s) {
                const u32x4 k = X::key_operand(cur.k[h], s);
                f32x4 step;
#pragma unroll
                for (int r = 0; r < 4; ++r)  // steps of tokens 4 g + r, group s
                    step[r] = X::half_of(cur.ks[h][(r * G + s) / 2], (r * G + s) & 1);
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) {
                    f32x4 c = init[rt][s];
#pragma unroll
                    for (int w = NT - 1; w >= 0; --w) c = mfma_bf16(k, q[rt][s][w], c);
#pragma unroll
                    for (int r = 0; r < 4; ++r) sc[rt][h][r] = fmaf(step[r], c[r], sc[rt][h][r]);
                }
            }
        }
        float vstep[2][4];
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int r = 0; r < 4; ++r) vstep[h][r] = X::half_of(cur.vs[h][r >> 1], r & 1);
        const bool masked = t + CA_TT > unmasked;
        uint32_t pw[RT][NT][4];
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            if (masked) {
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        if (t + 16 * h + 4 * g + r >= lim[rt]) sc[rt][h][r] = -INFINITY;
            }
            float mx = fmaxf(fmaxf(fmaxf(sc[rt][0][0], sc[rt][0][1]), fmaxf(sc[rt][0][2], sc[rt][0][3])),
                             fmaxf(fmaxf(sc[rt][1][0], sc[rt][1][1]), fmaxf(sc[rt][1][2], sc[rt][1][3])));
            mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
            mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
            mx *= p.scale_log2 * X::CODE;
            if (__any(mx > m[rt] + CA_RESCALE)) {
                const float mn = fmaxf(mx, m[rt]);
                const float f = mn == m[rt] ? 1.f : __builtin_amdgcn_exp2f(m[rt] - mn);
                l[rt] *= f;
                osum[rt] *= f;
#pragma unroll
                for (int j = 0; j < OT; ++j) o[rt][j] *= f;
                m[rt] = mn;
            }
            const float base = m[rt] == -INFINITY ? 0.f : m[rt];
            float pv[2][4];
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const float e = __builtin_amdgcn_exp2f(fmaf(sc[rt][h][r], p.scale_log2 * X::CODE, -base));
                    l[rt] += e;
                    pv[h][r] = e * vstep[h][r];
                    // a hidden key's value step may be anything
                    if (masked && t + 16 * h + 4 * g + r >= lim[rt]) pv[h][r] = 0.f;
                }
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int r = 0; r < 4; r += 2) {
                    if constexpr (F32) {
                        uint32_t w[3];
                        split3(pv[h][r], pv[h][r + 1], w);
#pragma unroll
                        for (int i = 0; i < 3; ++i) pw[rt][i][2 * h + r / 2] = w[i];
                    } else {
                        pw[rt][0][2 * h + r / 2] = pack_bf16x2(pv[h][r], pv[h][r + 1]);
                    }
                }
            if constexpr (!F32)
                osum[rt] = mfma_bf16(ones, u32x4{pw[rt][0][0], pw[rt][0][1], pw[rt][0][2], pw[rt][0][3]}, osum[rt]);
        }
#pragma unroll
        for (int j = 0; j < OT; ++j) {
            const u32x4 v = X::value_operand(cur, j);
#pragma unroll
            for (int rt = 0; rt < RT; ++rt)
#pragma unroll
                for (int w = NT - 1; w >= 0; --w)
                    o[rt][j] = mfma_bf16(v, u32x4{pw[rt][w][0], pw[rt][w][1], pw[rt][w][2], pw[rt][w][3]}, o[rt][j]);
        }
        cur = nxt;
    }

    // Join the four waves: the rows' common maximum, then the sums scaled to it, wave by wave in LDS.
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        l[rt] += __shfl_xor(l[rt], 16, 64);
        l[rt] += __shfl_xor(l[rt], 32, 64);
        if (g == 0) {
            sm[wave][16 * rt + col] = m[rt];
            sl[wave][16 * rt + col] = l[rt];
        }
    }
    __syncthreads();
    constexpr int R = D / 16;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        if (wave == w) {
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
                const int row = 16 * rt + col;
                const float mm = fmaxf(fmaxf(sm[0][row], sm[1][row]), fmaxf(sm[2][row], sm[3][row]));
                const float f = (m[rt] == mm ? 1.f : __builtin_amdgcn_exp2f(m[rt] - mm)) * X::CODE;
#pragma unroll
                for (int r = 0; r < 4; ++r)
#pragma unroll
                    for (int j = 0; j < OT; ++j) {
                        float *d = so + row * PITCH + R * (4 * g + r) + j;
                        const float x = (o[rt][j][r] - X::OFF * osum[rt][0]) * f;
                        *d = w == 0 ? x : *d + x;
                    }
            }
        }
        __syncthreads();
    }
    auto row_max = [&](int row) { return fmaxf(fmaxf(sm[0][row], sm[1][row]), fmaxf(sm[2][row], sm[3][row])); };
    auto row_sum = [&](int row, float mm) {
        float s = 0.f;
#pragma unroll
        for (int w = 0; w < 4; ++w) s += sl[w][row] * (sm[w][row] == mm ? 1.f : __builtin_amdgcn_exp2f(sm[w][row] - mm));
        return s;
    };

    // Thread's pieces of the block's output: four channels of a row.
    constexpr int Q = D / 4, PIECES = ROWS * Q;
    auto store = [&](int row, int c4, f32x4 x) {
        const int64_t i = (row0 + row) / p.share;
        T *dst = (T *)p.O + p.ol.at(b * p.heads + kvh * p.share + (row0 + row) % p.share) + i * p.ol.rs + 4 * c4;
        if (p.o_vec) {
            if constexpr (F32)
                *(f32x4 *)dst = x;
            else
                *(u32x2 *)dst = u32x2{pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3])};
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if constexpr (F32)
                    dst[e] = x[e];
                else
                    dst[e] = f32_to_bf16_rne(x[e]);
            }
        }
    };
    const f32x4 none = {0.f, 0.f, 0.f, 0.f};
    if (active == 1) {
        for (int e = tid; e < PIECES; e += CA_THREADS) {
            const int row = e / Q, c4 = e % Q;
            if (row0 + row >= p.rows) continue;
            const float mm = row_max(row), sum = row_sum(row, mm);
            const bool live = limit((row0 + row) / p.share) > 0;
            store(row, c4, live ? *(const f32x4 *)(so + row * PITCH + 4 * c4) * (1.f / sum) : none);
        }
        return;
    }
    // Partial results at device scope, [split][row][D + 2 floats]; the last block to arrive joins them.
    const int rows = min(ROWS, p.rows - row0);
    constexpr int PW = D + 4;
    const int64_t slots = (unit * p.row_blocks + rb) * p.splits;
    float *base = p.part + slots * (int64_t)(ROWS * PW);
    const __amdgpu_buffer_rsrc_t prt =
        __builtin_amdgcn_make_buffer_rsrc(base, (short)0, p.splits * ROWS * PW * 4, 0x00020000);
    for (int e = tid; e < rows * Q; e += CA_THREADS) {
        const int row = e / Q, c4 = e % Q;
        const uint32_t off = (uint32_t)(((split * ROWS + row) * PW + 4 * c4) * 4);
        __builtin_amdgcn_raw_buffer_store_b128(*(const u32x4 *)(so + row * PITCH + 4 * c4), prt, off, 0, CA_DEVICE_SCOPE);
        if (c4 == 0) {
            const float mm = row_max(row), sum = row_sum(row, mm);
            const u32x4 ml = {__float_as_uint(mm), __float_as_uint(sum), 0u, 0u};
            __builtin_amdgcn_raw_buffer_store_b128(ml, prt, off + D * 4, 0, CA_DEVICE_SCOPE);
        }
    }
    __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0): the partial results have reached device scope
    __syncthreads();
    if (tid == 0) {
        // Ordered by the device-scope stores waited for above and the device-scope loads below.
        int *cnt_at = p.counters + unit * p.row_blocks + rb;
        const int old = __hip_atomic_fetch_add(cnt_at, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        last = old == active - 1;
        if (last) __hip_atomic_store(cnt_at, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    __syncthreads();
    if (!last) return;
    for (int e = tid; e < rows * Q; e += CA_THREADS) {
        const int row = e / Q, c4 = e % Q;
        f32x4 x = none;
        float mm = -INFINITY, sum = 0.f;
        for (int s = 0; s < active; ++s) {
            const uint32_t off = (uint32_t)(((s * ROWS + row) * PW + 4 * c4) * 4);
            const u32x2 ml = __builtin_bit_cast(
                u32x2, __builtin_amdgcn_raw_buffer_load_b64(prt, off + (D - 4 * c4) * 4, 0, CA_DEVICE_SCOPE));
            const f32x4 v = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(prt, off, 0, CA_DEVICE_SCOPE));
            const float ms = __uint_as_float(ml[0]), mn = fmaxf(mm, ms);
            const float fo = mm == mn ? 1.f : __builtin_amdgcn_exp2f(mm - mn);
            const float fs = ms == mn ? 1.f : __builtin_amdgcn_exp2f(ms - mn);
            x = x * fo + v * fs;
            sum = sum * fo + __uint_as_float(ml[1]) * fs;
            mm = mn;
        }
        const bool live = limit((row0 + row) / p.share) > 0;
        store(row, c4, live ? x * (1.f / sum) : none);
    }
}

template <bool F32, int BITS, int D>
void launch_rt(hipStream_t s, const CachedAttnArgs &a) {
    const dim3 grid((unsigned)(a.c.batch * a.c.kv_heads * a.row_blocks * a.splits)), block(CA_THREADS);
    hipLaunchKernelGGL((cached_attn<F32, BITS, D, 1>), grid, block, 0, s, a);
}

template <bool F32, int BITS>
void launch_dim(hipStream_t s, const CachedAttnArgs &a) {
    if (a.c.head_dim == 64) launch_rt<F32, BITS, 64>(s, a);
    else if (a.c.head_dim == 128) launch_rt<F32, BITS, 128>(s, a);
    else launch_rt<F32, BITS, 256>(s, a);
}

}  // namespace

int64_t plan_cached_attention(CachedAttnArgs &a, bool bf16, int num_cus) {
    (void)bf16;
    constexpr int ROWS = 16;
    a.row_blocks = (a.rows + ROWS - 1) / ROWS;
    const int64_t units = a.c.batch * a.c.kv_heads * a.row_blocks;
    // Two blocks a CU, splits of CA_MIN_CHUNK keys at least.
    int64_t splits = (2 * num_cus + units - 1) / units;
    splits = std::min({splits, (a.c.capacity + CA_MIN_CHUNK - 1) / CA_MIN_CHUNK, (int64_t)256});
    if (units > COUNTERS || splits < 2) splits = 1;
    a.splits = (int)splits;
    return splits > 1 ? units * splits * ROWS * (a.c.head_dim + 4) : 0;
}

it_status launch_cached_attention(hipStream_t s, bool bf16, const CachedAttnArgs &a) {
    if (bf16)
        a.c.bits == 4 ? launch_dim<false, 4>(s, a) : launch_dim<false, 8>(s, a);
    else
        a.c.bits == 4 ? launch_dim<true, 4>(s, a) : launch_dim<true, 8>(s, a);
    IT_HIP_TRY(hipGetLastError());
    return IT_OK;
}

}  // namespace it
