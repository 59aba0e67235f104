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
//     16 + code. The offset (16 + 8) leaves by one more product, steps times -24 sum(q) of each group (a
//     BF16 matrix times three BF16 terms of the sums, 3 G <= 24 of an instruction's 32 k), and for the values
//     with the sum of the rounded probabilities (a product with ones). 8-bit codes are converted, 128 too
//     large. P is rounded to BF16 before its product: 2^-8 a term at most, as the output's own rounding, and the
//     keys' roundings average.
//   * FP32 queries: every operand that is not a code is the sum of three BF16 terms (24 bits, three
//     products), and codes are converted with their sign: an offset would cost digits by cancellation.
//   * Codes and steps stream global -> LDS (buffer_load .. lds) into a ring of every wave's own, several
//     32-token tiles ahead: 131072 tokens of 8 heads of 128 channels (145 MB in 4 bits) take 39.6 us, 57 with one
//     tile in registers ahead. A wave waits for its own loads only, so no barrier is in the loop.
//   * Keys of a row are split among the four waves of a block, and for few rows among blocks; the partial
//     (m, l, O) are joined by the waves through LDS and by the row block's last block to arrive.
#include <algorithm>
#include <cmath>

#include "mfma.hpp"
#include "quant.hpp"

namespace it {
namespace {

constexpr int CA_THREADS = 256;
constexpr int CA_TT = 32;              // tokens a wave takes at a time
constexpr float CA_RESCALE = 8.f;      // rows are rescaled when their maximum grew by more (log2 units)
constexpr int CA_DEVICE_SCOPE = 16;    // cache-policy bit sc1 of the buffer intrinsics: device scope
constexpr int64_t CA_MIN_CHUNK = 256;  // keys of a split, at least
constexpr int CA_MAX_SPLITS = 128;
constexpr int CA_JOIN = 16;            // partial results a thread loads at a time in the join
constexpr int CA_TARGET = 1;           // blocks a CU that the splits aim at
// Blocks that a CU holds, by registers and by their rings of LDS: four with one row tile of up to 128 BF16
// channels (three in FP32), two otherwise.
constexpr int ca_blocks(bool f32, int d, int rt) { return rt == 1 && d <= 128 ? (f32 ? 3 : 4) : 2; }
constexpr int CA_LDS_BYTES = 157 << 10;

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
        // One v_and_or_b32 (left alone the compiler takes an and and an or, whose literals save it registers).
        uint32_t v = k == 0 ? w << 3 : w >> (4 * k - 3), r;
        asm("v_and_or_b32 %0, %1, %2, %3" : "=v"(r) : "v"(v), "s"(0x00780078u), "v"(0x41804180u));
        return r;
    }
}

// Bytes 2 k and 2 k + 1 of w.
template <bool F32>
__device__ __forceinline__ uint32_t byte_pair(uint32_t w, int k) {
    const float o = F32 ? 128.f : 0.f;
    return pack_bf16x2((float)((w >> (16 * k)) & 255u) - o, (float)((w >> (16 * k + 8)) & 255u) - o);
}

typedef __attribute__((address_space(3))) void ca_lds_t;
// Vector accesses that need an element's alignment only.
typedef float f32x4_any __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t u32x4_any __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t u32x2_any __attribute__((ext_vector_type(2), aligned(2)));

// x over the lanes 16 and 32 apart: v_permlane*_swap gives each half (each pair of 16-lane rows) both.
template <typename F>
__device__ __forceinline__ float over_groups(float x, F f) {
    const uint32_t b = __float_as_uint(x);
    const auto p = __builtin_amdgcn_permlane32_swap(b, b, false, false);
    const uint32_t c = __float_as_uint(f(__uint_as_float(p[0]), __uint_as_float(p[1])));
    const auto q = __builtin_amdgcn_permlane16_swap(c, c, false, false);
    return f(__uint_as_float(q[0]), __uint_as_float(q[1]));
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

    // A slot of the ring: 32 tokens' key codes, value codes, key steps and value steps, as they lie in the
    // cache, each padded to whole load instructions.
    static constexpr int CODES = CA_TT * ROW;
    static constexpr int KS_AT = 2 * CODES, KS_LOADS = G > 4 ? G / 4 : 1;
    static constexpr int VS_AT = KS_AT + 256 * KS_LOADS;
    static constexpr int SLOT = VS_AT + 256;
    static constexpr int LOADS = 2 * (CODES / 1024) + KS_LOADS + 1;  // load instructions of a slot
    static constexpr int FIT = CA_LDS_BYTES / ca_blocks(F32, D, RT) / (4 * SLOT);
    static constexpr int NB = FIT > 6 ? 6 : FIT < 2 ? 2 : FIT;
    static_assert(CODES % 1024 == 0 && NB * LOADS < 64, "whole loads, counted by vmcnt");

    // Tokens t .. t + 31 (t a multiple of 32) into `slot`; an invalid tile loads nothing (zeros). A descriptor of
    // exactly the 32 tokens for each of the four arrays: scalar arithmetic, and a lane's offset never changes.
    __device__ __forceinline__ static void issue(const CacheGeom &c, const char *region, uint32_t t, bool valid, uint32_t slot,
                                                 int lane) {
        auto array = [&](int64_t at, int bytes) {
            return __builtin_amdgcn_make_buffer_rsrc(const_cast<char *>(region + at), (short)0, valid ? bytes : 0, 0x00020000);
        };
        auto to_lds = [&](uint32_t to) {
            uint32_t x = slot + to;
            asm("" : "+s"(x));  // opaque: the waits in the loop order these loads
            return (ca_lds_t *)(uintptr_t)x;
        };
        const __amdgpu_buffer_rsrc_t k = array((int64_t)t * ROW, CODES), v = array(c.v_off + (int64_t)t * ROW, CODES);
#pragma unroll
        for (int i = 0; i < CODES / 1024; ++i)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(k, to_lds(1024 * i), 16, 16 * lane + 1024 * i, 0, 0, 0);
#pragma unroll
        for (int i = 0; i < CODES / 1024; ++i)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(v, to_lds(CODES + 1024 * i), 16, 16 * lane + 1024 * i, 0, 0, 0);
        const __amdgpu_buffer_rsrc_t ks = array(c.ks_off + (int64_t)t * (2 * G), CA_TT * 2 * G), vs = array(c.vs_off + (int64_t)t * 2, CA_TT * 2);
#pragma unroll
        for (int i = 0; i < KS_LOADS; ++i)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(ks, to_lds(KS_AT + 256 * i), 4, 4 * lane + 256 * i, 0, 0, 0);
        __builtin_amdgcn_raw_ptr_buffer_load_lds(vs, to_lds(VS_AT), 4, 4 * lane, 0, 0, 0);
    }

    // Codes and steps of 16 tokens' keys (half h of a slot); the steps of token 4 g + r, group s at word
    // (r G + s) / 2, and of token `col` as the operand of the offsets' product.
    struct Keys {
        uint32_t k[W], ks[SW], own[G / 2];
    };
    // Values of 32 tokens.
    struct Values {
        uint32_t v[2][W];
    };

    template <int N>
    __device__ __forceinline__ static void words(const char *p, uint32_t (&w)[N]) {
        if constexpr (N % 4 == 0) {
#pragma unroll
            for (int i = 0; i < N; i += 4) {
                const u32x4 v = *(const u32x4 *)(p + 4 * i);
                w[i] = v[0], w[i + 1] = v[1], w[i + 2] = v[2], w[i + 3] = v[3];
            }
        } else if constexpr (N == 2) {
            const u32x2 v = *(const u32x2 *)p;
            w[0] = v[0], w[1] = v[1];
        } else {
            w[0] = *(const uint32_t *)p;
        }
    }

    __device__ __forceinline__ static void read(const char *slot, int h, int col, int g, Keys &x) {
        words(slot + (16 * h + col) * ROW + g * LB, x.k);
        words(slot + KS_AT + (16 * h + 4 * g) * (2 * G), x.ks);
        if constexpr (!F32) words(slot + KS_AT + (16 * h + col) * (2 * G), x.own);
    }

    __device__ __forceinline__ static void read(const char *slot, int col, int g, Values &x) {
#pragma unroll
        for (int h = 0; h < 2; ++h) words(slot + CODES + (4 * h + g) * (4 * ROW) + col * LB, x.v[h]);
    }

    __device__ __forceinline__ static u32x4 key_operand(const uint32_t (&w)[W], int s) {
        if constexpr (BITS == 4)
            return u32x4{nibbles<F32>(w[s], 0), nibbles<F32>(w[s], 1), nibbles<F32>(w[s], 2), nibbles<F32>(w[s], 3)};
        else
            return u32x4{byte_pair<F32>(w[2 * s], 0), byte_pair<F32>(w[2 * s], 1), byte_pair<F32>(w[2 * s + 1], 0),
                         byte_pair<F32>(w[2 * s + 1], 1)};
    }

    // Channel R i + j of row i = lane % 16, tokens 4 g .. + 3 of both halves.
    __device__ __forceinline__ static u32x4 value_operand(const Values &x, int j) {
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
__global__ __launch_bounds__(CA_THREADS) __attribute__((amdgpu_waves_per_eu(CachedAttn<F32, BITS, D, RT>::SLOT > 16384 ? 1 : ca_blocks(F32, D, RT))))
void cached_attn(const CachedAttnArgs p) {
    using X = CachedAttn<F32, BITS, D, RT>;
    using T = std::conditional_t<F32, float, uint16_t>;
    constexpr int G = X::G, OT = X::OT, NT = X::NT, ROWS = 16 * RT;
    constexpr int PITCH = D + 4;  // floats of a row of the joined output in LDS
    constexpr int RING = 4 * X::NB * X::SLOT;
    static_assert(ROWS * PITCH * 4 <= RING, "the join of the waves fits the rings");
    __shared__ __attribute__((aligned(1024))) char ring[RING];
    float *so = (float *)ring;  // after the loop
    __shared__ float sm[4][ROWS], sl[4][ROWS];
    __shared__ int last;
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int col = lane & 15, g = lane >> 4;

    // The block's place: row block fastest, split slowest. Splits that a sequence has no keys for end at once, and
    // in this order they are the last to be dispatched: between the others they left CUs empty beside CUs
    // with two blocks (131072 tokens of 8 heads: 51.7 us against 40). Row blocks share keys, so where there are
    // several every XCD (workgroup w runs on XCD w % 8) takes a contiguous range of places.
    uint32_t pid = blockIdx.x;
    if (p.row_blocks > 1 && gridDim.x % 8 == 0) pid = (pid % 8) * (gridDim.x / 8) + pid / 8;
    const uint32_t units = (uint32_t)(p.c.batch * p.c.kv_heads), rest = pid / (uint32_t)p.row_blocks;
    const int rb = (int)(pid % (uint32_t)p.row_blocks), split = (int)(rest / units);
    const uint32_t unit = rest % units;  // sequence * kv_heads + cache head
    const uint32_t b = unit / (uint32_t)p.c.kv_heads, kvh = unit % (uint32_t)p.c.kv_heads;
    const char *region = p.c.data + unit * p.c.region;
    const int row0 = rb * ROWS;

    // Keys that a query sees: limit(i) = start + i + 1 within the cache, 0 for i >= count.
    const int64_t start = p.start[b];
    int64_t cnt = p.n;
    if (p.count) cnt = min(cnt, max((int64_t)p.count[b], (int64_t)0));
    auto limit = [&](int64_t i) -> int64_t {
        return i < cnt ? min(max(start + i + 1, (int64_t)0), p.c.capacity) : 0;
    };
    auto query = [&](int row) -> int64_t { return (uint32_t)row / (uint32_t)p.share; };
    const int64_t i_first = query(row0), i_last = min(query(row0 + ROWS - 1), cnt - 1);
    const int64_t total = i_last >= i_first ? limit(i_last) : 0;
    const int64_t unmasked = limit(i_first);  // every live row sees the keys below this
    // The splits' shares of the keys, whole steps of the block. All sequences take the same share, that which
    // spreads the batch's keys over the blocks aimed at, so that long sequences take more blocks.
    constexpr int64_t STEP = 4 * CA_TT;
    int64_t share = total;
    if (p.splits > 1) {
        float keys = (float)total;
        if (p.c.batch > 1) {
            keys = 0.f;
            for (int64_t j = lane; j < p.c.batch; j += 64) {
                int64_t c = p.n;
                if (p.count) c = min(c, max((int64_t)p.count[j], (int64_t)0));
                if (c > 0) keys += (float)min(max((int64_t)p.start[j] + c, (int64_t)0), p.c.capacity);
            }
#pragma unroll
            for (int o = 32; o > 0; o >>= 1) keys += __shfl_xor(keys, o, 64);
        }
        // A shuffle's result counts as different in every lane until it is read from the first.
        const int even = __builtin_amdgcn_readfirstlane((int)fminf(keys * p.per_key, 2e9f));
        share = max(max((int64_t)even, CA_MIN_CHUNK), (int64_t)((uint32_t)(total + p.splits - 1) / (uint32_t)p.splits));
    }
    share = (share + STEP - 1) / STEP * STEP;
    const int active = total > share ? (int)((uint32_t)(total + share - 1) / (uint32_t)share) : 1;
    if (split >= active) return;
    const int64_t t0 = split * share, t1 = min(total, t0 + share);

    // The first tiles of this wave's keys on their way.
    constexpr int NB = X::NB;
    const uint32_t my_ring = (uint32_t)(uintptr_t)(ca_lds_t *)ring + wave * (NB * X::SLOT);
    const int tw = (int)t0 + wave * CA_TT, te = (int)t1;
#pragma unroll
    for (int i = 0; i < NB; ++i)
        X::issue(p.c, region, (uint32_t)(tw + i * STEP), tw + i * STEP < te, my_ring + i * X::SLOT, lane);

    // This lane's query row of each row tile, as the B operand: channels 32 s + 8 g .. + 7 of step s.
    u32x4 q[RT][G][NT];
    u32x4 off[RT];  // operand of the offsets: term g of -OFF sum(q) of every group, zeros for g = 3
    int lim[RT];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        const int row = row0 + 16 * rt + col;
        const int64_t i = query(row);
        lim[rt] = row < p.rows ? (int)limit(i) : 0;
        float z[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        const T *src = (const T *)p.Q + p.ql.at(b, kvh * p.share + (row - i * p.share)) + i * p.ql.rs + 8 * g;
#pragma unroll
        for (int s = 0; s < G; ++s) {
            if constexpr (F32) {
                float x[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) x[e] = 0.f;
                if (row < p.rows) {
                    const f32x4 lo = *(const f32x4_any *)(src + 32 * s), hi = *(const f32x4_any *)(src + 32 * s + 4);
#pragma unroll
                    for (int e = 0; e < 4; ++e) x[e] = lo[e], x[4 + e] = hi[e];
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
                if (row < p.rows) x = *(const u32x4_any *)(src + 32 * s);
                q[rt][s][0] = x;
                float sum = 0.f;
#pragma unroll
                for (int e = 0; e < 4; ++e) sum += __uint_as_float(x[e] << 16) + __uint_as_float(x[e] & 0xffff0000u);
                z[s] = -X::OFF * over_groups(sum, [](float x, float y) { return x + y; });
            }
        }
        if constexpr (!F32) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                uint32_t t[3];
                split3(z[2 * e], z[2 * e + 1], t);
                off[rt][e] = g == 0 ? t[0] : g == 1 ? t[1] : g == 2 ? t[2] : 0u;
            }
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

    int slot = 0;
    for (int t = tw; t < te; t += (int)STEP) {
        // This tile has landed; the later ones may be in flight.
        asm volatile("s_waitcnt vmcnt(%0)" ::"n"((NB - 1) * X::LOADS) : "memory");
        const char *at = ring + (wave * NB + slot) * X::SLOT;
        f32x4 sc[RT][2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            typename X::Keys key;
            X::read(at, h, col, g, key);
            if constexpr (F32) {
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) sc[rt][h] = f32x4{0.f, 0.f, 0.f, 0.f};
            } else {
                u32x4 own = {0u, 0u, 0u, 0u};
#pragma unroll
                for (int i = 0; i < G / 2; ++i) own[i] = key.own[i];
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) sc[rt][h] = mfma_bf16(own, off[rt], f32x4{0.f, 0.f, 0.f, 0.f});
            }
#pragma unroll
            for (int s = 0; s < G; ++s) {
                const u32x4 k = X::key_operand(key.k, s);
                f32x4 step;
#pragma unroll
                for (int r = 0; r < 4; ++r)  // steps of tokens 4 g + r, group s
                    step[r] = X::half_of(key.ks[(r * G + s) / 2], (r * G + s) & 1);
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) {
                    f32x4 c = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int w = NT - 1; w >= 0; --w) c = mfma_bf16(k, q[rt][s][w], c);
#pragma unroll
                    for (int r = 0; r < 4; ++r) sc[rt][h][r] = fmaf(step[r], c[r], sc[rt][h][r]);
                }
            }
        }
        float vstep[2][4];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const u32x2 w = *(const u32x2 *)(at + X::VS_AT + (16 * h + 4 * g) * 2);
#pragma unroll
            for (int r = 0; r < 4; ++r) vstep[h][r] = X::half_of(w[r >> 1], r & 1);
        }
        typename X::Values value;
        X::read(at, col, g, value);
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
            mx *= p.scale_log2 * X::CODE;
            if (__any(mx > m[rt] + CA_RESCALE)) {
                mx = over_groups(mx, [](float x, float y) { return fmaxf(x, y); });
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
                }
            if (masked) {
                asm volatile("");  // a branch, not 24 more operations in every tile
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int r = 0; r < 4; ++r)  // a hidden key's value step may be anything
                        if (t + 16 * h + 4 * g + r >= lim[rt]) pv[h][r] = 0.f;
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
        // The slot is in registers: the tile NB steps ahead may take it.
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        const int ta = t + NB * (int)STEP;
        X::issue(p.c, region, (uint32_t)ta, ta < te, my_ring + slot * X::SLOT, lane);
        slot = slot + 1 == NB ? 0 : slot + 1;
#pragma unroll
        for (int j = 0; j < OT; ++j) {
            const u32x4 v = X::value_operand(value, j);
#pragma unroll
            for (int rt = 0; rt < RT; ++rt)
#pragma unroll
                for (int w = NT - 1; w >= 0; --w)
                    o[rt][j] = mfma_bf16(v, u32x4{pw[rt][w][0], pw[rt][w][1], pw[rt][w][2], pw[rt][w][3]}, o[rt][j]);
        }
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // loads into dead slots, before the rings are reused

    // Join the four waves: the rows' common maximum, then the sums scaled to it, wave by wave in LDS.
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        l[rt] = over_groups(l[rt], [](float x, float y) { return x + y; });
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
        const int64_t i = query(row0 + row);
        T *dst = (T *)p.O + p.ol.at(b, kvh * p.share + (row0 + row - i * p.share)) + i * p.ol.rs + 4 * c4;
        if constexpr (F32)
            *(f32x4_any *)dst = x;
        else
            *(u32x2_any *)dst = u32x2{pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3])};
    };
    const f32x4 none = {0.f, 0.f, 0.f, 0.f};
    if (active == 1) {
        for (int e = tid; e < PIECES; e += CA_THREADS) {
            const int row = e / Q, c4 = e % Q;
            if (row0 + row >= p.rows) continue;
            const float mm = row_max(row), sum = row_sum(row, mm);
            const bool live = limit(query(row0 + row)) > 0;
            store(row, c4, live ? *(const f32x4 *)(so + row * PITCH + 4 * c4) * (1.f / sum) : none);
        }
        return;
    }
    // Partial results at device scope, [split][row][D + 2 floats]; the last block to arrive joins them.
    const int rows = min(ROWS, p.rows - row0);
    constexpr int PW = D + 4;
    const int64_t slots = ((int64_t)unit * p.row_blocks + rb) * p.splits;
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
        int *cnt_at = p.counters + (int64_t)unit * p.row_blocks + rb;
        const int old = __hip_atomic_fetch_add(cnt_at, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        last = old == active - 1;
        if (last) __hip_atomic_store(cnt_at, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    __syncthreads();
    if (!last) return;
    // Each piece by `per` threads that share its splits, CA_JOIN of them in flight at a time: a device-scope
    // load takes 1 to 2 us, so the joins cost as many of those as a thread has turns, and the row's (m, l) are
    // loaded with the outputs rather than before them.
    const int pieces = rows * Q;
    int per = 1;  // a power of two, neighbours in a wave
    while (per < 64 && pieces * per * 2 <= CA_THREADS && per * 2 <= active) per *= 2;
    for (int e0 = 0; e0 < pieces; e0 += CA_THREADS / per) {
        const int e = e0 + tid / per, sub = tid % per;
        const int row = e < pieces ? e / Q : 0, c4 = e < pieces ? e % Q : 0;
        f32x4 x = none;
        float mm = -INFINITY, sum = 0.f;
        for (int s0 = sub; s0 < active; s0 += per * CA_JOIN) {
            u32x2 ml[CA_JOIN];
            f32x4 v[CA_JOIN];
#pragma unroll
            for (int i = 0; i < CA_JOIN; ++i) {
                // past the last split: zeros, by the range check
                const uint32_t off = (uint32_t)(((s0 + i * per) * ROWS + row) * (PW * 4)) | (s0 + i * per < active ? 0u : 0x80000000u);
                ml[i] = __builtin_bit_cast(u32x2, __builtin_amdgcn_raw_buffer_load_b64(prt, off + D * 4, 0, CA_DEVICE_SCOPE));
                v[i] = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(prt, off + 16 * c4, 0, CA_DEVICE_SCOPE));
            }
            float mn = mm;
#pragma unroll
            for (int i = 0; i < CA_JOIN; ++i) mn = fmaxf(mn, s0 + i * per < active ? __uint_as_float(ml[i][0]) : -INFINITY);
            const float fo = mm == mn ? 1.f : __builtin_amdgcn_exp2f(mm - mn);
            x *= fo;
            sum *= fo;
#pragma unroll
            for (int i = 0; i < CA_JOIN; ++i) {
                const float ms = __uint_as_float(ml[i][0]), f = ms == mn ? 1.f : __builtin_amdgcn_exp2f(ms - mn);
                if (s0 + i * per < active) {
                    x += f * v[i];
                    sum += f * __uint_as_float(ml[i][1]);
                }
            }
            mm = mn;
        }
        for (int o = 1; o < per; o <<= 1) {
            const float mo = __shfl_xor(mm, o, 64), mn = fmaxf(mm, mo);
            const float fa = mm == mn ? 1.f : __builtin_amdgcn_exp2f(mm - mn), fb = mo == mn ? 1.f : __builtin_amdgcn_exp2f(mo - mn);
#pragma unroll
            for (int i = 0; i < 4; ++i) x[i] = x[i] * fa + __shfl_xor(x[i], o, 64) * fb;
            sum = sum * fa + __shfl_xor(sum, o, 64) * fb;
            mm = mn;
        }
        if (e < pieces && sub == 0) store(row, c4, limit(query(row0 + row)) > 0 ? x * (1.f / sum) : none);
    }
}

// Two row tiles fit the registers of two waves a SIMD (256) up to these widths.
constexpr bool ca_two_tiles(bool f32, int d) { return d <= (f32 ? 64 : 128); }

template <bool F32, int BITS, int D>
void launch_rt(hipStream_t s, const CachedAttnArgs &a) {
    const dim3 grid((unsigned)(a.c.batch * a.c.kv_heads * a.row_blocks * a.splits)), block(CA_THREADS);
    if constexpr (ca_two_tiles(F32, D))
        if (a.row_tiles == 2) {
            hipLaunchKernelGGL((cached_attn<F32, BITS, D, 2>), grid, block, 0, s, a);
            return;
        }
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
    // 32 rows a block share the unpacked codes of a tile; 16 where that leaves CUs without a block.
    const int64_t pairs = a.c.batch * a.c.kv_heads * ((a.rows + 31) / 32);
    a.row_tiles = a.rows > 16 && pairs >= num_cus && ca_two_tiles(!bf16, a.c.head_dim) ? 2 : 1;
    const int rows = 16 * a.row_tiles;
    a.row_blocks = (a.rows + rows - 1) / rows;
    const int64_t units = a.c.batch * a.c.kv_heads * a.row_blocks;
    // Splits for one block a CU, of CA_MIN_CHUNK keys at least, and twice as many in the grid, so that a ragged
    // batch's long sequences can take more than their even part. More blocks stream no faster and their joins
    // cost more: 32768 tokens of 8 heads take 19.6 us with one block a CU, 22.6 with two, 33 with four.
    const int64_t target = CA_TARGET * num_cus;
    a.per_key = (float)((double)(a.c.kv_heads * a.row_blocks) / (double)target);
    int64_t splits = 2 * target / units;
    splits = std::min({splits, (a.c.capacity + CA_MIN_CHUNK - 1) / CA_MIN_CHUNK, (int64_t)CA_MAX_SPLITS});
    if (units > COUNTERS || splits < 2) splits = 1;
    a.splits = (int)splits;
    return splits > 1 ? units * splits * rows * (a.c.head_dim + 4) : 0;
}

it_status launch_cached_attention(hipStream_t s, bool bf16, const CachedAttnArgs &a) {
    if (const it_status st = check_blocks("cached_attention", a.c.batch * a.c.kv_heads * a.row_blocks * a.splits); st != IT_OK) return st;
    if (bf16)
        a.c.bits == 4 ? launch_dim<false, 4>(s, a) : launch_dim<false, 8>(s, a);
    else
        a.c.bits == 4 ? launch_dim<true, 4>(s, a) : launch_dim<true, 8>(s, a);
    IT_HIP_TRY(hipGetLastError());
    return IT_OK;
}

}  // namespace it
