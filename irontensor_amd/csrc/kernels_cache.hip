// The quantised key/value cache: writing (quantising) new tokens and reading them back. No counterpart in
// the reference, which recomputes the whole prompt for every token (its inference has no cache).
//
// Both kernels move bytes: a write reads the new keys and values once and writes a quarter (8 bits) or an
// eighth (4 bits) of FP32's bytes. A thread handles 8 channels of a block of four positions, the unit in
// which value codes lie together, so it writes whole 16-byte (32-byte) pieces and no thread shares a word
// with another; a block that the call covers in part is read, merged and written back by its one owner. A
// key's 32-channel group is four neighbouring lanes, a value row head_dim / 8 of them.
#include <algorithm>

#include "quant.hpp"
#include "quantiser.hpp"

namespace it {
namespace {

constexpr int CM_THREADS = 256;

// Vector accesses that need an element's alignment only.
typedef float f32x4_any __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t u32x4_any __attribute__((ext_vector_type(4), aligned(2)));

// Eight channels as loaded.
template <typename T>
struct Raw8 {
    uint32_t w[2 * sizeof(T)];
    __device__ __forceinline__ void load(const T *p) {
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; ++i) {
            const u32x4 v = *(const u32x4_any *)((const char *)p + 16 * i);
#pragma unroll
            for (int j = 0; j < 4; ++j) w[4 * i + j] = v[j];
        }
    }
    __device__ __forceinline__ void zero() {
#pragma unroll
        for (int i = 0; i < 2 * (int)sizeof(T); ++i) w[i] = 0;
    }
    // Bits of the largest |x|.
    __device__ __forceinline__ uint32_t most() const {
        if constexpr (sizeof(T) == 4) {
            uint32_t m = 0;
#pragma unroll
            for (int e = 0; e < 8; ++e) m = max(m, w[e] & 0x7fffffffu);
            return m;
        } else {
            // two to a word: the high halves compare as the words they begin, the low ones shifted up
            uint32_t hi = 0, lo = 0;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                hi = max(hi, w[e] & 0x7fff0000u);
                lo = max(lo, w[e] & 0x7fffu);
            }
            return max(hi, lo << 16);
        }
    }
    __device__ __forceinline__ void values(float (&x)[8]) const {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            if constexpr (sizeof(T) == 4)
                x[e] = __uint_as_float(w[e]);
            else
                x[e] = __uint_as_float(e & 1 ? w[e / 2] & 0xffff0000u : w[e / 2] << 16);
        }
    }
};

template <typename T>
__device__ __forceinline__ void store8(T *p, const float (&x)[8]) {
    if constexpr (sizeof(T) == 4) {
        *(f32x4_any *)p = f32x4{x[0], x[1], x[2], x[3]};
        *(f32x4_any *)(p + 4) = f32x4{x[4], x[5], x[6], x[7]};
    } else {
        *(u32x4_any *)p = u32x4{pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]), pack_bf16x2(x[4], x[5]),
                                pack_bf16x2(x[6], x[7])};
    }
}

template <int WIDTH>
__device__ __forceinline__ uint32_t max_over(uint32_t v) {
#pragma unroll
    for (int o = 1; o < WIDTH; o <<= 1) {
        const uint32_t w = (uint32_t)__shfl_xor((int)v, o, 64);
        v = v > w ? v : w;
    }
    return v;
}

// Nibble of channel e of an octet in a key word.
__device__ __forceinline__ constexpr int key_nibble(int e) { return e / 2 + 4 * (e & 1); }

template <typename T, int BITS, int D>
__global__ __launch_bounds__(CM_THREADS) void cache_write(const CacheMoveArgs p) {
    constexpr int OCT = D / 8;                    // threads of one block of four positions
    constexpr int ROW = D * BITS / 8;             // bytes of a token's codes
    constexpr int BIAS = BITS == 4 ? 8 : 128;
    constexpr float L = BITS == 4 ? 7.f : 127.f;
    // Units (a block of a head of a sequence) of OCT threads; 32-bit divisions, the 64-bit ones take 1 us.
    const uint32_t unit = blockIdx.x * (uint32_t)(CM_THREADS / OCT) + threadIdx.x / OCT;
    const int c = threadIdx.x % OCT;
    const bool live = unit < p.units;  // the same for all lanes of a unit, which shuffles among themselves
    const uint32_t bh = live ? unit / (uint32_t)p.blocks : 0, blk = live ? unit % (uint32_t)p.blocks : 0;
    const uint32_t b = bh / (uint32_t)p.c.kv_heads, h = bh % (uint32_t)p.c.kv_heads;
    const int64_t p0 = p.start[b];
    int64_t cnt = p.n;
    if (p.count) cnt = min(cnt, max((int64_t)p.count[b], (int64_t)0));
    const int64_t pb = ((p0 >> 2) + blk) * 4;
    const T *Kp = (const T *)p.K + p.lay.at(b, h) + 8 * c, *Vp = (const T *)p.V + p.lay.at(b, h) + 8 * c;
    char *region = p.c.data + bh * p.c.region;
    Raw8<T> kx[4], vx[4];
    bool ok[4];
    int some = 0, all = 1;
#pragma unroll
    for (int t = 0; t < 4; ++t) {
        const int64_t pos = pb + t, i = pos - p0;
        ok[t] = live && i >= 0 && i < cnt && pos >= 0 && pos < p.c.capacity;
        some |= ok[t];
        all &= ok[t];
        if (ok[t]) {
            kx[t].load(Kp + i * p.lay.rs);
            vx[t].load(Vp + i * p.lay.rs);
        } else {
            kx[t].zero();
            vx[t].zero();
        }
    }
    const int s = c / 4, g = c % 4;
    constexpr int WORDS = BITS;  // 8 channels of four tokens
    u32x4 *vd = (u32x4 *)(region + p.c.v_off + (pb / 4) * (4 * ROW) + c * (4 * WORDS));
    // What a block that is covered in part holds, loaded beside the new tokens rather than after their codes.
    u32x4 old[WORDS / 4];
    if (some && !all) {
#pragma unroll
        for (int q = 0; q < WORDS / 4; ++q) old[q] = vd[q];
    }
    uint32_t vu[4][8];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
        const float ks = quant_step<true>(max_over<4>(kx[t].most()), L), ki = quant_inverse(ks);
        const float vs = quant_step<true>(max_over<OCT>(vx[t].most()), L), vi = quant_inverse(vs);
        float x[8];
        uint32_t ku[8];
        kx[t].values(x);
        quant_codes<BIAS>(x, ks, ki, ku);
        vx[t].values(x);
        quant_codes<BIAS>(x, vs, vi, vu[t]);
        if (!ok[t]) continue;
        const int64_t pos = pb + t;
        char *kd = region + pos * ROW + g * (ROW / 4);
        if constexpr (BITS == 4) {
            // key_nibble: bytes of channels (0, 2), (4, 6), (1, 3), (5, 7)
            *(uint32_t *)(kd + 4 * s) = bytes4(ku[0], ku[4], ku[1], ku[5]) | bytes4(ku[2], ku[6], ku[3], ku[7]) << 4;
        } else {
            *(u32x2 *)(kd + 8 * s) = u32x2{bytes4(ku[0], ku[1], ku[2], ku[3]), bytes4(ku[4], ku[5], ku[6], ku[7])};
        }
        if (g == 0) *(uint16_t *)(region + p.c.ks_off + (pos * (D / CACHE_GROUP) + s) * 2) = f32_to_bf16_rne(ks);
        if (c == 0) *(uint16_t *)(region + p.c.vs_off + pos * 2) = f32_to_bf16_rne(vs);
    }
    if (!some) return;
    uint32_t w[WORDS];
#pragma unroll
    for (int i = 0; i < WORDS; ++i) {
        if constexpr (BITS == 4) {
            const int e = 4 * (i / 2), t = 2 * (i & 1);
            w[i] = bytes4(vu[t][e], vu[t][e + 2], vu[t + 1][e], vu[t + 1][e + 2]) |
                   bytes4(vu[t][e + 1], vu[t][e + 3], vu[t + 1][e + 1], vu[t + 1][e + 3]) << 4;
        } else {
            w[i] = bytes4(vu[0][i], vu[1][i], vu[2][i], vu[3][i]);
        }
    }
#pragma unroll
    for (int q = 0; q < WORDS / 4; ++q) {
        u32x4 v = {w[4 * q], w[4 * q + 1], w[4 * q + 2], w[4 * q + 3]};
        if (!all) {
            // the other tokens' halves (bytes) of every word stay
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                uint32_t mine;
                if constexpr (BITS == 4)
                    mine = (ok[2 * (i & 1)] ? 0xffffu : 0u) | (ok[2 * (i & 1) + 1] ? 0xffff0000u : 0u);
                else
                    mine = (ok[0] ? 0xffu : 0u) | (ok[1] ? 0xff00u : 0u) | (ok[2] ? 0xff0000u : 0u) | (ok[3] ? 0xff000000u : 0u);
                v[i] = (v[i] & mine) | (old[q][i] & ~mine);
            }
        }
        vd[q] = v;
    }
}

template <typename T, int BITS, int D>
__global__ __launch_bounds__(CM_THREADS) void cache_read(const CacheMoveArgs p) {
    constexpr int OCT = D / 8;
    constexpr int ROW = D * BITS / 8;
    constexpr int BIAS = BITS == 4 ? 8 : 128;
    constexpr int WORDS = BITS;
    const uint32_t unit = blockIdx.x * (uint32_t)(CM_THREADS / OCT) + threadIdx.x / OCT;
    const int c = threadIdx.x % OCT;
    if (unit >= p.units) return;
    const uint32_t bh = unit / (uint32_t)p.blocks, b = bh / (uint32_t)p.c.kv_heads, h = bh % (uint32_t)p.c.kv_heads;
    const int64_t pb = ((p.begin >> 2) + unit % (uint32_t)p.blocks) * 4;
    const char *region = p.c.data + bh * p.c.region;
    T *Ko = (T *)p.Ko + p.lay.at(b, h) + 8 * c, *Vo = (T *)p.Vo + p.lay.at(b, h) + 8 * c;
    const int s = c / 4, g = c % 4;
    uint32_t w[WORDS];
    const u32x4 *vd = (const u32x4 *)(region + p.c.v_off + (pb / 4) * (4 * ROW) + c * (4 * WORDS));
#pragma unroll
    for (int q = 0; q < WORDS / 4; ++q)
#pragma unroll
        for (int i = 0; i < 4; ++i) w[4 * q + i] = vd[q][i];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
        const int64_t pos = pb + t;
        if (pos < p.begin || pos >= p.begin + p.n) continue;
        const float ks = bf16_to_f32(*(const uint16_t *)(region + p.c.ks_off + (pos * (D / CACHE_GROUP) + s) * 2));
        const float vs = bf16_to_f32(*(const uint16_t *)(region + p.c.vs_off + pos * 2));
        const char *kd = region + pos * ROW + g * (ROW / 4);
        uint32_t k0, k1;
        if constexpr (BITS == 4) {
            k0 = k1 = *(const uint32_t *)(kd + 4 * s);
        } else {
            const u32x2 kk = *(const u32x2 *)(kd + 8 * s);
            k0 = kk[0], k1 = kk[1];
        }
        float kx[8], vx[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const uint32_t ku = BITS == 4 ? (k0 >> (4 * key_nibble(e))) & 15u : ((e < 4 ? k0 : k1) >> (8 * (e & 3))) & 255u;
            const uint32_t vu = BITS == 4 ? (w[2 * (e / 4) + t / 2] >> (16 * (t & 1) + 4 * (e & 3))) & 15u
                                          : (w[e] >> (8 * t)) & 255u;
            kx[e] = (float)((int)ku - BIAS) * ks + 0.f;  // + 0: an untouched slot reads +0, not -8 * 0 = -0
            vx[e] = (float)((int)vu - BIAS) * vs + 0.f;
        }
        const int64_t i = pos - p.begin;
        store8(Ko + i * p.lay.rs, kx);
        store8(Vo + i * p.lay.rs, vx);
    }
}

template <bool WRITE, typename T, int BITS>
it_status launch_move(hipStream_t s, CacheMoveArgs a) {
    a.units = a.c.batch * a.c.kv_heads * a.blocks;  // below 2^31, checked by the caller
    const int64_t per = CM_THREADS / (a.c.head_dim / 8);
    const int64_t blocks = (a.units + per - 1) / per;
    if (const it_status st = check_blocks(WRITE ? "kv_cache_write" : "kv_cache_read", blocks); st != IT_OK) return st;
    const dim3 grid((unsigned)blocks), block(CM_THREADS);
    const int d = a.c.head_dim;
    if constexpr (WRITE) {
        if (d == 64) hipLaunchKernelGGL((cache_write<T, BITS, 64>), grid, block, 0, s, a);
        else if (d == 128) hipLaunchKernelGGL((cache_write<T, BITS, 128>), grid, block, 0, s, a);
        else hipLaunchKernelGGL((cache_write<T, BITS, 256>), grid, block, 0, s, a);
    } else {
        if (d == 64) hipLaunchKernelGGL((cache_read<T, BITS, 64>), grid, block, 0, s, a);
        else if (d == 128) hipLaunchKernelGGL((cache_read<T, BITS, 128>), grid, block, 0, s, a);
        else hipLaunchKernelGGL((cache_read<T, BITS, 256>), grid, block, 0, s, a);
    }
    IT_HIP_TRY(hipGetLastError());
    return IT_OK;
}

}  // namespace

it_status launch_cache_write(hipStream_t s, bool bf16, const CacheMoveArgs &a) {
    if (bf16) return a.c.bits == 4 ? launch_move<true, uint16_t, 4>(s, a) : launch_move<true, uint16_t, 8>(s, a);
    return a.c.bits == 4 ? launch_move<true, float, 4>(s, a) : launch_move<true, float, 8>(s, a);
}

it_status launch_cache_read(hipStream_t s, bool bf16, const CacheMoveArgs &a) {
    if (bf16) return a.c.bits == 4 ? launch_move<false, uint16_t, 4>(s, a) : launch_move<false, uint16_t, 8>(s, a);
    return a.c.bits == 4 ? launch_move<false, float, 4>(s, a) : launch_move<false, float, 8>(s, a);
}

}  // namespace it
