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

namespace it {
namespace {

constexpr int CM_THREADS = 256;

template <typename T>
__device__ __forceinline__ void load8(const T *p, int vec_ok, float (&x)[8]) {
    if constexpr (sizeof(T) == 4) {
        if (vec_ok) {
            const f32x4 a = *(const f32x4 *)p, b = *(const f32x4 *)(p + 4);
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] = a[e], x[4 + e] = b[e];
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = p[e];
        }
    } else {
        if (vec_ok) {
            const u32x4 h = *(const u32x4 *)p;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                x[2 * e] = __uint_as_float(h[e] << 16);
                x[2 * e + 1] = __uint_as_float(h[e] & 0xffff0000u);
            }
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = bf16_to_f32(p[e]);
        }
    }
}

template <typename T>
__device__ __forceinline__ void store8(T *p, int vec_ok, const float (&x)[8]) {
    if constexpr (sizeof(T) == 4) {
        if (vec_ok) {
            *(f32x4 *)p = f32x4{x[0], x[1], x[2], x[3]};
            *(f32x4 *)(p + 4) = f32x4{x[4], x[5], x[6], x[7]};
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) p[e] = x[e];
        }
    } else {
        if (vec_ok) {
            *(u32x4 *)p = u32x4{pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]), pack_bf16x2(x[4], x[5]),
                                pack_bf16x2(x[6], x[7])};
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) p[e] = f32_to_bf16_rne(x[e]);
        }
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

__device__ __forceinline__ uint32_t max8(const float (&x)[8]) {
    uint32_t m = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) m = max(m, abs_bits(x[e]));
    return m;
}

// Nibble of channel e of an octet in a key word.
__device__ __forceinline__ constexpr int key_nibble(int e) { return e / 2 + 4 * (e & 1); }

template <typename T, int BITS, int D>
__global__ __launch_bounds__(CM_THREADS) void cache_write(const CacheMoveArgs p) {
    constexpr int OCT = D / 8;                    // threads of one block of four positions
    constexpr int ROW = D * BITS / 8;             // bytes of a token's codes
    constexpr int BIAS = BITS == 4 ? 8 : 128;
    constexpr float L = BITS == 4 ? 7.f : 127.f;
    const int64_t item = (int64_t)blockIdx.x * CM_THREADS + threadIdx.x;
    const int c = (int)(item % OCT);
    const int64_t unit = item / OCT;
    const int64_t total = p.c.batch * p.c.kv_heads * p.blocks;
    const bool live = unit < total;  // the same for all lanes of a unit, which shuffles among themselves
    const int64_t bh = live ? unit / p.blocks : 0, blk = live ? unit % p.blocks : 0;
    const int64_t b = bh / p.c.kv_heads;
    const int64_t p0 = p.start[b];
    int64_t cnt = p.n;
    if (p.count) cnt = min(cnt, max((int64_t)p.count[b], (int64_t)0));
    const int64_t pb = ((p0 >> 2) + blk) * 4;
    const T *Kp = (const T *)p.K + p.lay.at(bh) + 8 * c, *Vp = (const T *)p.V + p.lay.at(bh) + 8 * c;
    char *region = p.c.data + bh * p.c.region;
    float kx[4][8], vx[4][8];
    bool ok[4];
    int some = 0, all = 1;
#pragma unroll
    for (int t = 0; t < 4; ++t) {
        const int64_t pos = pb + t, i = pos - p0;
        ok[t] = live && i >= 0 && i < cnt && pos >= 0 && pos < p.c.capacity;
        some |= ok[t];
        all &= ok[t];
        if (ok[t]) {
            load8(Kp + i * p.lay.rs, p.vec_ok, kx[t]);
            load8(Vp + i * p.lay.rs, p.vec_ok, vx[t]);
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) kx[t][e] = vx[t][e] = 0.f;
        }
    }
    float vn[4][8];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
        const float ks = quant_step<true>(max_over<4>(max8(kx[t])), L), ki = quant_inverse(ks);
        const float vs = quant_step<true>(max_over<OCT>(max8(vx[t])), L), vi = quant_inverse(vs);
        float kn[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            kn[e] = ki > 0.f ? quant_code(kx[t][e], ks, ki, L) : 0.f;
            vn[t][e] = vi > 0.f ? quant_code(vx[t][e], vs, vi, L) : 0.f;
        }
        if (!ok[t]) continue;
        const int64_t pos = pb + t;
        const int s = c / 4, g = c % 4;
        char *kd = region + pos * ROW + g * (ROW / 4);
        if constexpr (BITS == 4) {
            uint32_t w = 0;
#pragma unroll
            for (int e = 0; e < 8; ++e) w |= (uint32_t)((int)kn[e] + BIAS) << (4 * key_nibble(e));
            *(uint32_t *)(kd + 4 * s) = w;
        } else {
            u32x2 w = {0u, 0u};
#pragma unroll
            for (int e = 0; e < 8; ++e) w[e >> 2] |= (uint32_t)((int)kn[e] + BIAS) << (8 * (e & 3));
            *(u32x2 *)(kd + 8 * s) = w;
        }
        if (g == 0) *(uint16_t *)(region + p.c.ks_off + (pos * (D / CACHE_GROUP) + s) * 2) = f32_to_bf16_rne(ks);
        if (c == 0) *(uint16_t *)(region + p.c.vs_off + pos * 2) = f32_to_bf16_rne(vs);
    }
    if (!some) return;
    constexpr int WORDS = BITS;  // 8 channels of four tokens
    uint32_t w[WORDS], keep[WORDS];
#pragma unroll
    for (int i = 0; i < WORDS; ++i) w[i] = keep[i] = 0;
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const uint32_t u = (uint32_t)((int)vn[t][e] + BIAS);
            const int i = BITS == 4 ? 2 * (e / 4) + t / 2 : e;
            const int sh = BITS == 4 ? 16 * (t & 1) + 4 * (e & 3) : 8 * t;
            w[i] |= ok[t] ? u << sh : 0u;
            keep[i] |= ok[t] ? 0u : (BITS == 4 ? 15u : 255u) << sh;
        }
    u32x4 *vd = (u32x4 *)(region + p.c.v_off + (pb / 4) * (4 * ROW) + c * (4 * WORDS));
#pragma unroll
    for (int q = 0; q < WORDS / 4; ++q) {
        u32x4 v = {w[4 * q], w[4 * q + 1], w[4 * q + 2], w[4 * q + 3]};
        if (!all) {
            const u32x4 old = vd[q];
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] |= old[i] & keep[4 * q + i];
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
    const int64_t item = (int64_t)blockIdx.x * CM_THREADS + threadIdx.x;
    const int c = (int)(item % OCT);
    const int64_t unit = item / OCT;
    if (unit >= p.c.batch * p.c.kv_heads * p.blocks) return;
    const int64_t bh = unit / p.blocks, pb = ((p.begin >> 2) + unit % p.blocks) * 4;
    const char *region = p.c.data + bh * p.c.region;
    T *Ko = (T *)p.Ko + p.lay.at(bh) + 8 * c, *Vo = (T *)p.Vo + p.lay.at(bh) + 8 * c;
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
        store8(Ko + i * p.lay.rs, p.vec_ok, kx);
        store8(Vo + i * p.lay.rs, p.vec_ok, vx);
    }
}

template <bool WRITE, typename T, int BITS>
it_status launch_move(hipStream_t s, const CacheMoveArgs &a) {
    const int64_t items = a.c.batch * a.c.kv_heads * a.blocks * (a.c.head_dim / 8);
    const dim3 grid((unsigned)((items + CM_THREADS - 1) / CM_THREADS)), block(CM_THREADS);
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
