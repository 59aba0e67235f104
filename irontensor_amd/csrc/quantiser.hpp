// The quantiser of the cache and of the 8-bit products (device code).
#pragma once

#include "mfma.hpp"

namespace it {

// A group of values shares the step s = max|x| * (1 / L) (L: the largest code; FP32, 1 / L rounded) and keeps
// n = rne(x / s) of the step as it is stored. A step below the smallest normal number is stored as 0 (the
// group reads as zeros); a group that holds a NaN or an infinity gets s = NaN and codes 0, so that all of it
// reads as NaN.
constexpr float QUANT_TINY = 1.17549435e-38f;  // 2^-126

// The step from the largest |x|, given as its bits (compared as integers they order NaN above infinity
// above every number, so one integer maximum finds non-finite values too). BF16: the cache's steps are
// rounded to BF16, which costs no accuracy to speak of: codes are chosen for the step as stored, which is
// within 2^-8 of the unrounded one.
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

}  // namespace it
