// Products of 8-bit integers with a step for each token and output channel, and the row quantiser. No
// counterpart in the reference, whose weights are FP32 or BF16.
//
//   y[m, n] = (sum_k a[m, k] b[n, k]) sa[m] sb[n] + bias[n],   a, b whole numbers of 8 bits
//
// The sum is exact (32-bit integers; K below 2^17), so only the three last operations round, in FP32.
//
// Tiles: v_mfma_i32_32x32x32_i8 takes 16 bytes of a row per lane exactly as the BF16 instruction of half its
// k does, so the tile moves as the BF16 one: 128 bytes of k per k-tile, global -> LDS directly
// (buffer_load_dwordx4 ... lds), the 16-byte chunk c of row r at position c ^ ((r >> 1) & 7), and a fragment
// (32 rows x 16 k a lane) is one ds_read_b128. 128 x 128 tiles, 64 x 64 a wave, four LDS stages.
#include <algorithm>

#include "gemm_tiles.hpp"
#include "quant.hpp"

namespace it {
namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x16 __attribute__((ext_vector_type(16)));
typedef __attribute__((address_space(3))) void lds_void_t;

constexpr uint32_t I8_OOB = 0x80000000u;  // a buffer load's range check turns this offset into zeros

// ------------------------------------------------------------------ row quantiser

template <typename T>
__device__ __forceinline__ float value_of(T x) {
    if constexpr (sizeof(T) == 4)
        return x;
    else
        return bf16_to_f32(x);
}

// One block a row: the largest |x| first, then the codes. Codes from `cols` to the next multiple of 16 are 0.
template <typename T>
__global__ __launch_bounds__(256) void quantize_rows(const T *X, int64_t ldx, int64_t cols, int8_t *codes, int64_t ldc,
                                                     float *steps) {
    __shared__ uint32_t most[4];
    const int64_t row = blockIdx.x;
    const T *x = X + row * ldx;
    uint32_t mb = 0;
    for (int64_t c = threadIdx.x; c < cols; c += 256) mb = max(mb, abs_bits(value_of(x[c])));
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) mb = max(mb, (uint32_t)__shfl_xor((int)mb, o, 64));
    if ((threadIdx.x & 63) == 0) most[threadIdx.x >> 6] = mb;
    __syncthreads();
    mb = max(max(most[0], most[1]), max(most[2], most[3]));
    const float s = quant_step<false>(mb, 127.f), inv = quant_inverse(s);
    const int64_t padded = (cols + 15) / 16 * 16;
    for (int64_t c = threadIdx.x; c < padded; c += 256)
        codes[row * ldc + c] = c < cols && inv > 0.f ? (int8_t)quant_code(value_of(x[c]), s, inv, 127.f) : (int8_t)0;
    if (threadIdx.x == 0) steps[row] = s;
}

// ------------------------------------------------------------------ tiles

__device__ __forceinline__ __amdgpu_buffer_rsrc_t i8_rsrc(const void *base, int64_t bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void *>(base), (short)0, (int)bytes, 0x00020000);
}

// 128 rows of one operand.
struct I8Operand {
    static constexpr int BK = 128, NI = 4;  // load instructions a wave and k-tile (8 rows each)
    __amdgpu_buffer_rsrc_t rsrc;
    uint32_t voff[NI];
    uint32_t chunk[NI];  // byte of the lane's chunk within the k-tile
    __device__ __forceinline__ void init(const int8_t *base, int64_t ld, int64_t rows, int64_t K, int wave, int lane) {
        rows = min(rows, (int64_t)128);
        rsrc = i8_rsrc(base, (rows - 1) * ld + K);
#pragma unroll
        for (int j = 0; j < NI; ++j) {
            const int r = 8 * (NI * wave + j) + (lane >> 3);
            chunk[j] = 16u * ((lane & 7) ^ ((r >> 1) & 7));
            voff[j] = (uint32_t)(r * ld) + chunk[j];
        }
    }
    // The k-tile at byte kk; chunks at K and beyond are zeros.
    __device__ __forceinline__ void issue(char *stage, uint32_t kk, uint32_t K, int wave) const {
#pragma unroll
        for (int j = 0; j < NI; ++j) {
            const uint32_t off = kk + chunk[j] < K ? voff[j] : I8_OOB;
            uint32_t x = (uint32_t)(uintptr_t)(lds_void_t *)(stage + (NI * wave + j) * 1024);
            asm("" : "+s"(x));  // the explicit waits order the loads, not the compiler's
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (lds_void_t *)(uintptr_t)x, 16, off, kk, 0, 0);
        }
    }
    // Rows row .. + 31, k 32 ks .. + 31: lane l holds row + l % 32 at k 32 ks + 16 (l / 32) .. + 15.
    __device__ __forceinline__ static i32x4 frag(const char *st, int row, int ks, int lane) {
        const int fr = lane & 31, y = (lane >> 5) ^ ((fr >> 1) & 7);
        return *(const i32x4 *)(st + (row + fr) * 128 + (((2 * ks) ^ y) * 16));
    }
};

constexpr int i8_waitcnt(int vm, int lgkm) { return (vm & 15) | ((vm >> 4) << 14) | (7 << 4) | (lgkm << 8); }

__device__ __forceinline__ void i8_store(const GemmI8Args &p, int64_t row, int64_t col, int acc, float sa) {
    if (row >= p.M || col >= p.N) return;
    float v = (float)acc * sa * p.sB[col];
    if (p.bias) v += p.bias[col];
    if (p.out_bf16)
        ((uint16_t *)p.C)[row * p.ldc + col] = f32_to_bf16_rne(v);
    else
        ((float *)p.C)[row * p.ldc + col] = v;
}

__global__ __launch_bounds__(NTHREADS) void gemm_i8_128(const GemmI8Args p) {
    constexpr int TILE = 128 * 128, BK = 128;
    __shared__ __attribute__((aligned(1024))) char st[2][2 * TILE];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave >> 1, wn = wave & 1;
    int tm, tn;
    map_tile(blockIdx.x, p.tiles_m, p.tiles_n, tm, tn);
    const int64_t m0 = (int64_t)tm * 128, n0 = (int64_t)tn * 128;
    I8Operand oa, ob;
    oa.init(p.A + m0 * p.lda, p.lda, p.M - m0, p.K, wave, lane);
    ob.init(p.B + n0 * p.ldb, p.ldb, p.N - n0, p.K, wave, lane);
    i32x16 acc[2][2];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[i][j][r] = 0;
    const uint32_t K = (uint32_t)p.K;
    const int ntiles = (int)((p.K + BK - 1) / BK);
    auto issue = [&](int t) {
        char *s = st[t & 1];
        oa.issue(s, (uint32_t)t * BK, K, wave);
        ob.issue(s + TILE, (uint32_t)t * BK, K, wave);
    };
    if (ntiles > 0) issue(0);
    for (int t = 0; t < ntiles; ++t) {
        __builtin_amdgcn_s_waitcnt(i8_waitcnt(0, 0));  // tile t has landed, tile t - 1's fragments are read
        __syncthreads();
        if (t + 1 < ntiles) issue(t + 1);
        const char *s = st[t & 1];
#pragma unroll
        for (int ks = 0; ks < 4; ++ks) {
            i32x4 fa[2], fb[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) fa[i] = I8Operand::frag(s, wm * 64 + 32 * i, ks, lane);
#pragma unroll
            for (int j = 0; j < 2; ++j) fb[j] = I8Operand::frag(s + TILE, wn * 64 + 32 * j, ks, lane);
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int j = 0; j < 2; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(fa[i], fb[j], acc[i][j], 0, 0, 0);
        }
    }
    // acc[i][j][r]: row 32 i + 8 (r / 4) + 4 (lane / 32) + r % 4, column 32 j + lane % 32 of the wave's 64 x 64.
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            const int64_t row = m0 + wm * 64 + 32 * i + 8 * (r >> 2) + 4 * (lane >> 5) + (r & 3);
            const float sa = row < p.M ? p.sA[row] : 0.f;
#pragma unroll
            for (int j = 0; j < 2; ++j) i8_store(p, row, n0 + wn * 64 + 32 * j + (lane & 31), acc[i][j][r], sa);
        }
}

}  // namespace

it_status launch_quantize_i8(hipStream_t s, bool bf16, int64_t rows, int64_t cols, const void *X, int64_t ldx,
                             int8_t *codes, int64_t ldc, float *steps) {
    const dim3 grid((unsigned)rows), block(256);
    if (bf16)
        hipLaunchKernelGGL((quantize_rows<uint16_t>), grid, block, 0, s, (const uint16_t *)X, ldx, cols, codes, ldc, steps);
    else
        hipLaunchKernelGGL((quantize_rows<float>), grid, block, 0, s, (const float *)X, ldx, cols, codes, ldc, steps);
    IT_HIP_TRY(hipGetLastError());
    return IT_OK;
}

it_status launch_gemm_i8(it_context *ctx, GemmI8Args a) {
    a.tiles_m = (int)((a.M + 127) / 128);
    a.tiles_n = (int)((a.N + 127) / 128);
    hipLaunchKernelGGL(gemm_i8_128, dim3((unsigned)(a.tiles_m * a.tiles_n)), dim3(NTHREADS), 0, ctx->stream, a);
    IT_HIP_TRY(hipGetLastError());
    return IT_OK;
}

}  // namespace it
