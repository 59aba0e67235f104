// Products of 8-bit integers with a step for each token and output channel, and the row quantiser. No
// counterpart in the reference, whose weights are FP32 or BF16.
//
//   y[m, n] = (sum_k a[m, k] b[n, k]) sa[m] sb[n] + bias[n],   a, b whole numbers of 8 bits
//
// The sum is exact (32-bit integers; K below 2^17), so only the three last operations round, in FP32.
//
// Tiles: v_mfma_i32_32x32x32_i8 takes 16 bytes of a row per lane exactly as the BF16 instruction of half its
// k does, so the tiles move as the BF16 ones (gemm_bf16_dtl): 128 bytes of k per k-tile, global -> LDS
// directly (buffer_load_dwordx4 ... lds), the 16-byte chunk c of row r at position c ^ ((r >> 1) & 7), a
// fragment (32 rows x 16 k a lane) one ds_read_b128.
#include <algorithm>

#include "gemm_tiles.hpp"
#include "quant.hpp"
#include "quantiser.hpp"

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

// 8 values at x[c ..], zeros from `cols` on. Vector loads that need an element's alignment only.
typedef uint32_t u32x4_any __attribute__((ext_vector_type(4), aligned(2)));

template <typename T>
__device__ __forceinline__ void row8(const T *x, int64_t c, int64_t cols, float (&v)[8]) {
    if (c + 8 <= cols) {
        if constexpr (sizeof(T) == 4) {
            const f32x4 a = *(const f32x4_any *)(x + c), b = *(const f32x4_any *)(x + c + 4);
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = a[e], v[4 + e] = b[e];
        } else {
            const u32x4 h = *(const u32x4_any *)(x + c);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                v[2 * e] = __uint_as_float(h[e] << 16);
                v[2 * e + 1] = __uint_as_float(h[e] & 0xffff0000u);
            }
        }
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = c + e < cols ? value_of(x[c + e]) : 0.f;
    }
}

__device__ __forceinline__ u32x2 codes8(const float (&v)[8], float s, float inv) {
    uint32_t u[8];
    quant_codes<0>(v, s, inv, u);
    return u32x2{bytes4(u[0], u[1], u[2], u[3]), bytes4(u[4], u[5], u[6], u[7])};
}

// RL lanes a row (64: four rows a block; 256: a block a row), each with VN vectors of 8 values in registers, so
// that the row is read once; a longer row is read again from VN * 8 * RL on. Codes from `cols` to
// `padded` are 0. 8192 x 4096 BF16 (101 MB) takes 29 us: 3.5 TB/s.
template <typename T, int RL, int VN>
__global__ __launch_bounds__(256) void quantize_rows(const T *X, int64_t ldx, int64_t rows, int64_t cols, int64_t padded,
                                                     int8_t *codes, int64_t ldc, float *steps) {
    __shared__ uint32_t most[4];
    const int lane = threadIdx.x % RL;
    const int64_t row = (int64_t)blockIdx.x * (256 / RL) + threadIdx.x / RL;
    if (row >= rows) return;  // whole waves; RL 256: never
    const T *x = X + row * ldx;
    constexpr int64_t HELD = (int64_t)VN * 8 * RL;
    float v[VN][8];
    uint32_t mb = 0;
#pragma unroll
    for (int i = 0; i < VN; ++i) {
        row8(x, (int64_t)(i * RL + lane) * 8, cols, v[i]);
#pragma unroll
        for (int e = 0; e < 8; ++e) mb = max(mb, abs_bits(v[i][e]));
    }
    for (int64_t c = HELD + lane * 8; c < cols; c += RL * 8) {
        float t[8];
        row8(x, c, cols, t);
#pragma unroll
        for (int e = 0; e < 8; ++e) mb = max(mb, abs_bits(t[e]));
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) mb = max(mb, (uint32_t)__shfl_xor((int)mb, o, 64));
    if constexpr (RL == 256) {
        if ((threadIdx.x & 63) == 0) most[threadIdx.x >> 6] = mb;
        __syncthreads();
        mb = max(max(most[0], most[1]), max(most[2], most[3]));
    }
    const float s = quant_step<false>(mb, 127.f), inv = quant_inverse(s);
    int8_t *out = codes + row * ldc;
#pragma unroll
    for (int i = 0; i < VN; ++i) {
        const int64_t c = (int64_t)(i * RL + lane) * 8;
        if (c < padded) *(u32x2 *)(out + c) = codes8(v[i], s, inv);
    }
    for (int64_t c = HELD + lane * 8; c < padded; c += RL * 8) {
        float t[8];
        row8(x, c, cols, t);
        *(u32x2 *)(out + c) = codes8(t, s, inv);
    }
    if (lane == 0) steps[row] = s;
}

// ------------------------------------------------------------------ tiles

__device__ __forceinline__ __amdgpu_buffer_rsrc_t i8_rsrc(const void *base, int64_t bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void *>(base), (short)0, (int)bytes, 0x00020000);
}

// ROWS rows of one operand. WHOLE: K is a multiple of the k-tile.
template <int ROWS, bool WHOLE>
struct I8Operand {
    static constexpr int BK = 128, NI = ROWS / 32;  // load instructions a wave and k-tile (8 rows each)
    const void *base;
    int bytes;
    uint32_t voff[NI];
    int wave, lane;
    __device__ __forceinline__ void init(const int8_t *first, int64_t ld, int64_t rows, int64_t K, int w, int l) {
        rows = min(rows, (int64_t)ROWS);
        base = first;
        bytes = (int)((rows - 1) * ld + K);
        wave = w;
        lane = l;
#pragma unroll
        for (int j = 0; j < NI; ++j) voff[j] = (uint32_t)((8 * (NI * wave + j) + (lane >> 3)) * ld) + chunk(j);
    }
    // Byte of the lane's chunk within the k-tile.
    __device__ __forceinline__ uint32_t chunk(int j) const {
        const int r = 8 * (NI * wave + j) + (lane >> 3);
        return 16u * ((lane & 7) ^ ((r >> 1) & 7));
    }
    // The k-tile at byte kk; k-tiles at K and beyond are zeros (a descriptor of no bytes), and so are the last
    // one's chunks there. OPAQUE: the LDS address goes through an empty asm, so that the caller's waits order
    // these loads and the compiler adds none of its own before other LDS reads.
    template <bool OPAQUE>
    __device__ __forceinline__ void issue(char *stage, uint32_t kk, uint32_t K) const {
        const __amdgpu_buffer_rsrc_t rsrc = i8_rsrc(base, kk < K ? bytes : 0);
        const bool part = !WHOLE && kk + BK > K;
#pragma unroll
        for (int j = 0; j < NI; ++j) {
            uint32_t off = voff[j];
            if constexpr (!WHOLE)
                if (part && kk + chunk(j) >= K) off = I8_OOB;
            lds_void_t *dst = (lds_void_t *)(stage + (NI * wave + j) * 1024);
            if constexpr (OPAQUE) {
                uint32_t x = (uint32_t)(uintptr_t)dst;
                asm("" : "+s"(x));
                dst = (lds_void_t *)(uintptr_t)x;
            }
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, dst, 16, off, kk, 0, 0);
        }
    }
    // Rows row .. + 31, k 32 ks .. + 31: lane l holds row + l % 32 at k 32 ks + 16 (l / 32) .. + 15.
    __device__ __forceinline__ static i32x4 frag(const char *st, int row, int ks, int lane) {
        const int fr = lane & 31, y = (lane >> 5) ^ ((fr >> 1) & 7);
        return *(const i32x4 *)(st + (row + fr) * 128 + (((2 * ks) ^ y) * 16));
    }
};

constexpr int i8_waitcnt(int vm, int lgkm) { return (vm & 15) | ((vm >> 4) << 14) | (7 << 4) | (lgkm << 8); }

// Four columns of a row from their sums.
__device__ __forceinline__ void i8_store4(const GemmI8Args &p, i32x4 acc, int64_t row, int64_t col, float sa, f32x4 sb,
                                          f32x4 bias) {
    f32x4 v;
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = (float)acc[e] * sa * sb[e] + bias[e];
    const int64_t at = row * p.ldc + col;
    if (col + 4 <= p.N) {
        if (p.out_bf16)
            *(u32x2_any *)((uint16_t *)p.C + at) = u32x2{pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3])};
        else
            *(f32x4_any *)((float *)p.C + at) = v;
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (col + e < p.N) store_out(p.C, at + e, v[e], p.out_bf16);
    }
}

__device__ __forceinline__ void i8_column_terms(const GemmI8Args &p, int64_t col, f32x4 &sb, f32x4 &bias) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const bool ok = col + e < p.N;
        sb[e] = ok ? p.sB[col + e] : 0.f;
        bias[e] = ok && p.bias ? p.bias[col + e] : 0.f;
    }
}

// 64 FA x 64 FB output tiles, 2 x 2 waves of 32 FA x 32 FB, NS LDS stages. A k-tile is four k-steps; each
// step's products run with the next step's fragment reads, the last with the next tile's first reads and the
// loads of the tile NS ahead into the stage just read. Two stages are two LDS objects, which tell the compiler
// that loads into one never meet reads of the other; with more the loads are opaque.
template <int FA, int FB, int NS, bool WHOLE>
__global__ __launch_bounds__(NTHREADS) __attribute__((amdgpu_waves_per_eu(NS * (FA + FB) > 10 ? 1 : 2)))
void gemm_i8_tile(const GemmI8Args p) {
    constexpr int BM = 64 * FA, BN = 64 * FB, BK = 128, TILE = BM * BK, STAGE = (BM + BN) * BK;
    constexpr bool OPAQUE = NS > 2;
    constexpr int PIECE = 32 * (32 * FB + 4) * 4;  // bytes of a wave's piece of the epilogue
    static_assert((NS > 2 ? 4 : 2) * PIECE <= (NS > 2 ? NS : 1) * STAGE, "the epilogue's pieces fit the stages");
    __shared__ __attribute__((aligned(1024))) char st0[NS > 2 ? NS * STAGE : STAGE];
    __shared__ __attribute__((aligned(1024))) char st1[NS > 2 ? 16 : STAGE];
    auto stage = [&](int i) -> char * { return NS > 2 ? st0 + i * STAGE : i ? st1 : st0; };
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave >> 1, wn = wave & 1;
    int tm, tn;
    map_tile(blockIdx.x, p.tiles_m, p.tiles_n, tm, tn);
    const int64_t m0 = (int64_t)tm * BM, n0 = (int64_t)tn * BN;
    using OA = I8Operand<BM, WHOLE>;
    using OB = I8Operand<BN, WHOLE>;
    OA oa;
    OB ob;
    oa.init(p.A + m0 * p.lda, p.lda, p.M - m0, p.K, wave, lane);
    ob.init(p.B + n0 * p.ldb, p.ldb, p.N - n0, p.K, wave, lane);
    // The steps and the bias of the tile now: loaded in the epilogue, row by row, they cost it 12 us.
    __shared__ float row_steps[BM];
    if (tid < BM) row_steps[tid] = m0 + tid < p.M ? p.sA[m0 + tid] : 0.f;
    constexpr int EC = 32 * FB, EP = EC + 4, LPR = EC / 4, RPI = 64 / LPR;
    const int c4 = lane % LPR * 4, rl = lane / LPR;
    const int64_t col = n0 + wn * EC + c4;
    f32x4 sb, bias;
    i8_column_terms(p, col, sb, bias);
    i32x16 acc[FA][FB];
#pragma unroll
    for (int i = 0; i < FA; ++i)
#pragma unroll
        for (int j = 0; j < FB; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[i][j][r] = 0;
    const uint32_t K = (uint32_t)p.K;
    const int ntiles = (int)((p.K + BK - 1) / BK);
    auto issue = [&](int t, char *stage) {
        oa.template issue<OPAQUE>(stage, (uint32_t)t * BK, K);
        ob.template issue<OPAQUE>(stage + TILE, (uint32_t)t * BK, K);
    };
    i32x4 fa0[FA], fb0[FB], fa1[FA], fb1[FB];
    auto frags = [&](i32x4 (&fa)[FA], i32x4 (&fb)[FB], const char *s, int ks) {
#pragma unroll
        for (int i = 0; i < FA; ++i) fa[i] = OA::frag(s, wm * 32 * FA + 32 * i, ks, lane);
#pragma unroll
        for (int j = 0; j < FB; ++j) fb[j] = OB::frag(s + TILE, wn * 32 * FB + 32 * j, ks, lane);
    };
    auto products = [&](const i32x4 (&fa)[FA], const i32x4 (&fb)[FB]) {
#pragma unroll
        for (int i = 0; i < FA; ++i)
#pragma unroll
            for (int j = 0; j < FB; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(fa[i], fb[j], acc[i][j], 0, 0, 0);
    };
    constexpr int NLOAD = OA::NI + OB::NI;
    constexpr int PAIRS = FA * FB >= 2 ? FA * FB / 2 : 1;
    constexpr int DSR = (FA + FB + PAIRS - 1) / PAIRS, VMR = (NLOAD + PAIRS - 1) / PAIRS;
    auto body = [&](char *cur, const char *nxt, int t) {
        frags(fa1, fb1, cur, 1);
        products(fa0, fb0);
        frags(fa0, fb0, cur, 2);
        products(fa1, fb1);
        frags(fa1, fb1, cur, 3);
        products(fa0, fb0);
#pragma unroll
        for (int g = 0; g < 3 * PAIRS; ++g) {
            __builtin_amdgcn_sched_group_barrier(sg::DS_READ, DSR, 0);
            __builtin_amdgcn_sched_group_barrier(sg::MFMA, 2, 0);
        }
        // `cur` is read and tile t + 1 has landed (later ones may still be in flight); the barrier keeps the
        // block's reads of `cur` ahead of the loads into it, the fence the reads of `nxt` behind the barrier.
        __builtin_amdgcn_s_waitcnt(i8_waitcnt((NS - 2) * NLOAD, 0));
        if constexpr (NS == 2) {
            __syncthreads();
        } else {
            __builtin_amdgcn_s_barrier();
            __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
        }
        issue(t + NS, cur);  // past the last tile: zeros, so that the count in the wait holds
        frags(fa0, fb0, nxt, 0);
        products(fa1, fb1);
#pragma unroll
        for (int g = 0; g < PAIRS; ++g) {
            __builtin_amdgcn_sched_group_barrier(sg::DS_READ, DSR, 0);
            __builtin_amdgcn_sched_group_barrier(sg::VMEM_READ, VMR, 0);
            __builtin_amdgcn_sched_group_barrier(sg::MFMA, 2, 0);
        }
    };
    if (ntiles > 0) {
#pragma unroll
        for (int i = 0; i < NS - 1; ++i) issue(i, stage(i));
        __builtin_amdgcn_s_waitcnt(i8_waitcnt((NS - 2) * NLOAD, 15));  // tile 0 has landed
        __syncthreads();
        issue(NS - 1, stage(NS - 1));
        frags(fa0, fb0, stage(0), 0);
        // Whole rounds of the stages: tiles past the last are zeros.
        for (int t = 0; t < ntiles; t += NS) {
#pragma unroll
            for (int i = 0; i < NS; ++i) body(stage(i), stage((i + 1) % NS), t + i);
        }
        __builtin_amdgcn_s_waitcnt(i8_waitcnt(0, 0));  // the loads into dead stages, and the last fragment reads
    }
    __syncthreads();
    // Epilogue: 32 rows at a time through a piece of LDS of the wave's own, so that stores are whole lines.
    // acc[i][j][r]: row 32 i + 8 (r / 4) + 4 (lane / 32) + r % 4, column 32 j + lane % 32 of the wave's part.
    int *piece = (int *)(NS > 2 ? st0 + wave * PIECE : (wave & 1 ? st1 : st0) + (wave >> 1) * PIECE);
#pragma unroll
    for (int i = 0; i < FA; ++i) {
#pragma unroll
        for (int j = 0; j < FB; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r)
                piece[(8 * (r >> 2) + 4 * (lane >> 5) + (r & 3)) * EP + 32 * j + (lane & 31)] = acc[i][j][r];
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");  // a wave's LDS accesses complete in order
        if (col < p.N) {
#pragma unroll 8
            for (int q = 0; q < 32 / RPI; ++q) {
                const int rt = wm * 32 * FA + 32 * i + RPI * q + rl;
                if (m0 + rt < p.M)
                    i8_store4(p, *(const i32x4 *)(piece + (RPI * q + rl) * EP + c4), m0 + rt, col, row_steps[rt], sb, bias);
            }
        }
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    }
}

// ------------------------------------------------------------------ few rows

// M <= 16: every weight code is read once and used M times; reading it is the bound. As the BF16 kernel of the
// same shapes (gemv_nt): a block owns 16 output columns and splits K among its four waves; loads come in
// pairs, each instruction 8 whole 128-byte lines, and go through a 4 KB LDS slot of the wave into the layout
// of v_mfma_i32_16x16x64_i8 (lane l: row l % 16, 16 bytes at 16 (l / 16)).
constexpr int GI_UNROLL = 8;
__device__ __forceinline__ int gi_slot(int rr, int c) { return rr * 8 + (c ^ rr); }

template <bool XHI>
__global__ __launch_bounds__(NTHREADS) void gemv_i8(const GemmI8Args p) {
    constexpr int KCHUNK = 64;
    __shared__ u32x4 stage[4][2][4][64];  // a wave's two slots: W rows 0-7, 8-15, X rows 0-7, 8-15
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int r = lane & 15, g = lane >> 4;
    const int rl = lane >> 3, kc = lane & 7;
    const int64_t n0 = (int64_t)blockIdx.x * 16;
    const int64_t nrows = min((int64_t)16, p.N - n0);
    const __amdgpu_buffer_rsrc_t wrs = i8_rsrc(p.B + n0 * p.ldb, (nrows - 1) * p.ldb + p.K);
    const __amdgpu_buffer_rsrc_t xrs = i8_rsrc(p.A, (p.M - 1) * p.lda + p.K);
    const uint32_t wo0 = (uint32_t)(rl * p.ldb), wo1 = (uint32_t)((8 + rl) * p.ldb);
    const uint32_t xo0 = (uint32_t)(rl * p.lda), xo1 = (uint32_t)((8 + rl) * p.lda);
    const int wslot = gi_slot(rl, kc), rq = r >> 3, rr = r & 7;
    const int lo_slot = gi_slot(rr, g), hi_slot = gi_slot(rr, 4 + g), xq = XHI ? rq : 0;
    const int64_t span = (p.K + 4 * KCHUNK - 1) / (4 * KCHUNK) * KCHUNK;
    const int64_t kb = wave * span, ke = min(p.K, kb + span);
    i32x4 acc = {0, 0, 0, 0};
    for (int64_t k = kb; k < ke; k += GI_UNROLL * KCHUNK) {
        u32x4 wr[GI_UNROLL], xr[GI_UNROLL];
#pragma unroll
        for (int pr = 0; pr < GI_UNROLL / 2; ++pr) {
            const int64_t kk = k + 128 * pr + 16 * kc;
            const bool ok = kk < ke;
            const uint32_t ko = (uint32_t)kk;
            wr[2 * pr] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(wrs, ok ? wo0 + ko : I8_OOB, 0, 0));
            wr[2 * pr + 1] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(wrs, ok ? wo1 + ko : I8_OOB, 0, 0));
            xr[2 * pr] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(xrs, ok ? xo0 + ko : I8_OOB, 0, 0));
            if constexpr (XHI)
                xr[2 * pr + 1] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(xrs, ok ? xo1 + ko : I8_OOB, 0, 0));
        }
        __builtin_amdgcn_sched_barrier(0);  // every load before the first use
#pragma unroll
        for (int pr = 0; pr < GI_UNROLL / 2; ++pr) {
            u32x4(&s)[4][64] = stage[wave][pr & 1];
            s[0][wslot] = wr[2 * pr];
            s[1][wslot] = wr[2 * pr + 1];
            s[2][wslot] = xr[2 * pr];
            if constexpr (XHI) s[3][wslot] = xr[2 * pr + 1];
            __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
            const u32x4 wlo = s[rq][lo_slot], whi = s[rq][hi_slot];
            const u32x4 xlo = s[2 + xq][lo_slot], xhi = s[2 + xq][hi_slot];
            acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i32x4, xlo), __builtin_bit_cast(i32x4, wlo), acc, 0, 0, 0);
            acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i32x4, xhi), __builtin_bit_cast(i32x4, whi), acc, 0, 0, 0);
        }
    }
    stage[wave][0][0][lane] = __builtin_bit_cast(u32x4, acc);
    __syncthreads();
    if (wave != 0) return;
    i32x4 sum = __builtin_bit_cast(i32x4, stage[0][0][0][lane]);
#pragma unroll
    for (int w = 1; w < 4; ++w) sum += __builtin_bit_cast(i32x4, stage[w][0][0][lane]);
    const int64_t col = n0 + r;  // rows 4 g + i
    if (col >= p.N) return;
    const float sb = p.sB[col], bias = p.bias ? p.bias[col] : 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int64_t row = 4 * g + i;
        if (row < p.M) store_out(p.C, row * p.ldc + col, (float)sum[i] * p.sA[row] * sb + bias, p.out_bf16);
    }
}

// The same on activations that are not quantised yet, for few and short rows (M K <= GX_MAX): every block
// quantises them all into LDS while its first weight loads are in flight, instead of in a launch before: 7.3 ->
// 5.4 us for one row of 256 values (N 768). Every block does the same work, so it does not pay for more: 4 rows
// of 4096 values took 17.0 us this way (N 11008) and 12.2 in two launches.
constexpr int GX_MAX = 4096;

template <typename T>
__global__ __launch_bounds__(NTHREADS) void gemv_i8_x(const GemmI8Args p) {
    constexpr int KCHUNK = 64;
    __shared__ u32x4 stage[4][2][2][64];
    __shared__ __attribute__((aligned(16))) char xq[GX_MAX + 4 * 16 + 16 * 128];
    __shared__ uint32_t most[4];
    __shared__ float xs[16];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int r = lane & 15, g = lane >> 4;
    const int rl = lane >> 3, kc = lane & 7;
    const int64_t n0 = (int64_t)blockIdx.x * 16;
    const int64_t nrows = min((int64_t)16, p.N - n0);
    const __amdgpu_buffer_rsrc_t wrs = i8_rsrc(p.B + n0 * p.ldb, (nrows - 1) * p.ldb + p.K);
    const uint32_t wo0 = (uint32_t)(rl * p.ldb), wo1 = (uint32_t)((8 + rl) * p.ldb);
    const int wslot = gi_slot(rl, kc), rq = r >> 3, rr = r & 7;
    const int lo_slot = gi_slot(rr, g), hi_slot = gi_slot(rr, 4 + g);
    const int K = (int)p.K, M = (int)p.M, pitch = K + 16;
    const int span = (K + 4 * KCHUNK - 1) / (4 * KCHUNK) * KCHUNK;
    const int kb = wave * span, ke = min(K, kb + span);
    u32x4 wr[GI_UNROLL];
    auto load_w = [&](int k) {
#pragma unroll
        for (int pr = 0; pr < GI_UNROLL / 2; ++pr) {
            const int kk = k + 128 * pr + 16 * kc;
            const bool ok = kk < ke;
            wr[2 * pr] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(wrs, ok ? wo0 + kk : I8_OOB, 0, 0));
            wr[2 * pr + 1] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(wrs, ok ? wo1 + kk : I8_OOB, 0, 0));
        }
        __builtin_amdgcn_sched_barrier(0);
    };
    load_w(kb);
    // Row m by 256 / rows lanes: rows at once 1, 2 or 4.
    const int at_once = M >= 4 ? 4 : M >= 2 ? 2 : 1, lanes = NTHREADS / at_once, x0 = tid % lanes;
    for (int m0 = 0; m0 < M; m0 += at_once) {
        const int m = m0 + tid / lanes;
        const bool live = m < M;
        const T *x = (const T *)p.X + (int64_t)(live ? m : 0) * p.ldx;
        uint32_t mb = 0;
        if (live)
            for (int c = x0 * 8; c < p.xcols; c += lanes * 8) {
                float v[8];
                row8(x, c, p.xcols, v);
#pragma unroll
                for (int e = 0; e < 8; ++e) mb = max(mb, abs_bits(v[e]));
            }
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) mb = max(mb, (uint32_t)__shfl_xor((int)mb, o, 64));
        if (m0 > 0) __syncthreads();  // the last rows' maxima have been read
        if (lane == 0) most[wave] = mb;
        __syncthreads();
        if (at_once == 1) mb = max(max(most[0], most[1]), max(most[2], most[3]));
        if (at_once == 2) mb = max(most[wave & 2], most[wave | 1]);
        const float s = quant_step<false>(mb, 127.f), inv = quant_inverse(s);
        if (live) {
            for (int c = x0 * 8; c < K; c += lanes * 8) {
                float v[8];
                row8(x, c, p.xcols, v);
                *(u32x2 *)(xq + m * pitch + c) = codes8(v, s, inv);
            }
            if (x0 == 0) xs[m] = s;
        }
    }
    __syncthreads();
    const char *xrow = xq + (r < M ? r : 0) * pitch + 16 * g;  // rows past M repeat row 0; they are not stored
    i32x4 acc = {0, 0, 0, 0};
    for (int k = kb; k < ke; k += GI_UNROLL * KCHUNK) {
        if (k > kb) load_w(k);
#pragma unroll
        for (int pr = 0; pr < GI_UNROLL / 2; ++pr) {
            u32x4(&s)[2][64] = stage[wave][pr & 1];
            s[0][wslot] = wr[2 * pr];
            s[1][wslot] = wr[2 * pr + 1];
            __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
            const u32x4 wlo = s[rq][lo_slot], whi = s[rq][hi_slot];
            // Codes of X past this wave's k meet zeros of W; the buffer has room for them.
            const i32x4 xlo = *(const i32x4 *)(xrow + k + 128 * pr), xhi = *(const i32x4 *)(xrow + k + 128 * pr + 64);
            acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(xlo, __builtin_bit_cast(i32x4, wlo), acc, 0, 0, 0);
            acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(xhi, __builtin_bit_cast(i32x4, whi), acc, 0, 0, 0);
        }
    }
    stage[wave][0][0][lane] = __builtin_bit_cast(u32x4, acc);
    __syncthreads();
    if (wave != 0) return;
    i32x4 sum = __builtin_bit_cast(i32x4, stage[0][0][0][lane]);
#pragma unroll
    for (int w = 1; w < 4; ++w) sum += __builtin_bit_cast(i32x4, stage[w][0][0][lane]);
    const int64_t col = n0 + r;
    if (col >= p.N) return;
    const float sb = p.sB[col], bias = p.bias ? p.bias[col] : 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int64_t row = 4 * g + i;
        if (row < M) store_out(p.C, row * p.ldc + col, (float)sum[i] * xs[row] * sb + bias, p.out_bf16);
    }
}

template <int FA, int FB, int NS>
it_status launch_tile(hipStream_t s, GemmI8Args a) {
    a.tiles_m = (int)((a.M + 64 * FA - 1) / (64 * FA));
    a.tiles_n = (int)((a.N + 64 * FB - 1) / (64 * FB));
    if (const it_status st = check_blocks("gemm_i8", (int64_t)a.tiles_m * a.tiles_n); st != IT_OK) return st;
    const dim3 grid((unsigned)(a.tiles_m * a.tiles_n)), block(NTHREADS);
    if (a.K % 128 == 0)
        hipLaunchKernelGGL((gemm_i8_tile<FA, FB, NS, true>), grid, block, 0, s, a);
    else
        hipLaunchKernelGGL((gemm_i8_tile<FA, FB, NS, false>), grid, block, 0, s, a);
    IT_HIP_TRY(hipGetLastError());
    return IT_OK;
}

template <typename T, int RL, int VN>
it_status launch_rows(hipStream_t s, int64_t rows, int64_t cols, const void *X, int64_t ldx, int8_t *codes, int64_t ldc,
                      float *steps) {
    const int64_t blocks = (rows + 256 / RL - 1) / (256 / RL);
    if (const it_status st = check_blocks("quantize_i8", blocks); st != IT_OK) return st;
    hipLaunchKernelGGL((quantize_rows<T, RL, VN>), dim3((unsigned)blocks), dim3(256), 0, s, (const T *)X, ldx, rows, cols,
                       std::min((cols + 127) / 128 * 128, ldc), codes, ldc, steps);
    IT_HIP_TRY(hipGetLastError());
    return IT_OK;
}

template <typename T>
it_status launch_rows_of(hipStream_t s, int64_t rows, int64_t cols, const void *X, int64_t ldx, int8_t *codes, int64_t ldc,
                         float *steps) {
    // A wave a row where there are rows enough to fill the GPU: no block barrier (1999 x 1237 FP32: 6.1 us with a
    // block a row, 5.6 so). Fewer rows have a block each, for the time of one row.
    if (rows >= 1024) {
        if (cols <= 512) return launch_rows<T, 64, 1>(s, rows, cols, X, ldx, codes, ldc, steps);
        if (cols <= 2048) return launch_rows<T, 64, 4>(s, rows, cols, X, ldx, codes, ldc, steps);
        if (cols <= 4096) return launch_rows<T, 64, 8>(s, rows, cols, X, ldx, codes, ldc, steps);
        return launch_rows<T, 256, 4>(s, rows, cols, X, ldx, codes, ldc, steps);
    } else {
        if (cols <= 512) return launch_rows<T, 64, 1>(s, rows, cols, X, ldx, codes, ldc, steps);
        if (cols <= 2048) return launch_rows<T, 256, 1>(s, rows, cols, X, ldx, codes, ldc, steps);
        if (cols <= 4096) return launch_rows<T, 256, 2>(s, rows, cols, X, ldx, codes, ldc, steps);
        return launch_rows<T, 256, 4>(s, rows, cols, X, ldx, codes, ldc, steps);
    }
}

}  // namespace

it_status launch_quantize_i8(hipStream_t s, bool bf16, int64_t rows, int64_t cols, const void *X, int64_t ldx,
                             int8_t *codes, int64_t ldc, float *steps) {
    return bf16 ? launch_rows_of<uint16_t>(s, rows, cols, X, ldx, codes, ldc, steps)
                : launch_rows_of<float>(s, rows, cols, X, ldx, codes, ldc, steps);
}

it_status launch_gemm_i8(it_context *ctx, GemmI8Args a) {
    hipStream_t s = ctx->stream;
    if (a.M <= 16) {
        if (const it_status st = check_blocks("gemm_i8", (a.N + 15) / 16); st != IT_OK) return st;
        const dim3 grid((unsigned)((a.N + 15) / 16)), block(NTHREADS);
        if (a.M > 8)
            hipLaunchKernelGGL((gemv_i8<true>), grid, block, 0, s, a);
        else
            hipLaunchKernelGGL((gemv_i8<false>), grid, block, 0, s, a);
        IT_HIP_TRY(hipGetLastError());
        return IT_OK;
    }
    // Prices in us: a k-tile of every tile on a CU (one more for each of its tiles beyond the first), and
    // the launch with the tile's first loads and its epilogue. From 12 shapes of 20 .. 8192 rows.
    struct Config {
        int bm, bn;
        double kt, fixed;
    };
    static const Config configs[] = {{64, 64, 0.22, 3.5}, {128, 64, 0.40, 3.3}, {128, 64, 0.375, 3.5}, {256, 128, 1.0, 6.0}, {256, 256, 1.65, 13.0}};
    const double kt = (double)((a.K + 127) / 128);
    int best = 0;
    double best_t = 1e30;
    for (int i = 0; i < 5; ++i) {
        const Config &c = configs[i];
        const int64_t tiles = ((a.M + c.bm - 1) / c.bm) * ((a.N + c.bn - 1) / c.bn);
        // The two-stage 128 x 64 tile needs a second block on the CU to cover its loads.
        if (i == 2 && tiles < 2 * ctx->num_cus) continue;
        const double t = (double)((tiles + ctx->num_cus - 1) / ctx->num_cus) * kt * c.kt + c.fixed;
        if (t < best_t) best_t = t, best = i;
    }
    switch (best) {
    case 0: return launch_tile<1, 1, 4>(s, a);
    case 1: return launch_tile<2, 1, 3>(s, a);
    case 2: return launch_tile<2, 1, 2>(s, a);
    case 3: return launch_tile<4, 2, 3>(s, a);
    default: return launch_tile<4, 4, 2>(s, a);
    }
}

bool gemv_i8_x_applicable(int64_t M, int64_t K) { return M <= 16 && M * K <= GX_MAX; }

it_status launch_gemv_i8_x(hipStream_t s, bool bf16, const GemmI8Args &a) {
    if (const it_status st = check_blocks("linear_i8", (a.N + 15) / 16); st != IT_OK) return st;
    const dim3 grid((unsigned)((a.N + 15) / 16)), block(NTHREADS);
    if (bf16)
        hipLaunchKernelGGL((gemv_i8_x<uint16_t>), grid, block, 0, s, a);
    else
        hipLaunchKernelGGL((gemv_i8_x<float>), grid, block, 0, s, a);
    IT_HIP_TRY(hipGetLastError());
    return IT_OK;
}

}  // namespace it
