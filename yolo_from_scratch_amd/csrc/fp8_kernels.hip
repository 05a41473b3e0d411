// Matrix product in 8-bit floating point (e4m3) with a scale for each block of 128, and the quantisers that feed it.
//
// A block's scale is the smallest power of two s = 2^e, e >= -127, with max|x| <= 448 s over its finite elements (1 for a block
// of zeros); q = x / s rounded to e4m3 (exact division, to nearest, ties to even; Inf and NaN become NaN).  It is kept as the byte
// e + 127 (E8M0).  Powers of two are what the scaled matrix instruction takes as operands, so a product of two blocks needs
// no multiplication by its scales in the loop, and the transpose of a 128 x 128 block is the same bytes.
//
// Row scales (a scale per row and 128 columns: activations, gradients) are kept "packed": for each 128-column block kb a plane
// of bytes in which the four rows r, r + 16, r + 32, r + 48 of a group of 64 lie next to each other, i.e. row at
//     (kb * G + row / 64) * 64 + (row % 16) * 4 + (row % 64) / 16,       G = 4 * ceil(rows / 256):
// one dword per lane and 64 rows holds the scales of the four 16-row fragments that a wave multiplies, and the instruction
// selects the byte.
#include "yfs_common.h"
#include "yfs_vec.h"
#include <math.h>
#include <type_traits>

namespace {
typedef __bf16 bf16_t;
typedef __attribute__((ext_vector_type(8))) __bf16 bf16x8;
typedef __attribute__((ext_vector_type(2))) __bf16 bf16x2;
typedef __attribute__((ext_vector_type(4))) __bf16 bf16x4;
typedef __attribute__((ext_vector_type(4))) float f32x4;
typedef __attribute__((ext_vector_type(4))) int i32x4;
typedef __attribute__((ext_vector_type(8))) int i32x8;
typedef __attribute__((address_space(3))) void* lds_ptr;

__host__ __device__ inline long long pad128(long long n) { return (n + 127) & ~127LL; }
__host__ __device__ inline int groups64(long long rows) { return (int)((rows + 255) / 256 * 4); }
__host__ __device__ inline long long packed_bytes(long long rows, long long kblocks) { return kblocks * groups64(rows) * 64; }
__device__ __forceinline__ long long packed_at(long long row, long long kb, int groups) {
    return (kb * groups + (row >> 6)) * 64 + (row & 15) * 4 + ((row & 63) >> 4);
}

// e of the smallest power of two with amax <= 448 * 2^e = 0.875 * 2^(e + 9); amax finite and >= 0
__device__ __forceinline__ int scale_exponent(float amax) {
    const unsigned u = __float_as_uint(amax);
    const int e = (int)(u >> 23) - 126 - 9 + ((u & 0x7FFFFFu) > 0x600000u ? 1 : 0);   // a subnormal amax ends below -127
    return u == 0 ? 0 : (e < -127 ? -127 : e);
}
__device__ __forceinline__ float pow2(int e) { return __uint_as_float((unsigned)(e + 127) << 23); }   // -126 <= e <= 127
__device__ __forceinline__ float finite_abs(float v) {
    const float a = fabsf(v);
    return a < __builtin_inff() ? a : 0.0f;
}
__device__ __forceinline__ unsigned pack4(float a, float b, float c, float d) {
    int p = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    return (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, p, true);
}

// ---- quantisers ------------------------------------------------------------------------------------------------------
struct QuantArgs {
    const void* x;
    long long ld, M, K;        // x [M, K], ld elements from row to row
    unsigned char *q, *s;      // [M, pad128(K)] and its scales (packed row scales, or [ceil(M/128), ceil(K/128)])
    unsigned char *qt, *st;    // the transpose [K, pad128(M)] and its scales
    float* colsum;             // [ceil(M/128), K] sums of x over the rows of a tile, or NULL
    int groups, groups_t;      // 64-row groups of the packed planes of q and qt
};

// One workgroup per 128 x 128 tile, 8 x 8 elements per thread.  BLOCK: one scale for the tile.  Otherwise ROWQ: a scale per
// row; COLQ: a scale per column, written transposed.
template <typename T, bool BLOCK, bool ROWQ, bool COLQ>
__global__ void __launch_bounds__(256) quant_tile_kernel(QuantArgs g) {
    __shared__ float red[4][128];
    __shared__ __attribute__((aligned(16))) unsigned char tile[COLQ ? 128 * 144 : 16];
    const int cg = threadIdx.x & 15, rg = threadIdx.x >> 4, wave = threadIdx.x >> 6;
    const long long kb = blockIdx.x, mb = blockIdx.y;
    const long long k0 = kb * 128 + cg * 8, m0 = mb * 128 + rg * 8;
    float v[8][8];
#pragma unroll
    for (int i = 0; i < 8; ++i) load_vec8((const T*)g.x + (m0 + i) * g.ld + k0, m0 + i < g.M ? g.K - k0 : 0, v[i]);
    if (g.colsum) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            float s = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; ++i) s += v[i][j];
            s += __shfl_xor(s, 16, 64);
            s += __shfl_xor(s, 32, 64);
            if ((threadIdx.x & 48) == 0) red[wave][cg * 8 + j] = s;
        }
        __syncthreads();
        if (threadIdx.x < 128 && kb * 128 + threadIdx.x < g.K)
            g.colsum[mb * g.K + kb * 128 + threadIdx.x] =
                (red[0][threadIdx.x] + red[1][threadIdx.x]) + (red[2][threadIdx.x] + red[3][threadIdx.x]);
        __syncthreads();
    }
    const long long ldq = pad128(g.K), ldt = pad128(g.M);
    int eb = 0;
    if (BLOCK) {
        float a = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
            for (int j = 0; j < 8; ++j) a = fmaxf(a, finite_abs(v[i][j]));
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) a = fmaxf(a, __shfl_xor(a, o, 64));
        if ((threadIdx.x & 63) == 0) red[0][wave] = a;
        __syncthreads();
        eb = scale_exponent(fmaxf(fmaxf(red[0][0], red[0][1]), fmaxf(red[0][2], red[0][3])));
        if (threadIdx.x == 0) {
            if (ROWQ) g.s[mb * (ldq >> 7) + kb] = (unsigned char)(eb + 127);
            if (COLQ) g.st[kb * (ldt >> 7) + mb] = (unsigned char)(eb + 127);
        }
    }
    if (ROWQ) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            int e = eb;
            if (!BLOCK) {
                float a = 0.0f;
#pragma unroll
                for (int j = 0; j < 8; ++j) a = fmaxf(a, finite_abs(v[i][j]));
#pragma unroll
                for (int o = 8; o > 0; o >>= 1) a = fmaxf(a, __shfl_xor(a, o, 64));
                e = scale_exponent(a);
                if (cg == 0 && m0 + i < g.M) g.s[packed_at(m0 + i, kb, g.groups)] = (unsigned char)(e + 127);
            }
            const float f = pow2(-e);
            const uint2 p = make_uint2(pack4(v[i][0] * f, v[i][1] * f, v[i][2] * f, v[i][3] * f),
                                       pack4(v[i][4] * f, v[i][5] * f, v[i][6] * f, v[i][7] * f));
            if (m0 + i < g.M) *reinterpret_cast<uint2*>(g.q + (m0 + i) * ldq + k0) = p;
        }
    }
    if (COLQ) {
        if (!BLOCK) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                float a = 0.0f;
#pragma unroll
                for (int i = 0; i < 8; ++i) a = fmaxf(a, finite_abs(v[i][j]));
                a = fmaxf(a, __shfl_xor(a, 16, 64));
                a = fmaxf(a, __shfl_xor(a, 32, 64));
                if ((threadIdx.x & 48) == 0) red[wave][cg * 8 + j] = a;
            }
            __syncthreads();
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            int e = eb;
            if (!BLOCK) {
                const int c = cg * 8 + j;
                e = scale_exponent(fmaxf(fmaxf(red[0][c], red[1][c]), fmaxf(red[2][c], red[3][c])));
                if (rg == 0 && k0 + j < g.K) g.st[packed_at(k0 + j, mb, g.groups_t)] = (unsigned char)(e + 127);
            }
            const float f = pow2(-e);
            *reinterpret_cast<uint2*>(tile + (cg * 8 + j) * 144 + rg * 8) =
                make_uint2(pack4(v[0][j] * f, v[1][j] * f, v[2][j] * f, v[3][j] * f),
                           pack4(v[4][j] * f, v[5][j] * f, v[6][j] * f, v[7][j] * f));
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int c = i * 32 + (threadIdx.x >> 3), ch = threadIdx.x & 7;
            const long long k = kb * 128 + c;
            if (k < g.K)
                *reinterpret_cast<i32x4*>(g.qt + k * ldt + mb * 128 + ch * 16) = *reinterpret_cast<const i32x4*>(tile + c * 144 + ch * 16);
        }
    }
}

// sums over the tiles of quant_tile_kernel's colsum, in tile order
__global__ void __launch_bounds__(256) colsum_kernel(const float* __restrict__ part, long long tiles, long long K,
                                                     float* __restrict__ out, int accumulate) {
    const long long k = (long long)blockIdx.x * 256 + threadIdx.x;
    if (k >= K) return;
    float s = 0.0f;
    for (long long t = 0; t < tiles; ++t) s += part[t * K + k];
    out[k] = accumulate ? out[k] + s : s;
}

template <bool BLOCK, bool ROWQ, bool COLQ>
int quantize(const QuantArgs& g, int dtype, hipStream_t s) {
    const dim3 grid((unsigned)yfs_cdiv(g.K, 128), (unsigned)yfs_cdiv(g.M, 128));
    if (dtype == YFS_F32) quant_tile_kernel<float, BLOCK, ROWQ, COLQ><<<grid, 256, 0, s>>>(g);
    else if (dtype == YFS_BF16) quant_tile_kernel<bf16_t, BLOCK, ROWQ, COLQ><<<grid, 256, 0, s>>>(g);
    else quant_tile_kernel<_Float16, BLOCK, ROWQ, COLQ><<<grid, 256, 0, s>>>(g);
    YFS_CHECK_LAUNCH("quant_tile_kernel");
    return YFS_OK;
}

// ---- product ---------------------------------------------------------------------------------------------------------
struct GemmArgs {
    const unsigned char *a, *as;   // a [M, pad128(K)], packed row scales
    const unsigned char *b, *bs;   // b [N, pad128(K)], packed row scales or [ceil(N/128), K/128]
    const float* bias;             // [N] or NULL
    void* out;                     // [M, N]
    float* part;                   // [splits][M][N] when splits > 1
    long long M, N;
    int kblocks, splits, per_split;
    int groups_a, groups_b;
    float slope;                   // 1: no activation
    int accumulate;                // fp32 output only: add to what is there
};

__device__ __forceinline__ __amdgpu_buffer_rsrc_t rsrc(const void* p, long long bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), 0, (int)(unsigned)(bytes < 0xFFFFFFFFLL ? bytes : 0xFFFFFFFFLL), 0x00020000);
}

// 32 e4m3 values of a fragment -> bf16, times 2^(byte - 127) (exact: four significant bits and a shift of the exponent)
__device__ __forceinline__ void widen(const i32x8& f, float scale, bf16x8 (&w)[4]) {
#pragma unroll
    for (int q = 0; q < 4; ++q)
#pragma unroll
        for (int d = 0; d < 2; ++d) {
            const bf16x2 lo = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(f[q * 2 + d], scale, false);
            const bf16x2 hi = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(f[q * 2 + d], scale, true);
            w[q][d * 4 + 0] = lo[0];
            w[q][d * 4 + 1] = lo[1];
            w[q][d * 4 + 2] = hi[0];
            w[q][d * 4 + 3] = hi[1];
        }
}

template <int SA, int SB>
__device__ __forceinline__ f32x4 mfma_fp8(const i32x8& a, const i32x8& b, f32x4 c, int sa, int sb) {
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, c, 0, 0, SA, sa, SB, sb);
}

__device__ __forceinline__ float leaky(float v, float slope) { return v > 0.0f ? v : v * slope; }

// Four neighbouring outputs of row m: columns n .. n + 3, of which those below N exist
template <typename TO>
__device__ __forceinline__ void store4(const GemmArgs& g, long long m, long long n, f32x4 v) {
    if (g.bias) {
#pragma unroll
        for (int r = 0; r < 4; ++r) v[r] += n + r < g.N ? g.bias[n + r] : 0.0f;
    }
    TO t[4];
    TO* o = (TO*)g.out + m * g.N + n;
    if (sizeof(TO) == 4 && g.accumulate) {
#pragma unroll
        for (int r = 0; r < 4; ++r) v[r] += n + r < g.N ? (float)o[r] : 0.0f;
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) t[r] = (TO)leaky(v[r], g.slope);
    if (n + 4 <= g.N) __builtin_memcpy(o, t, sizeof(t));
    else {
#pragma unroll
        for (int r = 0; r < 4; ++r)
            if (n + r < g.N) o[r] = t[r];
    }
}

// out tile of (WM FM 16) x (WN FN 16), a wave FM x FN fragments of 16 x 16.  LDS holds two stages of the 128-byte rows of both
// operands, 16-byte chunks swizzled by the row, filled by direct loads.  The operands' lanes hold 32 of a block's 128 k in an
// order that is the same on both sides, which is all that the sum needs.  The b rows are the instruction's first operand, so
// that a lane owns four neighbouring columns of one output row.
// EXACT: the e4m3 instructions sum a block's products with about 16 bits behind the largest (measured: 1.5e-5 relative
// whatever K, 2^-16); where the output is fp32 the operands are widened in registers and multiplied by the bf16 instruction,
// whose sums are full fp32.
template <int FM, int FN, int WM, int WN, bool ROWB, bool EXACT, typename TO>
__global__ void __launch_bounds__(64 * WM * WN) fp8_gemm_kernel(GemmArgs g) {
    constexpr int BM = WM * FM * 16, BN = WN * FN * 16, NW = WM * WN;
    constexpr int STAGE = (BM + BN) * 128;
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const int wm = wave / WN, wn = wave % WN;
    const long long m0 = (long long)blockIdx.y * BM, n0 = (long long)blockIdx.x * BN;
    const long long ld = (long long)g.kblocks * 128;
    const int kb0 = (int)blockIdx.z * g.per_split;
    const int kb1 = kb0 + g.per_split < g.kblocks ? kb0 + g.per_split : g.kblocks;
    const long long ra = g.M - m0 < BM ? g.M - m0 : BM, rb = g.N - n0 < BN ? g.N - n0 : BN;
    const __amdgpu_buffer_rsrc_t rsa = rsrc(g.a + m0 * ld, ra * ld), rsb = rsrc(g.b + n0 * ld, rb * ld);
    const int srow = lane >> 3;
    const unsigned chunk = (unsigned)((lane & 7) ^ srow) * 16u;
    auto stage = [&](int kb, int buf) {   // rows outside the operands read as zeros
        unsigned char* base = smem + buf * STAGE;
        for (int r = wave; r < BM / 8; r += NW)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rsa, (lds_ptr)(base + r * 1024), 16, (unsigned)((r * 8 + srow) * ld) + chunk,
                                                     (unsigned)kb * 128u, 0, 0);
        for (int r = wave; r < BN / 8; r += NW)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rsb, (lds_ptr)(base + BM * 128 + r * 1024), 16,
                                                     (unsigned)((r * 8 + srow) * ld) + chunk, (unsigned)kb * 128u, 0, 0);
    };
    const int frow = lane & 15, fk = lane >> 4;
    auto fragment = [&](const unsigned char* base, int row) {
        const i32x4 lo = *reinterpret_cast<const i32x4*>(base + row * 128 + ((fk ^ (row & 7)) * 16));
        const i32x4 hi = *reinterpret_cast<const i32x4*>(base + row * 128 + (((4 + fk) ^ (row & 7)) * 16));
        return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    };
    f32x4 acc[FN][FM];
#pragma unroll
    for (int i = 0; i < FN; ++i)
#pragma unroll
        for (int j = 0; j < FM; ++j) acc[i][j] = (f32x4){0.f, 0.f, 0.f, 0.f};

    stage(kb0, 0);
    for (int kb = kb0; kb < kb1; ++kb) {
        const int buf = (kb - kb0) & 1;
        const int sa = *reinterpret_cast<const int*>(g.as + ((long long)kb * g.groups_a + ((m0 + wm * FM * 16) >> 6)) * 64 + frow * 4);
        int sb;
        if (ROWB) {
            sb = *reinterpret_cast<const int*>(g.bs + ((long long)kb * g.groups_b + ((n0 + wn * FN * 16) >> 6)) * 64 + frow * 4);
            if (FN == 2) sb = (wn & 1) ? (int)((unsigned)sb >> 16) : sb;
        } else {
            const long long nb = (n0 + wn * FN * 16) >> 7, last = (g.N - 1) >> 7;
            sb = g.bs[(nb < last ? nb : last) * g.kblocks + kb];
        }
        yfs_stage_wait();
        __syncthreads();
        if (kb + 1 < kb1) stage(kb + 1, buf ^ 1);
        const unsigned char* ab = smem + buf * STAGE;
        const unsigned char* bb = ab + BM * 128;
        i32x8 fa[FM], fb[FN];
#pragma unroll
        for (int j = 0; j < FM; ++j) fa[j] = fragment(ab, wm * FM * 16 + j * 16 + frow);
#pragma unroll
        for (int i = 0; i < FN; ++i) fb[i] = fragment(bb, wn * FN * 16 + i * 16 + frow);
        if constexpr (EXACT) {
            bf16x8 wa[FM][4];
#pragma unroll
            for (int j = 0; j < FM; ++j) widen(fa[j], __uint_as_float((((unsigned)sa >> (8 * j)) & 255u) << 23), wa[j]);
#pragma unroll
            for (int i = 0; i < FN; ++i) {
                bf16x8 wb[4];
                widen(fb[i], __uint_as_float((((unsigned)sb >> (ROWB ? 8 * i : 0)) & 255u) << 23), wb);
#pragma unroll
                for (int j = 0; j < FM; ++j)
#pragma unroll
                    for (int q = 0; q < 4; ++q) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wb[q], wa[j][q], acc[i][j], 0, 0, 0);
            }
        } else {
            auto row = [&](auto it) {
                constexpr int I = decltype(it)::value, SB = ROWB ? I : 0;
                if constexpr (I < FN) {
                    acc[I][0] = mfma_fp8<SB, 0>(fb[I], fa[0], acc[I][0], sb, sa);
                    if constexpr (FM > 1) acc[I][1] = mfma_fp8<SB, 1>(fb[I], fa[1], acc[I][1], sb, sa);
                    if constexpr (FM > 2) acc[I][2] = mfma_fp8<SB, 2>(fb[I], fa[2], acc[I][2], sb, sa);
                    if constexpr (FM > 3) acc[I][3] = mfma_fp8<SB, 3>(fb[I], fa[3], acc[I][3], sb, sa);
                }
            };
            row(std::integral_constant<int, 0>());
            row(std::integral_constant<int, 1>());
            row(std::integral_constant<int, 2>());
            row(std::integral_constant<int, 3>());
        }
        __syncthreads();
    }
#pragma unroll
    for (int j = 0; j < FM; ++j) {
        const long long m = m0 + wm * FM * 16 + j * 16 + frow;
        if (m >= g.M) continue;
#pragma unroll
        for (int i = 0; i < FN; ++i) {
            const long long n = n0 + wn * FN * 16 + i * 16 + fk * 4;
            if (n >= g.N) continue;
            if (g.splits > 1) {
                float* o = g.part + ((long long)blockIdx.z * g.M + m) * g.N + n;
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    if (n + r < g.N) o[r] = acc[i][j][r];
            } else store4<TO>(g, m, n, acc[i][j]);
        }
    }
}

// joins the partial sums of the splits in their order
template <typename TO>
__global__ void __launch_bounds__(256) fp8_join_kernel(GemmArgs g) {
    const long long per_row = (g.N + 3) / 4, total = g.M * per_row;
    for (long long id = (long long)blockIdx.x * 256 + threadIdx.x; id < total; id += (long long)gridDim.x * 256) {
        const long long m = id / per_row, n = (id - m * per_row) * 4;
        f32x4 v = {0.f, 0.f, 0.f, 0.f};
        for (int s = 0; s < g.splits; ++s) {
            const float* p = g.part + ((long long)s * g.M + m) * g.N + n;
#pragma unroll
            for (int r = 0; r < 4; ++r) v[r] += n + r < g.N ? p[r] : 0.0f;
        }
        store4<TO>(g, m, n, v);
    }
}

struct Plan { int bm, bn, splits, per_split; };
Plan plan(long long M, long long N, int kblocks) {
    Plan p;
    p.bm = M <= 64 ? 64 : 128;
    p.bn = 128;
    const long long tiles = yfs_cdiv(M, p.bm) * yfs_cdiv(N, p.bn);
    long long s = tiles >= 256 ? 1 : 512 / tiles;
    if (s > kblocks / 2) s = kblocks / 2;
    if (s < 1) s = 1;
    p.per_split = (int)yfs_cdiv(kblocks, s);
    p.splits = (int)yfs_cdiv(kblocks, p.per_split);
    return p;
}

template <int FM, int FN, int WM, int WN, bool ROWB, bool EXACT, typename TO>
int launch_tiles(const GemmArgs& g, hipStream_t s) {
    constexpr int BM = WM * FM * 16, BN = WN * FN * 16;
    const dim3 grid((unsigned)yfs_cdiv(g.N, BN), (unsigned)yfs_cdiv(g.M, BM), (unsigned)g.splits);
    fp8_gemm_kernel<FM, FN, WM, WN, ROWB, EXACT, TO><<<grid, 64 * WM * WN, 2 * (BM + BN) * 128, s>>>(g);
    YFS_CHECK_LAUNCH("fp8_gemm_kernel");
    if (g.splits > 1) {
        long long nb = yfs_cdiv(g.M * ((g.N + 3) / 4), 256);
        fp8_join_kernel<TO><<<dim3((unsigned)(nb < 4096 ? nb : 4096)), 256, 0, s>>>(g);
        YFS_CHECK_LAUNCH("fp8_join_kernel");
    }
    return YFS_OK;
}

template <bool ROWB, bool EXACT, typename TO>
int gemm(GemmArgs g, hipStream_t s) {
    const Plan p = plan(g.M, g.N, g.kblocks);
    g.splits = p.splits;
    g.per_split = p.per_split;
    g.groups_a = groups64(g.M);
    g.groups_b = groups64(g.N);
    if (p.bm == 64) return launch_tiles<4, 2, 1, 4, ROWB, EXACT, TO>(g, s);
    return launch_tiles<4, 4, 2, 2, ROWB, EXACT, TO>(g, s);
}
size_t part_bytes(long long M, long long N, int kblocks) {
    const Plan p = plan(M, N, kblocks);
    return p.splits > 1 ? (size_t)p.splits * M * N * sizeof(float) : 0;
}

bool known(int d) { return d == YFS_F32 || d == YFS_BF16 || d == YFS_F16; }
constexpr int64_t kMost = (1LL << 23) - 256;   // 65534 tiles of 128 rows; a tile's rows of pad128(K) bytes stay inside one buffer descriptor
size_t align256(size_t n) { return (n + 255) & ~(size_t)255; }
}  // namespace

#define REQUIRE_SIZES(name, M, N, K)                                                                                       \
    YFS_REQUIRE((M) > 0 && (N) > 0 && (K) > 0 && (M) <= kMost && (N) <= kMost && (K) <= kMost, YFS_ERR_INVALID_ARG,       \
                name ": sizes must lie in [1, %lld] (got %lld, %lld, %lld)", (long long)kMost, (long long)(M), (long long)(N), \
                (long long)(K))
#define REQUIRE_ALIGNED(name, p) \
    YFS_REQUIRE((reinterpret_cast<uintptr_t>(p) & 15) == 0, YFS_ERR_INVALID_ARG, name ": " #p " must be 16-byte aligned")

YFS_API int yfs_fp8_quantize_weight(const void* w, int dtype, int64_t ld, int64_t N, int64_t K, void* q, void* scale, void* qt,
                                    void* scale_t, void* stream) {
    YFS_REQUIRE(w && q && scale && !qt == !scale_t, YFS_ERR_INVALID_ARG, "yfs_fp8_quantize_weight: null pointer");
    REQUIRE_SIZES("yfs_fp8_quantize_weight", 1, N, K);
    YFS_REQUIRE(ld >= 0, YFS_ERR_INVALID_ARG, "yfs_fp8_quantize_weight: negative row stride");
    YFS_REQUIRE(known(dtype), YFS_ERR_UNSUPPORTED, "yfs_fp8_quantize_weight: unknown dtype %d", dtype);
    REQUIRE_ALIGNED("yfs_fp8_quantize_weight", q);
    REQUIRE_ALIGNED("yfs_fp8_quantize_weight", qt);
    const QuantArgs g = {w, ld, N, K, (unsigned char*)q, (unsigned char*)scale, (unsigned char*)qt, (unsigned char*)scale_t, nullptr, 0, 0};
    return qt ? quantize<true, true, true>(g, dtype, (hipStream_t)stream) : quantize<true, true, false>(g, dtype, (hipStream_t)stream);
}

YFS_API size_t yfs_fp8_packed_scale_bytes(int64_t rows, int64_t cols) {
    return rows > 0 && cols > 0 ? (size_t)packed_bytes(rows, yfs_cdiv(cols, 128)) : 0;
}

YFS_API int yfs_fp8_quantize_rows(const void* x, int dtype, int64_t ld, int64_t M, int64_t K, void* q, void* scale, void* qt,
                                  void* scale_t, float* colsum, void* stream) {
    YFS_REQUIRE(x && (q || qt) && !q == !scale && !qt == !scale_t, YFS_ERR_INVALID_ARG, "yfs_fp8_quantize_rows: null pointer");
    REQUIRE_SIZES("yfs_fp8_quantize_rows", M, 1, K);
    YFS_REQUIRE(ld >= 0, YFS_ERR_INVALID_ARG, "yfs_fp8_quantize_rows: negative row stride");
    YFS_REQUIRE(known(dtype), YFS_ERR_UNSUPPORTED, "yfs_fp8_quantize_rows: unknown dtype %d", dtype);
    REQUIRE_ALIGNED("yfs_fp8_quantize_rows", q);
    REQUIRE_ALIGNED("yfs_fp8_quantize_rows", qt);
    const QuantArgs g = {x, ld, M, K, (unsigned char*)q, (unsigned char*)scale, (unsigned char*)qt, (unsigned char*)scale_t, colsum,
                         groups64(M), groups64(K)};
    hipStream_t s = (hipStream_t)stream;
    if (q && qt) return quantize<false, true, true>(g, dtype, s);
    return q ? quantize<false, true, false>(g, dtype, s) : quantize<false, false, true>(g, dtype, s);
}

YFS_API size_t yfs_fp8_gemm_workspace_bytes(int64_t M, int64_t N, int64_t K) {
    if (M <= 0 || N <= 0 || K <= 0 || M > kMost || N > kMost || K > kMost) return 0;
    return part_bytes(M, N, (int)yfs_cdiv(K, 128));
}

YFS_API int yfs_fp8_gemm(const void* aq, const void* a_scale, const void* bq, const void* b_scale, int b_row_scales, const float* bias,
                         void* out, int out_dtype, int64_t M, int64_t N, int64_t K, float slope, int accumulate, void* workspace,
                         size_t workspace_bytes, void* stream) {
    YFS_REQUIRE(aq && a_scale && bq && b_scale && out, YFS_ERR_INVALID_ARG, "yfs_fp8_gemm: null pointer");
    REQUIRE_SIZES("yfs_fp8_gemm", M, N, K);
    YFS_REQUIRE(known(out_dtype), YFS_ERR_UNSUPPORTED, "yfs_fp8_gemm: unknown dtype %d", out_dtype);
    YFS_REQUIRE(!accumulate || out_dtype == YFS_F32, YFS_ERR_UNSUPPORTED, "yfs_fp8_gemm: only an fp32 output accumulates");
    YFS_REQUIRE(slope >= 0.0f && slope <= 1.0f, YFS_ERR_INVALID_ARG, "yfs_fp8_gemm: slope %g not in [0, 1]", slope);
    REQUIRE_ALIGNED("yfs_fp8_gemm", aq);
    REQUIRE_ALIGNED("yfs_fp8_gemm", a_scale);
    REQUIRE_ALIGNED("yfs_fp8_gemm", bq);
    const size_t need = yfs_fp8_gemm_workspace_bytes(M, N, K);
    YFS_REQUIRE(need == 0 || (workspace && workspace_bytes >= need), YFS_ERR_WORKSPACE, "yfs_fp8_gemm: workspace needs %zu bytes", need);
    GemmArgs g = {(const unsigned char*)aq, (const unsigned char*)a_scale, (const unsigned char*)bq, (const unsigned char*)b_scale, bias, out,
                  (float*)workspace, M, N, (int)yfs_cdiv(K, 128), 1, 0, 0, 0, slope, accumulate};
    hipStream_t s = (hipStream_t)stream;
    if (b_row_scales) {
        if (out_dtype == YFS_F32) return gemm<true, true, float>(g, s);
        return out_dtype == YFS_BF16 ? gemm<true, false, bf16_t>(g, s) : gemm<true, false, _Float16>(g, s);
    }
    if (out_dtype == YFS_F32) return gemm<false, true, float>(g, s);
    return out_dtype == YFS_BF16 ? gemm<false, false, bf16_t>(g, s) : gemm<false, false, _Float16>(g, s);
}

namespace {
struct MatmulSpace { size_t q, s, part; };
MatmulSpace matmul_space(long long M, long long N, long long K) {
    return {align256((size_t)(M * pad128(K))), align256((size_t)packed_bytes(M, yfs_cdiv(K, 128))), part_bytes(M, N, (int)yfs_cdiv(K, 128))};
}
}  // namespace

YFS_API size_t yfs_fp8_matmul_workspace_bytes(int64_t M, int64_t N, int64_t K) {
    if (M <= 0 || N <= 0 || K <= 0 || M > kMost || N > kMost || K > kMost) return 0;
    const MatmulSpace w = matmul_space(M, N, K);
    return w.q + w.s + w.part;
}

YFS_API int yfs_fp8_matmul(const void* x, int x_dtype, int64_t ld, const void* wq, const void* w_scale, const float* bias, void* y,
                           int out_dtype, int64_t M, int64_t N, int64_t K, float slope, void* workspace, size_t workspace_bytes,
                           void* stream) {
    YFS_REQUIRE(x && wq && w_scale && y, YFS_ERR_INVALID_ARG, "yfs_fp8_matmul: null pointer");
    REQUIRE_SIZES("yfs_fp8_matmul", M, N, K);
    const size_t need = yfs_fp8_matmul_workspace_bytes(M, N, K);
    YFS_REQUIRE(workspace && workspace_bytes >= need && (reinterpret_cast<uintptr_t>(workspace) & 255) == 0, YFS_ERR_WORKSPACE,
                "yfs_fp8_matmul: workspace needs %zu bytes, 256-byte aligned", need);
    const MatmulSpace w = matmul_space(M, N, K);
    unsigned char* q = (unsigned char*)workspace;
    const int rc = yfs_fp8_quantize_rows(x, x_dtype, ld, M, K, q, q + w.q, nullptr, nullptr, nullptr, stream);
    if (rc != YFS_OK) return rc;
    return yfs_fp8_gemm(q, q + w.q, wq, w_scale, 0, bias, y, out_dtype, M, N, K, slope, 0, q + w.q + w.s, workspace_bytes - w.q - w.s, stream);
}

YFS_API int yfs_fp8_colsum(const float* part, int64_t tiles, int64_t K, float* out, int accumulate, void* stream) {
    YFS_REQUIRE(part && out && tiles > 0 && K > 0, YFS_ERR_INVALID_ARG, "yfs_fp8_colsum: null pointer or size <= 0");
    colsum_kernel<<<dim3((unsigned)yfs_cdiv(K, 256)), 256, 0, (hipStream_t)stream>>>(part, tiles, K, out, accumulate);
    YFS_CHECK_LAUNCH("colsum_kernel");
    return YFS_OK;
}
