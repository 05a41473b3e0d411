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

// e of the smallest power of two with amax <= 448 * 2^e = 0.875 * 2^(e + 9); amax finite and >= 0, given by its bits
__device__ __forceinline__ int scale_exponent(unsigned u) {
    const int e = (int)(u >> 23) - 126 - 9 + ((u & 0x7FFFFFu) > 0x600000u ? 1 : 0);   // a subnormal amax ends below -127
    return u == 0 ? 0 : (e < -127 ? -127 : e);
}
__device__ __forceinline__ float pow2(int e) { return __uint_as_float((unsigned)(e + 127) << 23); }   // -126 <= e <= 127

// Weights that are quantised and weight gradients go past the caches from half of the 256 MB on that the last of them holds.  Weights of
// 822 MB read through it push out their 8-bit form, which the backward pass reads next (64 x 50176 x 4096: dx 57 us, 33 with the
// weights read past it), and as many bytes of gradients left in it are written back while the next kernels run (the quantiser behind
// them 251 us, 217).  Only where rows begin on a line: elsewhere parts of lines are fetched or written twice (a training step at
// 184 x 4965 x 35251: 718 us, 697 through the caches; its quantiser at 184 x 4992 x 35200 the other way round, 192 against 235).
constexpr long long kPastCaches = 128LL << 20;
__host__ __device__ inline bool past_caches(long long row_bytes, long long bytes) { return bytes >= kPastCaches && row_bytes % 128 == 0; }

// Largest magnitudes are found among the bits, which are in the same order: one three-operand maximum takes two values.  Only a thread
// that meets an Inf or NaN looks at its values again, one by one.
constexpr unsigned kInfBits = 0x7F800000u;
__device__ __forceinline__ unsigned umax(unsigned a, unsigned b) { return a > b ? a : b; }
__device__ __forceinline__ unsigned abs_bits(float v) { return __float_as_uint(v) & 0x7FFFFFFFu; }
__device__ __forceinline__ unsigned finite_bits(float v) {
    asm volatile("" : "+v"(v));   // (or the magnitudes of the first look are kept for this one: 62 registers more)
    return abs_bits(v) < kInfBits ? abs_bits(v) : 0u;
}
template <int N>
__device__ __forceinline__ unsigned top_bits(const float (&v)[N]) {
    unsigned a = 0;
#pragma unroll
    for (int j = 0; j < N; ++j) a = umax(a, abs_bits(v[j]));
    return a;
}
template <int N>
__device__ __forceinline__ unsigned finite_top(const float (&v)[N]) {
    unsigned a = top_bits(v);
    if (a >= kInfBits) {
        a = 0;
#pragma unroll
        for (int j = 0; j < N; ++j) a = umax(a, finite_bits(v[j]));
    }
    return a;
}
__device__ __forceinline__ unsigned finite_top(const float (&v)[8][8]) {
    unsigned a = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) a = umax(a, top_bits(v[i]));
    if (a >= kInfBits) {
        a = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) a = umax(a, finite_top(v[i]));
    }
    return a;
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
    float* colsum;             // [ceil(M/128), K] sums of x over 128 rows each, or NULL
    int groups, groups_t;      // 64-row groups of the packed planes of q and qt
    int row_blocks;            // workgroups that quantise by rows
    bool once;                 // weights: read past the caches
};

// 8 x 8 weights of a thread: rows m .. and columns k .. of [M, K], zeros outside
template <typename T>
__device__ __forceinline__ void load_block(const QuantArgs& g, long long m, long long k, float (&v)[8][8]) {
    const T* p = (const T*)g.x + m * g.ld + k;
    if (g.once) {
#pragma unroll
        for (int i = 0; i < 8; ++i) load_vec8_once(p + i * g.ld, m + i < g.M ? g.K - k : 0, v[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) load_vec8(p + i * g.ld, m + i < g.M ? g.K - k : 0, v[i]);
    }
}

// Weights: one workgroup and one scale per 128 x 128 tile, 8 x 8 elements per thread; the transpose leaves through LDS.
template <typename T, bool COLQ>
__global__ void __launch_bounds__(256) quant_block_kernel(QuantArgs g) {
    __shared__ unsigned red[4];
    __shared__ __attribute__((aligned(16))) unsigned char tile[COLQ ? 128 * 144 : 16];
    const int cg = threadIdx.x & 15, rg = threadIdx.x >> 4, wave = threadIdx.x >> 6;
    // Neighbouring workgroups take a patch of up to 32 tiles down by the rest across: rows of a power of two times an odd number
    // of bytes meet few channels along one axis, whichever it is
    const int across = (int)((g.K + 127) >> 7), down = (int)((g.M + 127) >> 7), grp = (int)blockIdx.x / (32 * across);
    const int in = (int)blockIdx.x - grp * 32 * across, high = down - grp * 32 < 32 ? down - grp * 32 : 32;
    const long long kb = in / high, mb = grp * 32 + in - (int)kb * high;
    const long long k0 = kb * 128 + cg * 8, m0 = mb * 128 + rg * 8;
    const long long ldq = pad128(g.K), ldt = pad128(g.M);
    float v[8][8];
    load_block<T>(g, m0, k0, v);
    unsigned a = finite_top(v);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) a = umax(a, (unsigned)__shfl_xor((int)a, o, 64));
    if ((threadIdx.x & 63) == 0) red[wave] = a;
    __syncthreads();
    const int e = scale_exponent(umax(umax(red[0], red[1]), umax(red[2], red[3])));
    const float f = pow2(-e);
    if (threadIdx.x == 0) {
        g.s[mb * (ldq >> 7) + kb] = (unsigned char)(e + 127);
        if (COLQ) g.st[kb * (ldt >> 7) + mb] = (unsigned char)(e + 127);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const uint2 p = make_uint2(pack4(v[i][0] * f, v[i][1] * f, v[i][2] * f, v[i][3] * f),
                                   pack4(v[i][4] * f, v[i][5] * f, v[i][6] * f, v[i][7] * f));
        if (m0 + i < g.M) *reinterpret_cast<uint2*>(g.q + (m0 + i) * ldq + k0) = p;
    }
    if (COLQ) {
#pragma unroll
        for (int j = 0; j < 8; ++j)
            *reinterpret_cast<uint2*>(tile + (cg * 8 + j) * 144 + rg * 8) =
                make_uint2(pack4(v[0][j] * f, v[1][j] * f, v[2][j] * f, v[3][j] * f),
                           pack4(v[4][j] * f, v[5][j] * f, v[6][j] * f, v[7][j] * f));
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

// Activations and gradients.  The last row_blocks workgroups quantise by rows, 16 lanes x 8 elements per block, blocks of a row
// next to each other (four rows per thread, whose scales fill a dword of the packed plane, were slower: 12544 x 4096 bf16 35 us
// against 29, 5.3 TB/s).  The others, first because each takes longer, have 128 rows x 64 columns: column sums, and the transpose by
// rows, through LDS.  The second read of x comes from the caches; one 128 x 128 tile for both took 14 us where this takes 8
// (64 x 50176 bf16): too few workgroups with too long a chain of reductions each.
template <typename T>
__global__ void __launch_bounds__(256) quant_rows_kernel(QuantArgs g) {
    __shared__ unsigned top[4][64];
    __shared__ float sum[4][64];
    __shared__ unsigned tile[64 * 33];   // [column][128 rows + 4 bytes]
    const int col_blocks = (int)gridDim.x - g.row_blocks;
    if ((int)blockIdx.x >= col_blocks) {
        const long long kblocks = (g.K + 127) >> 7, total = g.M * kblocks;
        const int l = threadIdx.x & 15;
        for (long long id = (long long)((int)blockIdx.x - col_blocks) * 16 + (threadIdx.x >> 4); id < total; id += (long long)g.row_blocks * 16) {
            const long long m = total >> 32 ? id / kblocks : (unsigned)id / (unsigned)kblocks, kb = id - m * kblocks, k = kb * 128 + l * 8;
            float v[8];
            load_vec8((const T*)g.x + m * g.ld + k, g.K - k, v);
            unsigned a = finite_top(v);
#pragma unroll
            for (int o = 8; o > 0; o >>= 1) a = umax(a, (unsigned)__shfl_xor((int)a, o, 64));
            const int e = scale_exponent(a);
            if (l == 0) g.s[(kb * g.groups + (m >> 6)) * 64 + (m & 15) * 4 + ((m & 63) >> 4)] = (unsigned char)(e + 127);
            const float f = pow2(-e);
            *reinterpret_cast<uint2*>(g.q + m * kblocks * 128 + k) =
                make_uint2(pack4(v[0] * f, v[1] * f, v[2] * f, v[3] * f), pack4(v[4] * f, v[5] * f, v[6] * f, v[7] * f));
        }
        return;
    }
    const unsigned strips = (unsigned)((g.K + 63) >> 6);
    const long long mb = blockIdx.x / strips, strip = blockIdx.x - (unsigned)mb * strips, k0 = strip * 64;
    const int cg = threadIdx.x & 7, rg = threadIdx.x >> 3, wave = threadIdx.x >> 6;
    const long long m0 = mb * 128 + rg * 4, kc = k0 + cg * 8, ldt = pad128(g.M);
    float v[4][8];
#pragma unroll
    for (int i = 0; i < 4; ++i) load_vec8((const T*)g.x + (m0 + i) * g.ld + kc, m0 + i < g.M ? g.K - kc : 0, v[i]);
    unsigned a[8], all = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        a[j] = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) a[j] = umax(a[j], abs_bits(v[i][j]));
        all = umax(all, a[j]);
    }
    if (all >= kInfBits) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            a[j] = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) a[j] = umax(a[j], finite_bits(v[i][j]));
        }
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        float s = (v[0][j] + v[1][j]) + (v[2][j] + v[3][j]);
#pragma unroll
        for (int o = 8; o < 64; o <<= 1) {
            a[j] = umax(a[j], (unsigned)__shfl_xor((int)a[j], o, 64));
            if (g.colsum) s += __shfl_xor(s, o, 64);
        }
        if ((threadIdx.x & 56) == 0) {
            top[wave][cg * 8 + j] = a[j];
            sum[wave][cg * 8 + j] = s;
        }
    }
    __syncthreads();
    if (g.colsum && threadIdx.x < 64 && k0 + threadIdx.x < g.K)
        g.colsum[mb * g.K + k0 + threadIdx.x] = (sum[0][threadIdx.x] + sum[1][threadIdx.x]) + (sum[2][threadIdx.x] + sum[3][threadIdx.x]);
    if (!g.qt) return;
    auto exponent = [&](int c) { return scale_exponent(umax(umax(top[0][c], top[1][c]), umax(top[2][c], top[3][c]))); };
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const float f = pow2(-exponent(cg * 8 + j));
        tile[(cg * 8 + j) * 33 + rg] = pack4(v[0][j] * f, v[1][j] * f, v[2][j] * f, v[3][j] * f);
    }
    if (threadIdx.x < 16) {   // the 64 columns are one line of the packed scales
        unsigned bytes = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) bytes |= (unsigned)(exponent(i * 16 + (int)threadIdx.x) + 127) << (8 * i);
        *reinterpret_cast<unsigned*>(g.st + (mb * g.groups_t + strip) * 64 + threadIdx.x * 4) = bytes;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int c = i * 32 + (threadIdx.x >> 3), ch = threadIdx.x & 7;
        if (k0 + c < g.K) {
            const unsigned* t = tile + c * 33 + ch * 4;
            *reinterpret_cast<uint4*>(g.qt + (k0 + c) * ldt + mb * 128 + ch * 16) = make_uint4(t[0], t[1], t[2], t[3]);
        }
    }
}

// Sums over quant_rows_kernel's colsum: 32 columns x 32 slices of the tiles (8 where there are at most 64 tiles: 5 x 50176 3.1 us
// against 3.8), joined in slice order.  A chain of roundings is tiles / 32 + 31 long and its loads are on their way together (1568 x
// 4096: 4 us; as one chain over the tiles 161 us, and equal values lost 240 half steps of their sum).
__global__ void __launch_bounds__(1024) colsum_kernel(const float* __restrict__ part, long long tiles, long long K,
                                                      float* __restrict__ out, int accumulate) {
    __shared__ float red[32][33];
    const int ct = threadIdx.x & 31, slice = threadIdx.x >> 5, slices = (int)blockDim.x >> 5;
    const long long k = (long long)blockIdx.x * 32 + ct;
    float s = 0.0f;
    if (k < K) {
#pragma unroll 4
        for (long long t = slice; t < tiles; t += slices) s += part[t * K + k];
    }
    red[slice][ct] = s;
    __syncthreads();
    if (slice == 0 && k < K) {
        for (int q = 1; q < slices; ++q) s += red[q][ct];
        out[k] = accumulate ? out[k] + s : s;
    }
}

template <bool COLQ>
int quantize_blocks(const QuantArgs& g, int dtype, hipStream_t s) {
    YFS_REQUIRE(yfs_cdiv(g.K, 128) * yfs_cdiv(g.M, 128) < (1LL << 31) - 64, YFS_ERR_UNSUPPORTED, "yfs_fp8_quantize_weight: %lld x %lld is too large",
                g.M, g.K);
    const dim3 grid((unsigned)(yfs_cdiv(g.K, 128) * yfs_cdiv(g.M, 128)));
    if (dtype == YFS_F32) quant_block_kernel<float, COLQ><<<grid, 256, 0, s>>>(g);
    else if (dtype == YFS_BF16) quant_block_kernel<bf16_t, COLQ><<<grid, 256, 0, s>>>(g);
    else quant_block_kernel<_Float16, COLQ><<<grid, 256, 0, s>>>(g);
    YFS_CHECK_LAUNCH("quant_block_kernel");
    return YFS_OK;
}
int quantize_rows(QuantArgs g, int dtype, hipStream_t s) {
    const long long all = g.q ? yfs_cdiv(g.M * yfs_cdiv(g.K, 128), 16) : 0, rows = all < 16384 ? all : 16384;
    const long long cols = g.qt || g.colsum ? yfs_cdiv(g.K, 64) * yfs_cdiv(g.M, 128) : 0;
    g.row_blocks = (int)rows;
    YFS_REQUIRE(rows + cols < (1LL << 31), YFS_ERR_UNSUPPORTED, "yfs_fp8_quantize_rows: %lld x %lld is too large", g.M, g.K);
    const dim3 grid((unsigned)(g.row_blocks + cols));
    if (dtype == YFS_F32) quant_rows_kernel<float><<<grid, 256, 0, s>>>(g);
    else if (dtype == YFS_BF16) quant_rows_kernel<bf16_t><<<grid, 256, 0, s>>>(g);
    else quant_rows_kernel<_Float16><<<grid, 256, 0, s>>>(g);
    YFS_CHECK_LAUNCH("quant_rows_kernel");
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
    long long row0;                // row of the scales' planes that a[0] is (a call for the last rows of a larger product)
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

__device__ __forceinline__ f32x4 load4(const float* p, long long n, long long N) {   // p[n .. n + 3], zeros from N on
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
    if (n + 4 <= N) __builtin_memcpy(&v, p + n, 16);
    else {
#pragma unroll
        for (int r = 0; r < 4; ++r)
            if (n + r < N) v[r] = p[n + r];
    }
    return v;
}
__device__ __forceinline__ f32x4 act4(f32x4 v, f32x4 bias, float slope) {
#pragma unroll
    for (int r = 0; r < 4; ++r) v[r] = leaky(v[r] + bias[r], slope);
    return v;
}

// Four neighbouring outputs of row m: columns n .. n + 3, of which those below N exist
template <typename TO>
__device__ __forceinline__ void store4(const GemmArgs& g, long long m, long long n, f32x4 v) {
    const f32x4 none = {0.f, 0.f, 0.f, 0.f};
    v = act4(v, g.bias ? load4(g.bias, n, g.N) : none, g.slope);
    TO* o = (TO*)g.out + m * g.N + n;
    TO t[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) t[r] = (TO)(sizeof(TO) == 4 && g.accumulate && n + r < g.N ? v[r] + (float)o[r] : v[r]);
    if (n + 4 <= g.N) __builtin_memcpy(o, t, sizeof(t));
    else {
#pragma unroll
        for (int r = 0; r < 4; ++r)
            if (n + r < g.N) o[r] = t[r];
    }
}

// A finished tile of BM x BN fp32 outputs leaves through LDS ([row][BN * 4 + 16 bytes]), whole rows at a time.  Straight from the
// accumulators a wave would write 16 rows x 64 bytes at once, and rows of a power of two times an odd number of bytes all fall
// on one channel of the L2 (50176 columns: 330 us for 822 MB, 157 through LDS).  16-bit outputs gain nothing by it.
template <int BM, int BN, int NT>
__device__ __forceinline__ void store_tile(const GemmArgs& g, const unsigned char* smem, long long m0, long long n0) {
    constexpr int PER = BN / 4, PITCH = BN * 4 + 16;
    const bool once = past_caches(g.N * 4, g.M * g.N * 4);
#pragma unroll 4
    for (int id = threadIdx.x; id < BM * PER; id += NT) {
        const int r = id / PER, ch = id % PER;
        const long long m = m0 + r, n = n0 + ch * 4;
        if (m >= g.M || n >= g.N) continue;
        f32x4 t = *reinterpret_cast<const f32x4*>(smem + r * PITCH + ch * 16);
        float* o = (float*)g.out + m * g.N + n;
        if (g.accumulate) t += load4((const float*)g.out + m * g.N, n, g.N);
        if (n + 4 <= g.N && once) __builtin_nontemporal_store(__builtin_bit_cast(i32x4, t), (yfs_int4_any*)o);
        else if (n + 4 <= g.N) __builtin_memcpy(o, &t, 16);
        else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (n + j < g.N) o[j] = t[j];
        }
    }
}

__device__ __forceinline__ void store_part(const GemmArgs& g, int split, long long m, long long n, f32x4 v) {
    float* o = g.part + ((long long)split * g.M + m) * g.N + n;
    if (n + 4 <= g.N) __builtin_memcpy(o, &v, 16);
    else {
#pragma unroll
        for (int r = 0; r < 4; ++r)
            if (n + r < g.N) o[r] = v[r];
    }
}

template <int N>
__device__ __forceinline__ void wait_vm() { asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory"); }
__device__ __forceinline__ void barrier() {
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_sched_barrier(0);
}

// The exponent byte of a 128-row block of b at k-block kb, through the scalar unit (the aligned dword that holds it: same page):
// no vector register, and nothing that the counted waits for vector loads would see.
__device__ __forceinline__ int block_scale(const unsigned char* row, int kb) {
    typedef const __attribute__((address_space(4))) unsigned* cptr;
    const uintptr_t p = reinterpret_cast<uintptr_t>(row) + (uintptr_t)(unsigned)kb;
    return (int)((*reinterpret_cast<cptr>(p & ~(uintptr_t)3) >> ((p & 3) * 8)) & 255u);
}

// out tile of (WM FM 16) x (WN FN 16), a wave FM x FN fragments of 16 x 16.  LDS holds a ring of S stages: the 128-byte rows of
// both operands, 16-byte chunks swizzled by the row, and the row scales, filled by direct loads.  S - 1 stages are on their
// way while one is multiplied; a stage is waited for by count (DPS loads per wave and stage, in order) and handed over with one
// barrier per k-block.  The operands' lanes hold 32 of a block's 128 k in an order that is the same on both sides, which is all
// that the sum needs.  The b rows are the instruction's first operand, so that a lane owns four neighbouring columns of one
// output row.
// EXACT: the e4m3 instructions align the 128 products of a block to the largest and keep 16 bits behind it, so an output is off by
// 2^-9 of the largest product of each block at most, 1.5e-5 of the outputs' norm whatever K (measured).  An output whose products
// cancel can lose more than its own last place by it; the operands' rounding to four significant bits, 2^-4 of each product, is far
// above it in any case.  Where the output is fp32 the operands are widened in registers and multiplied by the bf16 instruction,
// whose sums are full fp32.  For 16-bit outputs that would cost (us, 16-bit sums / fp32 sums): 12544 x 4096 x 4096 217 / 379,
// 4096 x 4096 x 4096 70 / 128, 300 x 4096 x 4096 21.5 / 28.7, 64 x 4096 x 50176 55 / 57.
template <int FM, int FN, int WM, int WN, int S, bool ROWB, bool EXACT, typename TO>
__global__ void __launch_bounds__(64 * WM * WN) fp8_gemm_kernel(GemmArgs g) {
    constexpr int BM = WM * FM * 16, BN = WN * FN * 16, NW = WM * WN;
    constexpr int TILE = (BM + BN) * 128, STAGE = TILE + NW * 256 * (ROWB ? 2 : 1);
    constexpr int DPS = (BM + BN) / 8 / NW + (ROWB ? 2 : 1);
    static_assert(BM % (8 * NW) == 0 && BN % (8 * NW) == 0 && FM * 16 <= 64 && FN * 16 <= 64, "rows per wave");
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const int wm = wave / WN, wn = wave % WN;
    int tm = (int)blockIdx.y, tn = (int)blockIdx.x;
    if constexpr (sizeof(TO) == 4) {
        // Workgroups go round the 8 XCDs.  Where the rows of a large output begin inside a line, neighbouring tiles share lines: each XCD then
        // takes tiles that are neighbours (4001 x 50001 x 64: 194 us against 267; whole lines, 4096 x 50176 x 64, 159 against 139)
        if (g.splits == 1 && g.N % 32 != 0 && g.M * g.N * 4 >= kPastCaches) {
            const int across = (int)gridDim.x, total = across * (int)gridDim.y, lin = tm * across + tn;
            const int q8 = total >> 3, r8 = total & 7, xcd = lin & 7;
            const int id = (xcd < r8 ? xcd * (q8 + 1) : r8 * (q8 + 1) + (xcd - r8) * q8) + (lin >> 3);
            tm = id / across;
            tn = id - tm * across;
        }
    }
    const long long m0 = (long long)tm * BM, n0 = (long long)tn * BN;
    const long long ld = (long long)g.kblocks * 128;
    const int kb0 = (int)blockIdx.z * g.per_split;
    const int kb1 = kb0 + g.per_split < g.kblocks ? kb0 + g.per_split : g.kblocks;
    const long long ra = g.M - m0 < BM ? g.M - m0 : BM, rb = g.N - n0 < BN ? g.N - n0 : BN;
    const __amdgpu_buffer_rsrc_t rsa = rsrc(g.a + m0 * ld, ra * ld), rsb = rsrc(g.b + n0 * ld, rb * ld);
    const int srow = lane >> 3;
    const unsigned chunk = (unsigned)((lane & 7) ^ srow) * 16u;
    auto stage = [&](int kb, int buf) {   // rows outside the operands read as zeros
        unsigned char* base = smem + buf * STAGE;
        const unsigned so = (unsigned)kb * 128u;
#pragma unroll
        for (int i = 0; i < BM / 8 / NW; ++i) {
            const int r = wave * (BM / 8 / NW) + i;
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rsa, (lds_ptr)(base + r * 1024), 16, (unsigned)((r * 8 + srow) * ld) + chunk, so, 0, 0);
        }
#pragma unroll
        for (int i = 0; i < BN / 8 / NW; ++i) {
            const int r = wave * (BN / 8 / NW) + i;
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rsb, (lds_ptr)(base + BM * 128 + r * 1024), 16,
                                                     (unsigned)((r * 8 + srow) * ld) + chunk, so, 0, 0);
        }
        // each wave its own copy of the scales: 4 groups of 64 rows; groups behind the plane's end are not used
        const long long ga = (long long)kb * g.groups_a + ((g.row0 + m0) >> 6);
        const __amdgpu_buffer_rsrc_t rs = rsrc(g.as + ga * 64, ((long long)g.kblocks * g.groups_a - ga) * 64);
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (lds_ptr)(base + TILE + wave * 256), 4, (unsigned)lane * 4u, 0, 0, 0);
        if (ROWB) {
            const long long gb = (long long)kb * g.groups_b + (n0 >> 6);
            const __amdgpu_buffer_rsrc_t rt = rsrc(g.bs + gb * 64, ((long long)g.kblocks * g.groups_b - gb) * 64);
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rt, (lds_ptr)(base + TILE + (NW + wave) * 256), 4, (unsigned)lane * 4u, 0, 0, 0);
        }
    };
    const int frow = lane & 15, fk = lane >> 4;
    auto fragment = [&](const unsigned char* base, int row) {
        const i32x4 lo = *reinterpret_cast<const i32x4*>(base + row * 128 + ((fk ^ (row & 7)) * 16));
        const i32x4 hi = *reinterpret_cast<const i32x4*>(base + row * 128 + (((4 + fk) ^ (row & 7)) * 16));
        return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    };
    // scales of a wave's F fragments: the dword of its 64-row group, shifted down to its first fragment
    auto scales = [&](const unsigned char* base, int row0) {
        const int d = *reinterpret_cast<const int*>(base + (row0 >> 6) * 64 + frow * 4);
        return (int)((unsigned)d >> ((row0 & 63) / 16 * 8));
    };
    const long long nb = (n0 + wn * FN * 16) >> 7, last = (g.N - 1) >> 7;
    const unsigned char* const bsrow = ROWB ? nullptr : g.bs + (nb < last ? nb : last) * g.kblocks;
    int sbn = ROWB ? 0 : block_scale(bsrow, kb0);
    f32x4 acc[FN][FM];
#pragma unroll
    for (int i = 0; i < FN; ++i)
#pragma unroll
        for (int j = 0; j < FM; ++j) acc[i][j] = (f32x4){0.f, 0.f, 0.f, 0.f};

    const int nit = kb1 - kb0;
#pragma unroll
    for (int t = 0; t < S - 1; ++t)
        if (t < nit) stage(kb0 + t, t);
    int buf = 0, into = S - 1;
    for (int t = 0; t < nit; ++t) {
        if (t + S - 2 < nit) wait_vm<DPS * (S - 2)>(); else wait_vm<0>();
        barrier();   // stage t is there for every wave; every wave has left the stage before it
        if (t + S - 1 < nit) stage(kb0 + t + S - 1, into);
        into = into + 1 == S ? 0 : into + 1;
        const unsigned char* ab = smem + buf * STAGE;
        const unsigned char* bb = ab + BM * 128;
        buf = buf + 1 == S ? 0 : buf + 1;
        const int sa = scales(ab + TILE + wave * 256, wm * FM * 16);
        const int sb = ROWB ? scales(ab + TILE + (NW + wave) * 256, wn * FN * 16) : sbn;
        if (!ROWB && t + 1 < nit) sbn = block_scale(bsrow, kb0 + t + 1);
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
    }
    if (sizeof(TO) == 4 && g.splits == 1) {
        barrier();   // every wave has read its last fragments: the ring becomes the tile
#pragma unroll
        for (int i = 0; i < FN; ++i) {
            const int col = wn * FN * 16 + i * 16 + fk * 4;
            const f32x4 none = {0.f, 0.f, 0.f, 0.f};
            const f32x4 bias = g.bias ? load4(g.bias, n0 + col, g.N) : none;
#pragma unroll
            for (int j = 0; j < FM; ++j)
                *reinterpret_cast<f32x4*>(smem + (wm * FM * 16 + j * 16 + frow) * (BN * 4 + 16) + col * 4) = act4(acc[i][j], bias, g.slope);
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        barrier();
        store_tile<BM, BN, 64 * NW>(g, smem, m0, n0);
        return;
    }
#pragma unroll
    for (int j = 0; j < FM; ++j) {
        const long long m = m0 + wm * FM * 16 + j * 16 + frow;
        if (m >= g.M) continue;
#pragma unroll
        for (int i = 0; i < FN; ++i) {
            const long long n = n0 + wn * FN * 16 + i * 16 + fk * 4;
            if (n >= g.N) continue;
            if (g.splits > 1) store_part(g, blockIdx.z, m, n, acc[i][j]);
            else if constexpr (sizeof(TO) < 4) store4<TO>(g, m, n, acc[i][j]);
        }
    }
}

// Large products: 256 x 256 outputs, 8 waves as 2 (row halves of a half-tile) x 4, one workgroup per CU.  The schedule of the
// convolutions' 8-wave kernel with 8-bit rows: a k-block is four half-tiles of 16 KiB (128 rows x 128 bytes: A0, A1, B0, B1),
// LDS holds two k-blocks, and the two row halves run one barrier apart, so that on every SIMD one wave multiplies while its
// partner reads fragments and sends loads:
//   phase A: read B0, A0, B1 | send A1 of block t + 1                       | 16 products with A0
//   phase B: read A1         | send B0, A0, B1 and the scales of block t + 2 | 16 products with A1
// A half-tile is sent again one phase after its fragments were read, every wave having retired its reads (lgkmcnt 0) before the
// phase's first barrier.  The only wait for loads is in phase B and leaves the seven just sent on their way.
// A wave's 128 x 64 outputs are 128 accumulators; a fragment pair read from LDS feeds 4 (2) products of 32 cycles.
constexpr int G8_HALF = 128 * 128, G8_BUF = 4 * G8_HALF, G8_SCALES = 2 * G8_BUF;
constexpr int G8_LDS = G8_SCALES + 2 * 8 * 256;

template <typename TO>
__global__ void __launch_bounds__(512, 2) fp8_gemm8_kernel(GemmArgs g) {
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const int wm = wave >> 2, wn = wave & 3, frow = lane & 15, fk = lane >> 4;
    // Workgroups go round the 8 XCDs: each XCD gets neighbouring tiles, in groups of 8 tile rows, so that the tiles that run on
    // it at one time share their operands' rows in its L2
    const int mt = (int)((g.M + 255) >> 8), nt = (int)((g.N + 255) >> 8), total = mt * nt;
    const int q8 = total >> 3, r8 = total & 7, xcd = (int)blockIdx.x & 7;
    const int id = (xcd < r8 ? xcd * (q8 + 1) : r8 * (q8 + 1) + (xcd - r8) * q8) + ((int)blockIdx.x >> 3);
    const int grp = id / (8 * nt), in = id - grp * 8 * nt, high = mt - grp * 8 < 8 ? mt - grp * 8 : 8;
    const int tn = in / high, tm = grp * 8 + in - tn * high;
    const long long m0 = __builtin_amdgcn_readfirstlane(tm) * 256LL, n0 = __builtin_amdgcn_readfirstlane(tn) * 256LL;
    const long long ld = (long long)g.kblocks * 128;
    const int nit = g.kblocks;
    const unsigned ra = (unsigned)((g.M - m0 < 256 ? g.M - m0 : 256) * ld), rb = (unsigned)((g.N - n0 < 256 ? g.N - n0 : 256) * ld);
    const unsigned char *const pa = g.a + m0 * ld, *const pb = g.b + n0 * ld, *const ps = g.as + (m0 >> 6) * 64;
    const int srow = lane >> 3;
    const unsigned off0 = (unsigned)((wave * 16 + srow) * ld) + (unsigned)((lane & 7) ^ srow) * 16u, off8 = (unsigned)(8 * ld), half = (unsigned)(128 * ld);
    // Rows outside the operands, and whole blocks behind the last one, read as zeros (a descriptor of no bytes): every pass of
    // the loop sends the same loads, without a branch.
    auto stage = [&](const unsigned char* p, unsigned bytes, int h, int slot, int kb, int buf) {
        const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(const_cast<unsigned char*>(p), 0, kb < nit ? (int)bytes : 0, 0x00020000);
        unsigned off = off0;
        asm volatile("" : "+v"(off));   // (four sums of a register and a scalar a phase instead of four registers all the way)
#pragma unroll
        for (int i = 0; i < 2; ++i)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_ptr)(smem + buf * G8_BUF + slot * G8_HALF + (wave * 2 + i) * 1024), 16,
                                                     off + (unsigned)i * off8 + (unsigned)h * half, (unsigned)kb * 128u, 0, 0);
    };
    auto stage_scales = [&](int kb, int buf) {   // each wave its own copy of the 256 rows' bytes
        const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(const_cast<unsigned char*>(ps + (long long)kb * g.groups_a * 64), 0,
                                                                            kb < nit ? 256 : 0, 0x00020000);
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (lds_ptr)(smem + G8_SCALES + (buf * 8 + wave) * 256), 4, (unsigned)lane * 4u, 0, 0, 0);
    };
    const long long last = (g.N - 1) >> 7, nb = n0 >> 7;
    const unsigned char *const bs0 = g.bs + nb * nit, *const bs1 = g.bs + (nb + 1 < last ? nb + 1 : last) * nit;
    int s0 = block_scale(bs0, 0), s1 = block_scale(bs1, 0), s0n, s1n;

    f32x4 acc[2][2][2][4];   // [A half][B half][fragment of B][fragment of A]
#pragma unroll
    for (int i = 0; i < 32; ++i) (&acc[0][0][0][0])[i] = (f32x4){0.f, 0.f, 0.f, 0.f};
    auto fragment = [&](const unsigned char* base, int row) {
        const i32x4 lo = *reinterpret_cast<const i32x4*>(base + row * 128 + ((fk ^ (row & 7)) * 16));
        const i32x4 hi = *reinterpret_cast<const i32x4*>(base + row * 128 + (((4 + fk) ^ (row & 7)) * 16));
        return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    };
    i32x8 fa[4], fb0[2], fb1[2];
    auto read_a = [&](const unsigned char* hb) {
#pragma unroll
        for (int b = 0; b < 4; ++b) fa[b] = fragment(hb, wm * 64 + b * 16 + frow);
    };
    auto read_b = [&](const unsigned char* hb, i32x8 (&f)[2]) {
#pragma unroll
        for (int a = 0; a < 2; ++a) f[a] = fragment(hb, wn * 32 + a * 16 + frow);
    };
    auto products = [&](f32x4 (&c)[2][4], const i32x8 (&f)[2], int sb, int sa) {
        __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int a = 0; a < 2; ++a) {
            c[a][0] = mfma_fp8<0, 0>(f[a], fa[0], c[a][0], sb, sa);
            c[a][1] = mfma_fp8<0, 1>(f[a], fa[1], c[a][1], sb, sa);
            c[a][2] = mfma_fp8<0, 2>(f[a], fa[2], c[a][2], sb, sa);
            c[a][3] = mfma_fp8<0, 3>(f[a], fa[3], c[a][3], sb, sa);
        }
        __builtin_amdgcn_s_setprio(0);
    };
    auto lgkm0 = [&]() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); };

    stage(pb, rb, 0, 2, 0, 0);
    stage(pb, rb, 1, 3, 0, 0);
    stage(pa, ra, 0, 0, 0, 0);
    stage(pa, ra, 1, 1, 0, 0);
    stage_scales(0, 0);
    stage(pb, rb, 0, 2, 1, 1);
    stage(pa, ra, 0, 0, 1, 1);
    stage(pb, rb, 1, 3, 1, 1);
    stage_scales(1, 1);
    wait_vm<7>();
    auto block = [&](int t, auto buf_tag) {
        constexpr int BUF = decltype(buf_tag)::value;
        const unsigned char* tb = smem + BUF * G8_BUF;
        read_b(tb + 2 * G8_HALF, fb0);
        read_a(tb);
        read_b(tb + 3 * G8_HALF, fb1);
        const unsigned char* sp = smem + G8_SCALES + (BUF * 8 + wave) * 256 + frow * 4;
        const int sa0 = *reinterpret_cast<const int*>(sp + wm * 64), sa1 = *reinterpret_cast<const int*>(sp + 128 + wm * 64);
        const int tn = t + 1 < nit ? t + 1 : nit - 1;
        s0n = block_scale(bs0, tn);
        s1n = block_scale(bs1, tn);
        stage(pa, ra, 1, 1, t + 1, BUF ^ 1);
        lgkm0();
        barrier();
        products(acc[0][0], fb0, s0, sa0);
        products(acc[0][1], fb1, s1, sa0);
        barrier();
        read_a(tb + G8_HALF);
        stage(pb, rb, 0, 2, t + 2, BUF);
        stage(pa, ra, 0, 0, t + 2, BUF);
        stage(pb, rb, 1, 3, t + 2, BUF);
        stage_scales(t + 2, BUF);
        wait_vm<7>();
        lgkm0();
        barrier();
        products(acc[1][1], fb1, s1, sa1);
        products(acc[1][0], fb0, s0, sa1);
        barrier();
        s0 = s0n;
        s1 = s1n;
    };
    barrier();
    if (wm == 1) barrier();   // waves 4-7 run one barrier behind waves 0-3 from here on
    for (int t = 0; t < nit; t += 2) {   // an odd count ends with a block of zeros
        block(t, std::integral_constant<int, 0>());
        block(t + 1, std::integral_constant<int, 1>());
    }
    if (wm == 0) barrier();
    wait_vm<0>();   // (the loads of no bytes still write their zeros)
    // Straight from the accumulators: through LDS, whole rows at a time, took 3-9 % longer here (one workgroup per CU: nothing
    // else runs meanwhile)
#pragma unroll
    for (int wh = 0; wh < 2; ++wh)
#pragma unroll
        for (int a = 0; a < 2; ++a) {
            const long long n = n0 + wh * 128 + wn * 32 + a * 16 + fk * 4;
            if (n >= g.N) continue;
#pragma unroll
            for (int ph = 0; ph < 2; ++ph)
#pragma unroll
                for (int b = 0; b < 4; ++b) {
                    const long long m = m0 + ph * 128 + wm * 64 + b * 16 + frow;
                    if (m < g.M) store4<TO>(g, m, n, acc[ph][wh][a][b]);
                }
        }
}

// Few rows (a server's single images): bound by the weights' bytes, each read once, straight into the registers of the one
// wave that multiplies them, so that nothing has to be shared before the end.  A workgroup owns 16 columns; its waves take the
// k-blocks in turn (neighbouring waves read neighbouring 128 bytes of the same 16 rows), U at a time with the next U on their
// way, and join their sums through LDS in wave order.  x comes in its own type and the workgroup first quantises what it
// multiplies into LDS, [block][row][128 bytes] with the exponent bytes behind: no second launch (measured on one row, 4096 x
// 50176: 43 us, 4.8 TB/s; quantising in the multiplying lanes instead took 77 us, 15 of 16 of them have no row of their own).
template <typename T, typename TO>
__global__ void __launch_bounds__(1024) fp8_rows_kernel(GemmArgs g, const T* x, long long ldx, long long K) {
    constexpr bool EXACT = sizeof(TO) == 4;
    constexpr int U = 4;
    __shared__ f32x4 red[16][64];
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    const int lane = threadIdx.x & 63, frow = lane & 15, fk = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6)), nw = (int)(blockDim.x >> 6);
    const long long n0 = (long long)blockIdx.x * 16, ld = (long long)g.kblocks * 128;
    const int kb0 = (int)blockIdx.y * g.per_split;
    const int kb1 = kb0 + g.per_split < g.kblocks ? kb0 + g.per_split : g.kblocks;
    const int rows = (int)g.M, nkb = kb1 - kb0;
    const long long nrow = n0 + frow < g.N ? n0 + frow : g.N - 1;   // (the last row again: its columns are not stored)
    const unsigned char* bp = g.b + nrow * ld + fk * 16;
    const unsigned char* bsp = g.bs + (n0 >> 7) * g.kblocks;
    const bool live = frow < rows;
    unsigned char* const sx = smem + (long long)nkb * rows * 128;

    i32x4 b[2][U][2];
    int sb[2][U];
    auto fetch = [&](int kb, auto into) {
        constexpr int I = decltype(into)::value;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int k = kb + u * nw;
            if (k >= kb1) break;
            b[I][u][0] = *reinterpret_cast<const i32x4*>(bp + (long long)k * 128);
            b[I][u][1] = *reinterpret_cast<const i32x4*>(bp + (long long)k * 128 + 64);
            sb[I][u] = bsp[k];
        }
    };
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    auto multiply = [&](int kb, auto from) {
        constexpr int I = decltype(from)::value;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int k = kb + u * nw;
            if (k >= kb1) break;
            const i32x4 none = {0, 0, 0, 0};
            i32x4 lo = none, hi = none;
            int s = 127;
            if (live) {
                const unsigned char* p = smem + ((long long)(k - kb0) * rows + frow) * 128 + fk * 16;
                lo = *reinterpret_cast<const i32x4*>(p);
                hi = *reinterpret_cast<const i32x4*>(p + 64);
                s = sx[(k - kb0) * rows + frow];
            }
            const i32x8 v = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
            const i32x8 w = __builtin_shufflevector(b[I][u][0], b[I][u][1], 0, 1, 2, 3, 4, 5, 6, 7);
            if constexpr (EXACT) {
                bf16x8 wa[4], wb[4];
                widen(v, __uint_as_float((unsigned)s << 23), wa);
                widen(w, __uint_as_float((unsigned)sb[I][u] << 23), wb);
#pragma unroll
                for (int q = 0; q < 4; ++q) acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wb[q], wa[q], acc, 0, 0, 0);
            } else acc = mfma_fp8<0, 0>(w, v, acc, sb[I][u], s);
        }
    };
    const std::integral_constant<int, 0> A;
    const std::integral_constant<int, 1> B;
    const int step = nw * U;
    fetch(kb0 + wave, A);
    {   // while the first weights are on their way: 16 lanes x 8 elements per block, as quant_rows_kernel
        const int l = threadIdx.x & 15, groups = (int)(blockDim.x >> 4);
        for (int id = (int)(threadIdx.x >> 4); id < nkb * rows; id += groups) {
            const int blk = id / rows, m = id - blk * rows;
            const long long k = (long long)(kb0 + blk) * 128 + l * 8;
            float v[8];
            load_vec8(x + m * ldx + k, K - k, v);
            unsigned top = finite_top(v);
#pragma unroll
            for (int o = 8; o > 0; o >>= 1) top = umax(top, (unsigned)__shfl_xor((int)top, o, 64));
            const int e = scale_exponent(top);
            const float f = pow2(-e);
            *reinterpret_cast<uint2*>(smem + (long long)id * 128 + l * 8) =
                make_uint2(pack4(v[0] * f, v[1] * f, v[2] * f, v[3] * f), pack4(v[4] * f, v[5] * f, v[6] * f, v[7] * f));
            if (l == 0) sx[id] = (unsigned char)(e + 127);
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        barrier();
    }
    for (int kb = kb0 + wave; kb < kb1; kb += 2 * step) {
        fetch(kb + step, B);
        multiply(kb, A);
        fetch(kb + 2 * step, A);
        multiply(kb + step, B);
    }
    red[wave][lane] = acc;
    __syncthreads();
    if (wave == 0) {
        for (int w = 1; w < nw; ++w) acc += red[w][lane];
        const long long n = n0 + fk * 4;
        if (live && n < g.N) {
            if (g.splits > 1) store_part(g, blockIdx.y, frow, n, acc);
            else store4<TO>(g, frow, n, acc);
        }
    }
}

// A training step's forward pass for at most 64 rows: bound by the bytes of the weights in their own type, so they are
// quantised, transposed for the backward pass and multiplied while they are on the chip.  A workgroup takes 128 columns of y and
// per_split blocks of the reduction; per block the 128 x 128 weights are read once, leave through LDS as 8-bit columns (qt, for dx),
// and from LDS as rows into the products: a wave owns 32 columns of all 64 rows.  The partial sums are joined by fp8_join_kernel.
// 64 x 4096 x 50176, fp32 weights: 232 us, 4.5 TB/s of 822 MB read and 222 MB written (quantiser and product one after the other: 251 + 48).
// Three workgroups per CU, the next block's weights ahead in registers, x straight from L2: 287, 264, 275 where two plain ones took 251.
template <typename T, typename TO>
__global__ void __launch_bounds__(256) fp8_train_rows_kernel(GemmArgs g, QuantArgs w) {
    constexpr bool EXACT = sizeof(TO) == 4;
    __shared__ unsigned red[4];
    __shared__ __attribute__((aligned(16))) unsigned char wt[128 * 128], xt[64 * 128], tt[128 * 144];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, frow = lane & 15, fk = lane >> 4;
    const int cg = threadIdx.x & 15, rg = threadIdx.x >> 4;
    const int down = (int)((g.N + 127) >> 7), nb = (int)blockIdx.x % down, split = (int)blockIdx.x / down;
    const int kb0 = split * g.per_split, kb1 = kb0 + g.per_split < g.kblocks ? kb0 + g.per_split : g.kblocks;
    const long long n0 = nb * 128LL, m0 = n0 + rg * 8, ldt = pad128(g.N), ldx = g.kblocks * 128LL;
    auto fragment = [&](const unsigned char* base, int row) {
        const i32x4 lo = *reinterpret_cast<const i32x4*>(base + row * 128 + ((fk ^ (row & 7)) * 16));
        const i32x4 hi = *reinterpret_cast<const i32x4*>(base + row * 128 + (((4 + fk) ^ (row & 7)) * 16));
        return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    };
    f32x4 acc[2][4];
#pragma unroll
    for (int i = 0; i < 8; ++i) (&acc[0][0])[i] = (f32x4){0.f, 0.f, 0.f, 0.f};
    for (int kb = kb0; kb < kb1; ++kb) {
        const long long k0 = kb * 128LL + cg * 8;
        float v[8][8];
        load_block<T>(w, m0, k0, v);
        i32x4 xv[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {   // 64 rows of x, 16 bytes a thread and half
            const int row = i * 32 + (threadIdx.x >> 3);
            xv[i] = (i32x4){0, 0, 0, 0};
            if (row < g.M) xv[i] = *reinterpret_cast<const i32x4*>(g.a + row * ldx + kb * 128LL + (threadIdx.x & 7) * 16);
        }
        const int sa = *reinterpret_cast<const int*>(g.as + (long long)kb * g.groups_a * 64 + frow * 4);
        unsigned a = finite_top(v);
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) a = umax(a, (unsigned)__shfl_xor((int)a, o, 64));
        if (lane == 0) red[wave] = a;
        __syncthreads();   // (and every wave has left the block before this one)
        const int e = scale_exponent(umax(umax(red[0], red[1]), umax(red[2], red[3])));
        const float f = pow2(-e);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int row = rg * 8 + i;
            *reinterpret_cast<uint2*>(wt + row * 128 + (((cg >> 1) ^ (row & 7)) * 16) + (cg & 1) * 8) =
                make_uint2(pack4(v[i][0] * f, v[i][1] * f, v[i][2] * f, v[i][3] * f), pack4(v[i][4] * f, v[i][5] * f, v[i][6] * f, v[i][7] * f));
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int row = i * 32 + (threadIdx.x >> 3);
            *reinterpret_cast<i32x4*>(xt + row * 128 + (((threadIdx.x & 7) ^ (row & 7)) * 16)) = xv[i];
        }
        if (w.qt) {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                *reinterpret_cast<uint2*>(tt + (cg * 8 + j) * 144 + rg * 8) =
                    make_uint2(pack4(v[0][j] * f, v[1][j] * f, v[2][j] * f, v[3][j] * f), pack4(v[4][j] * f, v[5][j] * f, v[6][j] * f, v[7][j] * f));
        }
        __syncthreads();
        if (w.qt) {
            if (threadIdx.x == 0) w.st[kb * (ldt >> 7) + nb] = (unsigned char)(e + 127);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int c = i * 32 + (threadIdx.x >> 3), ch = threadIdx.x & 7;
                const long long k = kb * 128LL + c;
                if (k < w.K)
                    *reinterpret_cast<i32x4*>(w.qt + k * ldt + n0 + ch * 16) = *reinterpret_cast<const i32x4*>(tt + c * 144 + ch * 16);
            }
        }
        i32x8 fa[4], fb[2];
#pragma unroll
        for (int j = 0; j < 4; ++j) fa[j] = fragment(xt, j * 16 + frow);
#pragma unroll
        for (int i = 0; i < 2; ++i) fb[i] = fragment(wt, wave * 32 + i * 16 + frow);
        const int sb = e + 127;
        if constexpr (EXACT) {
            bf16x8 wb[2][4];
#pragma unroll
            for (int i = 0; i < 2; ++i) widen(fb[i], __uint_as_float((unsigned)sb << 23), wb[i]);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                bf16x8 wa[4];
                widen(fa[j], __uint_as_float((((unsigned)sa >> (8 * j)) & 255u) << 23), wa);
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int q = 0; q < 4; ++q) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wb[i][q], wa[q], acc[i][j], 0, 0, 0);
            }
        } else {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                acc[i][0] = mfma_fp8<0, 0>(fb[i], fa[0], acc[i][0], sb, sa);
                acc[i][1] = mfma_fp8<0, 1>(fb[i], fa[1], acc[i][1], sb, sa);
                acc[i][2] = mfma_fp8<0, 2>(fb[i], fa[2], acc[i][2], sb, sa);
                acc[i][3] = mfma_fp8<0, 3>(fb[i], fa[3], acc[i][3], sb, sa);
            }
        }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const long long m = j * 16 + frow;
        if (m >= g.M) continue;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const long long n = n0 + wave * 32 + i * 16 + fk * 4;
            if (n >= g.N) continue;
            if (g.splits > 1) store_part(g, split, m, n, acc[i][j]);
            else store4<TO>(g, m, n, acc[i][j]);
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
        const float* p = g.part + m * g.N;
#pragma unroll 8
        for (int s = 0; s < g.splits; ++s) v += load4(p + s * g.M * g.N, n, g.N);
        store4<TO>(g, m, n, v);
    }
}

constexpr int kRows = 16;              // rows that fp8_rows_kernel can take
constexpr size_t kRowsLds = 128 * 1024;   // its quantised rows in LDS
constexpr int kCUs = 256;

// two: two workgroups per CU although the reduction is split; body: rows that kind 2 takes
struct Plan { int kind, bm, bn, splits, per_split; long long body; bool two = false; };   // kind 0: fp8_rows_kernel, 1: fp8_gemm_kernel, 2: fp8_gemm8_kernel
size_t rows_lds(long long M, int per_split) { return ((size_t)per_split * M * 129 + 15) & ~(size_t)15; }
void set_splits(Plan& p, long long s, int kblocks) {
    if (s < 1) s = 1;
    p.per_split = (int)yfs_cdiv(kblocks, s);
    p.splits = (int)yfs_cdiv(kblocks, p.per_split);
}
// Operands that are both in 8 bits.  The largest tile of which there are enough for the chip (measured on the sizes in
// brackets, us, against the next best):
//   256 x 256 from two thirds of a round of 256 on, where they are three quarters full (3000 x 4096 x 4096: 49 / 56; 2048 x 4096 x 4096,
//             half a round: 47 / 38), and where they fit one round and the next smaller do not (160 x 50176 x 4096: 61 / 87)
//   128 x 128 from three workgroups on two CUs on (300 x 16384 x 4096: 31 / 34; 1024 x 4096 x 8192, one per CU: 47 / 41); with fp32
//             sums, from seven on four (1470 x 4096 x 2009, three on two: 33 / 31)
//   64 x 128  from one per CU on (2048 x 2048 x 2048: 16 / 18; 64 x 50176 x 4096: 48 / 56)
// Fewer, and the reduction is split, 4 blocks or more each (more parts than these cost more in the join than they bring):
//   128 blocks or more: 128 x 128 with three stages, one per CU, up to 8 parts, where that leaves less than a quarter of the CUs
//             (128 x 4096 x 50176: 52 / 62; 2000 x 500 x 20000: 36 / 59; 100 x 300 x 50000, 79 parts: 20 / 16)
//   64 blocks or more: 64 x 128, two per CU, up to 8 parts (300 x 4096 x 16384: 37 / 57; 193 x 1678 x 10146, 9 parts: 25 / 21)
//   64 x 64 unsplit        where they are three quarters of one per CU (300 x 4096 x 4096: 17 / 21)
//   64 x 128, one per CU   (64 x 4096 x 50176: 44 / 47)
// `exact` (fp32 outputs): no 256 x 256 form; 8 waves on the 128 x 128 tile where the reduction is so short that the stores
// are what counts (4096 x 50176 x 64: 139 / 157; 4096 x 4096 x 4096: 126 / 116 the other way round).
Plan plan_tiles(long long M, long long N, int kblocks, bool exact) {
    Plan p = {1, 128, 128, 1, kblocks, 0};
    const long long mt = yfs_cdiv(M, 256), nt = yfs_cdiv(N, 256), t256 = mt * nt, t128 = yfs_cdiv(M, 128) * yfs_cdiv(N, 128);
    if (!exact && ((3 * t256 >= 2 * kCUs && 4 * M * N >= 3 * t256 * 65536) || (t256 <= kCUs && t128 > 2 * kCUs))) {
        p.kind = 2;
        p.bm = p.bn = 256;
        // A last round of fewer than half the CUs costs as much as a full one: its tile rows go to the small tiles instead.  One tile
        // row that is wider than the whole rounds stays in one piece (200 x 82944 x 4096: 131 / 163 by 128 x 128 tiles)
        const long long over = t256 % kCUs;
        const long long whole = t256 > kCUs && over > 0 && over <= kCUs / 2 && t256 - over >= nt ? (t256 - over) / nt : mt;
        p.body = whole * 256 < M ? whole * 256 : M;
        return p;
    }
    if (M > 64 && 4 * t128 >= (exact ? 7 : 6) * kCUs) return p;
    const long long deep = kCUs / t128;
    if (kblocks >= 128 && M > 64 && deep > 1 && deep <= 8 && 4 * deep * t128 > 3 * kCUs) {
        set_splits(p, deep < kblocks / 4 ? deep : kblocks / 4, kblocks);
        return p;
    }
    p.bm = 64;
    const long long wide = yfs_cdiv(M, 64) * yfs_cdiv(N, 128);
    long long s = kCUs / wide;
    if (kblocks >= 64 && M > 64 && wide > kCUs / 4) {
        p.two = true;
        s = 2 * kCUs / wide;
    } else if (wide >= kCUs) s = 1;
    else if (yfs_cdiv(M, 64) * yfs_cdiv(N, 64) >= kCUs - kCUs / 4) {
        p.bn = 64;
        return p;
    }
    if (s > kblocks / 4) s = kblocks / 4;
    set_splits(p, s, kblocks);
    return p;
}
// x in its own type: few enough rows are quantised by the workgroups that multiply them.
Plan plan_matmul(long long M, long long N, int kblocks, bool exact) {
    if (M <= kRows) {
        Plan p = {0, 16, 16, 1, kblocks, 0};
        const long long tiles = yfs_cdiv(N, 16);
        long long s = tiles >= kCUs ? 1 : kCUs / tiles;
        if (s > kblocks / 64) s = kblocks / 64;
        set_splits(p, s, kblocks);
        if (rows_lds(M, p.per_split) <= kRowsLds) return p;
    }
    return plan_tiles(M, N, kblocks, exact);
}
size_t part_bytes(const Plan& p, long long M, long long N) { return p.splits > 1 ? (size_t)p.splits * M * N * sizeof(float) : 0; }

template <typename TO>
int join(const GemmArgs& g, hipStream_t s) {
    if (g.splits > 1) {
        long long nb = yfs_cdiv(g.M * ((g.N + 3) / 4), 256);
        fp8_join_kernel<TO><<<dim3((unsigned)(nb < 4096 ? nb : 4096)), 256, 0, s>>>(g);
        YFS_CHECK_LAUNCH("fp8_join_kernel");
    }
    return YFS_OK;
}

template <int FM, int FN, int WM, int WN, int S, bool ROWB, bool EXACT, typename TO>
int launch_tiles(const GemmArgs& g, hipStream_t s) {
    constexpr int BM = WM * FM * 16, BN = WN * FN * 16, NW = WM * WN;
    constexpr int STAGE = (BM + BN) * 128 + NW * 256 * (ROWB ? 2 : 1);
    const dim3 grid((unsigned)yfs_cdiv(g.N, BN), (unsigned)yfs_cdiv(g.M, BM), (unsigned)g.splits);
    auto kern = fp8_gemm_kernel<FM, FN, WM, WN, S, ROWB, EXACT, TO>;
    // a short reduction leaves the rest of the ring to other workgroups
    constexpr int TILE_OUT = sizeof(TO) == 4 ? BM * (BN * 4 + 16) : 0, MOST = STAGE * S > TILE_OUT ? STAGE * S : TILE_OUT;
    const int ring = STAGE * (g.per_split < S ? g.per_split : S), lds = ring > TILE_OUT ? ring : TILE_OUT;
    const hipError_t e = hipFuncSetAttribute((const void*)kern, hipFuncAttributeMaxDynamicSharedMemorySize, MOST);
    YFS_REQUIRE(e == hipSuccess, YFS_ERR_LAUNCH, "fp8_gemm_kernel: cannot reserve %d bytes of LDS", MOST);
    kern<<<grid, 64 * NW, lds, s>>>(g);
    YFS_CHECK_LAUNCH("fp8_gemm_kernel");
    yfs_note_kernel("fp8_gemm_kernel<%d,%d,splits%d>", BM, BN, g.splits);
    return join<TO>(g, s);
}

template <typename TO>
int launch_gemm8(const GemmArgs& g, hipStream_t s) {
    auto kern = fp8_gemm8_kernel<TO>;
    const hipError_t e = hipFuncSetAttribute((const void*)kern, hipFuncAttributeMaxDynamicSharedMemorySize, G8_LDS);
    YFS_REQUIRE(e == hipSuccess, YFS_ERR_LAUNCH, "fp8_gemm8_kernel: cannot reserve %d bytes of LDS", G8_LDS);
    kern<<<dim3((unsigned)(yfs_cdiv(g.M, 256) * yfs_cdiv(g.N, 256))), 512, G8_LDS, s>>>(g);
    YFS_CHECK_LAUNCH("fp8_gemm8_kernel");
    return YFS_OK;
}

template <bool ROWB, bool EXACT, typename TO>
int gemm(GemmArgs g, hipStream_t s) {
    const Plan p = plan_tiles(g.M, g.N, g.kblocks, EXACT);
    g.splits = p.splits;
    g.per_split = p.per_split;
    g.groups_a = groups64(g.M);
    g.groups_b = groups64(g.N);
    if constexpr (!EXACT && !ROWB) {
        if (p.kind == 2) {
            // Whole rounds of 256 tiles by the large kernel; a few tile rows that would start another round by the small tiles
            const long long rest = g.M - p.body;
            if (rest > 0) {
                GemmArgs r = g;
                r.a += p.body * g.kblocks * 128;
                r.row0 = p.body;
                r.out = (TO*)g.out + p.body * g.N;
                r.M = rest;
                const bool wide = yfs_cdiv(rest, 64) * yfs_cdiv(g.N, 128) >= kCUs;
                const int rc = wide ? launch_tiles<4, 2, 1, 4, 2, ROWB, EXACT, TO>(r, s) : launch_tiles<2, 2, 2, 2, 3, ROWB, EXACT, TO>(r, s);
                if (rc != YFS_OK) return rc;
                g.M = p.body;
            }
            const int rc = launch_gemm8<TO>(g, s);
            if (rc == YFS_OK) yfs_note_kernel("fp8_gemm8_kernel<rest%lld>", rest);
            return rc;
        }
    }
    if (p.bm == 128) {
        if constexpr (EXACT) {
            if (g.kblocks <= 4) return launch_tiles<4, 2, 2, 4, 2, ROWB, EXACT, TO>(g, s);
        }
        if (p.splits > 1) return launch_tiles<4, 2, 2, 4, 3, ROWB, EXACT, TO>(g, s);
        return launch_tiles<4, 4, 2, 2, 2, ROWB, EXACT, TO>(g, s);
    }
    if (p.bn == 64) return launch_tiles<2, 2, 2, 2, 3, ROWB, EXACT, TO>(g, s);
    // (unsplit, four workgroups of two stages per CU; split to one per CU, three stages keep more on their way)
    if (p.splits == 1 || p.two) return launch_tiles<4, 2, 1, 4, 2, ROWB, EXACT, TO>(g, s);
    return launch_tiles<4, 2, 1, 4, 3, ROWB, EXACT, TO>(g, s);
}

template <typename T, typename TO>
int matmul_rows(GemmArgs g, const Plan& p, const void* x, long long ldx, long long K, hipStream_t s) {
    g.splits = p.splits;
    g.per_split = p.per_split;
    auto kern = fp8_rows_kernel<T, TO>;
    const hipError_t e = hipFuncSetAttribute((const void*)kern, hipFuncAttributeMaxDynamicSharedMemorySize, (int)kRowsLds);
    YFS_REQUIRE(e == hipSuccess, YFS_ERR_LAUNCH, "fp8_rows_kernel: cannot reserve %d bytes of LDS", (int)kRowsLds);
    const int waves = p.per_split >= 16 ? 16 : (p.per_split >= 8 ? 8 : 4);
    kern<<<dim3((unsigned)yfs_cdiv(g.N, 16), (unsigned)p.splits), 64 * waves, rows_lds(g.M, p.per_split), s>>>(g, (const T*)x, ldx, K);
    YFS_CHECK_LAUNCH("fp8_rows_kernel");
    yfs_note_kernel("fp8_rows_kernel<splits%d>", g.splits);
    return join<TO>(g, s);
}
template <typename T>
int matmul_rows(const GemmArgs& g, const Plan& p, const void* x, long long ldx, long long K, int out_dtype, hipStream_t s) {
    if (out_dtype == YFS_F32) return matmul_rows<T, float>(g, p, x, ldx, K, s);
    return out_dtype == YFS_BF16 ? matmul_rows<T, bf16_t>(g, p, x, ldx, K, s) : matmul_rows<T, _Float16>(g, p, x, ldx, K, s);
}

// Rows that fp8_train_rows_kernel takes, and its plan: two workgroups per CU, two blocks or more each
constexpr int kTrainRows = 64;
Plan plan_train_rows(long long N, int kblocks) {
    Plan p = {3, 64, 128, 1, kblocks, 0};
    long long s = 2 * kCUs / yfs_cdiv(N, 128);
    if (s > kblocks / 2) s = kblocks / 2;
    if (s > 128) s = 128;
    set_splits(p, s, kblocks);
    return p;
}
template <typename T>
int train_rows(GemmArgs g, const QuantArgs& w, int out_dtype, hipStream_t s) {
    const dim3 grid((unsigned)(yfs_cdiv(g.N, 128) * g.splits));
    if (out_dtype == YFS_F32) fp8_train_rows_kernel<T, float><<<grid, 256, 0, s>>>(g, w);
    else if (out_dtype == YFS_BF16) fp8_train_rows_kernel<T, bf16_t><<<grid, 256, 0, s>>>(g, w);
    else fp8_train_rows_kernel<T, _Float16><<<grid, 256, 0, s>>>(g, w);
    YFS_CHECK_LAUNCH("fp8_train_rows_kernel");
    yfs_note_kernel("fp8_train_rows_kernel<splits%d>", g.splits);
    if (out_dtype == YFS_F32) return join<float>(g, s);
    return out_dtype == YFS_BF16 ? join<bf16_t>(g, s) : join<_Float16>(g, s);
}

bool weight_once(const void* w, int dtype, long long ld, long long N, long long K) {
    const long long size = dtype == YFS_F32 ? 4 : 2;
    return past_caches((long long)(reinterpret_cast<uintptr_t>(w) & 127) + ld * size, N * K * size);
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
    const QuantArgs g = {w, ld, N, K, (unsigned char*)q, (unsigned char*)scale, (unsigned char*)qt, (unsigned char*)scale_t, nullptr, 0, 0, 0, weight_once(w, dtype, ld, N, K)};
    return qt ? quantize_blocks<true>(g, dtype, (hipStream_t)stream) : quantize_blocks<false>(g, dtype, (hipStream_t)stream);
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
    REQUIRE_ALIGNED("yfs_fp8_quantize_rows", scale);
    REQUIRE_ALIGNED("yfs_fp8_quantize_rows", scale_t);
    const QuantArgs g = {x, ld, M, K, (unsigned char*)q, (unsigned char*)scale, (unsigned char*)qt, (unsigned char*)scale_t, colsum,
                         groups64(M), groups64(K), 0, false};
    return quantize_rows(g, dtype, (hipStream_t)stream);
}

// (whatever the output's type: the larger of the two forms)
YFS_API size_t yfs_fp8_gemm_workspace_bytes(int64_t M, int64_t N, int64_t K) {
    if (M <= 0 || N <= 0 || K <= 0 || M > kMost || N > kMost || K > kMost) return 0;
    return part_bytes(plan_tiles(M, N, (int)yfs_cdiv(K, 128), true), M, N);
}

YFS_API int yfs_fp8_gemm_plan(int64_t M, int64_t N, int64_t K, int out_dtype, int64_t* plan) {
    YFS_REQUIRE(plan, YFS_ERR_INVALID_ARG, "yfs_fp8_gemm_plan: null pointer");
    REQUIRE_SIZES("yfs_fp8_gemm_plan", M, N, K);
    YFS_REQUIRE(known(out_dtype), YFS_ERR_UNSUPPORTED, "yfs_fp8_gemm_plan: unknown dtype %d", out_dtype);
    const Plan p = plan_tiles(M, N, (int)yfs_cdiv(K, 128), out_dtype == YFS_F32);
    const int64_t v[] = {p.bm, p.bn, p.splits, p.per_split, p.kind == 2 ? p.body : 0};
    for (int i = 0; i < YFS_FP8_PLAN_LEN; ++i) plan[i] = v[i];
    return YFS_OK;
}

YFS_API int yfs_fp8_gemm(const void* aq, const void* a_scale, const void* bq, const void* b_scale, int b_row_scales, const float* bias,
                         void* out, int out_dtype, int64_t M, int64_t N, int64_t K, float slope, int accumulate, void* workspace,
                         size_t workspace_bytes, void* stream) {
    YFS_REQUIRE(aq && a_scale && bq && b_scale && out, YFS_ERR_INVALID_ARG, "yfs_fp8_gemm: null pointer");
    REQUIRE_SIZES("yfs_fp8_gemm", M, N, K);
    YFS_REQUIRE(known(out_dtype), YFS_ERR_UNSUPPORTED, "yfs_fp8_gemm: unknown dtype %d", out_dtype);
    YFS_REQUIRE(!b_row_scales || out_dtype == YFS_F32, YFS_ERR_UNSUPPORTED, "yfs_fp8_gemm: row scales on both sides need an fp32 output");
    YFS_REQUIRE(!accumulate || (out_dtype == YFS_F32 && slope == 1.0f), YFS_ERR_UNSUPPORTED,
                "yfs_fp8_gemm: only an fp32 output without an activation accumulates");
    YFS_REQUIRE(slope >= 0.0f && slope <= 1.0f, YFS_ERR_INVALID_ARG, "yfs_fp8_gemm: slope %g not in [0, 1]", slope);
    REQUIRE_ALIGNED("yfs_fp8_gemm", aq);
    REQUIRE_ALIGNED("yfs_fp8_gemm", a_scale);
    REQUIRE_ALIGNED("yfs_fp8_gemm", bq);
    if (b_row_scales) REQUIRE_ALIGNED("yfs_fp8_gemm", b_scale);
    const size_t need = yfs_fp8_gemm_workspace_bytes(M, N, K);
    YFS_REQUIRE(need == 0 || (workspace && workspace_bytes >= need), YFS_ERR_WORKSPACE, "yfs_fp8_gemm: workspace needs %zu bytes", need);
    GemmArgs g = {(const unsigned char*)aq, (const unsigned char*)a_scale, (const unsigned char*)bq, (const unsigned char*)b_scale, bias, out,
                  (float*)workspace, M, N, (int)yfs_cdiv(K, 128), 1, 0, 0, 0, 0, slope, accumulate};
    hipStream_t s = (hipStream_t)stream;
    if (b_row_scales) return gemm<true, true, float>(g, s);
    if (out_dtype == YFS_F32) return gemm<false, true, float>(g, s);
    return out_dtype == YFS_BF16 ? gemm<false, false, bf16_t>(g, s) : gemm<false, false, _Float16>(g, s);
}

namespace {
struct MatmulSpace { size_t q, s, part; };
MatmulSpace matmul_space(long long M, long long N, long long K) {
    const int kb = (int)yfs_cdiv(K, 128);
    const Plan p = plan_matmul(M, N, kb, true);
    if (p.kind == 0) return {0, 0, part_bytes(p, M, N)};
    return {align256((size_t)(M * pad128(K))), align256((size_t)packed_bytes(M, kb)), part_bytes(p, M, N)};
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
    YFS_REQUIRE(known(x_dtype) && known(out_dtype), YFS_ERR_UNSUPPORTED, "yfs_fp8_matmul: unknown dtype %d or %d", x_dtype, out_dtype);
    YFS_REQUIRE(ld >= 0, YFS_ERR_INVALID_ARG, "yfs_fp8_matmul: negative row stride");
    YFS_REQUIRE(slope >= 0.0f && slope <= 1.0f, YFS_ERR_INVALID_ARG, "yfs_fp8_matmul: slope %g not in [0, 1]", slope);
    REQUIRE_ALIGNED("yfs_fp8_matmul", wq);
    const size_t need = yfs_fp8_matmul_workspace_bytes(M, N, K);
    YFS_REQUIRE(need == 0 || (workspace && workspace_bytes >= need && (reinterpret_cast<uintptr_t>(workspace) & 255) == 0),
                YFS_ERR_WORKSPACE, "yfs_fp8_matmul: workspace needs %zu bytes, 256-byte aligned", need);
    const Plan p = plan_matmul(M, N, (int)yfs_cdiv(K, 128), true);
    if (p.kind == 0) {
        const GemmArgs g = {nullptr, nullptr, (const unsigned char*)wq, (const unsigned char*)w_scale, bias, y, (float*)workspace,
                            M, N, (int)yfs_cdiv(K, 128), 1, 0, 0, 0, 0, slope, 0};
        hipStream_t s = (hipStream_t)stream;
        if (x_dtype == YFS_F32) return matmul_rows<float>(g, p, x, ld, K, out_dtype, s);
        if (x_dtype == YFS_BF16) return matmul_rows<bf16_t>(g, p, x, ld, K, out_dtype, s);
        return matmul_rows<_Float16>(g, p, x, ld, K, out_dtype, s);
    }
    const MatmulSpace w = matmul_space(M, N, K);
    unsigned char* q = (unsigned char*)workspace;
    const int rc = yfs_fp8_quantize_rows(x, x_dtype, ld, M, K, q, q + w.q, nullptr, nullptr, nullptr, stream);
    if (rc != YFS_OK) return rc;
    return yfs_fp8_gemm(q, q + w.q, wq, w_scale, 0, bias, y, out_dtype, M, N, K, slope, 0, q + w.q + w.s, workspace_bytes - w.q - w.s, stream);
}

YFS_API int yfs_fp8_colsum(const float* part, int64_t tiles, int64_t K, float* out, int accumulate, void* stream) {
    YFS_REQUIRE(part && out, YFS_ERR_INVALID_ARG, "yfs_fp8_colsum: null pointer");
    REQUIRE_SIZES("yfs_fp8_colsum", tiles, 1, K);
    colsum_kernel<<<dim3((unsigned)yfs_cdiv(K, 32)), tiles <= 64 ? 256 : 1024, 0, (hipStream_t)stream>>>(part, tiles, K, out, accumulate);
    YFS_CHECK_LAUNCH("colsum_kernel");
    return YFS_OK;
}

// ---- a linear layer's training step ----------------------------------------------------------------------------------
namespace {
// consecutive pieces of one buffer, each 256-byte aligned
struct Pieces {
    unsigned char* base;
    size_t used = 0;
    unsigned char* take(size_t bytes) {
        unsigned char* p = base + used;
        used += align256(bytes);
        return p;
    }
};
// What the backward pass multiplies: the weight's blocks transposed (for dx), x's columns in blocks of 128 rows (for dw).
struct Saved {
    unsigned char *wqt = nullptr, *wst = nullptr, *xqt = nullptr, *xst = nullptr;
    size_t bytes;
    Saved(void* buf, long long M, long long N, long long K, int needs) {
        Pieces p{(unsigned char*)buf};
        if (needs & YFS_NEED_DX) {
            wqt = p.take((size_t)(K * pad128(N)));
            wst = p.take((size_t)(yfs_cdiv(K, 128) * yfs_cdiv(N, 128)));
        }
        if (needs & YFS_NEED_DW) {
            xqt = p.take((size_t)(K * pad128(M)));
            xst = p.take((size_t)packed_bytes(K, yfs_cdiv(M, 128)));
        }
        bytes = p.used;
    }
};
struct ForwardSpace {
    unsigned char *wq = nullptr, *ws = nullptr, *xq, *xs, *part;
    size_t part_bytes, bytes;
    ForwardSpace(void* buf, long long M, long long N, long long K) {
        Pieces p{(unsigned char*)buf};
        const int kb = (int)yfs_cdiv(K, 128);
        if (M > kTrainRows) {
            wq = p.take((size_t)(N * pad128(K)));
            ws = p.take((size_t)(yfs_cdiv(N, 128) * kb));
        }
        xq = p.take((size_t)(M * pad128(K)));
        xs = p.take((size_t)packed_bytes(M, kb));
        part_bytes = M > kTrainRows ? yfs_fp8_gemm_workspace_bytes(M, N, K) : ::part_bytes(plan_train_rows(N, kb), M, N);
        part = p.take(part_bytes);
        bytes = p.used;
    }
};
struct BackwardSpace {
    unsigned char *dq = nullptr, *ds = nullptr, *dqt = nullptr, *dst = nullptr, *part;
    float* colsum = nullptr;
    size_t part_bytes = 0, bytes;
    BackwardSpace(void* buf, long long M, long long N, long long K, int needs) {
        Pieces p{(unsigned char*)buf};
        if (needs & YFS_NEED_DX) {
            dq = p.take((size_t)(M * pad128(N)));
            ds = p.take((size_t)packed_bytes(M, yfs_cdiv(N, 128)));
            part_bytes = yfs_fp8_gemm_workspace_bytes(M, K, N);
        }
        if (needs & YFS_NEED_DW) {
            dqt = p.take((size_t)(N * pad128(M)));
            dst = p.take((size_t)packed_bytes(N, yfs_cdiv(M, 128)));
            const size_t b = yfs_fp8_gemm_workspace_bytes(N, K, M);
            part_bytes = b > part_bytes ? b : part_bytes;
        }
        if (needs & YFS_NEED_DB) colsum = (float*)p.take((size_t)(yfs_cdiv(M, 128) * N * sizeof(float)));
        part = p.take(part_bytes);   // the two products use it one after the other
        bytes = p.used;
    }
};
bool sizes_ok(long long M, long long N, long long K) { return M > 0 && N > 0 && K > 0 && M <= kMost && N <= kMost && K <= kMost; }
bool aligned256(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 255) == 0; }
}  // namespace

YFS_API size_t yfs_fp8_linear_saved_bytes(int64_t M, int64_t N, int64_t K, int needs) {
    return sizes_ok(M, N, K) ? Saved(nullptr, M, N, K, needs).bytes : 0;
}
YFS_API size_t yfs_fp8_linear_fwd_workspace_bytes(int64_t M, int64_t N, int64_t K) {
    return sizes_ok(M, N, K) ? ForwardSpace(nullptr, M, N, K).bytes : 0;
}
YFS_API size_t yfs_fp8_linear_bwd_workspace_bytes(int64_t M, int64_t N, int64_t K, int needs) {
    return sizes_ok(M, N, K) ? BackwardSpace(nullptr, M, N, K, needs).bytes : 0;
}

YFS_API int yfs_fp8_linear_fwd(const void* x, int x_dtype, int64_t ldx, const void* w, int w_dtype, int64_t ldw, const float* bias, void* y,
                               int y_dtype, int64_t M, int64_t N, int64_t K, int needs, void* saved, size_t saved_bytes, void* workspace,
                               size_t workspace_bytes, void* stream) {
    YFS_REQUIRE(x && w && y, YFS_ERR_INVALID_ARG, "yfs_fp8_linear_fwd: null pointer");
    REQUIRE_SIZES("yfs_fp8_linear_fwd", M, N, K);
    const Saved k(saved, M, N, K, needs);
    const ForwardSpace f(workspace, M, N, K);
    YFS_REQUIRE(workspace && workspace_bytes >= f.bytes && aligned256(workspace), YFS_ERR_WORKSPACE,
                "yfs_fp8_linear_fwd: workspace needs %zu bytes, 256-byte aligned", f.bytes);
    YFS_REQUIRE(k.bytes == 0 || (saved && saved_bytes >= k.bytes && aligned256(saved)), YFS_ERR_WORKSPACE,
                "yfs_fp8_linear_fwd: saved needs %zu bytes, 256-byte aligned", k.bytes);
    YFS_REQUIRE(known(w_dtype) && known(y_dtype) && ldw >= 0, YFS_ERR_UNSUPPORTED, "yfs_fp8_linear_fwd: unknown dtype %d or %d, or a negative row stride",
                w_dtype, y_dtype);
    if (M <= kTrainRows) {
        const int rc = yfs_fp8_quantize_rows(x, x_dtype, ldx, M, K, f.xq, f.xs, k.xqt, k.xst, nullptr, stream);
        if (rc != YFS_OK) return rc;
        const Plan p = plan_train_rows(N, (int)yfs_cdiv(K, 128));
        const GemmArgs g = {f.xq, f.xs, nullptr, nullptr, bias, y, (float*)f.part, M, N, (int)yfs_cdiv(K, 128), p.splits, p.per_split,
                            groups64(M), 0, 0, 1.0f, 0};
        const QuantArgs q = {w, ldw, N, K, nullptr, nullptr, k.wqt, k.wst, nullptr, 0, 0, 0, weight_once(w, w_dtype, ldw, N, K)};
        hipStream_t s = (hipStream_t)stream;
        if (w_dtype == YFS_F32) return train_rows<float>(g, q, y_dtype, s);
        return w_dtype == YFS_BF16 ? train_rows<bf16_t>(g, q, y_dtype, s) : train_rows<_Float16>(g, q, y_dtype, s);
    }
    int rc = yfs_fp8_quantize_weight(w, w_dtype, ldw, N, K, f.wq, f.ws, k.wqt, k.wst, stream);
    if (rc == YFS_OK) rc = yfs_fp8_quantize_rows(x, x_dtype, ldx, M, K, f.xq, f.xs, k.xqt, k.xst, nullptr, stream);
    if (rc == YFS_OK)
        rc = yfs_fp8_gemm(f.xq, f.xs, f.wq, f.ws, 0, bias, y, y_dtype, M, N, K, 1.0f, 0, f.part, f.part_bytes, stream);
    return rc;
}

YFS_API int yfs_fp8_linear_bwd(const void* dy, int dy_dtype, int64_t lddy, void* dx, int dx_dtype, float* dw, int accumulate_w, float* db,
                               int accumulate_b, int64_t M, int64_t N, int64_t K, int needs, const void* saved, size_t saved_bytes,
                               void* workspace, size_t workspace_bytes, void* stream) {
    YFS_REQUIRE(dy && !dx == !(needs & YFS_NEED_DX) && !dw == !(needs & YFS_NEED_DW) && !db == !(needs & YFS_NEED_DB), YFS_ERR_INVALID_ARG,
                "yfs_fp8_linear_bwd: null pointer, or an output that `needs` does not ask for");
    YFS_REQUIRE(needs & (YFS_NEED_DX | YFS_NEED_DW), YFS_ERR_INVALID_ARG, "yfs_fp8_linear_bwd: neither dx nor dw is asked for");
    REQUIRE_SIZES("yfs_fp8_linear_bwd", M, N, K);
    const Saved k(const_cast<void*>(saved), M, N, K, needs);
    const BackwardSpace f(workspace, M, N, K, needs);
    YFS_REQUIRE(workspace && workspace_bytes >= f.bytes && aligned256(workspace), YFS_ERR_WORKSPACE,
                "yfs_fp8_linear_bwd: workspace needs %zu bytes, 256-byte aligned", f.bytes);
    YFS_REQUIRE(saved && saved_bytes >= k.bytes && aligned256(saved), YFS_ERR_WORKSPACE,
                "yfs_fp8_linear_bwd: saved needs %zu bytes, 256-byte aligned", k.bytes);
    const bool direct = db && M <= 128 && !accumulate_b;   // one tile of rows: its column sums are db
    int rc = yfs_fp8_quantize_rows(dy, dy_dtype, lddy, M, N, f.dq, f.ds, f.dqt, f.dst, direct ? db : f.colsum, stream);
    if (rc == YFS_OK && dx)
        rc = yfs_fp8_gemm(f.dq, f.ds, k.wqt, k.wst, 0, nullptr, dx, dx_dtype, M, K, N, 1.0f, 0, f.part, f.part_bytes, stream);
    if (rc == YFS_OK && dw)
        rc = yfs_fp8_gemm(f.dqt, f.dst, k.xqt, k.xst, 1, nullptr, dw, YFS_F32, N, K, M, 1.0f, accumulate_w, f.part, f.part_bytes, stream);
    if (rc == YFS_OK && db && !direct) rc = yfs_fp8_colsum(f.colsum, yfs_cdiv(M, 128), N, db, accumulate_b, stream);
    return rc;
}
