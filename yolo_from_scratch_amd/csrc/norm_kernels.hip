// Layer norm over the last axis, forward and backward.
//   mu = mean_c x,  v = mean_c (x - mu)^2,  r = 1 / sqrt(v + eps),  h = (x - mu) r,  y = h w + b
//   g = dy w,  dx = r (g - mean_c g - h mean_c (g h)),  dw = sum_rows dy h,  db = sum_rows dy
// Bound by HBM: forward x + y, backward x + dy + dx.  A row is held in registers between its statistics and its output, so
// it is read once; the variance is taken from the centred values (no cancellation), everything between the 16-bit ends is
// fp32 and each output is rounded once.
#include "yfs_common.h"
#include "yfs_vec.h"

namespace {
// Sum over the G threads that share a row: a power of two up to 64 lanes of a wave, or the whole workgroup.
// `red` holds two floats per wave; the caller alternates `slot` between consecutive sums so that one barrier a sum is enough.
template <bool BLOCK>
__device__ __forceinline__ float2 row_sum(float a, float b, int G, float2* red, int slot) {
    const int top = BLOCK ? 32 : G >> 1;
    for (int o = top; o > 0; o >>= 1) {
        a += __shfl_xor(a, o, 64);
        b += __shfl_xor(b, o, 64);
    }
    if (!BLOCK) return make_float2(a, b);
    const int nw = (int)(blockDim.x >> 6), wave = (int)(threadIdx.x >> 6);
    float2* r = red + slot * 16;
    if ((threadIdx.x & 63) == 0) r[wave] = make_float2(a, b);
    __syncthreads();
    a = b = 0.0f;
    for (int w = 0; w < nw; ++w) {   // the same order in every thread
        const float2 t = r[w];
        a += t.x;
        b += t.y;
    }
    return make_float2(a, b);
}

// One group of G threads per row (BLOCK: the workgroup), NV vectors of VE elements per thread.
template <typename T, int NV, bool BLOCK>
__global__ void __launch_bounds__(BLOCK ? 1024 : 256) ln_fwd_kernel(const T* __restrict__ x, long long xs, const float* __restrict__ w,
                                                                   const float* __restrict__ b, T* __restrict__ y,
                                                                   float* __restrict__ mean, float* __restrict__ rstd,
                                                                   long long rows, int cols, float eps, int lg) {
    constexpr int VE = 16 / sizeof(T);
    __shared__ float2 red[32];
    const int G = BLOCK ? (int)blockDim.x : 1 << lg;
    const int t = BLOCK ? (int)threadIdx.x : (int)threadIdx.x & (G - 1);
    const long long rpb = BLOCK ? 1 : 256 >> lg;
    const float inv = 1.0f / (float)cols;
    for (long long row = (long long)blockIdx.x * rpb + (BLOCK ? 0 : (int)threadIdx.x >> lg); row < rows; row += (long long)gridDim.x * rpb) {
        float v[NV][VE];
        float s = 0.0f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (i * G + t) * VE;
            load_vec(x + row * xs + c, cols - c, v[i]);
#pragma unroll
            for (int j = 0; j < VE; ++j) s += v[i][j];
        }
        const float mu = row_sum<BLOCK>(s, 0.0f, G, red, 0).x * inv;
        float q = 0.0f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int n = cols - (i * G + t) * VE;
#pragma unroll
            for (int j = 0; j < VE; ++j) {
                v[i][j] -= mu;
                q += j < n ? v[i][j] * v[i][j] : 0.0f;
            }
        }
        const float r = 1.0f / sqrtf(row_sum<BLOCK>(q, 0.0f, G, red, 1).x * inv + eps);
        if (t == 0) {
            if (mean) mean[row] = mu;
            if (rstd) rstd[row] = r;
        }
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (i * G + t) * VE;
            float wv[VE], bv[VE];
            load_vec_or(w, c, cols - c, wv, 1.0f);
            load_vec_or(b, c, cols - c, bv, 0.0f);
#pragma unroll
            for (int j = 0; j < VE; ++j) v[i][j] = v[i][j] * r * wv[j] + bv[j];
            store_vec(y + row * cols + c, cols - c, v[i]);
        }
    }
}

// Rows longer than a workgroup's registers: the row is read three times (the second and third time from L2).
template <typename T>
__global__ void __launch_bounds__(1024) ln_fwd_long_kernel(const T* __restrict__ x, long long xs, const float* __restrict__ w,
                                                          const float* __restrict__ b, T* __restrict__ y, float* __restrict__ mean,
                                                          float* __restrict__ rstd, long long rows, int cols, float eps) {
    constexpr int VE = 16 / sizeof(T);
    __shared__ float2 red[32];
    const float inv = 1.0f / (float)cols;
    for (long long row = blockIdx.x; row < rows; row += gridDim.x) {
        const T* xr = x + row * xs;
        float v[VE], s = 0.0f, q = 0.0f;
        for (long long c = (long long)threadIdx.x * VE; c < cols; c += 1024 * VE) {
            load_vec(xr + c, cols - c, v);
#pragma unroll
            for (int j = 0; j < VE; ++j) s += v[j];
        }
        const float mu = row_sum<true>(s, 0.0f, 1024, red, 0).x * inv;
        for (long long c = (long long)threadIdx.x * VE; c < cols; c += 1024 * VE) {
            load_vec(xr + c, cols - c, v);
#pragma unroll
            for (int j = 0; j < VE; ++j) q += j < cols - c ? (v[j] - mu) * (v[j] - mu) : 0.0f;
        }
        const float r = 1.0f / sqrtf(row_sum<true>(q, 0.0f, 1024, red, 1).x * inv + eps);
        if (threadIdx.x == 0) {
            if (mean) mean[row] = mu;
            if (rstd) rstd[row] = r;
        }
        for (long long c = (long long)threadIdx.x * VE; c < cols; c += 1024 * VE) {
            float wv[VE], bv[VE];
            load_vec(xr + c, cols - c, v);
            load_vec_or(w, c, cols - c, wv, 1.0f);
            load_vec_or(b, c, cols - c, bv, 0.0f);
#pragma unroll
            for (int j = 0; j < VE; ++j) v[j] = (v[j] - mu) * r * wv[j] + bv[j];
            store_vec(y + row * cols + c, cols - c, v);
        }
    }
}

struct BwdArgs {
    const void *dy, *x;
    long long dys, xs;
    const float *w, *mean, *rstd;
    void* dx;             // may be NULL
    float *dw, *db;       // results, or partial sums [parts][2][cols]
    long long rows;
    int cols, lg;
};

template <typename T, int NV, bool BLOCK>
__global__ void __launch_bounds__(BLOCK ? 1024 : 256) ln_dx_kernel(BwdArgs g) {
    constexpr int VE = 16 / sizeof(T);
    __shared__ float2 red[32];
    const int G = BLOCK ? (int)blockDim.x : 1 << g.lg;
    const int t = BLOCK ? (int)threadIdx.x : (int)threadIdx.x & (G - 1);
    const long long rpb = BLOCK ? 1 : 256 >> g.lg;
    const float inv = 1.0f / (float)g.cols;
    int slot = 0;
    for (long long row = (long long)blockIdx.x * rpb + (BLOCK ? 0 : (int)threadIdx.x >> g.lg); row < g.rows; row += (long long)gridDim.x * rpb) {
        const float mu = g.mean[row], r = g.rstd[row];
        float h[NV][VE], d[NV][VE], s1 = 0.0f, s2 = 0.0f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (i * G + t) * VE, n = g.cols - c;
            float wv[VE];
            load_vec((const T*)g.x + row * g.xs + c, n, h[i]);
            load_vec((const T*)g.dy + row * g.dys + c, n, d[i]);
            load_vec_or(g.w, c, n, wv, 1.0f);
#pragma unroll
            for (int j = 0; j < VE; ++j) {
                h[i][j] = j < n ? (h[i][j] - mu) * r : 0.0f;
                d[i][j] *= wv[j];
                s1 += d[i][j];
                s2 += d[i][j] * h[i][j];
            }
        }
        const float2 s = row_sum<BLOCK>(s1, s2, G, red, slot);
        slot ^= 1;
        const float m1 = s.x * inv, m2 = s.y * inv;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (i * G + t) * VE;
#pragma unroll
            for (int j = 0; j < VE; ++j) d[i][j] = r * (d[i][j] - m1 - h[i][j] * m2);
            store_vec((T*)g.dx + row * g.cols + c, g.cols - c, d[i]);
        }
    }
}

template <typename T>
__global__ void __launch_bounds__(1024) ln_dx_long_kernel(BwdArgs g) {
    constexpr int VE = 16 / sizeof(T);
    __shared__ float2 red[32];
    const float inv = 1.0f / (float)g.cols;
    int slot = 0;
    for (long long row = blockIdx.x; row < g.rows; row += gridDim.x) {
        const T *xr = (const T*)g.x + row * g.xs, *dr = (const T*)g.dy + row * g.dys;
        const float mu = g.mean[row], r = g.rstd[row];
        float h[VE], d[VE], wv[VE], s1 = 0.0f, s2 = 0.0f;
        for (long long c = (long long)threadIdx.x * VE; c < g.cols; c += 1024 * VE) {
            const long long n = g.cols - c;
            load_vec(xr + c, n, h);
            load_vec(dr + c, n, d);
            load_vec_or(g.w, c, n, wv, 1.0f);
#pragma unroll
            for (int j = 0; j < VE; ++j) {
                s1 += d[j] * wv[j];
                s2 += j < n ? d[j] * wv[j] * (h[j] - mu) * r : 0.0f;
            }
        }
        const float2 s = row_sum<true>(s1, s2, 1024, red, slot);
        slot ^= 1;
        const float m1 = s.x * inv, m2 = s.y * inv;
        for (long long c = (long long)threadIdx.x * VE; c < g.cols; c += 1024 * VE) {
            const long long n = g.cols - c;
            load_vec(xr + c, n, h);
            load_vec(dr + c, n, d);
            load_vec_or(g.w, c, n, wv, 1.0f);
#pragma unroll
            for (int j = 0; j < VE; ++j) d[j] = r * (d[j] * wv[j] - m1 - (h[j] - mu) * r * m2);
            store_vec((T*)g.dx + row * g.cols + c, n, d);
        }
    }
}

// dw, db of a strip of 32 * VE columns over the rows of one part: 32 column threads x 8 row slices, joined in slice order.
template <typename T>
__global__ void __launch_bounds__(256) ln_dwdb_kernel(BwdArgs g, long long rows_per_part) {
    constexpr int VE = 16 / sizeof(T);
    __shared__ float red[8][2][32 * VE + 4];
    const int ct = threadIdx.x & 31, rs = threadIdx.x >> 5;
    const long long c = ((long long)blockIdx.x * 32 + ct) * VE, n = g.cols - c;
    const long long lo = (long long)blockIdx.y * rows_per_part;
    const long long hi = lo + rows_per_part < g.rows ? lo + rows_per_part : g.rows;
    float aw[VE], ab[VE];
#pragma unroll
    for (int j = 0; j < VE; ++j) aw[j] = ab[j] = 0.0f;
    if (n > 0) {
        for (long long row = lo + rs; row < hi; row += 8) {
            const float mu = g.mean[row], r = g.rstd[row];
            float h[VE], d[VE];
            load_vec((const T*)g.x + row * g.xs + c, n, h);
            load_vec((const T*)g.dy + row * g.dys + c, n, d);
#pragma unroll
            for (int j = 0; j < VE; ++j) {
                aw[j] += j < n ? d[j] * ((h[j] - mu) * r) : 0.0f;
                ab[j] += d[j];
            }
        }
    }
#pragma unroll
    for (int j = 0; j < VE; ++j) {
        red[rs][0][ct * VE + j] = aw[j];
        red[rs][1][ct * VE + j] = ab[j];
    }
    __syncthreads();
    for (int k = threadIdx.x; k < 2 * 32 * VE; k += 256) {
        const int which = k / (32 * VE), cc = k % (32 * VE);
        const long long col = (long long)blockIdx.x * 32 * VE + cc;
        if (col >= g.cols) continue;
        float s = 0.0f;
#pragma unroll
        for (int q = 0; q < 8; ++q) s += red[q][which][cc];
        float* out = which ? g.db : g.dw;
        if (out) out[(long long)blockIdx.y * 2 * g.cols + col] = s;
    }
}

// dw, db from partial sums [parts][2][cols], in the order of the parts
__global__ void __launch_bounds__(256) ln_reduce_kernel(const float* __restrict__ part, int parts, int cols, float* __restrict__ dw,
                                                        float* __restrict__ db) {
    __shared__ float red[8][32];
    const int ct = threadIdx.x & 31, ps = threadIdx.x >> 5;
    const long long k = (long long)blockIdx.x * 32 + ct;   // column of [2][cols]
    float s = 0.0f;
    if (k < 2LL * cols)
        for (int p = ps; p < parts; p += 8) s += part[(long long)p * 2 * cols + k];
    red[ps][ct] = s;
    __syncthreads();
    if (ps == 0 && k < 2LL * cols) {
#pragma unroll
        for (int q = 1; q < 8; ++q) s += red[q][ct];
        float* out = k < cols ? dw : db;
        if (out) out[k < cols ? k : k - cols] = s;
    }
}

constexpr int kMaxParts = 256;
// Rows are summed by one workgroup per strip as long as they are few; the rest goes over up to kMaxParts parts.
int dwdb_parts(long long rows, int cols, int esize) {
    const long long strips = yfs_cdiv(cols, 32 * (16 / esize));
    long long parts = yfs_cdiv(2048, strips);
    const long long most = yfs_cdiv(rows, 64);
    if (parts > most) parts = most;
    if (parts > kMaxParts) parts = kMaxParts;
    return (int)(parts < 1 ? 1 : parts);
}

struct Shape { int nv, lg, threads; };   // threads > 256 or lg < 0: one workgroup per row; nv == 0: the long form
Shape ln_shape(int cols, int esize, int max_nv_block) {
    const long long vecs = yfs_cdiv(cols, 16 / esize);
    for (int lg = 3; lg <= 6; ++lg)
        if (vecs <= (1 << lg)) return {1, lg, 256};
    if (vecs <= 128) return {2, 6, 256};
    for (int th = 256; th <= 1024; th *= 2)
        if (vecs <= th) return {1, -1, th};
    for (int nv = 2; nv <= max_nv_block; nv *= 2)
        if (vecs <= 1024LL * nv) return {nv, -1, 1024};
    return {0, -1, 1024};
}
unsigned row_blocks(long long rows, const Shape& s) {
    const long long nb = s.lg >= 0 ? yfs_cdiv(rows, 256 >> s.lg) : rows;
    return (unsigned)(nb < 8192 ? nb : 8192);
}

template <typename T>
int fwd(const void* x, long long xs, const float* w, const float* b, void* y, float* mean, float* rstd, long long rows, int cols,
        float eps, hipStream_t s) {
    const Shape sh = ln_shape(cols, sizeof(T), sizeof(T) == 2 ? 4 : 8);
    const dim3 grid(row_blocks(rows, sh)), blk(sh.threads);
#define LN_FWD(NV, BLOCK) ln_fwd_kernel<T, NV, BLOCK><<<grid, blk, 0, s>>>((const T*)x, xs, w, b, (T*)y, mean, rstd, rows, cols, eps, sh.lg)
    if (sh.nv == 0)
        ln_fwd_long_kernel<T><<<grid, blk, 0, s>>>((const T*)x, xs, w, b, (T*)y, mean, rstd, rows, cols, eps);
    else if (sh.lg >= 0) {
        if (sh.nv == 1) LN_FWD(1, false); else LN_FWD(2, false);
    } else switch (sh.nv) {
        case 1: LN_FWD(1, true); break;
        case 2: LN_FWD(2, true); break;
        case 4: LN_FWD(4, true); break;
        default:
            if constexpr (sizeof(T) == 4) LN_FWD(8, true);
    }
#undef LN_FWD
    YFS_CHECK_LAUNCH("ln_fwd_kernel");
    return YFS_OK;
}

template <typename T>
int bwd(BwdArgs g, float* part, hipStream_t s) {
    if (g.dx) {
        const Shape sh = ln_shape(g.cols, sizeof(T), sizeof(T) == 2 ? 2 : 4);
        g.lg = sh.lg;
        const dim3 grid(row_blocks(g.rows, sh)), blk(sh.threads);
        if (sh.nv == 0) ln_dx_long_kernel<T><<<grid, blk, 0, s>>>(g);
        else if (sh.lg >= 0) {
            if (sh.nv == 1) ln_dx_kernel<T, 1, false><<<grid, blk, 0, s>>>(g);
            else ln_dx_kernel<T, 2, false><<<grid, blk, 0, s>>>(g);
        } else switch (sh.nv) {
            case 1: ln_dx_kernel<T, 1, true><<<grid, blk, 0, s>>>(g); break;
            case 2: ln_dx_kernel<T, 2, true><<<grid, blk, 0, s>>>(g); break;
            default:
                if constexpr (sizeof(T) == 4) ln_dx_kernel<T, 4, true><<<grid, blk, 0, s>>>(g);
        }
        YFS_CHECK_LAUNCH("ln_dx_kernel");
    }
    if (g.dw || g.db) {
        const int parts = dwdb_parts(g.rows, g.cols, sizeof(T));
        const long long per = yfs_cdiv(g.rows, parts);
        const dim3 grid((unsigned)yfs_cdiv(g.cols, 32 * (16 / sizeof(T))), (unsigned)parts);
        if (parts == 1) {
            ln_dwdb_kernel<T><<<grid, 256, 0, s>>>(g, per);
            YFS_CHECK_LAUNCH("ln_dwdb_kernel");
        } else {
            float *dw = g.dw, *db = g.db;
            g.dw = part;
            g.db = part + g.cols;
            ln_dwdb_kernel<T><<<grid, 256, 0, s>>>(g, per);
            YFS_CHECK_LAUNCH("ln_dwdb_kernel");
            ln_reduce_kernel<<<dim3((unsigned)yfs_cdiv(2LL * g.cols, 32)), 256, 0, s>>>(part, parts, g.cols, dw, db);
            YFS_CHECK_LAUNCH("ln_reduce_kernel");
        }
    }
    return YFS_OK;
}

bool known(int dtype) { return dtype == YFS_F32 || dtype == YFS_BF16 || dtype == YFS_F16; }
}  // namespace

YFS_API int yfs_layer_norm_fwd(const void* x, int64_t x_stride, const float* w, const float* b, void* y, float* mean, float* rstd,
                               int64_t rows, int64_t cols, float eps, int dtype, void* stream) {
    YFS_REQUIRE(x && y, YFS_ERR_INVALID_ARG, "yfs_layer_norm_fwd: null pointer");
    YFS_REQUIRE(rows > 0 && cols > 0 && cols < (1LL << 30) && x_stride >= 0, YFS_ERR_INVALID_ARG,
                "yfs_layer_norm_fwd: need rows > 0, 0 < cols < 2^30 and a row stride >= 0 (got rows=%lld cols=%lld stride=%lld)",
                (long long)rows, (long long)cols, (long long)x_stride);
    YFS_REQUIRE(eps >= 0.0f, YFS_ERR_INVALID_ARG, "yfs_layer_norm_fwd: eps %g is negative", eps);
    YFS_REQUIRE(known(dtype), YFS_ERR_UNSUPPORTED, "yfs_layer_norm_fwd: unknown dtype %d", dtype);
    hipStream_t s = (hipStream_t)stream;
    if (dtype == YFS_F32) return fwd<float>(x, x_stride, w, b, y, mean, rstd, rows, (int)cols, eps, s);
    if (dtype == YFS_BF16) return fwd<__bf16>(x, x_stride, w, b, y, mean, rstd, rows, (int)cols, eps, s);
    return fwd<_Float16>(x, x_stride, w, b, y, mean, rstd, rows, (int)cols, eps, s);
}

YFS_API size_t yfs_layer_norm_bwd_workspace_bytes(int64_t rows, int64_t cols, int dtype) {
    if (rows <= 0 || cols <= 0 || cols >= (1LL << 30) || !known(dtype)) return 0;
    const int parts = dwdb_parts(rows, (int)cols, dtype == YFS_F32 ? 4 : 2);
    return parts == 1 ? 0 : (size_t)parts * 2 * (size_t)cols * sizeof(float);
}

YFS_API int yfs_layer_norm_bwd(const void* dy, int64_t dy_stride, const void* x, int64_t x_stride, const float* w, const float* mean,
                               const float* rstd, void* dx, float* dw, float* db, int64_t rows, int64_t cols, int dtype,
                               void* workspace, size_t workspace_bytes, void* stream) {
    YFS_REQUIRE(dy && x && mean && rstd, YFS_ERR_INVALID_ARG, "yfs_layer_norm_bwd: null pointer");
    YFS_REQUIRE(rows > 0 && cols > 0 && cols < (1LL << 30) && x_stride >= 0 && dy_stride >= 0, YFS_ERR_INVALID_ARG,
                "yfs_layer_norm_bwd: need rows > 0, 0 < cols < 2^30 and row strides >= 0 (got rows=%lld cols=%lld)", (long long)rows,
                (long long)cols);
    YFS_REQUIRE(known(dtype), YFS_ERR_UNSUPPORTED, "yfs_layer_norm_bwd: unknown dtype %d", dtype);
    const size_t need = (dw || db) ? yfs_layer_norm_bwd_workspace_bytes(rows, cols, dtype) : 0;
    YFS_REQUIRE(need == 0 || (workspace && workspace_bytes >= need), YFS_ERR_WORKSPACE,
                "yfs_layer_norm_bwd: workspace needs %zu bytes", need);
    const BwdArgs g = {dy, x, dy_stride, x_stride, w, mean, rstd, dx, dw, db, rows, (int)cols, 0};
    hipStream_t s = (hipStream_t)stream;
    if (dtype == YFS_F32) return bwd<float>(g, (float*)workspace, s);
    if (dtype == YFS_BF16) return bwd<__bf16>(g, (float*)workspace, s);
    return bwd<_Float16>(g, (float*)workspace, s);
}
