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

// One group of G threads per row (BLOCK: the workgroup), NV vectors of VE elements per thread.  ODD: the width is no multiple of
// VE, and the row's last vector is cut off.  The workgroups stay, 16 waves a CU, with weight and bias in their registers (12544 x
// 4096 bf16: 36 us, 5.7 TB/s; one workgroup per row 43; reading weight and bias again for every row 44).
template <typename T, int NV, bool BLOCK, bool ODD>
__global__ void __launch_bounds__(BLOCK ? 512 : 256) ln_fwd_kernel(const T* __restrict__ x, long long xs, const float* __restrict__ w,
                                                                   const float* __restrict__ b, T* __restrict__ y,
                                                                   float* __restrict__ mean, float* __restrict__ rstd,
                                                                   long long rows, int cols, float eps, int lg) {
    constexpr int VE = 16 / sizeof(T);
    __shared__ float2 red[32];
    const int G = BLOCK ? (int)blockDim.x : 1 << lg;
    const int t = BLOCK ? (int)threadIdx.x : (int)threadIdx.x & (G - 1);
    const long long rpb = BLOCK ? 1 : 256 >> lg;
    const long long first = (long long)blockIdx.x * rpb + (BLOCK ? 0 : (int)threadIdx.x >> lg), stride = (long long)gridDim.x * rpb;
    bool whole[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) whole[i] = ODD && __all((i * G + t + 1) * VE <= cols);
    const float inv = 1.0f / (float)cols;
    // weight and bias stay in registers where there is room for them
    constexpr bool KEEP = NV <= 3;
    float wv[KEEP ? NV : 1][VE], bv[KEEP ? NV : 1][VE];
    auto params = [&](int i, float (&pw)[VE], float (&pb)[VE]) {
        const int c = (i * G + t) * VE;
        load_vec_or(w, c, cols, pw, 1.0f);
        load_vec_or(b, c, cols, pb, 0.0f);
    };
    if constexpr (KEEP) {
#pragma unroll
        for (int i = 0; i < NV; ++i) params(i, wv[i], bv[i]);
    }
    T ahead[NV][VE];
    auto fetch = [&](long long row) {   // the next row is on its way while one is reduced
#pragma unroll
        for (int i = 0; i < NV; ++i) load_row<ODD>(x + row * xs, (i * G + t) * VE, cols, whole[i], ahead[i]);
    };
    if (first < rows) fetch(first);
    for (long long row = first; row < rows; row += stride) {
        float v[NV][VE];
        float s = 0.0f;
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int j = 0; j < VE; ++j) {
                v[i][j] = (float)ahead[i][j];
                s += v[i][j];
            }
        if (row + stride < rows) fetch(row + stride);
        const float mu = row_sum<BLOCK>(s, 0.0f, G, red, 0).x * inv;
        float q = 0.0f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (i * G + t) * VE;
            if (!(ODD && whole[i])) {   // (what lies behind the row counts as its mean)
#pragma unroll
                for (int j = 0; j < VE; ++j) v[i][j] = (ODD ? c + j < cols : c < cols) ? v[i][j] : mu;
            }
#pragma unroll
            for (int j = 0; j < VE; ++j) {
                v[i][j] -= mu;
                q += v[i][j] * v[i][j];
            }
        }
        const float r = 1.0f / sqrtf(row_sum<BLOCK>(q, 0.0f, G, red, 1).x * inv + eps);
        if (t == 0) {
            if (mean) mean[row] = mu;
            if (rstd) rstd[row] = r;
        }
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int k = KEEP ? i : 0;
            if constexpr (!KEEP) params(i, wv[0], bv[0]);
#pragma unroll
            for (int j = 0; j < VE; ++j) v[i][j] = v[i][j] * r * wv[k][j] + bv[k][j];
            store_row<ODD>(y + row * cols, (i * G + t) * VE, cols, whole[i], v[i]);
        }
    }
}

// Weights of a thread's vectors, the next one's on their way while one is used: all at once would take the registers of the row itself
template <int VE>
struct Ahead {
    const float* p;
    int cols;
    float none, v[2][VE];
    __device__ __forceinline__ void fetch(int i, int at, int c) { load_vec_or(p ? p + at : p, c, cols - at, v[i & 1], none); }
};
__device__ __forceinline__ void no_loads_earlier() { asm volatile("" ::: "memory"); }

// Rows of more than 2048 vectors, up to 8192: one workgroup of up to 16 waves per row, NV vectors per thread, kept in their own type
// between the passes (an fp32 copy would be twice the registers of a 16-bit row and leave one workgroup per CU); weight and bias come
// from L2.
template <typename T, int NV, bool ODD>
__global__ void __launch_bounds__(1024) ln_fwd_wide_kernel(const T* __restrict__ x, long long xs, const float* __restrict__ w,
                                                           const float* __restrict__ b, T* __restrict__ y, float* __restrict__ mean,
                                                           float* __restrict__ rstd, long long rows, int cols, float eps) {
    constexpr int VE = 16 / sizeof(T);
    __shared__ float2 red[32];
    const int G = (int)blockDim.x, step = G * VE, c = (int)threadIdx.x * VE;   // vector i of the thread: i * step + c
    bool whole[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) whole[i] = ODD && __all(i * step + c + VE <= cols);
    const float inv = 1.0f / (float)cols;
    for (long long row = blockIdx.x; row < rows; row += gridDim.x) {
        yfs_int4 raw[NV];
#pragma unroll
        for (int i = 0; i < NV; ++i) raw[i] = load_raw<ODD>(x + row * xs + i * step, c, cols - i * step, whole[i]);
        float s = 0.0f, q = 0.0f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            float v[VE];
            widen_raw<T>(raw[i], v);
#pragma unroll
            for (int j = 0; j < VE; ++j) s += v[j];
        }
        const float mu = row_sum<true>(s, 0.0f, G, red, 0).x * inv;
        fence(raw);
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            float v[VE];
            widen_raw<T>(raw[i], v);
#pragma unroll
            for (int j = 0; j < VE; ++j) {
                const float d = v[j] - mu;
                q += (ODD ? whole[i] || c + j < cols - i * step : c < cols - i * step) ? d * d : 0.0f;
            }
        }
        const float r = 1.0f / sqrtf(row_sum<true>(q, 0.0f, G, red, 1).x * inv + eps);
        fence(raw);
        if (c == 0) {
            if (mean) mean[row] = mu;
            if (rstd) rstd[row] = r;
        }
        Ahead<VE> pw = {w, cols, 1.0f}, pb = {b, cols, 0.0f};
        pw.fetch(0, 0, c);
        pb.fetch(0, 0, c);
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            if (i + 1 < NV) {
                pw.fetch(i + 1, (i + 1) * step, c);
                pb.fetch(i + 1, (i + 1) * step, c);
                no_loads_earlier();
            }
            float v[VE];
            widen_raw<T>(raw[i], v);
#pragma unroll
            for (int j = 0; j < VE; ++j) v[j] = (v[j] - mu) * r * pw.v[i & 1][j] + pb.v[i & 1][j];
            store_row<ODD>(y + row * cols + i * step, c, cols - i * step, whole[i], v);
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
            load_vec_or(w, c, cols, wv, 1.0f);
            load_vec_or(b, c, cols, bv, 0.0f);
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
    int dx_blocks;        // workgroups before this index do dx, the others column sums
    int strips;           // of 32 vectors of columns
    long long part_rows;  // rows per partial sum
};

// dw, db of a strip of 32 * VE columns over the rows of one part: 32 column threads x (blockDim / 32) row slices, joined in
// slice order.
template <typename T>
__device__ __forceinline__ void column_sums(const BwdArgs& g, int block, float* red) {
    constexpr int VE = 16 / sizeof(T);
    const int ct = threadIdx.x & 31, rs = threadIdx.x >> 5, slices = (int)blockDim.x >> 5, wave = threadIdx.x >> 6;
    const int part = block / g.strips, strip = block - part * g.strips;
    const long long c = ((long long)strip * 32 + ct) * VE, n = g.cols - c;
    const long long lo = part * g.part_rows, hi = lo + g.part_rows < g.rows ? lo + g.part_rows : g.rows;
    float aw[VE], ab[VE];
#pragma unroll
    for (int j = 0; j < VE; ++j) aw[j] = ab[j] = 0.0f;
    if (n > 0) {
#pragma unroll 4
        for (long long row = lo + rs; row < hi; row += slices) {
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
        aw[j] += __shfl_xor(aw[j], 32, 64);
        ab[j] += __shfl_xor(ab[j], 32, 64);
        if ((threadIdx.x & 32) == 0) {
            red[(wave * 2 + 0) * 32 * VE + ct * VE + j] = aw[j];
            red[(wave * 2 + 1) * 32 * VE + ct * VE + j] = ab[j];
        }
    }
    __syncthreads();
    for (int k = threadIdx.x; k < 2 * 32 * VE; k += blockDim.x) {
        const int which = k / (32 * VE), cc = k % (32 * VE);
        const long long col = (long long)strip * 32 * VE + cc;
        if (col >= g.cols) continue;
        float s = 0.0f;
        for (int q = 0; q < slices / 2; ++q) s += red[(q * 2 + which) * 32 * VE + cc];
        float* out = which ? g.db : g.dw;
        if (out) out[(long long)part * 2 * g.cols + col] = s;
    }
}

// dx by rows as in the forward pass.  ACC: the thread that holds a column of dx sums its dw and db too, over the rows that its
// workgroup meets: x and dy are read once for all three (200704 x 256 bf16: 60 us, 5.1 TB/s; 53 + 114 as two kernels).  That needs
// many rows per workgroup, or the partial sums outgrow them; for few rows the column sums are other workgroups of the same launch.
// Four waves a SIMD at least, as the plan counts on: odd bf16 rows took 130 registers and then 188 us where 50000 x 1470 takes 130.
template <typename T, int NV, bool BLOCK, bool ACC, bool ODD>
__global__ void __launch_bounds__(BLOCK ? 512 : 256, 4) ln_bwd_kernel(BwdArgs g) {
    constexpr int VE = 16 / sizeof(T);
    __shared__ float2 red[32];
    extern __shared__ float sums[];
    if (!ACC && (int)blockIdx.x >= g.dx_blocks) {
        column_sums<T>(g, (int)blockIdx.x - g.dx_blocks, sums);
        return;
    }
    const int G = BLOCK ? (int)blockDim.x : 1 << g.lg;
    const int t = BLOCK ? (int)threadIdx.x : (int)threadIdx.x & (G - 1);
    const long long rpb = BLOCK ? 1 : 256 >> g.lg;
    const long long first = (long long)blockIdx.x * rpb + (BLOCK ? 0 : (int)threadIdx.x >> g.lg), stride = (long long)g.dx_blocks * rpb;
    bool whole[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) whole[i] = ODD && __all((i * G + t + 1) * VE <= g.cols);
    const float inv = 1.0f / (float)g.cols;
    float wv[NV][VE], aw[ACC ? NV : 1][VE], ab[ACC ? NV : 1][VE];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        load_vec_or(g.w, (i * G + t) * VE, g.cols, wv[i], 1.0f);
        if (ACC) {
#pragma unroll
            for (int j = 0; j < VE; ++j) aw[i][j] = ab[i][j] = 0.0f;
        }
    }
    int slot = 0;
    for (long long row = first; row < g.rows; row += stride) {   // (with the next row ahead, as in the forward pass, 200704 x 256 bf16 takes 75 us for 60)
        const float mu = g.mean[row], r = g.rstd[row];
        float h[NV][VE], d[NV][VE], s1 = 0.0f, s2 = 0.0f;
        T xr[NV][VE], dr[NV][VE];
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            load_row<ODD>((const T*)g.x + row * g.xs, (i * G + t) * VE, g.cols, whole[i], xr[i]);
            load_row<ODD>((const T*)g.dy + row * g.dys, (i * G + t) * VE, g.cols, whole[i], dr[i]);
        }
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (i * G + t) * VE;
#pragma unroll
            for (int j = 0; j < VE; ++j) h[i][j] = ((float)xr[i][j] - mu) * r;
            if (!(ODD && whole[i])) {
#pragma unroll
                for (int j = 0; j < VE; ++j) h[i][j] = (ODD ? c + j < g.cols : c < g.cols) ? h[i][j] : 0.0f;
            }
#pragma unroll
            for (int j = 0; j < VE; ++j) {
                d[i][j] = (float)dr[i][j];
                if (ACC) {
                    aw[i][j] += d[i][j] * h[i][j];
                    ab[i][j] += d[i][j];
                }
                d[i][j] *= wv[i][j];
                s1 += d[i][j];
                s2 += d[i][j] * h[i][j];
            }
        }
        const float2 s = row_sum<BLOCK>(s1, s2, G, red, slot);
        slot ^= 1;
        const float m1 = s.x * inv, m2 = s.y * inv;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
#pragma unroll
            for (int j = 0; j < VE; ++j) d[i][j] = r * (d[i][j] - m1 - h[i][j] * m2);
            store_row<ODD>((T*)g.dx + row * g.cols, (i * G + t) * VE, g.cols, whole[i], d[i]);
        }
    }
    if constexpr (ACC && BLOCK) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (i * G + t) * VE;
            store_vec(g.dw + (long long)blockIdx.x * 2 * g.cols + c, g.cols - c, aw[i]);
            store_vec(g.db + (long long)blockIdx.x * 2 * g.cols + c, g.cols - c, ab[i]);
        }
    } else if constexpr (ACC) {
        const int grp = (int)threadIdx.x >> g.lg, groups = 256 >> g.lg;
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int j = 0; j < VE; ++j) {
                const int c = (i * G + t) * VE + j;
                if (c < g.cols) {
                    sums[(grp * 2 + 0) * g.cols + c] = aw[i][j];
                    sums[(grp * 2 + 1) * g.cols + c] = ab[i][j];
                }
            }
        __syncthreads();
        for (int k = threadIdx.x; k < 2 * g.cols; k += 256) {
            float v = 0.0f;
            for (int q = 0; q < groups; ++q) v += sums[q * 2 * g.cols + k];
            g.dw[(long long)blockIdx.x * 2 * g.cols + k] = v;   // (db lies cols behind dw)
        }
    }
}

// Rows of more than 1024 vectors, up to 4096 (eight of x and of dy per thread do not fit).  ACC: with the sums of dw and db, in workgroups
// of up to 512 (2000 x 16384 bf16: 56 us, with column sums by other workgroups 80).  fp32 rows fit five waves a SIMD: 2500 x 9000
// 84 us against 131 with four.
template <typename T, int NV, bool ACC, bool ODD>
__global__ void __launch_bounds__(ACC ? 512 : 1024, ACC ? 1 : (sizeof(T) == 4 ? 5 : 4)) ln_bwd_wide_kernel(BwdArgs g) {
    constexpr int VE = 16 / sizeof(T);
    __shared__ float2 red[32];
    extern __shared__ float sums[];
    if (!ACC && (int)blockIdx.x >= g.dx_blocks) {
        column_sums<T>(g, (int)blockIdx.x - g.dx_blocks, sums);
        return;
    }
    const int G = (int)blockDim.x, step = G * VE, c = (int)threadIdx.x * VE;
    bool whole[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) whole[i] = ODD && __all(i * step + c + VE <= g.cols);
    const float inv = 1.0f / (float)g.cols;
    float aw[ACC ? NV : 1][VE], ab[ACC ? NV : 1][VE];
    if (ACC) {
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int j = 0; j < VE; ++j) aw[i][j] = ab[i][j] = 0.0f;
    }
    int slot = 0;
    for (long long row = blockIdx.x; row < g.rows; row += g.dx_blocks) {
        const float mu = g.mean[row], r = g.rstd[row];
        yfs_int4 xr[NV], dr[NV];
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            xr[i] = load_raw<ODD>((const T*)g.x + row * g.xs + i * step, c, g.cols - i * step, whole[i]);
            dr[i] = load_raw<ODD>((const T*)g.dy + row * g.dys + i * step, c, g.cols - i * step, whole[i]);
        }
        float s1 = 0.0f, s2 = 0.0f;
        Ahead<VE> pw = {g.w, g.cols, 1.0f};
        pw.fetch(0, 0, c);
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            if (i + 1 < NV) {
                pw.fetch(i + 1, (i + 1) * step, c);
                no_loads_earlier();
            }
            const float (&wv)[VE] = pw.v[i & 1];
            float xv[VE], dv[VE];
            widen_raw<T>(xr[i], xv);
            widen_raw<T>(dr[i], dv);
#pragma unroll
            for (int j = 0; j < VE; ++j) {   // (dy is 0 behind the row)
                const float h = (ODD ? whole[i] || c + j < g.cols - i * step : c < g.cols - i * step) ? (xv[j] - mu) * r : 0.0f, d = dv[j];
                if (ACC) {
                    aw[i][j] += d * h;
                    ab[i][j] += d;
                }
                s1 += d * wv[j];
                s2 += d * wv[j] * h;
            }
        }
        const float2 s = row_sum<true>(s1, s2, G, red, slot);
        slot ^= 1;
        const float m1 = s.x * inv, m2 = s.y * inv;
        fence(xr);
        fence(dr);
        pw.fetch(0, 0, c);
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            if (i + 1 < NV) {
                pw.fetch(i + 1, (i + 1) * step, c);
                no_loads_earlier();
            }
            const float (&wv)[VE] = pw.v[i & 1];
            float xv[VE], dv[VE];
            widen_raw<T>(xr[i], xv);
            widen_raw<T>(dr[i], dv);
#pragma unroll
            for (int j = 0; j < VE; ++j) dv[j] = r * (dv[j] * wv[j] - m1 - (xv[j] - mu) * r * m2);
            store_row<ODD>((T*)g.dx + row * g.cols + i * step, c, g.cols - i * step, whole[i], dv);
        }
    }
    if constexpr (ACC) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            store_vec(g.dw + (long long)blockIdx.x * 2 * g.cols + i * step + c, g.cols - i * step - c, aw[i]);
            store_vec(g.db + (long long)blockIdx.x * 2 * g.cols + i * step + c, g.cols - i * step - c, ab[i]);
        }
    }
}

template <typename T>
__global__ void __launch_bounds__(1024) ln_bwd_long_kernel(BwdArgs g) {
    constexpr int VE = 16 / sizeof(T);
    __shared__ float2 red[32];
    extern __shared__ float sums[];
    if ((int)blockIdx.x >= g.dx_blocks) {
        column_sums<T>(g, (int)blockIdx.x - g.dx_blocks, sums);
        return;
    }
    const float inv = 1.0f / (float)g.cols;
    int slot = 0;
    for (long long row = blockIdx.x; row < g.rows; row += g.dx_blocks) {
        const T *xr = (const T*)g.x + row * g.xs, *dr = (const T*)g.dy + row * g.dys;
        const float mu = g.mean[row], r = g.rstd[row];
        float h[VE], d[VE], wv[VE], s1 = 0.0f, s2 = 0.0f;
        for (long long c = (long long)threadIdx.x * VE; c < g.cols; c += 1024 * VE) {
            const long long n = g.cols - c;
            load_vec(xr + c, n, h);
            load_vec(dr + c, n, d);
            load_vec_or(g.w, c, g.cols, wv, 1.0f);
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
            load_vec_or(g.w, c, g.cols, wv, 1.0f);
#pragma unroll
            for (int j = 0; j < VE; ++j) d[j] = r * (d[j] * wv[j] - m1 - (h[j] - mu) * r * m2);
            store_vec((T*)g.dx + row * g.cols + c, n, d);
        }
    }
}

// dw, db from partial sums [parts][2][cols]: 32 columns x 32 slices of the parts, joined in slice order
__global__ void __launch_bounds__(1024) ln_reduce_kernel(const float* __restrict__ part, int parts, int cols, float* __restrict__ dw,
                                                         float* __restrict__ db) {
    __shared__ float red[32][33];
    const int ct = threadIdx.x & 31, ps = threadIdx.x >> 5;
    const long long k = (long long)blockIdx.x * 32 + ct;   // column of [2][cols]
    float s = 0.0f;
    if (k < 2LL * cols) {
#pragma unroll 8
        for (int p = ps; p < parts; p += 32) s += part[(long long)p * 2 * cols + k];
    }
    red[ps][ct] = s;
    __syncthreads();
    if (ps == 0 && k < 2LL * cols) {
#pragma unroll
        for (int q = 1; q < 32; ++q) s += red[q][ct];
        float* out = k < cols ? dw : db;
        if (out) out[k < cols ? k : k - cols] = s;
    }
}

constexpr int kCUs = 256;
// lg >= 0: groups of 2^lg lanes; lg < 0: one workgroup per row; nv == 0: the long form
struct Shape { int nv, lg, threads; bool wide = false; };
// A wave per row up to `wave_most` vectors a lane (three, with dw and db summed, are 186 registers: 1470 bf16 columns 160 us against
// 126 in workgroups of 128, 50000 rows backward; without sums three fit: 74 against 85 forward).  Longer rows have two vectors per
// thread (4096 bf16 columns: 43 us against 49 with one, 12544 rows forward), `block_most` in a workgroup of 512, and the wide kernels'
// four or eight (`wide_most`) in one of up to 1024 (forward, with four: 3000 x 12000 bf16 45 us against 52 in the wide form, which takes
// 2500 x 20000 in 76 us where three readings of the row take 135; backward, 104 in the wide form against 139).
Shape ln_shape(int cols, int esize, int wave_most, int block_most, int wide_most) {
    const long long vecs = yfs_cdiv(cols, 16 / esize);
    for (int lg = 3; lg <= 6; ++lg)
        if (vecs <= (1 << lg)) return {1, lg, 256};
    for (int nv = 2; nv <= wave_most; ++nv)
        if (vecs <= 64 * nv) return {nv, 6, 256};
    for (int nv = 2; nv <= block_most; nv *= 2)
        if (vecs <= 512 * nv) return {nv, -1, (int)(yfs_cdiv(vecs, 64 * nv) * 64)};
    for (int nv = 4; nv <= wide_most; nv *= 2)
        if (vecs <= 1024 * nv) return {nv, -1, (int)(yfs_cdiv(vecs, 64 * nv) * 64), true};
    return {0, -1, 1024};
}
// Workgroups that take the rows in turn: 32 waves a CU where a wave has a row, 16 where a workgroup has one
unsigned row_blocks(long long rows, const Shape& s) {
    const long long nb = s.lg >= 0 ? yfs_cdiv(rows, 256 >> s.lg) : rows, most = kCUs * (s.lg >= 0 ? 32 : 16) * 64 / s.threads;
    return (unsigned)(nb < most ? nb : most);
}

// How the backward pass goes over the chip.  acc: dx and the column sums by the same workgroups, one partial sum each; else
// column sums by workgroups of their own, over `parts` parts of the rows.
struct BwdPlan { Shape sh; bool acc; int dx_blocks, strips, parts; long long part_rows; };
BwdPlan bwd_plan(long long rows, int cols, int esize, bool need_dx) {
    BwdPlan p;
    p.sh = ln_shape(cols, esize, 2, 2, 4);
    p.strips = (int)yfs_cdiv(cols, 32 * (16 / esize));
    const long long rpb = p.sh.lg >= 0 ? 256 >> p.sh.lg : 1;
    // a partial sum is 8 bytes a column, written and read, a row of x, dy and dx 6 or 12: from 4 rows a workgroup on it is less than
    // reading x and dy again
    const long long nb = rows / (rpb * 4), vecs = yfs_cdiv(cols, 16 / esize);
    p.acc = need_dx && vecs <= 2048 && nb >= kCUs;
    const long long fill = kCUs * (p.sh.wide ? 8 : 16) * 64 / p.sh.threads;   // 16 waves per CU, 8 of the wide form
    p.dx_blocks = need_dx ? (int)row_blocks(rows, p.sh) : 0;
    if (p.acc) {
        p.dx_blocks = (int)(nb < fill ? nb : fill);
        p.parts = p.dx_blocks;
        p.part_rows = 0;
        return p;
    }
    const long long slices = p.sh.threads / 32;
    long long parts = yfs_cdiv(2048, p.strips), most = yfs_cdiv(rows, slices * 16);
    if (parts > most) parts = most;
    if (parts > 256) parts = 256;
    p.part_rows = yfs_cdiv(rows, parts);
    p.parts = (int)yfs_cdiv(rows, p.part_rows);
    return p;
}

template <typename T>
int fwd(const void* x, long long xs, const float* w, const float* b, void* y, float* mean, float* rstd, long long rows, int cols,
        float eps, hipStream_t s) {
    const bool odd = cols % (16 / (int)sizeof(T)) != 0;
    const Shape sh = ln_shape(cols, sizeof(T), 3, 4, 8);
    const dim3 grid(row_blocks(rows, sh)), blk(sh.threads);
#define LN_FWD(NV, BLOCK)                                                                                                              \
    do {                                                                                                                               \
        if (odd) ln_fwd_kernel<T, NV, BLOCK, true><<<grid, blk, 0, s>>>((const T*)x, xs, w, b, (T*)y, mean, rstd, rows, cols, eps, sh.lg);   \
        else ln_fwd_kernel<T, NV, BLOCK, false><<<grid, blk, 0, s>>>((const T*)x, xs, w, b, (T*)y, mean, rstd, rows, cols, eps, sh.lg);       \
    } while (0)
#define LN_WIDE(NV)                                                                                                                \
    do {                                                                                                                             \
        if (odd) ln_fwd_wide_kernel<T, NV, true><<<grid, blk, 0, s>>>((const T*)x, xs, w, b, (T*)y, mean, rstd, rows, cols, eps);      \
        else ln_fwd_wide_kernel<T, NV, false><<<grid, blk, 0, s>>>((const T*)x, xs, w, b, (T*)y, mean, rstd, rows, cols, eps);          \
    } while (0)
    if (sh.nv == 0)
        ln_fwd_long_kernel<T><<<grid, blk, 0, s>>>((const T*)x, xs, w, b, (T*)y, mean, rstd, rows, cols, eps);
    else if (sh.lg >= 0) {
        if (sh.nv == 1) LN_FWD(1, false);
        else if (sh.nv == 2) LN_FWD(2, false);
        else LN_FWD(3, false);
    } else if (sh.wide) {
        if (sh.nv == 4) LN_WIDE(4);
        else LN_WIDE(8);
    } else if (sh.nv == 2) LN_FWD(2, true);
    else LN_FWD(4, true);
#undef LN_WIDE
#undef LN_FWD
    YFS_CHECK_LAUNCH("ln_fwd_kernel");
    return YFS_OK;
}

template <typename T>
int bwd(BwdArgs g, float* part, hipStream_t s) {
    const bool sums = g.dw || g.db, odd = g.cols % (16 / (int)sizeof(T)) != 0;
    BwdPlan p = bwd_plan(g.rows, g.cols, sizeof(T), g.dx != nullptr);
    if (!sums) {
        p.acc = false;
        p.parts = 0;
        p.dx_blocks = (int)row_blocks(g.rows, p.sh);
    }
    g.lg = p.sh.lg;
    g.dx_blocks = p.dx_blocks;
    g.strips = p.strips;
    g.part_rows = p.part_rows;
    float *dw = g.dw, *db = g.db;
    const bool join = p.acc || p.parts > 1;
    if (join) {
        g.dw = part;
        g.db = part + g.cols;
    }
    if (!sums && !g.dx) return YFS_OK;
    const dim3 grid((unsigned)(p.dx_blocks + (p.acc ? 0 : (long long)p.strips * p.parts))), blk(p.sh.threads);
    // sums of the groups of a workgroup, or of the waves of a column strip
    const size_t lds = p.acc ? (p.sh.lg >= 0 ? (size_t)(256 >> p.sh.lg) * 2 * g.cols * sizeof(float) : 0)
                             : (sums ? (size_t)p.sh.threads / 64 * 2 * 32 * (16 / sizeof(T)) * sizeof(float) : 0);
#define LN_BWD(NV, BLOCK, ACC) \
    do { if (odd) ln_bwd_kernel<T, NV, BLOCK, ACC, true><<<grid, blk, lds, s>>>(g); else ln_bwd_kernel<T, NV, BLOCK, ACC, false><<<grid, blk, lds, s>>>(g); } while (0)
#define LN_WIDE(NV, ACC) \
    do { if (odd) ln_bwd_wide_kernel<T, NV, ACC, true><<<grid, blk, lds, s>>>(g); else ln_bwd_wide_kernel<T, NV, ACC, false><<<grid, blk, lds, s>>>(g); } while (0)
    if (p.sh.nv == 0) ln_bwd_long_kernel<T><<<grid, blk, lds, s>>>(g);
    else if (p.sh.lg >= 0) {
        if (p.sh.nv == 1 && p.acc) LN_BWD(1, false, true);
        else if (p.sh.nv == 1) LN_BWD(1, false, false);
        else if (p.acc) LN_BWD(2, false, true);
        else LN_BWD(2, false, false);
    } else if (p.sh.nv == 2) {
        if (p.acc) LN_BWD(2, true, true);
        else LN_BWD(2, true, false);
    } else {
        if (p.acc) LN_WIDE(4, true);
        else LN_WIDE(4, false);
    }
#undef LN_WIDE
#undef LN_BWD
    YFS_CHECK_LAUNCH("ln_bwd_kernel");
    if (sums && join) {
        ln_reduce_kernel<<<dim3((unsigned)yfs_cdiv(2LL * g.cols, 32)), 1024, 0, s>>>(part, p.parts, g.cols, dw, db);
        YFS_CHECK_LAUNCH("ln_reduce_kernel");
    }
    return YFS_OK;
}

bool known(int dtype) { return dtype == YFS_F32 || dtype == YFS_BF16 || dtype == YFS_F16; }
constexpr long long kMostCols = 1LL << 28;   // (a launch has fewer than 2^32 threads: 8 or 4 per column of the longest rows' sums)
}  // namespace

YFS_API int yfs_layer_norm_fwd(const void* x, int64_t x_stride, const float* w, const float* b, void* y, float* mean, float* rstd,
                               int64_t rows, int64_t cols, float eps, int dtype, void* stream) {
    YFS_REQUIRE(x && y, YFS_ERR_INVALID_ARG, "yfs_layer_norm_fwd: null pointer");
    YFS_REQUIRE(rows > 0 && cols > 0 && cols < kMostCols && x_stride >= 0, YFS_ERR_INVALID_ARG,
                "yfs_layer_norm_fwd: need rows > 0, 0 < cols < 2^28 and a row stride >= 0 (got rows=%lld cols=%lld stride=%lld)",
                (long long)rows, (long long)cols, (long long)x_stride);
    YFS_REQUIRE(eps >= 0.0f, YFS_ERR_INVALID_ARG, "yfs_layer_norm_fwd: eps %g is negative", eps);
    YFS_REQUIRE(known(dtype), YFS_ERR_UNSUPPORTED, "yfs_layer_norm_fwd: unknown dtype %d", dtype);
    hipStream_t s = (hipStream_t)stream;
    if (dtype == YFS_F32) return fwd<float>(x, x_stride, w, b, y, mean, rstd, rows, (int)cols, eps, s);
    if (dtype == YFS_BF16) return fwd<__bf16>(x, x_stride, w, b, y, mean, rstd, rows, (int)cols, eps, s);
    return fwd<_Float16>(x, x_stride, w, b, y, mean, rstd, rows, (int)cols, eps, s);
}

// (with or without dx: the larger of the two)
YFS_API size_t yfs_layer_norm_bwd_workspace_bytes(int64_t rows, int64_t cols, int dtype) {
    if (rows <= 0 || cols <= 0 || cols >= kMostCols || !known(dtype)) return 0;
    size_t most = 0;
    for (int dx = 0; dx < 2; ++dx) {
        const BwdPlan p = bwd_plan(rows, (int)cols, dtype == YFS_F32 ? 4 : 2, dx);
        const size_t need = p.acc || p.parts > 1 ? (size_t)p.parts * 2 * (size_t)cols * sizeof(float) : 0;
        most = need > most ? need : most;
    }
    return most;
}

YFS_API int yfs_layer_norm_bwd(const void* dy, int64_t dy_stride, const void* x, int64_t x_stride, const float* w, const float* mean,
                               const float* rstd, void* dx, float* dw, float* db, int64_t rows, int64_t cols, int dtype,
                               void* workspace, size_t workspace_bytes, void* stream) {
    YFS_REQUIRE(dy && x && mean && rstd, YFS_ERR_INVALID_ARG, "yfs_layer_norm_bwd: null pointer");
    YFS_REQUIRE(rows > 0 && cols > 0 && cols < kMostCols && x_stride >= 0 && dy_stride >= 0, YFS_ERR_INVALID_ARG,
                "yfs_layer_norm_bwd: need rows > 0, 0 < cols < 2^28 and row strides >= 0 (got rows=%lld cols=%lld)", (long long)rows,
                (long long)cols);
    YFS_REQUIRE(known(dtype), YFS_ERR_UNSUPPORTED, "yfs_layer_norm_bwd: unknown dtype %d", dtype);
    const size_t need = (dw || db) ? yfs_layer_norm_bwd_workspace_bytes(rows, cols, dtype) : 0;
    YFS_REQUIRE(need == 0 || (workspace && workspace_bytes >= need), YFS_ERR_WORKSPACE,
                "yfs_layer_norm_bwd: workspace needs %zu bytes", need);
    const BwdArgs g = {dy, x, dy_stride, x_stride, w, mean, rstd, dx, dw, db, rows, (int)cols, 0, 0, 0, 0};
    hipStream_t s = (hipStream_t)stream;
    if (dtype == YFS_F32) return bwd<float>(g, (float*)workspace, s);
    if (dtype == YFS_BF16) return bwd<__bf16>(g, (float*)workspace, s);
    return bwd<_Float16>(g, (float*)workspace, s);
}
