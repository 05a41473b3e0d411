// Dropout from a counter-based generator, with the LeakyReLU in front of it: no mask is stored, the backward pass draws the
// same numbers again.
//   element e of the tensor in row-major order is kept iff (philox4x32_10(key = seed, counter = e / 4)[e % 4] >> 8) 2^-24 >= p
//   y = keep ? leaky(x) / (1 - p) : 0          dx = keep ? dy / (1 - p) (y > 0 ? 1 : slope) : 0
// (the rule of yfs_fc_epilogue_fwd_bf16: the same seed and p keep the same elements there).
// (r >> 8) 2^-24 >= p  <=>  r >= ceil(p 2^24) 2^8, a comparison of whole numbers prepared on the host, with p rounded to fp32 (as
// there).  The scale is that of p itself: near 1 its fp32 neighbour is off by much more of 1 - p than a rounding (0.9999: 1.7e-4).
#include "yfs_common.h"
#include "yfs_vec.h"
#include <math.h>

// Reads and writes the tensor once; the generator's 20 products for four elements take about as long as their bytes, which is
// why its first round is folded and its exclusive-ors are three-operand instructions (200704 x 256 bf16: 50 -> 35 us a pass,
// 5.9 TB/s).
namespace {
constexpr int kThreads = 256;

struct DropArgs {
    const void *in, *y;          // x, or dy and (with a slope) y
    void* out;
    long long n;
    unsigned long long seed;
    const long long* seed_dev;   // overrides seed when not NULL
    unsigned ctr_hi;             // high word of the counters of these elements
    unsigned thr;                // kept iff r >= thr
    int none;                    // p == 1: nothing is kept
    float scale, slope;
};

template <typename T, bool BWD, bool ACT>
__device__ __forceinline__ void drop_vector(const DropArgs& g, unsigned long long seed, long long e, long long left) {
    constexpr int VE = 16 / sizeof(T);
    float v[VE], yv[VE];
    load_vec((const T*)g.in + e, left, v);
    if (BWD && ACT) load_vec((const T*)g.y + e, left, yv);
#pragma unroll
    for (int q = 0; q < VE / 4; ++q) {
        unsigned r[4];
        yfs_philox4(seed, (unsigned)(e >> 2) + q, g.ctr_hi, r);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int k = q * 4 + j;
            float t = v[k];
            if (ACT) t = (BWD ? yv[k] > 0.0f : t > 0.0f) ? t : t * g.slope;
            v[k] = r[j] >= g.thr && !g.none ? t * g.scale : 0.0f;   // a select: NaN and Inf in dropped places leave nothing
        }
    }
    store_vec((T*)g.out + e, left, v);
}

template <typename T, bool BWD, bool ACT>
__global__ void __launch_bounds__(kThreads) dropout_kernel(DropArgs g) {
    constexpr int VE = 16 / sizeof(T);
    const unsigned long long seed = g.seed_dev ? (unsigned long long)*g.seed_dev : g.seed;
    const long long whole = g.n / VE, stride = (long long)gridDim.x * kThreads;
    long long id = (long long)blockIdx.x * kThreads + threadIdx.x;
    for (; id < whole; id += stride) drop_vector<T, BWD, ACT>(g, seed, id * VE, VE);
    if (id == whole && g.n % VE) drop_vector<T, BWD, ACT>(g, seed, id * VE, g.n % VE);   // the last elements
}

template <bool BWD, bool ACT>
int launch(DropArgs g, int dtype, hipStream_t s) {
    // 2^34 elements at a time, so that the counters of a launch share their high word
    const long long n = g.n, chunk = 1LL << 34, size = dtype == YFS_F32 ? 4 : 2, vec = 16 / size;
    const char *in = (const char*)g.in, *y = (const char*)g.y;
    char* out = (char*)g.out;
    for (long long at = 0; at < n; at += chunk) {
        g.n = n - at < chunk ? n - at : chunk;
        g.in = in + at * size;
        g.y = y ? y + at * size : nullptr;
        g.out = out + at * size;
        g.ctr_hi = (unsigned)(at >> 34);
        long long nb = yfs_cdiv(yfs_cdiv(g.n, vec), kThreads);
        const dim3 grid((unsigned)(nb < (1 << 20) ? nb : 1 << 20));
        if (dtype == YFS_F32) dropout_kernel<float, BWD, ACT><<<grid, kThreads, 0, s>>>(g);
        else if (dtype == YFS_BF16) dropout_kernel<__bf16, BWD, ACT><<<grid, kThreads, 0, s>>>(g);
        else dropout_kernel<_Float16, BWD, ACT><<<grid, kThreads, 0, s>>>(g);
        YFS_CHECK_LAUNCH("dropout_kernel");
    }
    return YFS_OK;
}

int run(const char* name, bool bwd, const void* in, const void* y, void* out, int64_t n, double p, float slope, uint64_t seed,
        const int64_t* seed_dev, int dtype, void* stream) {
    YFS_REQUIRE(in && out, YFS_ERR_INVALID_ARG, "%s: null pointer", name);
    YFS_REQUIRE(n > 0, YFS_ERR_INVALID_ARG, "%s: n must be positive (got %lld)", name, (long long)n);
    YFS_REQUIRE(p >= 0.0 && p <= 1.0, YFS_ERR_INVALID_ARG, "%s: p %g not in [0, 1]", name, p);
    YFS_REQUIRE(slope >= 0.0f && slope <= 1.0f, YFS_ERR_INVALID_ARG, "%s: slope %g not in [0, 1]", name, slope);
    YFS_REQUIRE(dtype == YFS_F32 || dtype == YFS_BF16 || dtype == YFS_F16, YFS_ERR_UNSUPPORTED, "%s: unknown dtype %d", name, dtype);
    const bool act = slope != 1.0f;
    YFS_REQUIRE(!bwd || !act || y, YFS_ERR_INVALID_ARG, "%s: the gradient of an activation needs y", name);
    const float p32 = (float)p;
    DropArgs g = {in, y, out, n, seed, (const long long*)seed_dev, 0u, 0u, p32 >= 1.0f, 0.0f, slope};
    const double t = ceil((double)p32 * 16777216.0);
    g.thr = g.none ? 0xFFFFFFFFu : (unsigned)t << 8;
    g.scale = g.none ? 0.0f : (float)(1.0 / (1.0 - p));
    hipStream_t s = (hipStream_t)stream;
    if (bwd) return act ? launch<true, true>(g, dtype, s) : launch<true, false>(g, dtype, s);
    return act ? launch<false, true>(g, dtype, s) : launch<false, false>(g, dtype, s);
}
}  // namespace

YFS_API int yfs_dropout_fwd(const void* x, void* y, int64_t n, double p, float slope, uint64_t seed, const int64_t* seed_dev,
                            int dtype, void* stream) {
    return run("yfs_dropout_fwd", false, x, nullptr, y, n, p, slope, seed, seed_dev, dtype, stream);
}

YFS_API int yfs_dropout_bwd(const void* dy, const void* y, void* dx, int64_t n, double p, float slope, uint64_t seed,
                            const int64_t* seed_dev, int dtype, void* stream) {
    return run("yfs_dropout_bwd", true, dy, y, dx, n, p, slope, seed, seed_dev, dtype, stream);
}
