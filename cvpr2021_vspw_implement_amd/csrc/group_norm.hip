// Group normalisation with activation and dropout on channels-last activations [n][hw][c], fp32 / bf16 / fp16.
//
//   forward    mean, var over (hw, channels of a group);  a = w (x - mean) / sqrt(var + eps) + b;  y = drop(act(a))
//   backward   da = dy drop'(.) act'(a);  db = sum da;  dw = sum da xhat;  t = da w;
//              dx = rstd (t - mean(t) - xhat mean(t xhat))     (means over the group)
//
// Statistics, sums and the pre-activation are evaluated in fp64: a fp64 fma runs at the rate of a plain fp32 one on this
// chip and the kernels are bound by HBM, so it costs nothing, a mean far from zero loses no digits, and the ReLU border
// is decided on the exactly rounded pre-activation.  All sums have a fixed order: results are bit-reproducible.
//
// Three streaming passes' worth of kernels: stats -> apply, and bwd_stats -> bwd_reduce -> bwd_apply.
#include "elem.h"

enum { ACT_NONE = 0, ACT_RELU = 1, ACT_SILU = 2, ACT_GELU = 3 };

struct GnShape {
    long long hw;
    int n, c, groups, cpg;  // cpg: channels per group
    int tx, slabs, chunks;
};

__device__ __forceinline__ float act_value(float a, int act) {
    if (act == ACT_RELU) return a > 0.f ? a : (a != a ? a : 0.f);
    if (act == ACT_SILU) return a / (1.f + expf(-a));
    if (act == ACT_GELU) return 0.5f * a * erfcf(-a * 0.70710678118654752f);
    return a;
}
__device__ __forceinline__ float act_slope(float a, int act) {
    if (act == ACT_RELU) return a > 0.f ? 1.f : (a != a ? a : 0.f);
    if (act == ACT_SILU) {
        const float s = 1.f / (1.f + expf(-a));
        return s * (1.f + a * (1.f - s));
    }
    if (act == ACT_GELU) return 0.5f * erfcf(-a * 0.70710678118654752f) + a * 0.39894228040143268f * expf(-0.5f * a * a);
    return 1.f;
}

// block-wide: sums of s[e], q[e] over the pixel lanes of every channel, left in red[0..1][channel of the slab]
template <int V>
__device__ __forceinline__ void reduce_pixels(double* s, double* q, double (*red)[256 * V], int tx) {
    const int tid = threadIdx.x;
#pragma unroll
    for (int e = 0; e < V; ++e) {
        red[0][tid * V + e] = s[e];
        red[1][tid * V + e] = q[e];
    }
    __syncthreads();
    const int width = tx * V;
    for (int half = 128 / tx; half > 0; half >>= 1) {  // 256 / tx pixel lanes, a power of two
        for (int i = tid; i < half * width; i += 256) {
            red[0][i] += red[0][i + half * width];
            red[1][i] += red[1][i + half * width];
        }
        __syncthreads();
    }
}

// part[img][chunk][slab][k][2]: sum and sum of squares of x - x0 over the chunk's pixels of the slab's share of group (first
// group of the slab + k); gs entries per slab.  x0 = the group's first element: with it a mean of 10^6 standard deviations
// costs the variance nothing.
template <typename T, int V>
__global__ __launch_bounds__(256) void gn_stats_kernel(const T* __restrict__ x, GnShape g, int gs, double* __restrict__ part) {
    __shared__ double red[2][256 * V];
    const int slab = blockIdx.x % g.slabs;
    const int rest = blockIdx.x / g.slabs;
    const int chunk = rest % g.chunks, img = rest / g.chunks;
    const int c0 = (slab * g.tx + (int)threadIdx.x % g.tx) * V;
    const int ty = 256 / g.tx;
    double s[V], q[V];
#pragma unroll
    for (int e = 0; e < V; ++e) s[e] = q[e] = 0.0;
    if (c0 < g.c) {
        const T* xi = x + (size_t)img * g.hw * g.c;
        const T* xp = xi + c0;
        double x0[V];
#pragma unroll
        for (int e = 0; e < V; ++e) x0[e] = (double)(float)xi[(c0 + e) / g.cpg * g.cpg];
#pragma unroll 4
        for (long long p = (long long)chunk * ty + threadIdx.x / g.tx; p < g.hw; p += (long long)g.chunks * ty) {
            float f[V];
            Vec<T, V>::load(xp + (size_t)p * g.c, f);
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const double d = (double)f[e] - x0[e];
                s[e] += d;
                q[e] = fma(d, d, q[e]);
            }
        }
    }
    reduce_pixels<V>(s, q, red, g.tx);
    const int first = slab * g.tx * V, last = min(g.c, first + g.tx * V);
    const int g0 = first / g.cpg, g1 = (last - 1) / g.cpg;
    for (int k = threadIdx.x; k <= g1 - g0; k += 256) {
        const int lo = max(first, (g0 + k) * g.cpg), hi = min(last, (g0 + k + 1) * g.cpg);
        double a = 0, b = 0;
        for (int ch = lo; ch < hi; ++ch) {
            a += red[0][ch - first];
            b += red[1][ch - first];
        }
        double* o = part + ((((size_t)img * g.chunks + chunk) * g.slabs + slab) * gs + k) * 2;
        o[0] = a;
        o[1] = b;
    }
}

// mean and 1/sqrt(var + eps) of the groups that overlap the block's slab, into LDS ms[k][2]: entries of all chunks and of
// the slabs that share the group, summed in a fixed order by `lanes` lanes per group.
template <typename T>
__device__ __forceinline__ void group_stats(const T* __restrict__ x, const double* __restrict__ part, const GnShape& g,
                                            int gs, int img, int slab, int slabw, float eps, double* ms) {
    const int first = slab * slabw, last = min(g.c, first + slabw);
    const int g0 = first / g.cpg, count = (last - 1) / g.cpg - g0 + 1;
    int lanes = 64;
    while (lanes > 1 && 256 / lanes < count) lanes >>= 1;
    const int sub = threadIdx.x % lanes;
    const double inv = 1.0 / ((double)g.hw * g.cpg);
    for (int k0 = 0; k0 < count; k0 += 256 / lanes) {
        const int k = k0 + threadIdx.x / lanes;
        double a = 0, b = 0;
        if (k < count) {
            const int gr = g0 + k;
            const int s0 = gr * g.cpg / slabw, ns = ((gr + 1) * g.cpg - 1) / slabw - s0 + 1;
            for (int i = sub; i < g.chunks * ns; i += lanes) {
                const int sl = s0 + i % ns;
                const double* o = part + ((((size_t)img * g.chunks + i / ns) * g.slabs + sl) * gs + (gr - sl * slabw / g.cpg)) * 2;
                a += o[0];
                b += o[1];
            }
        }
        for (int o = lanes >> 1; o > 0; o >>= 1) {
            a += __shfl_xor(a, o, 64);
            b += __shfl_xor(b, o, 64);
        }
        if (k < count && sub == 0) {
            const double m = a * inv;
            double var = b * inv - m * m;
            if (var < 0) var = 0;
            ms[2 * k] = m + (double)(float)x[(size_t)img * g.hw * g.c + (size_t)(g0 + k) * g.cpg];
            ms[2 * k + 1] = 1.0 / sqrt(var + (double)eps);
        }
    }
    __syncthreads();
}

// The dropout factors of one pixel's channels c0 .. c0+V-1 (memory index e0); ck: the channel form's, computed once.
template <int V>
__device__ __forceinline__ void drop_factors(const Philox& gen, const DropRule& d, int mode, size_t e0, const float* ck, float* k) {
    if (mode == 1) {
        unsigned u[V];
        gen.run<V>(e0, u);  // V > 1 only where c % V == 0: e0 is a multiple of 4
#pragma unroll
        for (int e = 0; e < V; ++e) k[e] = d.factor(u[e]);
    } else {
#pragma unroll
        for (int e = 0; e < V; ++e) k[e] = ck[e];
    }
}

struct GnDrop {
    DropRule rule;
    int mode;  // 0: none, 1: per element, 2: per image and channel
    const long long* rng;
};

template <typename T, int V>
__global__ __launch_bounds__(256) void gn_apply_kernel(const T* __restrict__ x, T* __restrict__ y, GnShape g, int gs,
                                                       const double* __restrict__ part, const float* __restrict__ w,
                                                       const float* __restrict__ b, float eps, int act, GnDrop dr,
                                                       double* __restrict__ stats) {
    __shared__ double ms[2 * 64 * V];
    const int slab = blockIdx.x % g.slabs;
    const int rest = blockIdx.x / g.slabs;
    const int chunk = rest % g.chunks, img = rest / g.chunks;
    const int slabw = g.tx * V;
    group_stats(x, part, g, gs, img, slab, slabw, eps, ms);
    const int first = slab * slabw, g0 = first / g.cpg;
    if (chunk == 0 && stats) {  // for the backward pass; a group that spans slabs is written by the one it starts in
        const int last = min(g.c, first + slabw);
        for (int k = threadIdx.x; k <= (last - 1) / g.cpg - g0; k += 256)
            if ((g0 + k) * g.cpg >= first) {
                stats[((size_t)img * g.groups + g0 + k) * 2] = ms[2 * k];
                stats[((size_t)img * g.groups + g0 + k) * 2 + 1] = ms[2 * k + 1];
            }
    }
    const int c0 = first + ((int)threadIdx.x % g.tx) * V;
    if (c0 >= g.c) return;
    const int ty = 256 / g.tx;
    double A[V], B[V];
    float ck[V];
    const Philox gen(dr.rng);
#pragma unroll
    for (int e = 0; e < V; ++e) {
        const int k = (c0 + e) / g.cpg - g0;
        A[e] = ms[2 * k + 1] * (w ? (double)w[c0 + e] : 1.0);
        B[e] = (b ? (double)b[c0 + e] : 0.0) - ms[2 * k] * A[e];
        ck[e] = 1.f;
        if (dr.mode == 2) {
            unsigned u;
            gen.run<1>((unsigned long long)img * g.c + c0 + e, &u);
            ck[e] = dr.rule.factor(u);
        }
    }
    const size_t base = (size_t)img * g.hw * g.c + c0;
#pragma unroll 2
    for (long long p = (long long)chunk * ty + threadIdx.x / g.tx; p < g.hw; p += (long long)g.chunks * ty) {
        float f[V], k[V];
        const size_t e0 = base + (size_t)p * g.c;
        Vec<T, V>::load(x + e0, f);
        drop_factors<V>(gen, dr.rule, dr.mode, e0, ck, k);
#pragma unroll
        for (int e = 0; e < V; ++e) f[e] = drop_apply(act_value((float)fma((double)f[e], A[e], B[e]), act), k[e]);
        Vec<T, V>::store(y + e0, f);
    }
}

// part[img][chunk][2][c]: sum da, sum da xhat over the chunk's pixels
template <typename T, int V>
__global__ __launch_bounds__(256) void gn_bwd_stats_kernel(const T* __restrict__ x, const T* __restrict__ dy, GnShape g,
                                                           const double* __restrict__ stats, const float* __restrict__ w,
                                                           const float* __restrict__ b, int act, GnDrop dr,
                                                           double* __restrict__ part) {
    __shared__ double red[2][256 * V];
    const int slab = blockIdx.x % g.slabs;
    const int rest = blockIdx.x / g.slabs;
    const int chunk = rest % g.chunks, img = rest / g.chunks;
    const int first = slab * g.tx * V;
    const int c0 = first + ((int)threadIdx.x % g.tx) * V;
    const int ty = 256 / g.tx;
    double s[V], q[V];
#pragma unroll
    for (int e = 0; e < V; ++e) s[e] = q[e] = 0.0;
    if (c0 < g.c) {
        double R[V], M[V];
        float W[V], Bv[V], ck[V];
        const Philox gen(dr.rng);
#pragma unroll
        for (int e = 0; e < V; ++e) {
            const double* st = stats + ((size_t)img * g.groups + (c0 + e) / g.cpg) * 2;
            R[e] = st[1];
            M[e] = -st[0] * st[1];
            W[e] = w ? w[c0 + e] : 1.f;
            Bv[e] = b ? b[c0 + e] : 0.f;
            ck[e] = 1.f;
            if (dr.mode == 2) {
                unsigned u;
                gen.run<1>((unsigned long long)img * g.c + c0 + e, &u);
                ck[e] = dr.rule.factor(u);
            }
        }
        const size_t base = (size_t)img * g.hw * g.c + c0;
#pragma unroll 2
        for (long long p = (long long)chunk * ty + threadIdx.x / g.tx; p < g.hw; p += (long long)g.chunks * ty) {
            float f[V], d[V], k[V];
            const size_t e0 = base + (size_t)p * g.c;
            Vec<T, V>::load(x + e0, f);
            Vec<T, V>::load(dy + e0, d);
            drop_factors<V>(gen, dr.rule, dr.mode, e0, ck, k);
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const double xh = fma((double)f[e], R[e], M[e]);
                const double da = (double)(drop_apply(d[e], k[e]) * act_slope((float)fma(xh, (double)W[e], (double)Bv[e]), act));
                s[e] += da;
                q[e] = fma(da, xh, q[e]);
            }
        }
    }
    reduce_pixels<V>(s, q, red, g.tx);
    for (int i = threadIdx.x; i < g.tx * V; i += 256)
        if (first + i < g.c) {
            double* o = part + ((size_t)img * g.chunks + chunk) * 2 * g.c + first + i;
            o[0] = red[0][i];
            o[g.c] = red[1][i];
        }
}

// csum[img][2][c] = sum over chunks of part: one workgroup per image and 32 columns, 8 row lanes
__global__ __launch_bounds__(256) void gn_bwd_reduce_kernel(const double* __restrict__ part, int chunks, int c2,
                                                            double* __restrict__ csum) {
    __shared__ double red[8][32];
    const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
    const int blocks = (c2 + 31) / 32;
    const int img = blockIdx.x / blocks, col = (blockIdx.x % blocks) * 32 + tx;
    double a = 0;
    if (col < c2) {
        const double* p = part + (size_t)img * chunks * c2 + col;
#pragma unroll 4
        for (int z = ty; z < chunks; z += 8) a += p[(size_t)z * c2];
    }
    red[ty][tx] = a;
    __syncthreads();
    if (ty == 0 && col < c2) {
        a = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) a += red[j][tx];
        csum[(size_t)img * c2 + col] = a;
    }
}

template <typename T, int V>
__global__ __launch_bounds__(256) void gn_bwd_apply_kernel(const T* __restrict__ x, const T* __restrict__ dy,
                                                           T* __restrict__ dx, GnShape g, const double* __restrict__ stats,
                                                           const float* __restrict__ w, const float* __restrict__ b, int act,
                                                           GnDrop dr, const double* __restrict__ csum,
                                                           float* __restrict__ dw, float* __restrict__ db) {
    __shared__ double ts[2 * 64 * V];
    const int slab = blockIdx.x % g.slabs;
    const int rest = blockIdx.x / g.slabs;
    const int chunk = rest % g.chunks, img = rest / g.chunks;
    const int first = slab * g.tx * V, last = min(g.c, first + g.tx * V);
    if (img == 0 && chunk == 0)  // the parameter gradients of the slab's channels
        for (int ch = first + threadIdx.x; ch < last; ch += 256) {
            double a = 0, q = 0;
            for (int i = 0; i < g.n; ++i) {
                a += csum[(size_t)i * 2 * g.c + ch];
                q += csum[((size_t)i * 2 + 1) * g.c + ch];
            }
            if (db) db[ch] = (float)a;
            if (dw) dw[ch] = (float)q;
        }
    if (!dx) return;
    // mean(t), mean(t xhat) of the groups of this slab
    const int g0 = first / g.cpg, count = (last - 1) / g.cpg - g0 + 1;
    const double inv = 1.0 / ((double)g.hw * g.cpg);
    int lanes = 64;
    while (lanes > 1 && 256 / lanes < count) lanes >>= 1;
    for (int k0 = 0; k0 < count; k0 += 256 / lanes) {
        const int k = k0 + threadIdx.x / lanes, sub = threadIdx.x % lanes;
        double a = 0, q = 0;
        if (k < count)
            for (int ch = (g0 + k) * g.cpg + sub; ch < (g0 + k + 1) * g.cpg; ch += lanes) {
                const double wt = w ? (double)w[ch] : 1.0;
                a = fma(wt, csum[(size_t)img * 2 * g.c + ch], a);
                q = fma(wt, csum[((size_t)img * 2 + 1) * g.c + ch], q);
            }
        for (int o = lanes >> 1; o > 0; o >>= 1) {
            a += __shfl_xor(a, o, 64);
            q += __shfl_xor(q, o, 64);
        }
        if (k < count && sub == 0) {
            ts[2 * k] = a * inv;
            ts[2 * k + 1] = q * inv;
        }
    }
    __syncthreads();
    const int c0 = first + ((int)threadIdx.x % g.tx) * V;
    if (c0 >= g.c) return;
    const int ty = 256 / g.tx;
    double R[V], M[V];
    float W[V], Bv[V], T1[V], T2[V], ck[V];
    const Philox gen(dr.rng);
#pragma unroll
    for (int e = 0; e < V; ++e) {
        const int gr = (c0 + e) / g.cpg;
        const double* st = stats + ((size_t)img * g.groups + gr) * 2;
        R[e] = st[1];
        M[e] = -st[0] * st[1];
        W[e] = w ? w[c0 + e] : 1.f;
        Bv[e] = b ? b[c0 + e] : 0.f;
        T1[e] = (float)ts[2 * (gr - g0)];
        T2[e] = (float)ts[2 * (gr - g0) + 1];
        ck[e] = 1.f;
        if (dr.mode == 2) {
            unsigned u;
            gen.run<1>((unsigned long long)img * g.c + c0 + e, &u);
            ck[e] = dr.rule.factor(u);
        }
    }
    const size_t base = (size_t)img * g.hw * g.c + c0;
#pragma unroll 2
    for (long long p = (long long)chunk * ty + threadIdx.x / g.tx; p < g.hw; p += (long long)g.chunks * ty) {
        float f[V], d[V], k[V];
        const size_t e0 = base + (size_t)p * g.c;
        Vec<T, V>::load(x + e0, f);
        Vec<T, V>::load(dy + e0, d);
        drop_factors<V>(gen, dr.rule, dr.mode, e0, ck, k);
#pragma unroll
        for (int e = 0; e < V; ++e) {
            const double xh = fma((double)f[e], R[e], M[e]);
            const float da = drop_apply(d[e], k[e]) * act_slope((float)fma(xh, (double)W[e], (double)Bv[e]), act);
            f[e] = (float)R[e] * (fmaf(da, W[e], -T1[e]) - (float)xh * T2[e]);
        }
        Vec<T, V>::store(dx + e0, f);
    }
}

// ------------------------------------------------------------------------------------------------------------- host
static bool gn_shape_ok(int n, long long hw, int c, int groups, int dtype) {
    return n > 0 && hw > 0 && c > 0 && groups > 0 && c % groups == 0 && vspw_dtype_ok(dtype) &&
           hw <= (0x7fffffffffffffffLL / n) / c / 8;
}
// 16-byte accesses when rows keep the alignment; the plan is a function of the shape alone
static int gn_vec(int c, int dtype) {
    const int v = 16 / vspw_dtype_size(dtype);
    return c % v == 0 ? v : 1;
}
static GnShape gn_plan(int n, long long hw, int c, int groups, int dtype) {
    const SlabPlan s = vspw_slab_plan(n, hw, c, gn_vec(c, dtype), 8);
    GnShape g;
    g.hw = hw;
    g.n = n;
    g.c = c;
    g.groups = groups;
    g.cpg = c / groups;
    g.tx = s.tx;
    g.slabs = s.slabs;
    g.chunks = s.chunks;
    return g;
}
static int gn_gs(const GnShape& g, int v) {  // groups that a slab can overlap
    const int w = g.tx * v;
    const int most = (w + g.cpg - 1) / g.cpg + 1;
    return most < g.groups ? most : g.groups;
}

extern "C" size_t vspw_group_norm_fwd_workspace(int n, long long hw, int c, int groups, int dtype) {
    if (!gn_shape_ok(n, hw, c, groups, dtype)) return 0;
    const GnShape g = gn_plan(n, hw, c, groups, dtype);
    return (size_t)n * g.chunks * g.slabs * gn_gs(g, gn_vec(c, dtype)) * 2 * sizeof(double);
}

extern "C" size_t vspw_group_norm_bwd_workspace(int n, long long hw, int c, int groups, int dtype) {
    if (!gn_shape_ok(n, hw, c, groups, dtype)) return 0;
    const GnShape g = gn_plan(n, hw, c, groups, dtype);
    return (size_t)n * (g.chunks + 1) * 2 * c * sizeof(double);
}

static bool gn_args(int act, double p, const long long* rng, int channelwise, GnDrop& dr) {
    if (act < ACT_NONE || act > ACT_GELU || !(p >= 0.0 && p <= 1.0) || (p > 0.0 && !rng)) return false;
    dr.rule = DropRule::of(p);
    dr.mode = p > 0.0 ? (channelwise ? 2 : 1) : 0;
    dr.rng = p > 0.0 ? rng : nullptr;
    return true;
}

template <typename T, int V>
static int gn_fwd_launch(const void* x, void* y, const GnShape& g, const float* w, const float* b, float eps, int act,
                         const GnDrop& dr, double* stats, double* part, hipStream_t st) {
    const int gs = gn_gs(g, V);
    const dim3 grid((unsigned)(g.slabs * g.chunks * g.n));
    hipLaunchKernelGGL((gn_stats_kernel<T, V>), grid, dim3(256), 0, st, (const T*)x, g, gs, part);
    const int rc = vspw_launch_status();
    if (rc != VSPW_OK) return rc;
    hipLaunchKernelGGL((gn_apply_kernel<T, V>), grid, dim3(256), 0, st, (const T*)x, (T*)y, g, gs, part, w, b, eps, act, dr,
                       stats);
    return vspw_launch_status();
}

template <typename T, int V>
static int gn_bwd_launch(const void* x, const void* dy, void* dx, const GnShape& g, const float* w, const float* b, int act,
                         const GnDrop& dr, const double* stats, float* dw, float* db, double* part, hipStream_t st) {
    const dim3 grid((unsigned)(g.slabs * g.chunks * g.n));
    double* csum = part + (size_t)g.n * g.chunks * 2 * g.c;
    hipLaunchKernelGGL((gn_bwd_stats_kernel<T, V>), grid, dim3(256), 0, st, (const T*)x, (const T*)dy, g, stats, w, b, act,
                       dr, part);
    int rc = vspw_launch_status();
    if (rc != VSPW_OK) return rc;
    hipLaunchKernelGGL(gn_bwd_reduce_kernel, dim3((unsigned)(((2 * g.c + 31) / 32) * g.n)), dim3(256), 0, st, part, g.chunks,
                       2 * g.c, csum);
    rc = vspw_launch_status();
    if (rc != VSPW_OK) return rc;
    hipLaunchKernelGGL((gn_bwd_apply_kernel<T, V>), grid, dim3(256), 0, st, (const T*)x, (const T*)dy, (T*)dx, g, stats, w, b,
                       act, dr, csum, dw, db);
    return vspw_launch_status();
}

static bool gn_grid_ok(const GnShape& g) {
    return (long long)g.slabs * g.chunks * g.n <= 0x7fffffffLL && (long long)((2LL * g.c + 31) / 32) * g.n <= 0x7fffffffLL;
}

extern "C" int vspw_group_norm_fwd(const void* x, void* y, int n, long long hw, int c, int groups, int dtype, const float* w,
                                   const float* b, float eps, int act, double p, const long long* rng, int channelwise,
                                   double* stats, void* ws, size_t ws_bytes, void* stream) {
    GnDrop dr;
    if (!x || !y || !gn_shape_ok(n, hw, c, groups, dtype) || !(eps >= 0.f) || !gn_args(act, p, rng, channelwise, dr))
        return VSPW_EINVAL;
    const GnShape g = gn_plan(n, hw, c, groups, dtype);
    if (!gn_grid_ok(g) || !ws || ws_bytes < vspw_group_norm_fwd_workspace(n, hw, c, groups, dtype)) return VSPW_EINVAL;
    const bool vec = gn_vec(c, dtype) > 1;
    if (vec && (((uintptr_t)x | (uintptr_t)y) & 15)) return VSPW_EINVAL;
    double* part = reinterpret_cast<double*>(ws);
    hipStream_t st = vspw_stream(stream);
#define GN_FWD(T, V) gn_fwd_launch<T, V>(x, y, g, w, b, eps, act, dr, stats, part, st)
    if (dtype == VSPW_F32) return vec ? GN_FWD(float, 4) : GN_FWD(float, 1);
    if (dtype == VSPW_BF16) return vec ? GN_FWD(bf16_t, 8) : GN_FWD(bf16_t, 1);
    return vec ? GN_FWD(f16_t, 8) : GN_FWD(f16_t, 1);
#undef GN_FWD
}

extern "C" int vspw_group_norm_bwd(const void* x, const void* dy, void* dx, int n, long long hw, int c, int groups, int dtype,
                                   const float* w, const float* b, int act, double p, const long long* rng, int channelwise,
                                   const double* stats, float* dw, float* db, void* ws, size_t ws_bytes, void* stream) {
    GnDrop dr;
    if (!x || !dy || !stats || !gn_shape_ok(n, hw, c, groups, dtype) || !gn_args(act, p, rng, channelwise, dr))
        return VSPW_EINVAL;
    const GnShape g = gn_plan(n, hw, c, groups, dtype);
    if (!gn_grid_ok(g) || !ws || ws_bytes < vspw_group_norm_bwd_workspace(n, hw, c, groups, dtype)) return VSPW_EINVAL;
    const bool vec = gn_vec(c, dtype) > 1;
    if (vec && (((uintptr_t)x | (uintptr_t)dy | (uintptr_t)dx) & 15)) return VSPW_EINVAL;
    double* part = reinterpret_cast<double*>(ws);
    hipStream_t st = vspw_stream(stream);
#define GN_BWD(T, V) gn_bwd_launch<T, V>(x, dy, dx, g, w, b, act, dr, stats, dw, db, part, st)
    if (dtype == VSPW_F32) return vec ? GN_BWD(float, 4) : GN_BWD(float, 1);
    if (dtype == VSPW_BF16) return vec ? GN_BWD(bf16_t, 8) : GN_BWD(bf16_t, 1);
    return vec ? GN_BWD(f16_t, 8) : GN_BWD(f16_t, 1);
#undef GN_BWD
}
