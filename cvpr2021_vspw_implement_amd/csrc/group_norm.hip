// Group normalisation with activation and dropout on channels-last activations [n][hw][c], fp32 / bf16 / fp16.
//
//   forward    mean, var over (hw, channels of a group);  a = w (x - mean) / sqrt(var + eps) + b;  y = drop(act(a))
//   backward   da = dy drop'(.) act'(a);  db = sum da;  dw = sum da xhat;  t = da w;
//              dx = rstd (t - mean(t) - xhat mean(t xhat))     (means over the group)
//
// Sums are fp32 over four terms at a time and fp64 from there on, on values less the group's first element, so that a mean far
// from zero costs no digits.  The mean enters the fp32 arithmetic as two terms; ReLU's border is decided on the fp64
// pre-activation (the same in both directions).  All sums have a fixed order: results are bit-reproducible.
//
// Large images: streaming kernels, stats -> finish -> apply and bwd_stats -> bwd_reduce -> bwd_apply, bound by HBM.
// [10,512,60,60] fp32 (74 MB), ReLU, dropout: 26 (2.8 TB/s, x comes from memory) + 4 + 28 us (5.3 TB/s), 30 (5.0) + 5 + 38 us
// (5.9 TB/s); [4,256,119,119] bf16 (29 MB), SiLU: 12 + 4 + 16, 21 + 5 + 21 us.  The two small kernels cost a launch each.  Images whose
// groups fit the registers of a workgroup: one workgroup per image and group, which reads its elements once.
#include <type_traits>

#include "elem.h"

enum { ACT_NONE = 0, ACT_RELU = 1, ACT_SILU = 2, ACT_GELU = 3 };

struct GnShape {
    long long hw;
    int n, c, groups, cpg;  // cpg: channels per group
    int tx, slabs, chunks;  // streaming kernels
    int fx;                 // vectors per pixel of a group
    bool group;             // one workgroup per image and group
};
// Where a streaming workgroup stands.
struct GnPlace {
    int slab, chunk, img;
    __device__ __forceinline__ GnPlace(const GnShape& g) {
        slab = blockIdx.x % g.slabs;
        const int rest = blockIdx.x / g.slabs;
        chunk = rest % g.chunks;
        img = rest / g.chunks;
    }
};

// 1 / (1 + exp(-a)): the rounding of the exponent's argument is carried along, 2 units in the last place
__device__ __forceinline__ float sigmoid(float a) {
    const float L = -1.44269504088896340736f, hi = a * L;
    const float e = __builtin_amdgcn_exp2f(hi), rest = fmaf(a, L, -hi);
    return __builtin_amdgcn_rcpf(1.f + (fabsf(hi) < 128.f ? fmaf(e, rest * 0.69314718f, e) : e));
}
template <int ACT>
__device__ __forceinline__ float act_value(float a) {
    if (ACT == ACT_RELU) return a > 0.f ? a : (a != a ? a : 0.f);
    if (ACT == ACT_SILU) return a * sigmoid(a);
    if (ACT == ACT_GELU) return 0.5f * a * erfcf(-a * 0.70710678118654752f);
    return a;
}
template <int ACT>
__device__ __forceinline__ float act_slope(float a) {
    if (ACT == ACT_RELU) return a > 0.f ? 1.f : (a != a ? a : 0.f);
    if (ACT == ACT_SILU) {
        const float s = sigmoid(a);
        return s * (1.f + a * (1.f - s));
    }
    if (ACT == ACT_GELU) return 0.5f * erfcf(-a * 0.70710678118654752f) + a * 0.39894228040143268f * expf(-0.5f * a * a);
    return 1.f;
}

// What a thread keeps of one channel, and the pre-activation of an element of it.
template <int ACT>
struct Channel {
    float mh, ml, r, w, b;  // mean = mh + ml, 1 / sqrt(var + eps), weight, bias
    double A, B;            // ReLU: pre-activation = A x + B in fp64
    __device__ __forceinline__ void set(double mean, double rstd, float weight, float bias) {
        mh = (float)mean;
        ml = (float)(mean - (double)mh);
        r = (float)rstd;
        w = weight;
        b = bias;
        A = rstd * (double)weight;
        B = (double)bias - mean * A;
    }
    __device__ __forceinline__ float xhat(float x) const { return ((x - mh) - ml) * r; }
    __device__ __forceinline__ float pre(float x, float xh) const {
        return ACT == ACT_RELU ? (float)fma((double)x, A, B) : fmaf(xh, w, b);
    }
};

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

// Calls run(p, U) for U pixels at a time and run(p, 1) for the rest, so that U loads of every tensor are in flight.
template <int U, typename F>
__device__ __forceinline__ void walk(long long p, long long step, long long hw, F run) {
    for (; p + (U - 1) * step < hw; p += U * step) run(p, std::integral_constant<int, U>());
    for (; p < hw; p += step) run(p, std::integral_constant<int, 1>());
}

// part[img][chunk][slab][k][2]: sum and sum of squares of x - x0 over the chunk's pixels of the slab's share of group (first
// group of the slab + k); gs entries per slab.  x0 = the group's first element.
template <typename T, int V>
__global__ __launch_bounds__(256) void gn_stats_kernel(const T* __restrict__ x, GnShape g, int gs, double* __restrict__ part) {
    __shared__ double red[2][256 * V];
    const GnPlace at(g);
    const int c0 = (at.slab * g.tx + (int)threadIdx.x % g.tx) * V;
    const int ty = 256 / g.tx;
    double s[V], q[V];
#pragma unroll
    for (int e = 0; e < V; ++e) s[e] = q[e] = 0.0;
    if (c0 < g.c) {
        const T* xi = x + (size_t)at.img * g.hw * g.c;
        float x0[V];
#pragma unroll
        for (int e = 0; e < V; ++e) x0[e] = (float)xi[(c0 + e) / g.cpg * g.cpg];
        const long long step = (long long)g.chunks * ty;
        walk<4>((long long)at.chunk * ty + threadIdx.x / g.tx, step, g.hw, [&](long long p, auto nn) {
            constexpr int N = decltype(nn)::value;
            float f[N][V];
#pragma unroll
            for (int i = 0; i < N; ++i) Vec<T, V>::load(xi + c0 + (size_t)(p + i * step) * g.c, f[i]);
#pragma unroll
            for (int e = 0; e < V; ++e) {
                float a = 0.f, b = 0.f;
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    const float d = f[i][e] - x0[e];
                    a += d;
                    b = fmaf(d, d, b);
                }
                s[e] += (double)a;
                q[e] += (double)b;
            }
        });
    }
    reduce_pixels<V>(s, q, red, g.tx);
    const int first = at.slab * g.tx * V, last = min(g.c, first + g.tx * V);
    const int g0 = first / g.cpg, g1 = (last - 1) / g.cpg;
    for (int k = threadIdx.x; k <= g1 - g0; k += 256) {
        const int lo = max(first, (g0 + k) * g.cpg), hi = min(last, (g0 + k + 1) * g.cpg);
        double a = 0, b = 0;
        for (int ch = lo; ch < hi; ++ch) {
            a += red[0][ch - first];
            b += red[1][ch - first];
        }
        double* o = part + ((((size_t)at.img * g.chunks + at.chunk) * g.slabs + at.slab) * gs + k) * 2;
        o[0] = a;
        o[1] = b;
    }
}

// stats[img][group] = mean, 1/sqrt(var + eps): one wave per image and group sums the entries of all chunks and of the slabs
// that share the group, in a fixed order.  (Every workgroup of the apply kernel doing it for itself read 0.5 GB of partial
// sums at [4,256,119,119]: 32 us where this and the bare apply kernel take 20.)
template <typename T>
__global__ __launch_bounds__(256) void gn_finish_kernel(const T* __restrict__ x, const double* __restrict__ part, GnShape g,
                                                        int gs, int slabw, float eps, double* __restrict__ stats) {
    const long long id = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (id >= (long long)g.n * g.groups) return;
    const int img = (int)(id / g.groups), gr = (int)(id % g.groups), lane = threadIdx.x & 63;
    const int s0 = gr * g.cpg / slabw, ns = ((gr + 1) * g.cpg - 1) / slabw - s0 + 1;
    double a = 0, b = 0;
#pragma unroll 4
    for (int i = lane; i < g.chunks * ns; i += 64) {
        const int sl = s0 + i % ns;
        const double* o = part + ((((size_t)img * g.chunks + i / ns) * g.slabs + sl) * gs + (gr - sl * slabw / g.cpg)) * 2;
        a += o[0];
        b += o[1];
    }
    a = wave_sum_d(a);
    b = wave_sum_d(b);
    if (lane == 0) {
        const double inv = 1.0 / ((double)g.hw * g.cpg), m = a * inv;
        const double var = b * inv - m * m;
        stats[2 * id] = m + (double)(float)x[(size_t)img * g.hw * g.c + (size_t)gr * g.cpg];
        stats[2 * id + 1] = 1.0 / sqrt((var < 0 ? 0 : var) + (double)eps);
    }
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

// The channel form's factors of a thread's channels (1 when there is none).
template <int V>
__device__ __forceinline__ void channel_drops(const Philox& gen, const GnDrop& dr, unsigned long long e0, float* ck) {
#pragma unroll
    for (int e = 0; e < V; ++e) {
        ck[e] = 1.f;
        if (dr.mode == 2) {
            unsigned u;
            gen.run<1>(e0 + e, &u);
            ck[e] = dr.rule.factor(u);
        }
    }
}

template <typename T, int V, int ACT>
__global__ __launch_bounds__(256) void gn_apply_kernel(const T* __restrict__ x, T* __restrict__ y, GnShape g,
                                                       const float* __restrict__ w, const float* __restrict__ b, GnDrop dr,
                                                       const double* __restrict__ stats) {
    const GnPlace at(g);
    const int c0 = (at.slab * g.tx + (int)threadIdx.x % g.tx) * V;
    if (c0 >= g.c) return;
    const int ty = 256 / g.tx;
    Channel<ACT> ch[V];
    float ck[V];
    const Philox gen(dr.rng);
#pragma unroll
    for (int e = 0; e < V; ++e) {
        const double* st = stats + ((size_t)at.img * g.groups + (c0 + e) / g.cpg) * 2;
        ch[e].set(st[0], st[1], w ? w[c0 + e] : 1.f, b ? b[c0 + e] : 0.f);
    }
    channel_drops<V>(gen, dr, (unsigned long long)at.img * g.c + c0, ck);
    const size_t base = (size_t)at.img * g.hw * g.c + c0;
    const long long step = (long long)g.chunks * ty;
    walk<4>((long long)at.chunk * ty + threadIdx.x / g.tx, step, g.hw, [&](long long p, auto nn) {
        constexpr int N = decltype(nn)::value;
        float f[N][V];
#pragma unroll
        for (int i = 0; i < N; ++i) Vec<T, V>::load(x + base + (size_t)(p + i * step) * g.c, f[i]);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const size_t e0 = base + (size_t)(p + i * step) * g.c;
            float k[V];
            drop_factors<V>(gen, dr.rule, dr.mode, e0, ck, k);
#pragma unroll
            for (int e = 0; e < V; ++e) f[i][e] = drop_apply(act_value<ACT>(ch[e].pre(f[i][e], ch[e].xhat(f[i][e]))), k[e]);
            Vec<T, V>::store(y + e0, f[i]);
        }
    });
}

// da of one element and its xhat
template <int ACT>
__device__ __forceinline__ float gn_da(const Channel<ACT>& ch, float x, float dy, float k, float& xh) {
    xh = ch.xhat(x);
    return drop_apply(dy, k) * act_slope<ACT>(ch.pre(x, xh));
}

// part[img][chunk][2][c]: sum da, sum da xhat over the chunk's pixels
template <typename T, int V, int ACT>
__global__ __launch_bounds__(256) void gn_bwd_stats_kernel(const T* __restrict__ x, const T* __restrict__ dy, GnShape g,
                                                           const double* __restrict__ stats, const float* __restrict__ w,
                                                           const float* __restrict__ b, GnDrop dr, double* __restrict__ part) {
    __shared__ double red[2][256 * V];
    const GnPlace at(g);
    const int first = at.slab * g.tx * V;
    const int c0 = first + ((int)threadIdx.x % g.tx) * V;
    const int ty = 256 / g.tx;
    double s[V], q[V];
#pragma unroll
    for (int e = 0; e < V; ++e) s[e] = q[e] = 0.0;
    if (c0 < g.c) {
        Channel<ACT> ch[V];
        float ck[V];
        const Philox gen(dr.rng);
#pragma unroll
        for (int e = 0; e < V; ++e) {
            const double* st = stats + ((size_t)at.img * g.groups + (c0 + e) / g.cpg) * 2;
            ch[e].set(st[0], st[1], w ? w[c0 + e] : 1.f, b ? b[c0 + e] : 0.f);
        }
        channel_drops<V>(gen, dr, (unsigned long long)at.img * g.c + c0, ck);
        const size_t base = (size_t)at.img * g.hw * g.c + c0;
        const long long step = (long long)g.chunks * ty;
        walk<2>((long long)at.chunk * ty + threadIdx.x / g.tx, step, g.hw, [&](long long p, auto nn) {
            constexpr int N = decltype(nn)::value;
            float f[N][V], d[N][V], sa[V], sq[V];
#pragma unroll
            for (int i = 0; i < N; ++i) {
                Vec<T, V>::load(x + base + (size_t)(p + i * step) * g.c, f[i]);
                Vec<T, V>::load(dy + base + (size_t)(p + i * step) * g.c, d[i]);
            }
#pragma unroll
            for (int e = 0; e < V; ++e) sa[e] = sq[e] = 0.f;
#pragma unroll
            for (int i = 0; i < N; ++i) {
                float k[V];
                drop_factors<V>(gen, dr.rule, dr.mode, base + (size_t)(p + i * step) * g.c, ck, k);
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    float xh;
                    const float da = gn_da(ch[e], f[i][e], d[i][e], k[e], xh);
                    sa[e] += da;
                    sq[e] = fmaf(da, xh, sq[e]);
                }
            }
#pragma unroll
            for (int e = 0; e < V; ++e) {
                s[e] += (double)sa[e];
                q[e] += (double)sq[e];
            }
        });
    }
    reduce_pixels<V>(s, q, red, g.tx);
    for (int i = threadIdx.x; i < g.tx * V; i += 256)
        if (first + i < g.c) {
            double* o = part + ((size_t)at.img * g.chunks + at.chunk) * 2 * g.c + first + i;
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

// dw, db of channels [first, last): the images' sums, in image order
__device__ __forceinline__ void parameter_gradients(const double* __restrict__ csum, const GnShape& g, int first, int last,
                                                    float* __restrict__ dw, float* __restrict__ db) {
    for (int ch = first + threadIdx.x; ch < last; ch += blockDim.x) {
        double a = 0, q = 0;
        for (int i = 0; i < g.n; ++i) {
            a += csum[(size_t)i * 2 * g.c + ch];
            q += csum[((size_t)i * 2 + 1) * g.c + ch];
        }
        if (db) db[ch] = (float)a;
        if (dw) dw[ch] = (float)q;
    }
}
__global__ __launch_bounds__(256) void gn_params_kernel(const double* __restrict__ csum, GnShape g, float* __restrict__ dw,
                                                        float* __restrict__ db) {
    parameter_gradients(csum, g, blockIdx.x * 256, min(g.c, (int)blockIdx.x * 256 + 256), dw, db);
}

template <typename T, int V, int ACT>
__global__ __launch_bounds__(256) void gn_bwd_apply_kernel(const T* __restrict__ x, const T* __restrict__ dy,
                                                           T* __restrict__ dx, GnShape g, const double* __restrict__ stats,
                                                           const float* __restrict__ w, const float* __restrict__ b, GnDrop dr,
                                                           const double* __restrict__ csum, float* __restrict__ dw,
                                                           float* __restrict__ db) {
    __shared__ double ts[2 * 64 * V];
    const GnPlace at(g);
    const int first = at.slab * g.tx * V, last = min(g.c, first + g.tx * V);
    if (at.img == 0 && at.chunk == 0) parameter_gradients(csum, g, first, last, dw, db);
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
                a = fma(wt, csum[(size_t)at.img * 2 * g.c + ch], a);
                q = fma(wt, csum[((size_t)at.img * 2 + 1) * g.c + ch], q);
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
    Channel<ACT> ch[V];
    float T1[V], T2[V], ck[V];
    const Philox gen(dr.rng);
#pragma unroll
    for (int e = 0; e < V; ++e) {
        const int gr = (c0 + e) / g.cpg;
        const double* st = stats + ((size_t)at.img * g.groups + gr) * 2;
        ch[e].set(st[0], st[1], w ? w[c0 + e] : 1.f, b ? b[c0 + e] : 0.f);
        T1[e] = (float)ts[2 * (gr - g0)];
        T2[e] = (float)ts[2 * (gr - g0) + 1];
    }
    channel_drops<V>(gen, dr, (unsigned long long)at.img * g.c + c0, ck);
    const size_t base = (size_t)at.img * g.hw * g.c + c0;
    const long long step = (long long)g.chunks * ty;
    walk<2>((long long)at.chunk * ty + threadIdx.x / g.tx, step, g.hw, [&](long long p, auto nn) {
        constexpr int N = decltype(nn)::value;
        float f[N][V], d[N][V];
#pragma unroll
        for (int i = 0; i < N; ++i) {
            Vec<T, V>::load(x + base + (size_t)(p + i * step) * g.c, f[i]);
            Vec<T, V>::load(dy + base + (size_t)(p + i * step) * g.c, d[i]);
        }
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const size_t e0 = base + (size_t)(p + i * step) * g.c;
            float k[V];
            drop_factors<V>(gen, dr.rule, dr.mode, e0, ck, k);
#pragma unroll
            for (int e = 0; e < V; ++e) {
                float xh;
                const float da = gn_da(ch[e], f[i][e], d[i][e], k[e], xh);
                f[i][e] = ch[e].r * (fmaf(da, ch[e].w, -T1[e]) - xh * T2[e]);
            }
            Vec<T, V>::store(dx + e0, f[i]);
        }
    });
}

// ---- one workgroup per image and group ----
// sums of a and b over the workgroup, the same in every thread
template <int THREADS>
__device__ __forceinline__ void block_sum2(double& a, double& b, double (*red)[THREADS / 64]) {
    a = wave_sum_d(a);
    b = wave_sum_d(b);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) {
        red[0][threadIdx.x >> 6] = a;
        red[1][threadIdx.x >> 6] = b;
    }
    __syncthreads();
    a = b = 0;
#pragma unroll
    for (int i = 0; i < THREADS / 64; ++i) {
        a += red[0][i];
        b += red[1][i];
    }
}

// Which elements of the group a thread holds: channel vector `vec` of pixels p0, p0 + step, ...
template <int V>
struct GnHold {
    int img, c0;
    long long p0, step;
    size_t base;
    bool on;
    __device__ __forceinline__ GnHold(const GnShape& g, int threads) {
        const int id = xcd_remap(blockIdx.x, gridDim.x);  // neighbouring groups share cache lines: keep them on one XCD
        img = id / g.groups;
        const int ty = threads / g.fx;
        on = (int)threadIdx.x < ty * g.fx;
        c0 = id % g.groups * g.cpg + (int)threadIdx.x % g.fx * V;
        p0 = (int)threadIdx.x / g.fx;
        step = ty;
        base = (size_t)img * g.hw * g.c + c0;
    }
};

template <typename T, int V, int ACT, int TRIPS, int THREADS>
__global__ __launch_bounds__(THREADS) void gn_group_kernel(const T* __restrict__ x, T* __restrict__ y, GnShape g,
                                                           const float* __restrict__ w, const float* __restrict__ b, float eps,
                                                           GnDrop dr, double* __restrict__ stats) {
    typedef typename Raw<T, V>::type R;
    __shared__ double red[2][THREADS / 64];
    const GnHold<V> at(g, THREADS);
    R v[TRIPS];
#pragma unroll
    for (int i = 0; i < TRIPS; ++i)
        if (at.on && at.p0 + i * at.step < g.hw) v[i] = *reinterpret_cast<const R*>(x + at.base + (size_t)(at.p0 + i * at.step) * g.c);
    // mean, then the squares of the deviations: both from the registers
    const double inv = 1.0 / ((double)g.hw * g.cpg);
    double a = 0, none = 0;
#pragma unroll
    for (int i = 0; i < TRIPS; ++i)
        if (at.on && at.p0 + i * at.step < g.hw) {
            float f[V], s = 0.f;
            Raw<T, V>::floats(v[i], f);
            if (V > 1) {
#pragma unroll
                for (int e = 0; e < V; ++e) a += (double)f[e];
            } else {
                s = f[0];
                a += (double)s;
            }
        }
    block_sum2<THREADS>(a, none, red);
    const double mean = a * inv;
    const float mh = (float)mean, ml = (float)(mean - (double)mh);
    double q = 0;
    none = 0;
#pragma unroll
    for (int i = 0; i < TRIPS; ++i)
        if (at.on && at.p0 + i * at.step < g.hw) {
            float f[V], s = 0.f;
            Raw<T, V>::floats(v[i], f);
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const float d = (f[e] - mh) - ml;
                s = fmaf(d, d, s);
            }
            q += (double)s;
        }
    block_sum2<THREADS>(q, none, red);
    const double rstd = 1.0 / sqrt(q * inv + (double)eps);
    if (stats && threadIdx.x == 0) {
        const size_t k = (size_t)at.img * g.groups + at.c0 / g.cpg;
        stats[2 * k] = mean;
        stats[2 * k + 1] = rstd;
    }
    if (!at.on) return;
    Channel<ACT> ch[V];
    float ck[V];
    const Philox gen(dr.rng);
#pragma unroll
    for (int e = 0; e < V; ++e) ch[e].set(mean, rstd, w ? w[at.c0 + e] : 1.f, b ? b[at.c0 + e] : 0.f);
    channel_drops<V>(gen, dr, (unsigned long long)at.img * g.c + at.c0, ck);
#pragma unroll
    for (int i = 0; i < TRIPS; ++i)
        if (at.p0 + i * at.step < g.hw) {
            const size_t e0 = at.base + (size_t)(at.p0 + i * at.step) * g.c;
            float f[V], k[V];
            Raw<T, V>::floats(v[i], f);
            drop_factors<V>(gen, dr.rule, dr.mode, e0, ck, k);
#pragma unroll
            for (int e = 0; e < V; ++e) f[e] = drop_apply(act_value<ACT>(ch[e].pre(f[e], ch[e].xhat(f[e]))), k[e]);
            Vec<T, V>::store(y + e0, f);
        }
}

template <typename T, int V, int ACT, int TRIPS, int THREADS>
__global__ __launch_bounds__(THREADS) void gn_bwd_group_kernel(const T* __restrict__ x, const T* __restrict__ dy,
                                                               T* __restrict__ dx, GnShape g, const double* __restrict__ stats,
                                                               const float* __restrict__ w, const float* __restrict__ b,
                                                               GnDrop dr, double* __restrict__ csum, float* __restrict__ dw,
                                                               float* __restrict__ db) {
    typedef typename Raw<T, V>::type R;
    __shared__ double red[2][THREADS / 64];
    __shared__ float cs[2][THREADS * V];
    const GnHold<V> at(g, THREADS);
    const size_t kg = (size_t)at.img * g.groups + at.c0 / g.cpg;
    const double mean = stats[2 * kg], rstd = stats[2 * kg + 1];
    R vx[TRIPS], vd[TRIPS];
#pragma unroll
    for (int i = 0; i < TRIPS; ++i)
        if (at.on && at.p0 + i * at.step < g.hw) {
            const size_t e0 = at.base + (size_t)(at.p0 + i * at.step) * g.c;
            vx[i] = *reinterpret_cast<const R*>(x + e0);
            vd[i] = *reinterpret_cast<const R*>(dy + e0);
        }
    Channel<ACT> ch[V];
    float ck[V], sa[V], sq[V];
    const Philox gen(dr.rng);
#pragma unroll
    for (int e = 0; e < V; ++e) {
        sa[e] = sq[e] = 0.f;
        ch[e].set(mean, rstd, at.on && w ? w[at.c0 + e] : 1.f, at.on && b ? b[at.c0 + e] : 0.f);
    }
    channel_drops<V>(gen, dr, (unsigned long long)at.img * g.c + at.c0, ck);
#pragma unroll
    for (int i = 0; i < TRIPS; ++i)
        if (at.on && at.p0 + i * at.step < g.hw) {
            float f[V], d[V], k[V];
            Raw<T, V>::floats(vx[i], f);
            Raw<T, V>::floats(vd[i], d);
            drop_factors<V>(gen, dr.rule, dr.mode, at.base + (size_t)(at.p0 + i * at.step) * g.c, ck, k);
#pragma unroll
            for (int e = 0; e < V; ++e) {
                float xh;
                const float da = gn_da(ch[e], f[e], d[e], k[e], xh);
                sa[e] += da;  // at most TRIPS terms in fp32
                sq[e] = fmaf(da, xh, sq[e]);
            }
        }
    // per channel over the pixel lanes (fp64, fixed order), then over the group's channels with their weights
#pragma unroll
    for (int e = 0; e < V; ++e) {
        cs[0][threadIdx.x * V + e] = sa[e];
        cs[1][threadIdx.x * V + e] = sq[e];
    }
    __syncthreads();
    double t1 = 0, t2 = 0;
    const int ty = THREADS / g.fx;
    for (int i = threadIdx.x; i < g.cpg; i += THREADS) {
        double a = 0, q = 0;
        for (int r = 0; r < ty; ++r) {
            a += (double)cs[0][r * g.cpg + i];
            q += (double)cs[1][r * g.cpg + i];
        }
        const int c = (int)(kg % g.groups) * g.cpg + i;
        if (g.n == 1) {
            if (db) db[c] = (float)a;
            if (dw) dw[c] = (float)q;
        } else {
            csum[(size_t)at.img * 2 * g.c + c] = a;
            csum[((size_t)at.img * 2 + 1) * g.c + c] = q;
        }
        const double wt = w ? (double)w[c] : 1.0;
        t1 = fma(wt, a, t1);
        t2 = fma(wt, q, t2);
    }
    if (!dx) return;
    block_sum2<THREADS>(t1, t2, red);
    const double inv = 1.0 / ((double)g.hw * g.cpg);
    const float T1 = (float)(t1 * inv), T2 = (float)(t2 * inv);
    if (!at.on) return;
#pragma unroll
    for (int i = 0; i < TRIPS; ++i)
        if (at.p0 + i * at.step < g.hw) {
            const size_t e0 = at.base + (size_t)(at.p0 + i * at.step) * g.c;
            float f[V], d[V], k[V];
            Raw<T, V>::floats(vx[i], f);
            Raw<T, V>::floats(vd[i], d);
            drop_factors<V>(gen, dr.rule, dr.mode, e0, ck, k);
#pragma unroll
            for (int e = 0; e < V; ++e) {
                float xh;
                const float da = gn_da(ch[e], f[e], d[e], k[e], xh);
                f[e] = ch[e].r * (fmaf(da, ch[e].w, -T1) - xh * T2);
            }
            Vec<T, V>::store(dx + e0, f);
        }
}

// ------------------------------------------------------------------------------------------------------------- host
static bool gn_shape_ok(int n, long long hw, int c, int groups, int dtype) {
    return n > 0 && hw > 0 && c > 0 && groups > 0 && c % groups == 0 && vspw_dtype_ok(dtype) &&
           hw <= (0x7fffffffffffffffLL / n) / c / 8;
}
// Four elements per access where rows (for the group kernels: groups) allow it.  (Eight 16-bit elements need twice the
// registers per thread: [4,256,119,119] bf16 84 us in the four streaming kernels, four elements 69 us.)  The plan is a
// function of the shape alone.
static int gn_vec(int c) { return c % 4 == 0 ? 4 : 1; }
#define GN_TRIPS 4
#define GN_THREADS 256
static GnShape gn_plan(int n, long long hw, int c, int groups) {
    const SlabPlan s = vspw_slab_plan(n, hw, c, gn_vec(c), 8, 1024);
    GnShape g;
    g.hw = hw;
    g.n = n;
    g.c = c;
    g.groups = groups;
    g.cpg = c / groups;
    g.tx = s.tx;
    g.slabs = s.slabs;
    g.chunks = s.chunks;
    const int v = gn_vec(g.cpg);
    g.fx = g.cpg / v;
    // Where it fits, one workgroup per image and group is one launch instead of three ([2,512,6,6]: 4.6 us against 12.6).  The
    // same with 1024 threads for images up to 64 x 64 lost: [10,512,60,60] 61 us against 58 (320 workgroups on 256 CUs).
    g.group = g.fx <= GN_THREADS && hw <= (long long)GN_TRIPS * (GN_THREADS / g.fx) && (long long)n * groups <= 0x7fffffffLL;
    return g;
}
static int gn_gs(const GnShape& g, int v) {  // groups that a slab can overlap
    const int w = g.tx * v;
    const int most = (w + g.cpg - 1) / g.cpg + 1;
    return most < g.groups ? most : g.groups;
}

extern "C" size_t vspw_group_norm_fwd_workspace(int n, long long hw, int c, int groups, int dtype) {
    if (!gn_shape_ok(n, hw, c, groups, dtype)) return 0;
    const GnShape g = gn_plan(n, hw, c, groups);
    if (g.group) return 0;
    return ((size_t)n * g.chunks * g.slabs * gn_gs(g, gn_vec(c)) + (size_t)n * groups) * 2 * sizeof(double);
}

extern "C" size_t vspw_group_norm_bwd_workspace(int n, long long hw, int c, int groups, int dtype) {
    if (!gn_shape_ok(n, hw, c, groups, dtype)) return 0;
    const GnShape g = gn_plan(n, hw, c, groups);
    return (size_t)n * ((g.group ? 0 : g.chunks) + 1) * 2 * c * sizeof(double);
}

struct GnCall {
    const void *x, *dy;
    void* out;  // y or dx
    GnShape g;
    const float *w, *b;
    float eps;
    int act;
    GnDrop dr;
    double *stats, *ws;
    float *dw, *db;
    hipStream_t st;
};
static bool gn_args(int act, double p, const long long* rng, int channelwise, GnDrop& dr) {
    if (act < ACT_NONE || act > ACT_GELU || !(p >= 0.0 && p <= 1.0) || (p > 0.0 && !rng)) return false;
    dr.rule = DropRule::of(p);
    dr.mode = p > 0.0 ? (channelwise ? 2 : 1) : 0;
    dr.rng = p > 0.0 ? rng : nullptr;
    return true;
}

template <typename T, int V, int ACT>
static int gn_fwd_launch(const GnCall& a) {
    const int gs = gn_gs(a.g, V);
    const dim3 grid((unsigned)(a.g.slabs * a.g.chunks * a.g.n));
    hipLaunchKernelGGL((gn_stats_kernel<T, V>), grid, dim3(256), 0, a.st, (const T*)a.x, a.g, gs, a.ws);
    int rc = vspw_launch_status();
    if (rc != VSPW_OK) return rc;
    double* stats = a.stats ? a.stats : a.ws + (size_t)a.g.n * a.g.chunks * a.g.slabs * gs * 2;
    const long long groups = (long long)a.g.n * a.g.groups;
    hipLaunchKernelGGL((gn_finish_kernel<T>), dim3((unsigned)((groups + 3) / 4)), dim3(256), 0, a.st, (const T*)a.x, a.ws, a.g, gs,
                       a.g.tx * V, a.eps, stats);
    rc = vspw_launch_status();
    if (rc != VSPW_OK) return rc;
    hipLaunchKernelGGL((gn_apply_kernel<T, V, ACT>), grid, dim3(256), 0, a.st, (const T*)a.x, (T*)a.out, a.g, a.w, a.b, a.dr, stats);
    return vspw_launch_status();
}
template <typename T, int V, int ACT>
static int gn_fwd_group_launch(const GnCall& a) {
    hipLaunchKernelGGL((gn_group_kernel<T, V, ACT, GN_TRIPS, GN_THREADS>), dim3((unsigned)(a.g.n * a.g.groups)), dim3(GN_THREADS), 0,
                       a.st, (const T*)a.x, (T*)a.out, a.g, a.w, a.b, a.eps, a.dr, a.stats);
    return vspw_launch_status();
}

template <typename T, int V, int ACT>
static int gn_bwd_launch(const GnCall& a) {
    const dim3 grid((unsigned)(a.g.slabs * a.g.chunks * a.g.n));
    double* csum = a.ws + (size_t)a.g.n * a.g.chunks * 2 * a.g.c;
    hipLaunchKernelGGL((gn_bwd_stats_kernel<T, V, ACT>), grid, dim3(256), 0, a.st, (const T*)a.x, (const T*)a.dy, a.g, a.stats, a.w,
                       a.b, a.dr, a.ws);
    int rc = vspw_launch_status();
    if (rc != VSPW_OK) return rc;
    hipLaunchKernelGGL(gn_bwd_reduce_kernel, dim3((unsigned)(((2 * a.g.c + 31) / 32) * a.g.n)), dim3(256), 0, a.st, a.ws, a.g.chunks,
                       2 * a.g.c, csum);
    rc = vspw_launch_status();
    if (rc != VSPW_OK) return rc;
    hipLaunchKernelGGL((gn_bwd_apply_kernel<T, V, ACT>), grid, dim3(256), 0, a.st, (const T*)a.x, (const T*)a.dy, (T*)a.out, a.g,
                       a.stats, a.w, a.b, a.dr, csum, a.dw, a.db);
    return vspw_launch_status();
}
template <typename T, int V, int ACT>
static int gn_bwd_group_launch(const GnCall& a) {
    hipLaunchKernelGGL((gn_bwd_group_kernel<T, V, ACT, GN_TRIPS, GN_THREADS>), dim3((unsigned)(a.g.n * a.g.groups)),
                       dim3(GN_THREADS), 0, a.st, (const T*)a.x, (const T*)a.dy, (T*)a.out, a.g, a.stats, a.w, a.b, a.dr, a.ws, a.dw,
                       a.db);
    const int rc = vspw_launch_status();
    if (rc != VSPW_OK || a.g.n == 1 || (!a.dw && !a.db)) return rc;
    hipLaunchKernelGGL(gn_params_kernel, dim3((unsigned)((a.g.c + 255) / 256)), dim3(256), 0, a.st, a.ws, a.g, a.dw, a.db);
    return vspw_launch_status();
}

template <typename T, int V, int ACT, bool GROUP, bool BWD>
static int gn_pick(const GnCall& a) {
    if constexpr (GROUP)
        return BWD ? gn_bwd_group_launch<T, V, ACT>(a) : gn_fwd_group_launch<T, V, ACT>(a);
    else
        return BWD ? gn_bwd_launch<T, V, ACT>(a) : gn_fwd_launch<T, V, ACT>(a);
}
template <typename T, int V, bool GROUP, bool BWD>
static int gn_act(const GnCall& a) {
    switch (a.act) {
        case ACT_RELU: return gn_pick<T, V, ACT_RELU, GROUP, BWD>(a);
        case ACT_SILU: return gn_pick<T, V, ACT_SILU, GROUP, BWD>(a);
        case ACT_GELU: return gn_pick<T, V, ACT_GELU, GROUP, BWD>(a);
        default: return gn_pick<T, V, ACT_NONE, GROUP, BWD>(a);
    }
}
template <typename T, bool BWD>
static int gn_type(const GnCall& a, int v, int vg) {
    if (a.g.group) return vg > 1 ? gn_act<T, 4, true, BWD>(a) : gn_act<T, 1, true, BWD>(a);
    return v > 1 ? gn_act<T, 4, false, BWD>(a) : gn_act<T, 1, false, BWD>(a);
}
template <bool BWD>
static int gn_dispatch(const GnCall& a, int dtype) {
    const int v = gn_vec(a.g.c), vg = gn_vec(a.g.cpg);
    if ((long long)a.g.slabs * a.g.chunks * a.g.n > 0x7fffffffLL || ((2LL * a.g.c + 31) / 32) * a.g.n > 0x7fffffffLL) return VSPW_EINVAL;
    if (v > 1 && (((uintptr_t)a.x | (uintptr_t)a.dy | (uintptr_t)a.out) & 15)) return VSPW_EINVAL;  // storage on 16 bytes
    if (dtype == VSPW_F32) return gn_type<float, BWD>(a, v, vg);
    if (dtype == VSPW_BF16) return gn_type<bf16_t, BWD>(a, v, vg);
    return gn_type<f16_t, BWD>(a, v, vg);
}

extern "C" int vspw_group_norm_fwd(const void* x, void* y, int n, long long hw, int c, int groups, int dtype, const float* w,
                                   const float* b, float eps, int act, double p, const long long* rng, int channelwise,
                                   double* stats, void* ws, size_t ws_bytes, void* stream) {
    GnCall a = GnCall();
    if (!x || !y || !gn_shape_ok(n, hw, c, groups, dtype) || !(eps >= 0.f) || !gn_args(act, p, rng, channelwise, a.dr))
        return VSPW_EINVAL;
    a.g = gn_plan(n, hw, c, groups);
    const size_t need = vspw_group_norm_fwd_workspace(n, hw, c, groups, dtype);
    if (ws_bytes < need || (need && !ws)) return VSPW_EINVAL;
    a.x = x;
    a.out = y;
    a.w = w;
    a.b = b;
    a.eps = eps;
    a.act = act;
    a.stats = stats;
    a.ws = reinterpret_cast<double*>(ws);
    a.st = vspw_stream(stream);
    return gn_dispatch<false>(a, dtype);
}

extern "C" int vspw_group_norm_bwd(const void* x, const void* dy, void* dx, int n, long long hw, int c, int groups, int dtype,
                                   const float* w, const float* b, int act, double p, const long long* rng, int channelwise,
                                   const double* stats, float* dw, float* db, void* ws, size_t ws_bytes, void* stream) {
    GnCall a = GnCall();
    if (!x || !dy || !stats || !gn_shape_ok(n, hw, c, groups, dtype) || !gn_args(act, p, rng, channelwise, a.dr))
        return VSPW_EINVAL;
    a.g = gn_plan(n, hw, c, groups);
    if (!ws || ws_bytes < vspw_group_norm_bwd_workspace(n, hw, c, groups, dtype)) return VSPW_EINVAL;
    a.x = x;
    a.dy = dy;
    a.out = dx;
    a.w = w;
    a.b = b;
    a.act = act;
    a.stats = const_cast<double*>(stats);
    a.dw = dw;
    a.db = db;
    a.ws = reinterpret_cast<double*>(ws);
    a.st = vspw_stream(stream);
    return gn_dispatch<true>(a, dtype);
}
