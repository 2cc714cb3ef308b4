// Dropout from a counter-based generator: y = x * keep / (1 - p), the mask is recomputed from (seed, offset, index) wherever
// it is needed and never stored.  Element form (one 32-bit word per element, counted in memory order) and channel form (one
// word per image and channel: nn.Dropout2d).  The backward pass is the same call on the gradient.
//
// Bound: HBM (one read, one write).  The generator costs 20 32x32->64 multiplies per four elements.
// Measured: [2,4096,60,60] fp32, 118 MB in and out: 41 us, 5.7 TB/s; channel form, [10,2048,60,60] bf16, 147 MB in and out: 57 us,
// 5.2 TB/s.
#include "elem.h"

// Element form.  One trip handles 16 bytes (VEC) or the same elements one by one (ragged tail, unaligned storage).
template <typename T, bool VEC>
__global__ __launch_bounds__(256) void dropout_kernel(const T* __restrict__ x, T* __restrict__ y, long long n, DropRule d,
                                                      const long long* __restrict__ rng) {
    constexpr int V = 16 / (int)sizeof(T);
    const Philox g(rng);
    const long long trips = (n + V - 1) / V;
    for (long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x; i < trips; i += (long long)gridDim.x * blockDim.x) {
        const long long e0 = i * V;
        unsigned u[V];
        if (VEC && e0 + V <= n) {
            float f[V];
            Vec<T, V>::load(x + e0, f);
            g.run<V>((unsigned long long)e0, u);
#pragma unroll
            for (int e = 0; e < V; ++e) f[e] = drop_apply(f[e], d.factor(u[e]));
            Vec<T, V>::store(y + e0, f);
        } else {
            g.run<V>((unsigned long long)e0, u);
#pragma unroll
            for (int e = 0; e < V; ++e)
                if (e0 + e < n) y[e0 + e] = (T)drop_apply((float)x[e0 + e], d.factor(u[e]));
        }
    }
}

// Channel form on [n][hw][c]: a thread keeps its channels, so it asks the generator once.
template <typename T, int V>
__global__ __launch_bounds__(256) void dropout_channels_kernel(const T* __restrict__ x, T* __restrict__ y, long long hw,
                                                               int c, int tx, int slabs, int chunks, DropRule d,
                                                               const long long* __restrict__ rng) {
    const int slab = blockIdx.x % slabs;
    const int rest = blockIdx.x / slabs;
    const int chunk = rest % chunks, img = rest / chunks;
    const int c0 = (slab * tx + (int)threadIdx.x % tx) * V;
    if (c0 >= c) return;
    const int ty = 256 / tx;
    const Philox g(rng);
    float k[V];
#pragma unroll
    for (int e = 0; e < V; ++e) {
        unsigned u;
        g.run<1>((unsigned long long)img * c + c0 + e, &u);
        k[e] = d.factor(u);
    }
    const size_t base = (size_t)img * hw * c + c0;
#pragma unroll 4
    for (long long p = (long long)chunk * ty + threadIdx.x / tx; p < hw; p += (long long)chunks * ty) {
        float f[V];
        Vec<T, V>::load(x + base + (size_t)p * c, f);
#pragma unroll
        for (int e = 0; e < V; ++e) f[e] = drop_apply(f[e], k[e]);
        Vec<T, V>::store(y + base + (size_t)p * c, f);
    }
}

// offset state of a dropout module: used = state; state.offset += 1 (one thread; stream-ordered, so a replayed graph draws
// a new mask every time)
__global__ void rng_next_kernel(long long* state, long long* used) {
    used[0] = state[0];
    used[1] = state[1];
    state[1] += 1;
}

template <typename T>
static int dropout_launch(const void* x, void* y, long long n, long long hw, int c, DropRule d, const long long* rng,
                          bool channelwise, hipStream_t st) {
    constexpr int V = 16 / (int)sizeof(T);
    const T* xp = reinterpret_cast<const T*>(x);
    T* yp = reinterpret_cast<T*>(y);
    const bool aligned = (((uintptr_t)x | (uintptr_t)y) & 15) == 0;
    if (!channelwise) {
        const long long total = n * hw * c;
        // one trip per thread up to 2^16 workgroups: 236 MB in and out at 5.7 TB/s, 1024 workgroups of many trips 5.2 TB/s
        const long long trips = (total + V - 1) / V;
        const dim3 grid((unsigned)(trips < (256LL << 16) ? (trips + 255) / 256 : 1 << 16));
        if (aligned)
            hipLaunchKernelGGL((dropout_kernel<T, true>), grid, dim3(256), 0, st, xp, yp, total, d, rng);
        else
            hipLaunchKernelGGL((dropout_kernel<T, false>), grid, dim3(256), 0, st, xp, yp, total, d, rng);
        return vspw_launch_status();
    }
    const bool vec = aligned && c % V == 0;
    const SlabPlan s = vspw_slab_plan((int)n, hw, c, vec ? V : 1, 4, 4096);
    const long long blocks = (long long)s.slabs * s.chunks * n;
    if (blocks > 0x7fffffffLL) return VSPW_EINVAL;
    if (vec)
        hipLaunchKernelGGL((dropout_channels_kernel<T, V>), dim3((unsigned)blocks), dim3(256), 0, st, xp, yp, hw, c, s.tx,
                           s.slabs, s.chunks, d, rng);
    else
        hipLaunchKernelGGL((dropout_channels_kernel<T, 1>), dim3((unsigned)blocks), dim3(256), 0, st, xp, yp, hw, c, s.tx,
                           s.slabs, s.chunks, d, rng);
    return vspw_launch_status();
}

extern "C" int vspw_dropout(const void* x, void* y, long long n, long long hw, int c, int dtype, double p,
                            const long long* rng, int channelwise, void* stream) {
    if (!x || !y || !rng || n <= 0 || hw <= 0 || c <= 0 || !vspw_dtype_ok(dtype) || !(p >= 0.0 && p <= 1.0)) return VSPW_EINVAL;
    if (n > 0x7fffffffLL || hw > (0x7fffffffffffffffLL / n) / c) return VSPW_EINVAL;
    const DropRule d = DropRule::of(p);
    hipStream_t st = vspw_stream(stream);
    if (dtype == VSPW_F32) return dropout_launch<float>(x, y, n, hw, c, d, rng, channelwise != 0, st);
    if (dtype == VSPW_BF16) return dropout_launch<bf16_t>(x, y, n, hw, c, d, rng, channelwise != 0, st);
    return dropout_launch<f16_t>(x, y, n, hw, c, d, rng, channelwise != 0, st);
}

extern "C" int vspw_rng_next(long long* state, long long* used, void* stream) {
    if (!state || !used) return VSPW_EINVAL;
    hipLaunchKernelGGL(rng_next_kernel, dim3(1), dim3(1), 0, vspw_stream(stream), state, used);
    return vspw_launch_status();
}
