// Element types of the operators that take 16-bit activations next to fp32 (group norm, dropout, differential attention)
// and the counter-based generator the dropout masks come from.
#pragma once
#include <hip/hip_fp16.h>
#include "common.h"

typedef __bf16 bf16_t;
typedef _Float16 f16_t;

// V elements of type T <-> floats.  16-byte accesses when V * sizeof(T) == 16; V == 1 is the unaligned / ragged path.
// Rounding to 16 bits is round-to-nearest-even (hardware conversions).
template <typename T, int V>
struct Vec {
    typedef T type __attribute__((ext_vector_type(V)));
    static __device__ __forceinline__ void load(const T* p, float* f) {
        const type v = *reinterpret_cast<const type*>(p);
#pragma unroll
        for (int e = 0; e < V; ++e) f[e] = (float)v[e];
    }
    static __device__ __forceinline__ void store(T* p, const float* f) {
        type v;
#pragma unroll
        for (int e = 0; e < V; ++e) v[e] = (T)f[e];
        *reinterpret_cast<type*>(p) = v;
    }
};
template <typename T>
struct Vec<T, 1> {
    static __device__ __forceinline__ void load(const T* p, float* f) { f[0] = (float)p[0]; }
    static __device__ __forceinline__ void store(T* p, const float* f) { p[0] = (T)f[0]; }
};

// V elements as one register value, unpacked when they are used.
template <typename T, int V>
struct Raw {
    typedef T type __attribute__((ext_vector_type(V)));
    static __device__ __forceinline__ void floats(const type& v, float* f) {
#pragma unroll
        for (int e = 0; e < V; ++e) f[e] = (float)v[e];
    }
};
template <typename T>
struct Raw<T, 1> {
    typedef T type;
    static __device__ __forceinline__ void floats(const type& v, float* f) { f[0] = (float)v; }
};

// Philox4x32-10 (Salmon, Moraes, Dror, Shaw: "Parallel random numbers: as easy as 1, 2, 3", 2011): four independent
// 32-bit words per 128-bit counter (ctr, offset) under the 64-bit key `seed`.  A word is a function of its index alone, so
// forward and backward regenerate the same mask and nothing is stored.
struct Philox {
    unsigned k0, k1, o0, o1;
    __device__ __forceinline__ Philox(const long long* rng) {  // rng: (seed, offset) in device memory; NULL: unused
        const unsigned long long seed = rng ? (unsigned long long)rng[0] : 0ull, off = rng ? (unsigned long long)rng[1] : 0ull;
        k0 = (unsigned)seed;
        k1 = (unsigned)(seed >> 32);
        o0 = (unsigned)off;
        o1 = (unsigned)(off >> 32);
    }
    __device__ __forceinline__ void words(unsigned long long ctr, unsigned w[4]) const {
        unsigned x0 = (unsigned)ctr, x1 = (unsigned)(ctr >> 32), x2 = o0, x3 = o1, a = k0, b = k1;
#pragma unroll
        for (int r = 0; r < 10; ++r) {
            const unsigned long long p0 = (unsigned long long)x0 * 0xD2511F53u, p1 = (unsigned long long)x2 * 0xCD9E8D57u;
            x0 = (unsigned)(p1 >> 32) ^ x1 ^ a;
            x1 = (unsigned)p1;
            x2 = (unsigned)(p0 >> 32) ^ x3 ^ b;
            x3 = (unsigned)p0;
            a += 0x9E3779B9u;
            b += 0xBB67AE85u;
        }
        w[0] = x0;
        w[1] = x1;
        w[2] = x2;
        w[3] = x3;
    }
    // words e .. e+V-1 (V = 1, 4 or 8; e % 4 == 0 for V > 1)
    template <int V>
    __device__ __forceinline__ void run(unsigned long long e, unsigned* u) const {
        if (V == 1) {
            unsigned w[4];
            words(e >> 2, w);
            const int s = (int)(e & 3);
            u[0] = s == 0 ? w[0] : s == 1 ? w[1] : s == 2 ? w[2] : w[3];
        } else {
#pragma unroll
            for (int i = 0; i < V / 4; ++i) words((e >> 2) + i, u + 4 * i);
        }
    }
};

// keep[u >= floor(p 2^32)] / (1 - p); p == 1 drops everything (its threshold does not fit 32 bits).
struct DropRule {
    unsigned thr;
    float scale;  // 0: everything is dropped
    __host__ static DropRule of(double p) {
        DropRule d;
        if (p >= 1.0) {
            d.thr = 0xffffffffu;
            d.scale = 0.f;
        } else {
            d.thr = (unsigned)(p * 4294967296.0);
            d.scale = (float)(1.0 / (1.0 - p));
        }
        return d;
    }
    __device__ __forceinline__ float factor(unsigned u) const { return u >= thr ? scale : 0.f; }
};
__device__ __forceinline__ float drop_apply(float v, float f) { return f != 0.f ? v * f : 0.f; }  // a dropped inf / NaN is 0

static inline bool vspw_dtype_ok(int dtype) { return dtype == VSPW_F32 || dtype == VSPW_BF16 || dtype == VSPW_F16; }
static inline int vspw_dtype_size(int dtype) { return dtype == VSPW_F32 ? 4 : 2; }

// Thread layout of the channels-last streaming kernels: a block owns `slab` = tx * v channels of one image and walks its
// pixels with 256 / tx of them in flight; tx is the power of two that covers c (at most 64 lanes = 1 KiB per pixel), so a
// thread keeps its channels (and their coefficients and channel masks) for its whole life.
struct SlabPlan {
    int v, tx, slabs, chunks;
};
// min_trips: pixels per thread that a workgroup is worth; blocks: how many workgroups fill the chip.
static inline SlabPlan vspw_slab_plan(int n, long long hw, int c, int v, int min_trips, int blocks) {
    SlabPlan s;
    s.v = v;
    const int cv = (c + v - 1) / v;
    s.tx = 1;
    while (s.tx < cv && s.tx < 64) s.tx *= 2;
    s.slabs = (cv + s.tx - 1) / s.tx;
    const int ty = 256 / s.tx;
    long long want = blocks / ((long long)s.slabs * n);
    const long long most = (hw + (long long)ty * min_trips - 1) / ((long long)ty * min_trips);
    if (want > most) want = most;
    if (want < 1) want = 1;
    s.chunks = (int)want;
    return s;
}
