// Differential attention for gfx950, fp32 and bf16:
//
//   S_m = s q_m k_m^T,  P_m = softmax over the visible keys (m = 1, 2),   out = (P_1 - lam_h P_2) v
//   dP = dO v^T,  D_m = rowsum(P_m o dP) = dO . (P_m v)
//   dS_1 = P_1 o (dP - D_1),  dS_2 = -lam P_2 o (dP - D_2),  dq_m = s dS_m k_m,  dk_m = s dS_m^T q_m,
//   dv = (P_1 - lam P_2)^T dO,   dlam_h = -sum_rows D_2
//
// q [B,Nq,H,2,D], k [B,Nk,Hk,2,D], v [B,Nk,Hk,2D]; the G = H / Hk query heads of a key/value head are packed into the row
// dimension (row r = query * G + head of the group), so that they share every key tile that is read and the gradients of a
// shared head need no extra pass.  Visible: key_mask, and with `frame` > 0 only the keys of the query's frame and of earlier
// ones.  A row without visible keys is zero and has zero gradients.
//
// No map is ever written.  Forward: a wave owns 32 rows and streams 32-key tiles of k and v through LDS with a running
// maximum and sum per map.  The scores are computed transposed (S^T[key][row] = k_tile q^T), so that their accumulator
// registers ARE an operand of the second product (out^T[ch][row] += v_tile^T P^T): no LDS round trip, no shuffles.
// Backward: one kernel owns rows and streams keys (dq), one owns keys and streams rows (dk, dv); both recompute the scores
// from the saved log-sum-exp.  Long axes are split over workgroups when there are few rows (or keys); the partial results are
// joined in a fixed order, so every result is bit-reproducible.
//
// All softmax statistics and sums are fp32.  bf16 inputs: P and dS are rounded to bf16 (half a step, 2^-9 relative, of
// positive weights or of differences whose errors average over the keys) because the matrix unit takes both operands in the
// same type; everything else stays fp32 until the one rounding of each result.
#include <limits.h>
#include <math.h>

#include "elem.h"

typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

#define DA_TILE 32  // keys (or rows) per streamed tile, and rows (or keys) per wave
#define DA_INF __builtin_inff()

// One operand fragment of a 32 x 32 product over 16 terms.  Lane l: index l % 32 of its side, lh = l / 32 selects terms.
// row(): 16 consecutive elements of a row-major row.  col(): rows k0..k0+15 of column c0 + l % 32 of a row-major LDS tile.
// reg(): terms 16 t .. 16 t + 15 from a 32 x 32 result (register r of lane l = term (r & 3) + 8 (r >> 2) + 4 lh of index
// l % 32); col() and reg() deal the terms out alike: 4 lh + e and 8 + 4 lh + e.
template <typename T>
struct Mx;

template <>
struct Mx<float> {
    struct Frag {
        f32x4 a, b;
    };
    static constexpr int PAD = 4;  // LDS row padding (elements): 16 rows hit 16 different 16-byte bank groups
    static __device__ __forceinline__ Frag zero() {
        Frag f;
        f.a = f.b = f32x4{0.f, 0.f, 0.f, 0.f};
        return f;
    }
    static __device__ __forceinline__ Frag row(const float* p, int lh) {
        Frag f;
        f.a = *reinterpret_cast<const f32x4*>(p + 4 * lh);
        f.b = *reinterpret_cast<const f32x4*>(p + 8 + 4 * lh);
        return f;
    }
    static __device__ __forceinline__ Frag col(const float* tile, int ld, int k0, int c0, int lane) {
        const float* p = tile + (k0 + 4 * (lane >> 5)) * ld + c0 + (lane & 31);
        Frag f;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            f.a[e] = p[e * ld];
            f.b[e] = p[(8 + e) * ld];
        }
        return f;
    }
    static __device__ __forceinline__ Frag reg(const f32x16& s, int t) {
        Frag f;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            f.a[e] = s[8 * t + e];
            f.b[e] = s[8 * t + 4 + e];
        }
        return f;
    }
    static __device__ __forceinline__ void mma(f32x16& acc, const Frag& x, const Frag& y) {
#pragma unroll
        for (int e = 0; e < 4; ++e) acc = __builtin_amdgcn_mfma_f32_32x32x2f32(x.a[e], y.a[e], acc, 0, 0, 0);
#pragma unroll
        for (int e = 0; e < 4; ++e) acc = __builtin_amdgcn_mfma_f32_32x32x2f32(x.b[e], y.b[e], acc, 0, 0, 0);
    }
    static __device__ __forceinline__ void store4(float* p, f32x4 v) { *reinterpret_cast<f32x4*>(p) = v; }
};

template <>
struct Mx<bf16_t> {
    typedef bf16x8 Frag;
    static constexpr int PAD = 16;  // 32 bytes: the four rows of a transposed read hit different banks
    static __device__ __forceinline__ Frag zero() {
        Frag f;
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] = (bf16_t)0.f;
        return f;
    }
    static __device__ __forceinline__ Frag row(const bf16_t* p, int lh) { return *reinterpret_cast<const bf16x8*>(p + 8 * lh); }
    static __device__ __forceinline__ Frag col(const bf16_t* tile, int ld, int k0, int c0, int lane) {
        // transposing LDS read: 16 lanes name a 4 x 16 block (row i / 4, 4 elements from column 4 (i % 4)) and get a column each
        const int i = lane & 15;
        const bf16_t* p = tile + (k0 + 4 * (lane >> 5) + (i >> 2)) * ld + c0 + 16 * ((lane >> 4) & 1) + 4 * (i & 3);
        typedef __attribute__((address_space(3))) s16x4 lds4;
        const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)p);
        const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)(p + 8 * ld));
        typedef short s16x8 __attribute__((ext_vector_type(8)));
        const s16x8 ab = __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
        return __builtin_bit_cast(bf16x8, ab);
    }
    static __device__ __forceinline__ Frag reg(const f32x16& s, int t) {
        Frag f;
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] = (bf16_t)s[8 * t + e];
        return f;
    }
    static __device__ __forceinline__ void mma(f32x16& acc, const Frag& x, const Frag& y) {
        acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(x, y, acc, 0, 0, 0);
    }
    static __device__ __forceinline__ void store4(bf16_t* p, f32x4 v) {
        bf16x4 o;
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = (bf16_t)v[e];
        *reinterpret_cast<bf16x4*>(p) = o;
    }
};

struct DaArgs {
    const void *q, *k, *v, *lam, *go;
    const unsigned char* mask;
    void *out, *o2;             // [B,Nq,H,2D]
    float* lse;                 // [2][B*Hk][rows]: log2-sum-exp2 of s log2(e) S (+inf: no visible key)
    float* delta;               // [2][B*Hk][rows]: D_m
    void *dq, *dk, *dv, *dlam;
    float* part;                // partial results of a split axis
    float* ml;                  // forward: [chunks][B*Hk][rows][2] running maximum and sum per map: [..][2 m], [..][2 m + 1]
    double* lpart;              // [B*H][lchunks]: sums of D_2
    long long q_sb, q_sn, q_sh, q_sm, k_sb, k_sn, k_sh, k_sm, v_sb, v_sn, v_sh;
    int b, nq, nk, h, hk, g, rows, frame, lam_bf16, lchunks;
    int tiles, parts, span;     // workgroups along the owned axis; split of the streamed axis: parts of `span` entries
    float c, scale;             // scale * log2(e), scale
};

__device__ __forceinline__ float da_lambda(const DaArgs& a, int head) {
    return a.lam_bf16 ? (float)reinterpret_cast<const bf16_t*>(a.lam)[head] : reinterpret_cast<const float*>(a.lam)[head];
}
// keys [0, lim) are within the frames that the row's query sees
__device__ __forceinline__ int da_limit(const DaArgs& a, int row) {
    if (!a.frame) return a.nk;
    const long long pos = (long long)(row / a.g) + a.nk - a.nq;
    if (pos < 0) return 0;
    const long long lim = (pos / a.frame + 1) * a.frame;
    return lim < a.nk ? (int)lim : a.nk;
}
__device__ __forceinline__ f32x16 zero16() {
    f32x16 z;
#pragma unroll
    for (int r = 0; r < 16; ++r) z[r] = 0.f;
    return z;
}
__device__ __forceinline__ int acc_index(int r, int lh) { return (r & 3) + 8 * (r >> 2) + 4 * lh; }

// Streams [32][2D] tiles of two tensors (k and v, or q and dO) through registers into LDS: 16-byte vectors, thread t moves
// number t + threads * i; entries that take no part arrive as zeros whatever their memory holds.
template <typename T, int D, int THREADS>
struct Stager {
    static constexpr int VE = 16 / (int)sizeof(T);
    static constexpr int VROW = 2 * D / VE;             // vectors per row
    static constexpr int TOTAL = DA_TILE * VROW;
    static constexpr int F = (TOTAL + THREADS - 1) / THREADS;
    static constexpr int LD = 2 * D + Mx<T>::PAD;
    u32x4 x[F], y[F];

    template <typename PX, typename PY>
    __device__ __forceinline__ void load(int tid, PX px, PY py) {  // p?(row of the tile, column, ok) -> address
#pragma unroll
        for (int i = 0; i < F; ++i) {
            const int idx = tid + THREADS * i;
            const int row = TOTAL % THREADS == 0 || idx < TOTAL ? idx / VROW : 0;
            const int col = (idx % VROW) * VE;
            bool ok;
            const T* a = px(row, col, ok);
            const T* b = py(row, col);
            const u32x4 va = *reinterpret_cast<const u32x4*>(a), vb = *reinterpret_cast<const u32x4*>(b);
            const u32x4 z = {0, 0, 0, 0};
            x[i] = ok ? va : z;
            y[i] = ok ? vb : z;
        }
    }
    __device__ __forceinline__ void store(int tid, T* X, T* Y) const {
#pragma unroll
        for (int i = 0; i < F; ++i) {
            const int idx = tid + THREADS * i;
            if (TOTAL % THREADS == 0 || idx < TOTAL) {
                const int o = (idx / VROW) * LD + (idx % VROW) * VE;
                *reinterpret_cast<u32x4*>(X + o) = x[i];
                *reinterpret_cast<u32x4*>(Y + o) = y[i];
            }
        }
    }
};

// ---------------------------------------------------------------------------------------------------------- forward
template <typename T, int D, int WN>
__global__ __launch_bounds__(64 * WN, WN == 1 ? 1 : 2) void da_fwd_kernel(const DaArgs a) {
    typedef Mx<T> M;
    typedef Stager<T, D, 64 * WN> St;
    constexpr int W = 2 * D, LD = St::LD, KC = D / 16, CB = W / 32;
    __shared__ __attribute__((aligned(16))) T Ks[2][DA_TILE * LD];
    __shared__ __attribute__((aligned(16))) T Vs[2][DA_TILE * LD];
    __shared__ __attribute__((aligned(16))) float Kb[2][DA_TILE];  // 0, or -inf for keys that take no part

    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, l31 = lane & 31, lh = lane >> 5;
    const int tile = blockIdx.x % a.tiles;
    const int rest = blockIdx.x / a.tiles;
    const int part = rest % a.parts, bh = rest / a.parts;
    const int bi = bh / a.hk, kh = bh % a.hk;
    const int block0 = tile * 32 * WN;
    const int row0 = block0 + wave * 32;
    const int row = min(row0 + l31, a.rows - 1);  // rows past the end repeat the last one and are not stored
    const int head = kh * a.g + row % a.g, qi = row / a.g;

    const T* qrow = reinterpret_cast<const T*>(a.q) + bi * a.q_sb + qi * a.q_sn + head * a.q_sh;
    typename M::Frag q1[KC], q2[KC];
#pragma unroll
    for (int i = 0; i < KC; ++i) {
        q1[i] = M::row(qrow + 16 * i, lh);
        q2[i] = M::row(qrow + a.q_sm + 16 * i, lh);
    }
    const int lim = da_limit(a, row);
    const int lim_min = __shfl(lim, 0, 64);  // limits grow with the row
    const int key_begin = part * a.span;
    const int key_end = min(min(a.nk, key_begin + a.span), da_limit(a, min(block0 + 32 * WN, a.rows) - 1));
    const T* kb = reinterpret_cast<const T*>(a.k) + bi * a.k_sb + kh * a.k_sh;
    const T* vb = reinterpret_cast<const T*>(a.v) + bi * a.v_sb + kh * a.v_sh;
    const unsigned char* mb = a.mask ? a.mask + (size_t)bi * a.nk : nullptr;

    St st;
    float rb = 0.f;
    auto load_tile = [&](int key0) {
        st.load(
            tid,
            [&](int r, int c, bool& ok) {
                const int key = min(key0 + r, a.nk - 1);
                ok = key0 + r < key_end && (!mb || mb[key]);
                return kb + key * a.k_sn + (c >= D ? a.k_sm + c - D : c);
            },
            [&](int r, int c) { return vb + min(key0 + r, a.nk - 1) * a.v_sn + c; });
        if (tid < DA_TILE) rb = key0 + tid < key_end && (!mb || mb[key0 + tid]) ? 0.f : -DA_INF;
    };
    auto store_tile = [&](int buf) {
        st.store(tid, Ks[buf], Vs[buf]);
        if (tid < DA_TILE) Kb[buf][tid] = rb;
    };

    f32x16 o1[CB], o2[CB];
#pragma unroll
    for (int j = 0; j < CB; ++j) o1[j] = o2[j] = zero16();
    float m1 = -DA_INF, m2 = -DA_INF, l1 = 0.f, l2 = 0.f;

    // scores -> weights 2^(c S - m), running maximum m of every lane's row (both lane halves hold the same one).  The
    // accumulators are rescaled only when the maximum has grown by more than 2^8: weights stay below 256.
    auto softmax = [&](f32x16& s, float& m, float& l, f32x16* o, int cur, int key0) {
        if (mb || key0 + DA_TILE > key_end) {
#pragma unroll
            for (int g4 = 0; g4 < 4; ++g4) {
                const f32x4 kbias = *reinterpret_cast<const f32x4*>(&Kb[cur][8 * g4 + 4 * lh]);
#pragma unroll
                for (int e = 0; e < 4; ++e) s[4 * g4 + e] += kbias[e];
            }
        }
        if (key0 + DA_TILE > lim_min) {
#pragma unroll
            for (int r = 0; r < 16; ++r)
                if (key0 + acc_index(r, lh) >= lim) s[r] = -DA_INF;
        }
        float mx = s[0];
#pragma unroll
        for (int r = 1; r < 16; ++r) mx = fmaxf(mx, s[r]);
        mx = fmaxf(mx, __shfl_xor(mx, 32, 64)) * a.c;
        if (__any(mx > m + 8.f)) {
            const float mn = fmaxf(m, mx);
            const float f = m == -DA_INF ? 0.f : exp2f(m - mn);
            m = mn;
            l *= f;
#pragma unroll
            for (int j = 0; j < CB; ++j)
#pragma unroll
                for (int r = 0; r < 16; ++r) o[j][r] *= f;
        }
        const float mu = m == -DA_INF ? 0.f : m;
        float sum = 0.f;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            s[r] = __builtin_amdgcn_exp2f(fmaf(s[r], a.c, -mu));
            sum += s[r];
        }
        l += sum;
    };

    const int ntiles = key_end > key_begin ? (key_end - key_begin + DA_TILE - 1) / DA_TILE : 0;
    if (ntiles > 0) {
        load_tile(key_begin);
        store_tile(0);
        if (ntiles > 1) load_tile(key_begin + DA_TILE);
    }
    __syncthreads();
    for (int t = 0; t < ntiles; ++t) {
        const int cur = t & 1, key0 = key_begin + t * DA_TILE;
        const T* Kc = Ks[cur] + l31 * LD;
        f32x16 s1 = zero16(), s2 = zero16();
#pragma unroll
        for (int i = 0; i < KC; ++i) {
            M::mma(s1, M::row(Kc + 16 * i, lh), q1[i]);
            M::mma(s2, M::row(Kc + D + 16 * i, lh), q2[i]);
        }
        if (t + 1 < ntiles) {  // tile t+1 has been in flight since the last trip; its buffer's readers passed the barrier
            store_tile(cur ^ 1);
            if (t + 2 < ntiles) load_tile(key0 + 2 * DA_TILE);
        }
        softmax(s1, m1, l1, o1, cur, key0);
        softmax(s2, m2, l2, o2, cur, key0);
#pragma unroll
        for (int t2 = 0; t2 < 2; ++t2) {
            const typename M::Frag p1 = M::reg(s1, t2), p2 = M::reg(s2, t2);
#pragma unroll
            for (int j = 0; j < CB; ++j) {
                const typename M::Frag vf = M::col(Vs[cur], LD, 16 * t2, 32 * j, lane);
                M::mma(o1[j], vf, p1);
                M::mma(o2[j], vf, p2);
            }
        }
        __syncthreads();
    }
    l1 += __shfl_xor(l1, 32, 64);
    l2 += __shfl_xor(l2, 32, 64);
    if (row0 + l31 >= a.rows) return;
    if (a.parts > 1) {  // unnormalised sums with their maximum, joined by da_join_kernel
        const size_t e = ((size_t)part * a.b * a.hk + bh) * a.rows + row;
        float* po = a.part + e * 2 * W;
#pragma unroll
        for (int j = 0; j < CB; ++j)
#pragma unroll
            for (int g4 = 0; g4 < 4; ++g4) {
                const int ch = 32 * j + 8 * g4 + 4 * lh;
                f32x4 x, y;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    x[i] = o1[j][4 * g4 + i];
                    y[i] = o2[j][4 * g4 + i];
                }
                *reinterpret_cast<f32x4*>(po + ch) = x;
                *reinterpret_cast<f32x4*>(po + W + ch) = y;
            }
        if (lh == 0) *reinterpret_cast<f32x4*>(a.ml + e * 4) = f32x4{m1, l1, m2, l2};
        return;
    }
    const float i1 = l1 == 0.f ? 0.f : 1.f / l1, i2 = l2 == 0.f ? 0.f : 1.f / l2, lam = da_lambda(a, head);
    T* out = reinterpret_cast<T*>(a.out) + (((size_t)bi * a.nq + qi) * a.h + head) * W;
    T* out2 = a.o2 ? reinterpret_cast<T*>(a.o2) + (((size_t)bi * a.nq + qi) * a.h + head) * W : nullptr;
#pragma unroll
    for (int j = 0; j < CB; ++j)
#pragma unroll
        for (int g4 = 0; g4 < 4; ++g4) {
            const int ch = 32 * j + 8 * g4 + 4 * lh;
            f32x4 x, y;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                y[i] = o2[j][4 * g4 + i] * i2;
                x[i] = o1[j][4 * g4 + i] * i1 - lam * y[i];
            }
            M::store4(out + ch, x);
            if (out2) M::store4(out2 + ch, y);
        }
    if (a.lse && lh == 0) {
        const size_t e = (size_t)bh * a.rows + row, n = (size_t)a.b * a.hk * a.rows;
        a.lse[e] = l1 == 0.f ? DA_INF : m1 + log2f(l1);
        a.lse[n + e] = l2 == 0.f ? DA_INF : m2 + log2f(l2);
    }
}

// Joins the parts of a row: one workgroup per row, W / 4 threads across the channels, the rest across the parts.
template <typename T, int D>
__global__ __launch_bounds__(256) void da_join_kernel(const DaArgs a) {
    constexpr int W = 2 * D, CT = 2 * W / 4, PT = 256 / CT;  // CT threads hold one part's two sums
    __shared__ float red[4][256];
    __shared__ f32x4 sum[256];
    const int tid = threadIdx.x;
    const size_t n = (size_t)a.b * a.hk * a.rows, e = blockIdx.x;
    const int bh = (int)(e / a.rows), row = (int)(e % a.rows);
    const int head = (bh % a.hk) * a.g + row % a.g;
    float M[2] = {-DA_INF, -DA_INF}, L[2] = {0.f, 0.f};
    for (int p = tid; p < a.parts; p += 256) {
        const f32x4 v = *reinterpret_cast<const f32x4*>(a.ml + (p * n + e) * 4);
        M[0] = fmaxf(M[0], v[0]);
        M[1] = fmaxf(M[1], v[2]);
    }
    red[0][tid] = M[0];
    red[1][tid] = M[1];
    __syncthreads();
    for (int h = 128; h > 0; h >>= 1) {
        if (tid < h) {
            red[0][tid] = fmaxf(red[0][tid], red[0][tid + h]);
            red[1][tid] = fmaxf(red[1][tid], red[1][tid + h]);
        }
        __syncthreads();
    }
    M[0] = red[0][0] == -DA_INF ? 0.f : red[0][0];
    M[1] = red[1][0] == -DA_INF ? 0.f : red[1][0];
    for (int p = tid; p < a.parts; p += 256) {
        const f32x4 v = *reinterpret_cast<const f32x4*>(a.ml + (p * n + e) * 4);
        L[0] += v[1] * exp2f(v[0] - M[0]);
        L[1] += v[3] * exp2f(v[2] - M[1]);
    }
    red[2][tid] = L[0];
    red[3][tid] = L[1];
    __syncthreads();
    for (int h = 128; h > 0; h >>= 1) {
        if (tid < h) {
            red[2][tid] += red[2][tid + h];
            red[3][tid] += red[3][tid + h];
        }
        __syncthreads();
    }
    L[0] = red[2][0];
    L[1] = red[3][0];
    const int ch = tid % CT, map = ch >= CT / 2 ? 1 : 0;
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    for (int p = tid / CT; p < a.parts; p += PT) {
        const float w = exp2f(a.ml[(p * n + e) * 4 + 2 * map] - M[map]);
        const f32x4 v = *reinterpret_cast<const f32x4*>(a.part + (p * n + e) * 2 * W + 4 * ch);
        if (w != 0.f) acc += v * w;
    }
    sum[tid] = acc;
    __syncthreads();
    if (tid < CT / 2) {
        f32x4 x = {0.f, 0.f, 0.f, 0.f}, y = x;
        for (int p = 0; p < PT; ++p) {
            x += sum[p * CT + tid];
            y += sum[p * CT + CT / 2 + tid];
        }
        x *= L[0] == 0.f ? 0.f : 1.f / L[0];
        y *= L[1] == 0.f ? 0.f : 1.f / L[1];
        const size_t o = (((size_t)(bh / a.hk) * a.nq + row / a.g) * a.h + head) * W + 4 * tid;
        if (a.o2) Mx<T>::store4(reinterpret_cast<T*>(a.o2) + o, y);
        x -= y * da_lambda(a, head);
        Mx<T>::store4(reinterpret_cast<T*>(a.out) + o, x);
    }
    if (a.lse && tid < 2) a.lse[tid * n + e] = L[tid] == 0.f ? DA_INF : M[tid] + log2f(L[tid]);
}

// --------------------------------------------------------------------------------------------------------- backward
// D_1, D_2 of every row, and partial sums of D_2 per head: a workgroup owns 256 / LPR rows per trip of one (batch, head)
template <typename T, int D>
__global__ __launch_bounds__(256) void da_delta_kernel(const DaArgs a) {
    constexpr int W = 2 * D, V = 4, LPR = W / V;
    __shared__ double red[256];
    const int chunk = blockIdx.x % a.lchunks, bh = blockIdx.x / a.lchunks;
    const int bi = bh / a.h, head = bh % a.h;
    const int kh = head / a.g, g = head % a.g;
    const int sub = threadIdx.x % LPR;
    const float lam = da_lambda(a, head);
    const size_t n = (size_t)a.b * a.hk * a.rows;
    double total = 0.0;
    for (int q = chunk * (256 / LPR) + threadIdx.x / LPR; q < a.nq; q += a.lchunks * (256 / LPR)) {
        const size_t o = (((size_t)bi * a.nq + q) * a.h + head) * W + V * sub;
        float go[V], ou[V], o2[V];
        Vec<T, V>::load(reinterpret_cast<const T*>(a.go) + o, go);
        Vec<T, V>::load(reinterpret_cast<const T*>(a.out) + o, ou);
        Vec<T, V>::load(reinterpret_cast<const T*>(a.o2) + o, o2);
        float d1 = 0.f, d2 = 0.f;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            d2 = fmaf(go[i], o2[i], d2);
            d1 = fmaf(go[i], fmaf(lam, o2[i], ou[i]), d1);
        }
        for (int s = LPR / 2; s > 0; s >>= 1) {
            d1 += __shfl_xor(d1, s, 64);
            d2 += __shfl_xor(d2, s, 64);
        }
        if (sub == 0) {
            const size_t e = ((size_t)bi * a.hk + kh) * a.rows + (size_t)q * a.g + g;
            a.delta[e] = d1;
            a.delta[n + e] = d2;
            total += (double)d2;
        }
    }
    red[threadIdx.x] = total;
    __syncthreads();
    for (int h = 128; h > 0; h >>= 1) {
        if ((int)threadIdx.x < h) red[threadIdx.x] += red[threadIdx.x + h];
        __syncthreads();
    }
    if (threadIdx.x == 0) a.lpart[(size_t)bh * a.lchunks + chunk] = red[0];
}

// dlam[h] = - sum over batch and chunks: one workgroup per head
__global__ __launch_bounds__(256) void da_dlam_kernel(const DaArgs a) {
    __shared__ double red[256];
    const int head = blockIdx.x, n = a.b * a.lchunks;
    double s = 0.0;
    for (int i = threadIdx.x; i < n; i += 256)
        s += a.lpart[((size_t)(i / a.lchunks) * a.h + head) * a.lchunks + i % a.lchunks];
    red[threadIdx.x] = s;
    __syncthreads();
    for (int h = 128; h > 0; h >>= 1) {
        if ((int)threadIdx.x < h) red[threadIdx.x] += red[threadIdx.x + h];
        __syncthreads();
    }
    if (threadIdx.x == 0) {
        if (a.lam_bf16)
            reinterpret_cast<bf16_t*>(a.dlam)[head] = (bf16_t)(float)-red[0];
        else
            reinterpret_cast<float*>(a.dlam)[head] = (float)-red[0];
    }
}

// dq: a wave owns 32 rows (everything about them is one value per lane) and streams key tiles.
template <typename T, int D>
__global__ __launch_bounds__(256, 1) void da_dq_kernel(const DaArgs a) {
    typedef Mx<T> M;
    typedef Stager<T, D, 256> St;
    constexpr int W = 2 * D, LD = St::LD, KC = D / 16, VC = W / 16, DB = (D + 31) / 32;
    constexpr int LDT = LD;
    __shared__ __attribute__((aligned(16))) T Ks[2][DA_TILE * LD];
    __shared__ __attribute__((aligned(16))) T Vs[2][DA_TILE * LD];
    __shared__ __attribute__((aligned(16))) float Kb[2][DA_TILE];

    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, l31 = lane & 31, lh = lane >> 5;
    const int tile = blockIdx.x % a.tiles;
    const int rest = blockIdx.x / a.tiles;
    const int part = rest % a.parts, bh = rest / a.parts;
    const int bi = bh / a.hk, kh = bh % a.hk;
    const int block0 = tile * 128;
    const int row0 = block0 + wave * 32;
    const int row = min(row0 + l31, a.rows - 1);
    const int head = kh * a.g + row % a.g, qi = row / a.g;
    const size_t n = (size_t)a.b * a.hk * a.rows, e = (size_t)bh * a.rows + row;

    const T* qrow = reinterpret_cast<const T*>(a.q) + bi * a.q_sb + qi * a.q_sn + head * a.q_sh;
    const T* grow = reinterpret_cast<const T*>(a.go) + (((size_t)bi * a.nq + qi) * a.h + head) * W;
    typename M::Frag q1[KC], q2[KC], go[VC];
#pragma unroll
    for (int i = 0; i < KC; ++i) {
        q1[i] = M::row(qrow + 16 * i, lh);
        q2[i] = M::row(qrow + a.q_sm + 16 * i, lh);
    }
#pragma unroll
    for (int i = 0; i < VC; ++i) go[i] = M::row(grow + 16 * i, lh);
    const float e1 = a.lse[e], e2 = a.lse[n + e], d1 = a.delta[e], d2 = a.delta[n + e];
    const int lim = da_limit(a, row);
    const int lim_min = __shfl(lim, 0, 64);
    const int key_begin = part * a.span;
    const int key_end = min(min(a.nk, key_begin + a.span), da_limit(a, min(block0 + 128, a.rows) - 1));
    const T* kb = reinterpret_cast<const T*>(a.k) + bi * a.k_sb + kh * a.k_sh;
    const T* vb = reinterpret_cast<const T*>(a.v) + bi * a.v_sb + kh * a.v_sh;
    const unsigned char* mb = a.mask ? a.mask + (size_t)bi * a.nk : nullptr;

    St st;
    float rb = 0.f;
    auto load_tile = [&](int key0) {
        st.load(
            tid,
            [&](int r, int c, bool& ok) {
                const int key = min(key0 + r, a.nk - 1);
                ok = key0 + r < key_end && (!mb || mb[key]);
                return kb + key * a.k_sn + (c >= D ? a.k_sm + c - D : c);
            },
            [&](int r, int c) { return vb + min(key0 + r, a.nk - 1) * a.v_sn + c; });
        if (tid < DA_TILE) rb = key0 + tid < key_end && (!mb || mb[key0 + tid]) ? 0.f : -DA_INF;
    };
    auto store_tile = [&](int buf) {
        st.store(tid, Ks[buf], Vs[buf]);
        if (tid < DA_TILE) Kb[buf][tid] = rb;
    };
    f32x16 g1[DB], g2[DB];
#pragma unroll
    for (int j = 0; j < DB; ++j) g1[j] = g2[j] = zero16();

    const int ntiles = key_end > key_begin ? (key_end - key_begin + DA_TILE - 1) / DA_TILE : 0;
    if (ntiles > 0) {
        load_tile(key_begin);
        store_tile(0);
        if (ntiles > 1) load_tile(key_begin + DA_TILE);
    }
    __syncthreads();
    for (int t = 0; t < ntiles; ++t) {
        const int cur = t & 1, key0 = key_begin + t * DA_TILE;
        const T* Kc = Ks[cur] + l31 * LD;
        const T* Vc = Vs[cur] + l31 * LD;
        f32x16 s1 = zero16(), s2 = zero16(), dp = zero16();
#pragma unroll
        for (int i = 0; i < KC; ++i) {
            M::mma(s1, M::row(Kc + 16 * i, lh), q1[i]);
            M::mma(s2, M::row(Kc + D + 16 * i, lh), q2[i]);
        }
#pragma unroll
        for (int i = 0; i < VC; ++i) M::mma(dp, M::row(Vc + 16 * i, lh), go[i]);
        if (t + 1 < ntiles) {
            store_tile(cur ^ 1);
            if (t + 2 < ntiles) load_tile(key0 + 2 * DA_TILE);
        }
        if (mb || key0 + DA_TILE > key_end) {
#pragma unroll
            for (int g4 = 0; g4 < 4; ++g4) {
                const f32x4 kbias = *reinterpret_cast<const f32x4*>(&Kb[cur][8 * g4 + 4 * lh]);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    s1[4 * g4 + i] += kbias[i];
                    s2[4 * g4 + i] += kbias[i];
                }
            }
        }
        if (key0 + DA_TILE > lim_min) {
#pragma unroll
            for (int r = 0; r < 16; ++r)
                if (key0 + acc_index(r, lh) >= lim) s1[r] = s2[r] = -DA_INF;
        }
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            s1[r] = __builtin_amdgcn_exp2f(fmaf(s1[r], a.c, -e1)) * (dp[r] - d1);
            s2[r] = __builtin_amdgcn_exp2f(fmaf(s2[r], a.c, -e2)) * (dp[r] - d2);
        }
#pragma unroll
        for (int t2 = 0; t2 < 2; ++t2) {
            const typename M::Frag p1 = M::reg(s1, t2), p2 = M::reg(s2, t2);
#pragma unroll
            for (int j = 0; j < DB; ++j) {
                // D = 16: the upper 16 columns of the fragment belong to the other map (or the padding) and are not stored
                M::mma(g1[j], M::col(Ks[cur], LDT, 16 * t2, 32 * j, lane), p1);
                M::mma(g2[j], M::col(Ks[cur], LDT, 16 * t2, (D < 32 ? 0 : D) + 32 * j, lane), p2);
            }
        }
        __syncthreads();
    }
    if (row0 + l31 >= a.rows) return;
    const float f2 = -da_lambda(a, head) * a.scale;
    const size_t o = (((size_t)bi * a.nq + qi) * a.h + head) * W;
#pragma unroll
    for (int j = 0; j < DB; ++j)
#pragma unroll
        for (int g4 = 0; g4 < 4; ++g4) {
            const int ch = 32 * j + 8 * g4 + 4 * lh;
            f32x4 x, y;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                x[i] = g1[j][4 * g4 + i] * a.scale;
                y[i] = g2[j][4 * g4 + i] * f2;
            }
            // D = 16: map 1 sits in channels 0..15 of its product, map 2 in channels 16..31 of its own
            const int c1 = ch, c2 = D < 32 ? ch : D + ch;
            const bool ok1 = D >= 32 || ch < D, ok2 = D >= 32 || ch >= D;
            if (a.parts > 1) {
                float* p = a.part + (size_t)part * a.b * a.nq * a.h * W + o;
                if (ok1) *reinterpret_cast<f32x4*>(p + c1) = x;
                if (ok2) *reinterpret_cast<f32x4*>(p + c2) = y;
            } else {
                T* p = reinterpret_cast<T*>(a.dq) + o;
                if (ok1) M::store4(p + c1, x);
                if (ok2) M::store4(p + c2, y);
            }
        }
}

// dk, dv: a wave owns 32 keys and streams row tiles; row statistics come from LDS, four at a time.
template <typename T, int D>
__global__ __launch_bounds__(256, 1) void da_dkv_kernel(const DaArgs a) {
    typedef Mx<T> M;
    typedef Stager<T, D, 256> St;
    constexpr int W = 2 * D, LD = St::LD, KC = D / 16, VC = W / 16, DB = (D + 31) / 32, CB = W / 32;
    __shared__ __attribute__((aligned(16))) T Qs[2][DA_TILE * LD];
    __shared__ __attribute__((aligned(16))) T Gs[2][DA_TILE * LD];
    __shared__ __attribute__((aligned(16))) float Rs[2][6][DA_TILE];  // lse 1, lse 2, D_1, D_2, lambda, key limit (int)

    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, l31 = lane & 31, lh = lane >> 5;
    const int tile = blockIdx.x % a.tiles;
    const int rest = blockIdx.x / a.tiles;
    const int part = rest % a.parts, bh = rest / a.parts;
    const int bi = bh / a.hk, kh = bh % a.hk;
    const int block0 = tile * 128;
    const int key = block0 + wave * 32 + l31;
    const bool live = key < a.nk && (!a.mask || a.mask[(size_t)bi * a.nk + min(key, a.nk - 1)]);
    const size_t n = (size_t)a.b * a.hk * a.rows;

    typename M::Frag k1[KC], k2[KC], v[VC];
    {
        const int kc = min(key, a.nk - 1);
        const T* kp = reinterpret_cast<const T*>(a.k) + bi * a.k_sb + kh * a.k_sh + kc * a.k_sn;
        const T* vp = reinterpret_cast<const T*>(a.v) + bi * a.v_sb + kh * a.v_sh + kc * a.v_sn;
#pragma unroll
        for (int i = 0; i < KC; ++i) {
            k1[i] = live ? M::row(kp + 16 * i, lh) : M::zero();
            k2[i] = live ? M::row(kp + a.k_sm + 16 * i, lh) : M::zero();
        }
#pragma unroll
        for (int i = 0; i < VC; ++i) v[i] = live ? M::row(vp + 16 * i, lh) : M::zero();
    }
    int row_begin = part * a.span;
    const int row_end = min(a.rows, row_begin + a.span);
    const int key_last = min(block0 + 128, a.nk);  // keys of the block: [block0, key_last)
    if (a.frame) {  // the first query that sees the block's first key
        const long long q0 = (long long)block0 / a.frame * a.frame - (a.nk - a.nq);
        const long long r0 = q0 > 0 ? q0 * a.g / DA_TILE * DA_TILE : 0;
        if (r0 > row_begin) row_begin = r0 < row_end ? (int)r0 : row_end;
    }
    const T* qb = reinterpret_cast<const T*>(a.q) + bi * a.q_sb;
    const T* gb = reinterpret_cast<const T*>(a.go) + (size_t)bi * a.nq * a.h * W;

    St st;
    float rs = 0.f;
    auto load_tile = [&](int r0) {
        st.load(
            tid,
            [&](int r, int c, bool& ok) {
                const int row = min(r0 + r, a.rows - 1);
                ok = r0 + r < row_end;
                return qb + row / a.g * a.q_sn + (kh * a.g + row % a.g) * a.q_sh + (c >= D ? a.q_sm + c - D : c);
            },
            [&](int r, int c) {
                const int row = min(r0 + r, a.rows - 1);
                return gb + ((size_t)(row / a.g) * a.h + kh * a.g + row % a.g) * W + c;
            });
        if (tid < 6 * DA_TILE) {
            const int which = tid / DA_TILE, row = r0 + tid % DA_TILE;
            const size_t e = (size_t)bh * a.rows + min(row, a.rows - 1);
            if (which < 2)
                rs = row < row_end ? a.lse[which * n + e] : DA_INF;  // rows past the end: weight 0
            else if (which < 4)
                rs = row < row_end ? a.delta[(which - 2) * n + e] : 0.f;
            else if (which == 4)
                rs = da_lambda(a, kh * a.g + min(row, a.rows - 1) % a.g);
            else
                rs = __int_as_float(da_limit(a, min(row, a.rows - 1)));
        }
    };
    auto store_tile = [&](int buf) {
        st.store(tid, Qs[buf], Gs[buf]);
        if (tid < 6 * DA_TILE) Rs[buf][tid / DA_TILE][tid % DA_TILE] = rs;
    };
    f32x16 gk1[DB], gk2[DB], gv[CB];
#pragma unroll
    for (int j = 0; j < DB; ++j) gk1[j] = gk2[j] = zero16();
#pragma unroll
    for (int j = 0; j < CB; ++j) gv[j] = zero16();

    const int ntiles = row_end > row_begin ? (row_end - row_begin + DA_TILE - 1) / DA_TILE : 0;
    if (ntiles > 0) {
        load_tile(row_begin);
        store_tile(0);
        if (ntiles > 1) load_tile(row_begin + DA_TILE);
    }
    __syncthreads();
    for (int t = 0; t < ntiles; ++t) {
        const int cur = t & 1, r0 = row_begin + t * DA_TILE;
        const T* Qc = Qs[cur] + l31 * LD;
        const T* Gc = Gs[cur] + l31 * LD;
        f32x16 s1 = zero16(), s2 = zero16(), dp = zero16();
#pragma unroll
        for (int i = 0; i < KC; ++i) {
            M::mma(s1, M::row(Qc + 16 * i, lh), k1[i]);
            M::mma(s2, M::row(Qc + D + 16 * i, lh), k2[i]);
        }
#pragma unroll
        for (int i = 0; i < VC; ++i) M::mma(dp, M::row(Gc + 16 * i, lh), v[i]);
        if (t + 1 < ntiles) {
            store_tile(cur ^ 1);
            if (t + 2 < ntiles) load_tile(r0 + 2 * DA_TILE);
        }
        const bool edge = a.frame && __float_as_int(Rs[cur][5][0]) < key_last;
        f32x16 mix;
#pragma unroll
        for (int g4 = 0; g4 < 4; ++g4) {
            const int o = 8 * g4 + 4 * lh;
            const f32x4 e1 = *reinterpret_cast<const f32x4*>(&Rs[cur][0][o]), e2 = *reinterpret_cast<const f32x4*>(&Rs[cur][1][o]);
            const f32x4 d1 = *reinterpret_cast<const f32x4*>(&Rs[cur][2][o]), d2 = *reinterpret_cast<const f32x4*>(&Rs[cur][3][o]);
            const f32x4 lam = *reinterpret_cast<const f32x4*>(&Rs[cur][4][o]);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int r = 4 * g4 + i;
                float p1 = __builtin_amdgcn_exp2f(fmaf(s1[r], a.c, -e1[i])), p2 = __builtin_amdgcn_exp2f(fmaf(s2[r], a.c, -e2[i]));
                if (edge && key >= __float_as_int(Rs[cur][5][o + i])) p1 = p2 = 0.f;
                p2 *= lam[i];
                mix[r] = p1 - p2;
                s1[r] = p1 * (dp[r] - d1[i]);
                s2[r] = p2 * (d2[i] - dp[r]);
            }
        }
#pragma unroll
        for (int t2 = 0; t2 < 2; ++t2) {
            const typename M::Frag pm = M::reg(mix, t2), p1 = M::reg(s1, t2), p2 = M::reg(s2, t2);
#pragma unroll
            for (int j = 0; j < CB; ++j) M::mma(gv[j], M::col(Gs[cur], LD, 16 * t2, 32 * j, lane), pm);
#pragma unroll
            for (int j = 0; j < DB; ++j) {
                M::mma(gk1[j], M::col(Qs[cur], LD, 16 * t2, 32 * j, lane), p1);
                M::mma(gk2[j], M::col(Qs[cur], LD, 16 * t2, (D < 32 ? 0 : D) + 32 * j, lane), p2);
            }
        }
        __syncthreads();
    }
    if (key >= a.nk) return;
    const size_t o = (((size_t)bi * a.nk + key) * a.hk + kh) * W;
    const size_t np = (size_t)a.b * a.nk * a.hk * W;
    auto put = [&](int which, int ch, f32x4 x) {
        if (!live) x = f32x4{0.f, 0.f, 0.f, 0.f};  // its column never left this lane
        if (a.parts > 1)
            *reinterpret_cast<f32x4*>(a.part + ((size_t)part * 2 + which) * np + o + ch) = x;
        else if (which == 0)
            M::store4(reinterpret_cast<T*>(a.dk) + o + ch, x);
        else
            M::store4(reinterpret_cast<T*>(a.dv) + o + ch, x);
    };
#pragma unroll
    for (int g4 = 0; g4 < 4; ++g4) {
        const int c4 = 8 * g4 + 4 * lh;
        f32x4 x;
#pragma unroll
        for (int j = 0; j < CB; ++j) {
#pragma unroll
            for (int i = 0; i < 4; ++i) x[i] = gv[j][4 * g4 + i];
            put(1, 32 * j + c4, x);
        }
#pragma unroll
        for (int j = 0; j < DB; ++j) {
            const int ch = 32 * j + c4;
#pragma unroll
            for (int i = 0; i < 4; ++i) x[i] = gk1[j][4 * g4 + i] * a.scale;
            if (D >= 32 || ch < D) put(0, ch, x);
#pragma unroll
            for (int i = 0; i < 4; ++i) x[i] = gk2[j][4 * g4 + i] * a.scale;
            if (D >= 32 || ch >= D) put(0, D < 32 ? ch : D + ch, x);
        }
    }
}

// out = sum over parts of part[p * stride + i], rounded once
template <typename T>
__global__ __launch_bounds__(256) void da_sum_kernel(const float* __restrict__ part, T* __restrict__ out, long long n4,
                                                     int parts, long long stride) {
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < n4; i += (long long)gridDim.x * 256) {
        f32x4 s = *reinterpret_cast<const f32x4*>(part + 4 * i);
        for (int p = 1; p < parts; ++p) s += *reinterpret_cast<const f32x4*>(part + p * stride + 4 * i);
        Mx<T>::store4(out + 4 * i, s);
    }
}

// lam[h] = exp(q1.k1) - exp(q2.k2) + init, one wave per head; with g: the gradients of the four vectors
__global__ __launch_bounds__(64) void diff_lambda_kernel(const float* __restrict__ q1, const float* __restrict__ k1,
                                                         const float* __restrict__ q2, const float* __restrict__ k2,
                                                         float init, float* __restrict__ lam, const float* __restrict__ g,
                                                         float* __restrict__ gq1, float* __restrict__ gk1,
                                                         float* __restrict__ gq2, float* __restrict__ gk2, int d) {
    const size_t o = (size_t)blockIdx.x * d;
    float a = 0.f, b = 0.f;
    for (int i = threadIdx.x; i < d; i += 64) {
        a = fmaf(q1[o + i], k1[o + i], a);
        b = fmaf(q2[o + i], k2[o + i], b);
    }
    a = expf(wave_sum(a));
    b = expf(wave_sum(b));
    if (!g) {
        if (threadIdx.x == 0) lam[blockIdx.x] = a - b + init;
        return;
    }
    const float ga = g[blockIdx.x] * a, gb = -g[blockIdx.x] * b;
    for (int i = threadIdx.x; i < d; i += 64) {
        gq1[o + i] = ga * k1[o + i];
        gk1[o + i] = ga * q1[o + i];
        gq2[o + i] = gb * k2[o + i];
        gk2[o + i] = gb * q2[o + i];
    }
}

// ------------------------------------------------------------------------------------------------------------- host
// Splits the streamed axis (nt tiles) of nb workgroups into parts so that the rounds of `slots` resident workgroups are
// well filled; a part costs about `extra` tiles of prologue, epilogue and joining.
static int da_parts(long long nb, int nt, int slots, int extra, int most) {
    int best = 1;
    double cost = 1e300;
    for (int p = 1; p <= most && p <= nt; ++p) {
        const long long rounds = (nb * p + slots - 1) / slots;
        const double c = (double)rounds * ((nt + p - 1) / p + (p > 1 ? extra : 0)) + (p > 1 ? 0.02 * p : 0.0);
        if (c < cost * 0.98) {
            cost = c;
            best = p;
        }
    }
    return best;
}
static int da_span(int n, int parts) { return vspw_cdiv(vspw_cdiv(n, DA_TILE), parts) * DA_TILE; }

struct DaPlan {
    int g, rows, wn, tiles, parts, span;              // forward
    int qt, qparts, qspan, kt, kparts, kspan, lchunks;  // backward
    long long bhk;
    size_t fwd_bytes, bwd_bytes;
};
static bool da_plan(const vspw_dattn_desc* d, DaPlan& p) {
    if (!d || d->b <= 0 || d->nq <= 0 || d->nk <= 0 || d->h <= 0 || d->hk <= 0 || d->h % d->hk || d->frame < 0) return false;
    if (d->d != 16 && d->d != 32 && d->d != 64) return false;
    if (d->dtype != VSPW_F32 && d->dtype != VSPW_BF16) return false;
    if (d->lam_dtype != VSPW_F32 && d->lam_dtype != VSPW_BF16) return false;
    if (!(d->scale > 0.f) || !(d->scale < DA_INF)) return false;
    p.g = d->h / d->hk;
    const long long rows = (long long)d->nq * p.g;
    p.bhk = (long long)d->b * d->hk;
    if (rows > INT_MAX - 256 || d->nk > INT_MAX - 256 || p.bhk * rows > (1LL << 40) || (long long)d->b * d->nk * d->hk > (1LL << 40))
        return false;
    p.rows = (int)rows;
    const int W = 2 * d->d, nt = vspw_cdiv(d->nk, DA_TILE);
    // up to 32 rows: single-wave workgroups, many parts of the key axis; else four waves share a key tile
    p.wn = p.rows <= 32 ? 1 : 4;
    p.tiles = vspw_cdiv(p.rows, 32 * p.wn);
    p.parts = p.wn == 1 ? da_parts(p.tiles * p.bhk, nt, 1024, 1, 256) : da_parts(p.tiles * p.bhk, nt, 512, 4, 32);
    p.span = da_span(d->nk, p.parts);
    p.parts = vspw_cdiv(d->nk, p.span);
    p.fwd_bytes = p.parts > 1 ? (size_t)p.parts * p.bhk * p.rows * (2 * W + 4) * sizeof(float) : 0;
    const int slots = d->dtype == VSPW_F32 ? 256 : 512;
    p.qt = vspw_cdiv(p.rows, 128);
    p.qparts = da_parts(p.qt * p.bhk, nt, slots, 4, 16);
    p.qspan = da_span(d->nk, p.qparts);
    p.qparts = vspw_cdiv(d->nk, p.qspan);
    p.kt = vspw_cdiv(d->nk, 128);
    p.kparts = da_parts(p.kt * p.bhk, vspw_cdiv(p.rows, DA_TILE), slots, 4, 16);
    p.kspan = da_span(p.rows, p.kparts);
    p.kparts = vspw_cdiv(p.rows, p.kspan);
    const long long bh = (long long)d->b * d->h;
    long long lc = 2048 / bh;
    const long long most = vspw_cdiv(d->nq, 4 * (256 / (W / 4)));
    if (lc > most) lc = most;
    if (lc < 1) lc = 1;
    p.lchunks = (int)lc;
    if (p.tiles * p.bhk * p.parts > INT_MAX || p.qt * p.bhk * p.qparts > INT_MAX || p.kt * p.bhk * p.kparts > INT_MAX ||
        bh * p.lchunks > INT_MAX || p.bhk * p.rows > INT_MAX)
        return false;
    size_t parts = 0;  // dq and dk/dv run one after the other and share the partial sums' memory
    if (p.qparts > 1) parts = (size_t)p.qparts * p.bhk * p.rows * W;
    if (p.kparts > 1 && (size_t)p.kparts * 2 * p.bhk * d->nk * W > parts) parts = (size_t)p.kparts * 2 * p.bhk * d->nk * W;
    p.bwd_bytes = (size_t)bh * p.lchunks * sizeof(double) + ((size_t)2 * p.bhk * p.rows + parts) * sizeof(float);
    p.bwd_bytes += 32;  // alignment of the pieces
    return true;
}
static bool da_strides_ok(const vspw_dattn_desc* d, const void* q, const void* k, const void* v) {
    const long long ve = d->dtype == VSPW_F32 ? 4 : 8;
    const long long s[] = {d->q_sb, d->q_sn, d->q_sh, d->q_sm, d->k_sb, d->k_sn, d->k_sh, d->k_sm, d->v_sb, d->v_sn, d->v_sh};
    for (long long x : s)
        if (x % ve) return false;
    return (((uintptr_t)q | (uintptr_t)k | (uintptr_t)v) & 15) == 0;
}
static void da_fill(DaArgs& a, const vspw_dattn_desc* d, const DaPlan& p, const void* q, const void* k, const void* v,
                    const void* lam, const unsigned char* mask) {
    a = DaArgs();
    a.q = q;
    a.k = k;
    a.v = v;
    a.lam = lam;
    a.mask = mask;
    a.q_sb = d->q_sb;
    a.q_sn = d->q_sn;
    a.q_sh = d->q_sh;
    a.q_sm = d->q_sm;
    a.k_sb = d->k_sb;
    a.k_sn = d->k_sn;
    a.k_sh = d->k_sh;
    a.k_sm = d->k_sm;
    a.v_sb = d->v_sb;
    a.v_sn = d->v_sn;
    a.v_sh = d->v_sh;
    a.b = d->b;
    a.nq = d->nq;
    a.nk = d->nk;
    a.h = d->h;
    a.hk = d->hk;
    a.g = p.g;
    a.rows = p.rows;
    a.frame = d->frame;
    a.lam_bf16 = d->lam_dtype == VSPW_BF16;
    a.lchunks = p.lchunks;
    a.scale = d->scale;
    a.c = d->scale * 1.4426950408889634f;
}

extern "C" size_t vspw_diff_attn_fwd_workspace(const vspw_dattn_desc* d) {
    DaPlan p;
    return da_plan(d, p) ? p.fwd_bytes : 0;
}
extern "C" size_t vspw_diff_attn_bwd_workspace(const vspw_dattn_desc* d) {
    DaPlan p;
    return da_plan(d, p) ? p.bwd_bytes : 0;
}

template <typename T, int D>
static int da_fwd_launch(const DaArgs& a, const DaPlan& p, hipStream_t st) {
    const dim3 grid((unsigned)(p.tiles * p.bhk * p.parts));
    if (p.wn == 1)
        hipLaunchKernelGGL((da_fwd_kernel<T, D, 1>), grid, dim3(64), 0, st, a);
    else
        hipLaunchKernelGGL((da_fwd_kernel<T, D, 4>), grid, dim3(256), 0, st, a);
    const int rc = vspw_launch_status();
    if (rc != VSPW_OK || p.parts == 1) return rc;
    hipLaunchKernelGGL((da_join_kernel<T, D>), dim3((unsigned)(p.bhk * p.rows)), dim3(256), 0, st, a);
    return vspw_launch_status();
}

template <typename T, int D>
static int da_bwd_launch(DaArgs a, const DaPlan& p, hipStream_t st) {
    hipLaunchKernelGGL((da_delta_kernel<T, D>), dim3((unsigned)((long long)a.b * a.h * p.lchunks)), dim3(256), 0, st, a);
    int rc = vspw_launch_status();
    if (rc == VSPW_OK && a.dlam) {
        hipLaunchKernelGGL(da_dlam_kernel, dim3((unsigned)a.h), dim3(256), 0, st, a);
        rc = vspw_launch_status();
    }
    if (rc == VSPW_OK && a.dq) {
        a.tiles = p.qt;
        a.parts = p.qparts;
        a.span = p.qspan;
        hipLaunchKernelGGL((da_dq_kernel<T, D>), dim3((unsigned)(p.qt * p.bhk * p.qparts)), dim3(256), 0, st, a);
        rc = vspw_launch_status();
        if (rc == VSPW_OK && p.qparts > 1) {
            const long long n = (long long)a.b * a.nq * a.h * 2 * D;
            hipLaunchKernelGGL((da_sum_kernel<T>), dim3(vspw_stream_grid(n / 4, 256)), dim3(256), 0, st, a.part,
                               reinterpret_cast<T*>(a.dq), n / 4, p.qparts, n);
            rc = vspw_launch_status();
        }
    }
    if (rc == VSPW_OK && a.dk) {
        a.tiles = p.kt;
        a.parts = p.kparts;
        a.span = p.kspan;
        hipLaunchKernelGGL((da_dkv_kernel<T, D>), dim3((unsigned)(p.kt * p.bhk * p.kparts)), dim3(256), 0, st, a);
        rc = vspw_launch_status();
        if (rc == VSPW_OK && p.kparts > 1) {
            const long long n = (long long)a.b * a.nk * a.hk * 2 * D;
            hipLaunchKernelGGL((da_sum_kernel<T>), dim3(vspw_stream_grid(n / 4, 256)), dim3(256), 0, st, a.part,
                               reinterpret_cast<T*>(a.dk), n / 4, p.kparts, 2 * n);
            rc = vspw_launch_status();
            if (rc == VSPW_OK)
                hipLaunchKernelGGL((da_sum_kernel<T>), dim3(vspw_stream_grid(n / 4, 256)), dim3(256), 0, st, a.part + n,
                                   reinterpret_cast<T*>(a.dv), n / 4, p.kparts, 2 * n);
            if (rc == VSPW_OK) rc = vspw_launch_status();
        }
    }
    return rc;
}

#define DA_DISPATCH(FN, ...)                                                                       \
    (d->dtype == VSPW_F32 ? (d->d == 16 ? FN<float, 16>(__VA_ARGS__)                               \
                                        : d->d == 32 ? FN<float, 32>(__VA_ARGS__) : FN<float, 64>(__VA_ARGS__)) \
                          : (d->d == 16 ? FN<bf16_t, 16>(__VA_ARGS__)                              \
                                        : d->d == 32 ? FN<bf16_t, 32>(__VA_ARGS__) : FN<bf16_t, 64>(__VA_ARGS__)))

extern "C" int vspw_diff_attn_fwd(const vspw_dattn_desc* d, const void* q, const void* k, const void* v, const void* lam,
                                  const unsigned char* key_mask, void* out, void* o2, float* lse, void* ws, size_t ws_bytes,
                                  void* stream) {
    DaPlan p;
    if (!q || !k || !v || !lam || !out || !da_plan(d, p) || !da_strides_ok(d, q, k, v)) return VSPW_EINVAL;
    if ((((uintptr_t)out | (uintptr_t)o2 | (uintptr_t)ws) & 15) || ws_bytes < p.fwd_bytes || (p.fwd_bytes && !ws)) return VSPW_EINVAL;
    DaArgs a;
    da_fill(a, d, p, q, k, v, lam, key_mask);
    a.out = out;
    a.o2 = o2;
    a.lse = lse;
    a.tiles = p.tiles;
    a.parts = p.parts;
    a.span = p.span;
    a.part = reinterpret_cast<float*>(ws);
    if (p.parts > 1) a.ml = a.part + (size_t)p.parts * p.bhk * p.rows * 4 * d->d;
    return DA_DISPATCH(da_fwd_launch, a, p, vspw_stream(stream));
}

extern "C" int vspw_diff_attn_bwd(const vspw_dattn_desc* d, const void* q, const void* k, const void* v, const void* lam,
                                  const unsigned char* key_mask, const void* out, const void* o2, const float* lse,
                                  const void* go, void* dq, void* dk, void* dv, void* dlam, void* ws, size_t ws_bytes,
                                  void* stream) {
    DaPlan p;
    if (!q || !k || !v || !lam || !out || !o2 || !lse || !go || !da_plan(d, p) || !da_strides_ok(d, q, k, v)) return VSPW_EINVAL;
    if ((dk == nullptr) != (dv == nullptr) || !ws || ws_bytes < p.bwd_bytes) return VSPW_EINVAL;
    if (((uintptr_t)out | (uintptr_t)o2 | (uintptr_t)go | (uintptr_t)dq | (uintptr_t)dk | (uintptr_t)dv | (uintptr_t)ws) & 15)
        return VSPW_EINVAL;
    DaArgs a;
    da_fill(a, d, p, q, k, v, lam, key_mask);
    a.out = const_cast<void*>(out);
    a.o2 = const_cast<void*>(o2);
    a.lse = const_cast<float*>(lse);
    a.go = go;
    a.dq = dq;
    a.dk = dk;
    a.dv = dv;
    a.dlam = dlam;
    // [lpart doubles][delta][partial sums], every piece on 16 bytes
    a.lpart = reinterpret_cast<double*>(ws);
    size_t off = ((size_t)d->b * d->h * p.lchunks * sizeof(double) + 15) / 16 * 16;
    a.delta = reinterpret_cast<float*>(reinterpret_cast<char*>(ws) + off);
    off += ((size_t)2 * p.bhk * p.rows * sizeof(float) + 15) / 16 * 16;
    a.part = reinterpret_cast<float*>(reinterpret_cast<char*>(ws) + off);
    return DA_DISPATCH(da_bwd_launch, a, p, vspw_stream(stream));
}

extern "C" int vspw_diff_lambda_fwd(const float* lq1, const float* lk1, const float* lq2, const float* lk2, float init,
                                    float* lam, int h, int d, void* stream) {
    if (!lq1 || !lk1 || !lq2 || !lk2 || !lam || h <= 0 || d <= 0) return VSPW_EINVAL;
    hipLaunchKernelGGL(diff_lambda_kernel, dim3((unsigned)h), dim3(64), 0, vspw_stream(stream), lq1, lk1, lq2, lk2, init, lam,
                       nullptr, nullptr, nullptr, nullptr, nullptr, d);
    return vspw_launch_status();
}

extern "C" int vspw_diff_lambda_bwd(const float* lq1, const float* lk1, const float* lq2, const float* lk2, const float* g,
                                    float* gq1, float* gk1, float* gq2, float* gk2, int h, int d, void* stream) {
    if (!lq1 || !lk1 || !lq2 || !lk2 || !g || !gq1 || !gk1 || !gq2 || !gk2 || h <= 0 || d <= 0) return VSPW_EINVAL;
    hipLaunchKernelGGL(diff_lambda_kernel, dim3((unsigned)h), dim3(64), 0, vspw_stream(stream), lq1, lk1, lq2, lk2, 0.f,
                       nullptr, g, gq1, gk1, gq2, gk2, d);
    return vspw_launch_status();
}
