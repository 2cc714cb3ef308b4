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
// All softmax statistics and sums are fp32.  bf16 inputs: P and dS enter the matrix unit, which takes both operands in the same
// type, as two bf16 terms (16 bits: rounded to one term alone they cost as much as the rounding of the result does, measured
// 2.4e-3 against 1.7e-3 relative); everything else stays fp32 until the one rounding of each result.
#include <limits.h>
#include <math.h>

#include <type_traits>

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
    typedef Frag RegFrag;
    static constexpr int STEPS = 8, RSTEPS = 8;  // matrix instructions per product of two fragments
    // The frame rule in every tile and the scores of one tile too many are hidden behind the matrix instructions here, and a
    // second or third copy of the loop costs registers that spill.
    static constexpr bool ONE_LOOP = true;
    static __device__ __forceinline__ RegFrag reg(const f32x16& s, int t) {
        Frag f;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            f.a[e] = s[8 * t + e];
            f.b[e] = s[8 * t + 4 + e];
        }
        return f;
    }
    static __device__ __forceinline__ void step(f32x16& acc, const Frag& x, const Frag& y, int e) {
        acc = __builtin_amdgcn_mfma_f32_32x32x2f32(e < 4 ? x.a[e & 3] : x.b[e & 3], e < 4 ? y.a[e & 3] : y.b[e & 3], acc, 0, 0, 0);
    }
    static __device__ __forceinline__ f32x16 first(const Frag& x, const Frag& y, const f32x16& c) {  // step 0 onto c
        return __builtin_amdgcn_mfma_f32_32x32x2f32(x.a[0], y.a[0], c, 0, 0, 0);
    }
    static __device__ __forceinline__ void rstep(f32x16& acc, const Frag& x, const RegFrag& y, int e) { step(acc, x, y, e); }
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
    struct RegFrag {
        Frag hi, lo;
    };
    static __device__ __forceinline__ unsigned pack(float x, float y) {  // two at a time: one instruction
        typedef float f32x2 __attribute__((ext_vector_type(2)));
        typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
        return __builtin_bit_cast(unsigned, __builtin_convertvector(f32x2{x, y}, bf16x2));
    }
    static constexpr int STEPS = 1, RSTEPS = 2;
    static constexpr bool ONE_LOOP = false;
    static __device__ __forceinline__ RegFrag reg(const f32x16& s, int t) {
        u32x4 hi, lo;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float x = s[8 * t + 2 * i], y = s[8 * t + 2 * i + 1];
            hi[i] = pack(x, y);
            lo[i] = pack(x - __uint_as_float(hi[i] << 16), y - __uint_as_float(hi[i] & 0xffff0000u));
        }
        RegFrag f;
        f.hi = __builtin_bit_cast(Frag, hi);
        f.lo = __builtin_bit_cast(Frag, lo);
        return f;
    }
    static __device__ __forceinline__ void step(f32x16& acc, const Frag& x, const Frag& y, int) {
        acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(x, y, acc, 0, 0, 0);
    }
    static __device__ __forceinline__ f32x16 first(const Frag& x, const Frag& y, const f32x16& c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(x, y, c, 0, 0, 0);
    }
    static __device__ __forceinline__ void rstep(f32x16& acc, const Frag& x, const RegFrag& y, int e) {
        acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(x, e ? y.lo : y.hi, acc, 0, 0, 0);
    }
    static __device__ __forceinline__ void store4(bf16_t* p, f32x4 v) {
        bf16x4 o;
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = (bf16_t)v[e];
        *reinterpret_cast<bf16x4*>(p) = o;
    }
};

// Holds the order of the instruction stream: the vector work of a tile is dealt out between matrix instructions (64 cycles each
// in fp32) and operand fragments are read one step ahead; left to itself the compiler moves all reads up and runs out of
// registers, or gathers the vector work in one place, where the matrix unit waits for it.
__device__ __forceinline__ void da_pin() { __builtin_amdgcn_sched_barrier(0); }

struct DaArgs {
    const void *q, *k, *v, *lam, *go;
    const unsigned char* mask;
    void* out;                  // [B,Nq,H,2D]
    float* maps;                // [B,Nq,H,2,2D]: P_1 v and P_2 v in fp32, for D_m
    float* lse;                 // [2][B*Hk][rows]: log2-sum-exp2 of s log2(e) S (+inf: no visible key)
    float* stat;                // [6][B*Hk][rows]: both log-sum-exps, D_1, D_2, lambda, key limit (int): a row's constants
    void *dq, *dk, *dv, *dlam;
    float* part;                // partial results of a split axis
    float* ml;                  // forward: [chunks][B*Hk][rows][2] running maximum and sum per map: [..][2 m], [..][2 m + 1]
    double* lpart;              // [B*H][lchunks]: sums of D_2
    int* alone;                 // [B]: at most one key takes part
    long long q_sb, q_sn, q_sh, q_sm, k_sb, k_sn, k_sh, k_sm, v_sb, v_sn, v_sh;
    int b, nq, nk, h, hk, g, rows, frame, lam_bf16, lchunks;
    int tiles, parts, span;     // workgroups along the owned axis; split of the streamed axis: parts of `span` entries
    float c, scale;             // scale * log2(e), scale
    unsigned gm, gs;            // x / g = x * gm >> gs for 0 <= x < 2^31
};

__device__ __forceinline__ float da_lambda(const DaArgs& a, int head) {
    return a.lam_bf16 ? (float)reinterpret_cast<const bf16_t*>(a.lam)[head] : reinterpret_cast<const float*>(a.lam)[head];
}
__device__ __forceinline__ int da_div(const DaArgs& a, int x) { return (int)(((unsigned long long)(unsigned)x * a.gm) >> a.gs); }
// keys [0, lim) are within the frames that the row's query sees
__device__ __forceinline__ int da_limit(const DaArgs& a, int row) {
    if (!a.frame) return a.nk;
    const long long pos = (long long)(row / a.g) + a.nk - a.nq;
    if (pos < 0) return 0;
    const long long lim = (pos / a.frame + 1) * a.frame;
    return lim < a.nk ? (int)lim : a.nk;
}
// The first row (a multiple of DA_TILE) that sees keys from `key` on, which may lie behind the last one.
__device__ __forceinline__ long long da_first_row(const DaArgs& a, int key) {
    const long long q0 = (long long)(key / a.frame) * a.frame - a.nk + a.nq;
    return q0 > 0 ? q0 * a.g / DA_TILE * DA_TILE : 0;
}
// With frames the parts that stream nothing write nothing, and a tile with a single part left writes its result itself.
// Parts [0, n) of the rows' tile that ends with row `last`, and [n, parts) of the keys' tile that begins with `key`:
__device__ __forceinline__ int da_row_parts(const DaArgs& a, int last) {
    return a.frame ? max(0, da_limit(a, last) - 1) / a.span + 1 : a.parts;
}
__device__ __forceinline__ int da_key_parts(const DaArgs& a, int key) {
    return a.frame ? (int)min(da_first_row(a, key) / a.span, (long long)a.parts - 1) : 0;
}
// The workgroup's place.  With frames the parts that every tile has come first, and among them the longest tiles (rows: the
// last, keys: the first); neighbours, which go to different XCDs, then have like lengths.
__device__ __forceinline__ void da_place(const DaArgs& a, bool keys, int& tile, int& part, int& bh) {
    const int x = blockIdx.x;
    if (a.frame) {
        const int nb = a.b * a.hk;
        bh = x % nb;
        tile = x / nb % a.tiles;
        part = x / nb / a.tiles;
        if (keys)
            part = a.parts - 1 - part;
        else
            tile = a.tiles - 1 - tile;
    } else {
        tile = x % a.tiles;
        part = x / a.tiles % a.parts;
        bh = x / a.tiles / a.parts;
    }
}
__device__ __forceinline__ f32x16 zero16() {
    f32x16 z;
#pragma unroll
    for (int r = 0; r < 16; ++r) z[r] = 0.f;
    return z;
}
// maximum over the two lane halves
__device__ __forceinline__ float half_max(float x) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ int acc_index(int r, int lh) { return (r & 3) + 8 * (r >> 2) + 4 * lh; }
// x - lam y as the same two roundings whether or not the maps are stored too
__device__ __forceinline__ f32x4 da_mix(f32x4 x, f32x4 y, float lam) {
#pragma clang fp contract(off)
    return x - y * lam;
}
__device__ __forceinline__ f32x4 da_scaled(f32x4 x, float f) {
#pragma clang fp contract(off)
    return x * f;
}
__device__ __forceinline__ f32x4 quad(const f32x16& s, int g4) { return f32x4{s[4 * g4], s[4 * g4 + 1], s[4 * g4 + 2], s[4 * g4 + 3]}; }

// A streamed [32][2D] tile on its way from global memory through registers into LDS: 16-byte vectors, thread t moves the
// vectors t + THREADS * i (a tile smaller than the workgroup is moved more than once).  Nothing here branches or looks at what
// a load brought before put(): a branch would part the vector work from the matrix instructions it is dealt out between, a
// look would wait for memory.
template <typename T, int D, int THREADS>
struct Stager {
    static constexpr int VE = 16 / (int)sizeof(T);
    static constexpr int VROW = 2 * D / VE;  // vectors per row
    static constexpr int TOTAL = DA_TILE * VROW;
    static constexpr int F = (TOTAL + THREADS - 1) / THREADS;
    static constexpr int STEP = THREADS / VROW;  // rows between a thread's vectors
    static constexpr int LD = 2 * D + Mx<T>::PAD;
    static_assert((TOTAL % THREADS == 0 || THREADS % TOTAL == 0) && THREADS % VROW == 0, "");
    u32x4 x[F];

    static __device__ __forceinline__ int row(int tid, int i) { return tid % TOTAL / VROW + STEP * i; }
    static __device__ __forceinline__ int col(int tid) { return tid % VROW * VE; }
    __device__ __forceinline__ void get(int i, const char* base, unsigned off) { x[i] = *reinterpret_cast<const u32x4*>(base + off); }
    __device__ __forceinline__ void put(int tid, int i, T* X, bool ok) const {  // rows that take no part: zeros
        *reinterpret_cast<u32x4*>(X + row(tid, i) * LD + col(tid)) = ok ? x[i] : u32x4{0, 0, 0, 0};
    }
};

// The key side of a workgroup that owns rows: its share of the keys, and tiles of k and v on their way into LDS.
template <typename T, int D, int THREADS>
struct KeyStream {
    typedef Stager<T, D, THREADS> St;
    St k, v;
    const char *kp, *vp;      // the next tile to fetch; the last one of the tensor is fetched again and again
    const unsigned char* mb;  // the mask's row, or any readable byte when there is none
    long long ks, vs;         // bytes from key to key
    unsigned k0, v0, kc, vc;  // this thread's first row and column in bytes
    unsigned live1, live2;    // which keys of the last two tiles of k take part
    int begin, end, nk, krem, vrem, ktile, mstep, open;  // ?rem: keys of the tensor behind the first of the next tile
    unsigned char raw;

    __device__ __forceinline__ void init(const DaArgs& a, int tid, int bi, int kh, int part, int last_row) {
        constexpr int E = (int)sizeof(T);
        begin = part * a.span;  // below nk
        kp = reinterpret_cast<const char*>(reinterpret_cast<const T*>(a.k) + bi * a.k_sb + kh * a.k_sh + begin * a.k_sn);
        vp = reinterpret_cast<const char*>(reinterpret_cast<const T*>(a.v) + bi * a.v_sb + kh * a.v_sh + begin * a.v_sn);
        open = a.mask == nullptr;
        mb = open ? reinterpret_cast<const unsigned char*>(kp) : a.mask + (size_t)bi * a.nk;
        mstep = open ? 0 : 1;
        ks = a.k_sn * E;
        vs = a.v_sn * E;
        const int c = St::col(tid), r = St::row(tid, 0);
        k0 = r * (unsigned)ks;
        v0 = r * (unsigned)vs;
        kc = (c >= D ? (unsigned)a.k_sm + c - D : c) * E;
        vc = c * E;
        nk = a.nk;
        krem = vrem = nk - 1 - begin;
        ktile = begin - DA_TILE;
        end = min(min(a.nk, begin + a.span), da_limit(a, last_row));
        live1 = live2 = 0;
    }
    __device__ __forceinline__ int tiles() const { return end > begin ? (end - begin + DA_TILE - 1) / DA_TILE : 0; }
    // leading tiles of which every row of the workgroup sees all frames (rows see more and more keys: the first row decides)
    __device__ __forceinline__ int plain(const DaArgs& a, int first_row) const {
        return a.frame ? max(0, da_limit(a, first_row) - begin) / DA_TILE : tiles();
    }
    // vector i of the next tile; the last vector moves on
    __device__ __forceinline__ void get_k(int tid, int i) {
        if (i == 0) {
            ktile += DA_TILE;
            raw = mb[(unsigned)(min(ktile + tid % DA_TILE, nk - 1) * mstep)];
        }
        k.get(i, kp, min(k0 + i * St::STEP * (unsigned)ks, (unsigned)min(krem, DA_TILE) * (unsigned)ks) + kc);
        if (i == St::F - 1) {
            kp += krem >= DA_TILE ? DA_TILE * ks : 0;
            krem -= krem >= DA_TILE ? DA_TILE : 0;
        }
    }
    __device__ __forceinline__ void get_v(int i) {
        v.get(i, vp, min(v0 + i * St::STEP * (unsigned)vs, (unsigned)min(vrem, DA_TILE) * (unsigned)vs) + vc);
        if (i == St::F - 1) {
            vp += vrem >= DA_TILE ? DA_TILE * vs : 0;
            vrem -= vrem >= DA_TILE ? DA_TILE : 0;
        }
    }
    __device__ __forceinline__ void put_k(int tid, int i, T* K, float* B) {
        if (i == 0) {
            live1 = live2;
            const bool on = (ktile + tid % DA_TILE < end) & ((open | raw) != 0);
            live2 = (unsigned)__ballot(on);  // lanes 0..31: the tile's keys
            B[tid % DA_TILE] = on ? 0.f : -DA_INF;  // the same value from every thread of that key
        }
        k.put(tid, i, K, (live2 >> St::row(tid, i)) & 1);
    }
    __device__ __forceinline__ void put_v(int tid, int i, T* V, unsigned live) { v.put(tid, i, V, (live >> St::row(tid, i)) & 1); }
};

// What a tile's scores start from: 0, or -inf for the keys that take no part.
__device__ __forceinline__ f32x16 da_bias(const float* B, int lh) {
    f32x16 s;
#pragma unroll
    for (int g4 = 0; g4 < 4; ++g4) {
        const f32x4 b = *reinterpret_cast<const f32x4*>(B + 8 * g4 + 4 * lh);
#pragma unroll
        for (int i = 0; i < 4; ++i) s[4 * g4 + i] = b[i];
    }
    return s;
}

// Which row of the problem a lane of a row-owning workgroup stands for.
struct RowOf {
    int bi, kh, part, block0, row0, row, head, qi;
    bool live;
    __device__ __forceinline__ RowOf(const DaArgs& a, int wn, int wave, int l31) {
        int tile, bh;
        da_place(a, false, tile, part, bh);
        bi = bh / a.hk;
        kh = bh % a.hk;
        block0 = tile * 32 * wn;
        row0 = block0 + wave * 32;
        live = row0 + l31 < a.rows;
        row = min(row0 + l31, a.rows - 1);  // rows past the end repeat the last one and are not stored
        head = kh * a.g + row % a.g;
        qi = row / a.g;
    }
    __device__ __forceinline__ int last(const DaArgs& a, int wn) const { return min(block0 + 32 * wn, a.rows) - 1; }
};

#define DA_BOOL(x) std::integral_constant<bool, x>()

// ---------------------------------------------------------------------------------------------------------- forward
// Software pipeline.  A: the scores of tile t + 1 on the matrix unit, tile t's weights 2^(c S - m) on the vector unit; B: tile
// t's weights times v, and the maximum of tile t + 1.  One barrier per tile, between A and B.  k of tile t + 2 is put into
// LDS in A (its buffer was last read in the A before), v of tile t + 1 in B: both are read behind the next barrier only.
// Four waves of 32 rows share a key tile; up to 32 rows are one wave, and the keys are cut into more parts instead.
// Measured (12 D operations per row and key): fp32, 2 x 18000 rows and keys, D = 64: 4.33 ms, 115 TFLOP/s, matrix unit busy
// 76 - 80 %, its rate is the bound.  bf16, 6420 rows and keys, 4 heads, D = 32: 154 us, 411 TFLOP/s (the second term of the
// weights comes on top): the vector unit's two exponentials, roundings and maxima per row and key are the bound (74 % busy).
template <typename T, int D, int WN>
__global__ __launch_bounds__(64 * WN, WN == 1 || D == 64 ? 1 : 2) void da_fwd_kernel(const DaArgs a) {
    typedef Mx<T> M;
    typedef typename M::Frag Frag;
    typedef Stager<T, D, 64 * WN> St;
    constexpr int W = 2 * D, LD = St::LD, KC = D / 16, CB = W / 32;
    __shared__ __attribute__((aligned(16))) T Ks[2][DA_TILE * LD];
    __shared__ __attribute__((aligned(16))) T Vs[2][DA_TILE * LD];
    __shared__ __attribute__((aligned(16))) float Kb[2][DA_TILE];  // 0, or -inf for keys that take no part

    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, l31 = lane & 31, lh = lane >> 5;
    const RowOf ro(a, WN, wave, l31);
    const int nparts = da_row_parts(a, ro.last(a, WN));
    if (ro.part >= nparts) return;
    const T* qrow = reinterpret_cast<const T*>(a.q) + ro.bi * a.q_sb + ro.qi * a.q_sn + ro.head * a.q_sh;
    Frag q1[KC], q2[KC];
#pragma unroll
    for (int i = 0; i < KC; ++i) {
        q1[i] = M::row(qrow + 16 * i, lh);
        q2[i] = M::row(qrow + a.q_sm + 16 * i, lh);
    }
    const int lim = da_limit(a, ro.row);
    KeyStream<T, D, 64 * WN> ks;
    ks.init(a, tid, ro.bi, ro.kh, ro.part, ro.last(a, WN));
    const int ntiles = ks.tiles(), nplain = ks.plain(a, min(ro.block0, a.rows - 1));

    f32x16 o1[CB], o2[CB], s1, s2, n1, n2;
#pragma unroll
    for (int j = 0; j < CB; ++j) o1[j] = o2[j] = zero16();
    float m1 = -DA_INF, m2 = -DA_INF, l1 = 0.f, l2 = 0.f, x1 = -DA_INF, x2 = -DA_INF;
    Frag ga, gb;  // the first operands of the next A
    f32x16 bias;

    // one entry of both maps' scores of the tile at key0: later frames to -inf (EDGE), running maximum
    auto entry = [&](auto edge, f32x16& u, f32x16& w, int r, int key0) {
        if (decltype(edge)::value) {
            const bool hide = key0 + acc_index(r, lh) >= lim;
            u[r] = hide ? -DA_INF : u[r];
            w[r] = hide ? -DA_INF : w[r];
        }
        x1 = fmaxf(x1, u[r]);
        x2 = fmaxf(x2, w[r]);
    };
    auto finish_max = [&]() {  // over both lane halves, in the exponent's units
        x1 = half_max(x1) * a.c;
        x2 = half_max(x2) * a.c;
    };
    auto ready = [&](int buf) {  // what the next A starts from
        bias = da_bias(Kb[buf], lh);
        ga = M::row(Ks[buf] + l31 * LD, lh);
        gb = M::row(Ks[buf] + l31 * LD + D, lh);
    };
    // one tile: its scores in (s1, s2), those of the next left in (n1, n2); two calls in turn save the copy (bf16: 8 %)
    auto body = [&](auto next, auto edge, int t, f32x16& s1, f32x16& s2, f32x16& n1, f32x16& n2) {
        constexpr bool NEXT = decltype(next)::value;
        const int cur = t & 1, nxt = cur ^ 1, key1 = ks.begin + (t + 1) * DA_TILE;
        // The sums are rescaled only when a maximum has grown by more than 2^8: weights stay below 256.
        if (__any(x1 > m1 + 8.f || x2 > m2 + 8.f)) {
            const float a1 = fmaxf(m1, x1), a2 = fmaxf(m2, x2);
            const float f1 = m1 == -DA_INF ? 0.f : exp2f(m1 - a1), f2 = m2 == -DA_INF ? 0.f : exp2f(m2 - a2);
            m1 = a1;
            m2 = a2;
            l1 *= f1;
            l2 *= f2;
#pragma unroll
            for (int j = 0; j < CB; ++j)
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    o1[j][r] *= f1;
                    o2[j][r] *= f2;
                }
        }
        const float u1 = m1 == -DA_INF ? 0.f : m1, u2 = m2 == -DA_INF ? 0.f : m2;
        const T* Kn = Ks[nxt] + l31 * LD;
        constexpr int SL = KC * M::STEPS;
#pragma unroll
        for (int i = 0; i < KC; ++i) {
            const Frag fa = ga, fb = gb;
            if (NEXT && i + 1 < KC) {
                ga = M::row(Kn + 16 * (i + 1), lh);
                gb = M::row(Kn + D + 16 * (i + 1), lh);
            }
#pragma unroll
            for (int e = 0; e < M::STEPS; ++e) {
                if (NEXT && i + e == 0) {
                    n1 = M::first(fa, q1[0], bias);
                    n2 = M::first(fb, q2[0], bias);
                } else if (NEXT) {
                    M::step(n1, fa, q1[i], e);
                    M::step(n2, fb, q2[i], e);
                }
                const int slot = i * M::STEPS + e;
#pragma unroll
                for (int it = slot * 32 / SL; it < (slot + 1) * 32 / SL; ++it) {
                    const int r = it >> 1;
                    if (it & 1) {
                        s2[r] = __builtin_amdgcn_exp2f(fmaf(s2[r], a.c, -u2));
                        l2 += s2[r];
                    } else {
                        s1[r] = __builtin_amdgcn_exp2f(fmaf(s1[r], a.c, -u1));
                        l1 += s1[r];
                    }
                }
                if (NEXT) {
#pragma unroll
                    for (int f = slot * St::F / SL; f < (slot + 1) * St::F / SL; ++f) {
                        ks.put_k(tid, f, Ks[cur], Kb[cur]);
                        ks.get_k(tid, f);
                    }
                }
                da_pin();
            }
        }
        __syncthreads();
        Frag vn = M::col(Vs[cur], LD, 0, 0, lane);  // put by all waves in the B before
        da_pin();
        x1 = x2 = -DA_INF;
        constexpr int SB = 2 * CB * M::RSTEPS, S0 = SB >= 16 ? 2 : 0;  // the scores' last products are still in flight
#pragma unroll
        for (int t2 = 0; t2 < 2; ++t2) {
            const typename M::RegFrag p1 = M::reg(s1, t2), p2 = M::reg(s2, t2);
#pragma unroll
            for (int j = 0; j < CB; ++j) {
                const Frag vf = vn;
                if (t2 * CB + j + 1 < 2 * CB) vn = M::col(Vs[cur], LD, 16 * ((t2 * CB + j + 1) / CB), 32 * ((j + 1) % CB), lane);
#pragma unroll
                for (int e = 0; e < M::RSTEPS; ++e) {
                    M::rstep(o1[j], vf, p1, e);
                    M::rstep(o2[j], vf, p2, e);
                    const int slot = (t2 * CB + j) * M::RSTEPS + e;
                    if (NEXT && slot >= S0) {
#pragma unroll
                        for (int r = (slot - S0) * 16 / (SB - S0); r < (slot - S0 + 1) * 16 / (SB - S0); ++r) entry(edge, n1, n2, r, key1);
                    }
                    if (NEXT) {
#pragma unroll
                        for (int f = slot * St::F / SB; f < (slot + 1) * St::F / SB; ++f) {
                            ks.put_v(tid, f, Vs[nxt], ks.live1);
                            ks.get_v(f);
                        }
                    }
                    da_pin();
                }
            }
        }
        if (NEXT) {
            finish_max();
            ready(cur);
        }
    };

    if (ntiles > 0) {
#pragma unroll
        for (int f = 0; f < St::F; ++f) {
            ks.get_k(tid, f);
            ks.get_v(f);
        }
#pragma unroll
        for (int f = 0; f < St::F; ++f) {
            ks.put_k(tid, f, Ks[0], Kb[0]);
            ks.put_v(tid, f, Vs[0], ks.live2);
            ks.get_v(f);
        }
#pragma unroll
        for (int f = 0; f < St::F; ++f) ks.get_k(tid, f);
        __syncthreads();
        s1 = s2 = da_bias(Kb[0], lh);
        const T* K0 = Ks[0] + l31 * LD;
#pragma unroll
        for (int i = 0; i < KC; ++i) {
            const Frag fa = M::row(K0 + 16 * i, lh), fb = M::row(K0 + D + 16 * i, lh);
#pragma unroll
            for (int e = 0; e < M::STEPS; ++e) {
                M::step(s1, fa, q1[i], e);
                M::step(s2, fb, q2[i], e);
            }
        }
#pragma unroll
        for (int r = 0; r < 16; ++r) entry(DA_BOOL(true), s1, s2, r, ks.begin);
        finish_max();
#pragma unroll
        for (int f = 0; f < St::F; ++f) {
            ks.put_k(tid, f, Ks[1], Kb[1]);
            ks.get_k(tid, f);
        }
        __syncthreads();
        ready(1);
        int t = 0;
        if (M::ONE_LOOP) {
            for (; t < ntiles; ++t) {  // the tile past the end has weights 0
                body(DA_BOOL(true), DA_BOOL(true), t, s1, s2, n1, n2);
                s1 = n1;
                s2 = n2;
            }
        } else {  // tiles that every row of the workgroup sees whole come first
            for (; t + 2 < min(nplain, ntiles); t += 2) {
                body(DA_BOOL(true), DA_BOOL(false), t, s1, s2, n1, n2);
                body(DA_BOOL(true), DA_BOOL(false), t + 1, n1, n2, s1, s2);
            }
            for (; t + 1 < ntiles; ++t) {
                body(DA_BOOL(true), DA_BOOL(true), t, s1, s2, n1, n2);
                s1 = n1;
                s2 = n2;
            }
            body(DA_BOOL(false), DA_BOOL(false), t, s1, s2, n1, n2);
        }
    }
    l1 += __shfl_xor(l1, 32, 64);
    l2 += __shfl_xor(l2, 32, 64);
    if (!ro.live) return;
    const size_t e = ((size_t)ro.bi * a.hk + ro.kh) * a.rows + ro.row, n = (size_t)a.b * a.hk * a.rows;
    if (nparts > 1) {  // unnormalised sums with their maximum, joined by da_join_kernel
        float* po = a.part + (ro.part * n + e) * 2 * W;
#pragma unroll
        for (int j = 0; j < CB; ++j)
#pragma unroll
            for (int g4 = 0; g4 < 4; ++g4) {
                const int ch = 32 * j + 8 * g4 + 4 * lh;
                *reinterpret_cast<f32x4*>(po + ch) = quad(o1[j], g4);
                *reinterpret_cast<f32x4*>(po + W + ch) = quad(o2[j], g4);
            }
        if (lh == 0) *reinterpret_cast<f32x4*>(a.ml + (ro.part * n + e) * 4) = f32x4{m1, l1, m2, l2};
        return;
    }
    const float i1 = l1 == 0.f ? 0.f : 1.f / l1, i2 = l2 == 0.f ? 0.f : 1.f / l2, lam = da_lambda(a, ro.head);
    const size_t o = (((size_t)ro.bi * a.nq + ro.qi) * a.h + ro.head) * W;
    T* out = reinterpret_cast<T*>(a.out) + o;
#pragma unroll
    for (int j = 0; j < CB; ++j)
#pragma unroll
        for (int g4 = 0; g4 < 4; ++g4) {
            const int ch = 32 * j + 8 * g4 + 4 * lh;
            const f32x4 x = da_scaled(quad(o1[j], g4), i1), y = da_scaled(quad(o2[j], g4), i2);
            M::store4(out + ch, da_mix(x, y, lam));
            if (a.maps) {
                *reinterpret_cast<f32x4*>(a.maps + 2 * o + ch) = x;
                *reinterpret_cast<f32x4*>(a.maps + 2 * o + W + ch) = y;
            }
        }
    if (a.lse && lh == 0) {
        a.lse[e] = l1 == 0.f ? DA_INF : m1 + log2f(l1);
        a.lse[n + e] = l2 == 0.f ? DA_INF : m2 + log2f(l2);
    }
}

#define DA_JOIN_PARTS 32
#define DA_ROW_PARTS 512
// Joins the parts of a row.  Up to 32 parts: W / 4 threads per row, each goes over the parts by itself (every thread of a row
// reads the same maxima and sums of weights, from the cache).
__device__ __forceinline__ int da_last_of(const DaArgs& a, int row) {  // the last row of the forward kernel's tile
    const int n = a.rows <= 32 ? 32 : 128;
    return min(row / n * n + n, a.rows) - 1;
}
template <typename T, int D>
__global__ __launch_bounds__(256) void da_join_kernel(const DaArgs a) {
    constexpr int W = 2 * D, CT = W / 4;
    const size_t n = (size_t)a.b * a.hk * a.rows, e = (size_t)blockIdx.x * (256 / CT) + threadIdx.x / CT;
    if (e >= n) return;
    const int ch = 4 * (threadIdx.x % CT);
    const int bh = (int)(e / a.rows), row = (int)(e % a.rows);
    const int head = (bh % a.hk) * a.g + row % a.g;
    const int nparts = da_row_parts(a, da_last_of(a, row));
    if (nparts == 1) return;
    float M1 = -DA_INF, M2 = -DA_INF, L1 = 0.f, L2 = 0.f;
    for (int p = 0; p < nparts; ++p) {
        const f32x4 v = *reinterpret_cast<const f32x4*>(a.ml + (p * n + e) * 4);
        M1 = fmaxf(M1, v[0]);
        M2 = fmaxf(M2, v[2]);
    }
    const float u1 = M1 == -DA_INF ? 0.f : M1, u2 = M2 == -DA_INF ? 0.f : M2;
    f32x4 x = {0.f, 0.f, 0.f, 0.f}, y = x;
#pragma unroll 4
    for (int p = 0; p < nparts; ++p) {
        const f32x4 v = *reinterpret_cast<const f32x4*>(a.ml + (p * n + e) * 4);
        const float* s = a.part + (p * n + e) * 2 * W + ch;
        const float w1 = exp2f(v[0] - u1), w2 = exp2f(v[2] - u2);
        x += *reinterpret_cast<const f32x4*>(s) * w1;
        y += *reinterpret_cast<const f32x4*>(s + W) * w2;
        L1 = fmaf(v[1], w1, L1);
        L2 = fmaf(v[3], w2, L2);
    }
    x = da_scaled(x, L1 == 0.f ? 0.f : 1.f / L1);
    y = da_scaled(y, L2 == 0.f ? 0.f : 1.f / L2);
    const size_t o = (((size_t)(bh / a.hk) * a.nq + row / a.g) * a.h + head) * W + ch;
    Mx<T>::store4(reinterpret_cast<T*>(a.out) + o, da_mix(x, y, da_lambda(a, head)));
    if (a.maps) {
        *reinterpret_cast<f32x4*>(a.maps + 2 * (o - ch) + ch) = x;
        *reinterpret_cast<f32x4*>(a.maps + 2 * (o - ch) + W + ch) = y;
    }
    if (a.lse && ch == 0) {
        a.lse[e] = L1 == 0.f ? DA_INF : u1 + log2f(L1);
        a.lse[n + e] = L2 == 0.f ? DA_INF : u2 + log2f(L2);
    }
}

// More parts (few rows, a long axis): a workgroup takes 8 columns of both maps of a row and deals the parts out over 64 groups
// of its threads, sums in a fixed tree.  4 rows on 25200 keys of 2 x 64, bf16: 394 parts cost 12.5 us and 6.1 us for joining, 197
// parts 14.3 us and 5.1 us (8.6 us with one workgroup per row).
template <typename T, int D>
__global__ __launch_bounds__(256) void da_join_row_kernel(const DaArgs a) {
    constexpr int W = 2 * D, COLS = 8, CT = 2 * COLS / 4, PT = 256 / CT;  // CT threads hold one part's columns of both maps
    __shared__ float red[4][4];
    __shared__ f32x4 sum[4][CT];
    const int tid = threadIdx.x, wave = tid >> 6;
    const size_t n = (size_t)a.b * a.hk * a.rows, e = blockIdx.x / (W / COLS);
    const int col0 = blockIdx.x % (W / COLS) * COLS;
    const int bh = (int)(e / a.rows), row = (int)(e % a.rows);
    const int head = (bh % a.hk) * a.g + row % a.g;
    const int nparts = da_row_parts(a, da_last_of(a, row));
    if (nparts == 1) return;
    f32x4 mine[DA_ROW_PARTS / 256];
    float u[2] = {-DA_INF, -DA_INF}, L[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < DA_ROW_PARTS / 256; ++i) {
        const int p = tid + 256 * i;
        mine[i] = p < nparts ? *reinterpret_cast<const f32x4*>(a.ml + (p * n + e) * 4) : f32x4{-DA_INF, 0.f, -DA_INF, 0.f};
        u[0] = fmaxf(u[0], mine[i][0]);
        u[1] = fmaxf(u[1], mine[i][2]);
    }
#pragma unroll
    for (int m = 0; m < 2; ++m) {
        u[m] = wave_max(u[m]);
        if ((tid & 63) == 0) red[m][wave] = u[m];
    }
    __syncthreads();
#pragma unroll
    for (int m = 0; m < 2; ++m) {
        u[m] = fmaxf(fmaxf(red[m][0], red[m][1]), fmaxf(red[m][2], red[m][3]));
        if (u[m] == -DA_INF) u[m] = 0.f;
#pragma unroll
        for (int i = 0; i < DA_ROW_PARTS / 256; ++i) L[m] = fmaf(mine[i][2 * m + 1], exp2f(mine[i][2 * m] - u[m]), L[m]);
        L[m] = wave_sum(L[m]);
        if ((tid & 63) == 0) red[2 + m][wave] = L[m];
    }
    const int c = tid % CT, map = c / (CT / 2), ch = map * W + col0 + c % (CT / 2) * 4;
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < DA_ROW_PARTS / PT; ++i) {
        const int p = tid / CT + PT * i;
        if (p < nparts)
            acc += *reinterpret_cast<const f32x4*>(a.part + (p * n + e) * 2 * W + ch) *
                   exp2f(a.ml[(p * n + e) * 4 + 2 * map] - u[map]);
    }
#pragma unroll
    for (int s = CT; s < 64; s *= 2)
#pragma unroll
        for (int x = 0; x < 4; ++x) acc[x] += __shfl_xor(acc[x], s, 64);
    if ((tid & 63) < CT) sum[wave][c] = acc;
    __syncthreads();
#pragma unroll
    for (int m = 0; m < 2; ++m) L[m] = (red[2 + m][0] + red[2 + m][1]) + (red[2 + m][2] + red[2 + m][3]);
    if (tid < CT / 2) {
        f32x4 x = (sum[0][tid] + sum[1][tid]) + (sum[2][tid] + sum[3][tid]);
        f32x4 y = (sum[0][CT / 2 + tid] + sum[1][CT / 2 + tid]) + (sum[2][CT / 2 + tid] + sum[3][CT / 2 + tid]);
        x = da_scaled(x, L[0] == 0.f ? 0.f : 1.f / L[0]);
        y = da_scaled(y, L[1] == 0.f ? 0.f : 1.f / L[1]);
        const size_t o = (((size_t)(bh / a.hk) * a.nq + row / a.g) * a.h + head) * W;
        const int oc = col0 + 4 * tid;
        Mx<T>::store4(reinterpret_cast<T*>(a.out) + o + oc, da_mix(x, y, da_lambda(a, head)));
        if (a.maps) {
            *reinterpret_cast<f32x4*>(a.maps + 2 * o + oc) = x;
            *reinterpret_cast<f32x4*>(a.maps + 2 * o + W + oc) = y;
        }
    }
    if (a.lse && col0 == 0 && tid < 2) a.lse[tid * n + e] = L[tid] == 0.f ? DA_INF : u[tid] + log2f(L[tid]);
}

// --------------------------------------------------------------------------------------------------------- backward
// The constants of every row for the backward pass (D_1, D_2 among them), and partial sums of D_2 per head: a workgroup owns
// 256 / LPR rows per trip of one (batch, head).  One read of both maps' outputs and of dO: 15 us for 2 x 18000 rows of 128.
template <typename T, int D>
__global__ __launch_bounds__(256) void da_delta_kernel(const DaArgs a) {
    constexpr int W = 2 * D, V = 4, LPR = W / V;
    __shared__ double red[4];
    const int chunk = blockIdx.x % a.lchunks, bh = blockIdx.x / a.lchunks;
    const int bi = bh / a.h, head = bh % a.h;
    const int kh = head / a.g, g = head % a.g;
    const int sub = threadIdx.x % LPR;
    const float lam = da_lambda(a, head);
    const size_t n = (size_t)a.b * a.hk * a.rows;
    if (chunk == 0 && head == 0) {  // counts the keys that take part, up to two
        int seen = a.mask ? 0 : a.nk;
        const unsigned char* m = a.mask ? a.mask + (size_t)bi * a.nk : nullptr;
        for (int j0 = 0; m && j0 < a.nk && seen < 2; j0 += 16 * 256) {
            int here = 0;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const int j = j0 + 256 * i + (int)threadIdx.x;
                here += (j < a.nk) & (m[min(j, a.nk - 1)] != 0);
            }
            seen += __syncthreads_count(here == 1) + 2 * (__syncthreads_count(here > 1) != 0);
        }
        if (threadIdx.x == 0) a.alone[bi] = seen < 2;
    }
    double total = 0.0;
    for (int q = chunk * (256 / LPR) + threadIdx.x / LPR; q < a.nq; q += a.lchunks * (256 / LPR)) {
        const size_t o = (((size_t)bi * a.nq + q) * a.h + head) * W;
        float go[V];
        Vec<T, V>::load(reinterpret_cast<const T*>(a.go) + o + V * sub, go);
        const f32x4 x = *reinterpret_cast<const f32x4*>(a.maps + 2 * o + V * sub);
        const f32x4 y = *reinterpret_cast<const f32x4*>(a.maps + 2 * o + W + V * sub);
        double d1 = 0.0, d2 = 0.0;  // dlam's sum over the rows may cancel: nothing is rounded on the way to it
#pragma unroll
        for (int i = 0; i < V; ++i) {
            d1 = fma((double)go[i], (double)x[i], d1);
            d2 = fma((double)go[i], (double)y[i], d2);
        }
        for (int s = LPR / 2; s > 0; s >>= 1) {
            d1 += __shfl_xor(d1, s, 64);
            d2 += __shfl_xor(d2, s, 64);
        }
        if (sub == 0) {
            const int row = q * a.g + g;
            const size_t e = ((size_t)bi * a.hk + kh) * a.rows + row;
            a.stat[e] = a.lse[e];
            a.stat[n + e] = a.lse[n + e];
            a.stat[2 * n + e] = (float)d1;
            a.stat[3 * n + e] = (float)d2;
            a.stat[4 * n + e] = lam;
            a.stat[5 * n + e] = __int_as_float(da_limit(a, row));
            total += d2;
        }
    }
    total = wave_sum_d(total);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = total;
    __syncthreads();
    if (threadIdx.x == 0) a.lpart[(size_t)bh * a.lchunks + chunk] = (red[0] + red[1]) + (red[2] + red[3]);
}

// dlam[h] = - sum over batch and chunks: one workgroup per head
__global__ __launch_bounds__(256) void da_dlam_kernel(const DaArgs a) {
    __shared__ double red[4];
    const int head = blockIdx.x, n = a.b * a.lchunks;
    double s = 0.0;
    for (int i = threadIdx.x; i < n; i += 256)
        s += a.lpart[((size_t)(i / a.lchunks) * a.h + head) * a.lchunks + i % a.lchunks];
    s = wave_sum_d(s);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
        const float r = (float)-((red[0] + red[1]) + (red[2] + red[3]));
        if (a.lam_bf16)
            reinterpret_cast<bf16_t*>(a.dlam)[head] = (bf16_t)r;
        else
            reinterpret_cast<float*>(a.dlam)[head] = r;
    }
}

// dq: a wave owns 32 rows (everything about them is one value per lane) and streams key tiles.  A: S and dP of tile t + 1, dS of
// tile t; B: dq += dS k of tile t.  One barrier per tile, between A and B.  k: two tiles in use, one being put, and one that a
// slower wave may still be reading: four buffers; v is read in A only: two.
// Measured (12 D operations): fp32, 2 x 18000 rows and keys, D = 64: 4.27 ms, 117 TFLOP/s; bf16, the 2 x 4 frames below: 144 us,
// 395 TFLOP/s and the second term of dS.
template <typename T, int D>
__global__ __launch_bounds__(256, D >= 32 ? 1 : 2) void da_dq_kernel(const DaArgs a) {
    typedef Mx<T> M;
    typedef typename M::Frag Frag;
    typedef Stager<T, D, 256> St;
    constexpr int W = 2 * D, LD = St::LD, KC = D / 16, DB = (D + 31) / 32, C2 = D < 32 ? 0 : D;
    __shared__ __attribute__((aligned(16))) T Ks[4][DA_TILE * LD];
    __shared__ __attribute__((aligned(16))) T Vs[2][DA_TILE * LD];
    __shared__ __attribute__((aligned(16))) float Kb[4][DA_TILE];

    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, l31 = lane & 31, lh = lane >> 5;
    const RowOf ro(a, 4, wave, l31);
    const int nparts = da_row_parts(a, ro.last(a, 4));
    if (ro.part >= nparts) return;
    const size_t n = (size_t)a.b * a.hk * a.rows, e0 = ((size_t)ro.bi * a.hk + ro.kh) * a.rows + ro.row;
    const size_t o = (((size_t)ro.bi * a.nq + ro.qi) * a.h + ro.head) * W;
    const T* qrow = reinterpret_cast<const T*>(a.q) + ro.bi * a.q_sb + ro.qi * a.q_sn + ro.head * a.q_sh;
    const T* grow = reinterpret_cast<const T*>(a.go) + o;
    Frag q1[KC], q2[KC], go[2 * KC];
#pragma unroll
    for (int i = 0; i < KC; ++i) {
        q1[i] = M::row(qrow + 16 * i, lh);
        q2[i] = M::row(qrow + a.q_sm + 16 * i, lh);
        go[2 * i] = M::row(grow + 32 * i, lh);
        go[2 * i + 1] = M::row(grow + 32 * i + 16, lh);
    }
    const float e1 = a.stat[e0], e2 = a.stat[n + e0], d1 = a.stat[2 * n + e0], d2 = a.stat[3 * n + e0];
    const int lim = da_limit(a, ro.row);
    KeyStream<T, D, 256> ks;
    ks.init(a, tid, ro.bi, ro.kh, ro.part, ro.last(a, 4));
    const int ntiles = ks.tiles(), nplain = ks.plain(a, min(ro.block0, a.rows - 1));

    f32x16 g1[DB], g2[DB], s1, s2, dp = zero16(), n1, n2, np;
#pragma unroll
    for (int j = 0; j < DB; ++j) g1[j] = g2[j] = zero16();
    Frag ga, gb, gc, gd;  // the first operands of the next A
    f32x16 bias;

    auto ready = [&](int kbuf, int vbuf) {
        bias = da_bias(Kb[kbuf], lh);
        ga = M::row(Ks[kbuf] + l31 * LD, lh);
        gb = M::row(Ks[kbuf] + l31 * LD + D, lh);
        gc = M::row(Vs[vbuf] + l31 * LD, lh);
        gd = M::row(Vs[vbuf] + l31 * LD + 16, lh);
    };
    auto body = [&](auto next, auto edge, int t, f32x16& s1, f32x16& s2, f32x16& dp, f32x16& n1, f32x16& n2, f32x16& np) {
        constexpr bool NEXT = decltype(next)::value;
        const int key0 = ks.begin + t * DA_TILE, b0 = t & 3, b2 = (t + 2) & 3;
        const T *Kn = Ks[(t + 1) & 3] + l31 * LD, *Vn = Vs[(t + 1) & 1] + l31 * LD;
        constexpr int SL = KC * M::STEPS;
#pragma unroll
        for (int i = 0; i < KC; ++i) {
            const Frag fa = ga, fb = gb, fc = gc, fd = gd;
            if (NEXT && i + 1 < KC) {
                ga = M::row(Kn + 16 * (i + 1), lh);
                gb = M::row(Kn + D + 16 * (i + 1), lh);
                gc = M::row(Vn + 32 * (i + 1), lh);
                gd = M::row(Vn + 32 * (i + 1) + 16, lh);
            }
#pragma unroll
            for (int e = 0; e < M::STEPS; ++e) {
                if (NEXT && i + e == 0) {
                    n1 = M::first(fa, q1[0], bias);
                    np = M::first(fc, go[0], zero16());
                    n2 = M::first(fb, q2[0], bias);
                    M::step(np, fd, go[1], 0);
                } else if (NEXT) {
                    M::step(n1, fa, q1[i], e);
                    M::step(np, fc, go[2 * i], e);
                    M::step(n2, fb, q2[i], e);
                    M::step(np, fd, go[2 * i + 1], e);
                }
                const int slot = i * M::STEPS + e;
#pragma unroll
                for (int it = slot * 32 / SL; it < (slot + 1) * 32 / SL; ++it) {
                    const int r = it >> 1;
                    f32x16& s = it & 1 ? s2 : s1;
                    if (decltype(edge)::value) s[r] = key0 + acc_index(r, lh) >= lim ? -DA_INF : s[r];
                    s[r] = __builtin_amdgcn_exp2f(fmaf(s[r], a.c, it & 1 ? -e2 : -e1)) * (dp[r] - (it & 1 ? d2 : d1));
                }
                if (NEXT) {
#pragma unroll
                    for (int f = slot * St::F / SL; f < (slot + 1) * St::F / SL; ++f) {
                        ks.put_k(tid, f, Ks[b2], Kb[b2]);
                        ks.put_v(tid, f, Vs[t & 1], ks.live2);
                        ks.get_k(tid, f);
                        ks.get_v(f);
                    }
                }
                da_pin();
            }
        }
        Frag k1 = M::col(Ks[b0], LD, 0, 0, lane), k2 = M::col(Ks[b0], LD, 0, C2, lane);
        __syncthreads();
        da_pin();
#pragma unroll
        for (int t2 = 0; t2 < 2; ++t2) {
            const typename M::RegFrag p1 = M::reg(s1, t2), p2 = M::reg(s2, t2);
#pragma unroll
            for (int j = 0; j < DB; ++j) {
                const Frag c1 = k1, c2 = k2;
                if (t2 * DB + j + 1 < 2 * DB) {
                    k1 = M::col(Ks[b0], LD, 16 * ((t2 * DB + j + 1) / DB), 32 * ((j + 1) % DB), lane);
                    k2 = M::col(Ks[b0], LD, 16 * ((t2 * DB + j + 1) / DB), C2 + 32 * ((j + 1) % DB), lane);
                }
                // D = 16: each product holds 16 columns of the other map's keys too; they are not stored
#pragma unroll
                for (int e = 0; e < M::RSTEPS; ++e) {
                    M::rstep(g1[j], c1, p1, e);
                    M::rstep(g2[j], c2, p2, e);
                }
                da_pin();
            }
        }
        if (NEXT) ready(b2, t & 1);
    };

    if (ntiles > 0) {
#pragma unroll
        for (int f = 0; f < St::F; ++f) {
            ks.get_k(tid, f);
            ks.get_v(f);
        }
#pragma unroll
        for (int f = 0; f < St::F; ++f) {
            ks.put_k(tid, f, Ks[0], Kb[0]);
            ks.put_v(tid, f, Vs[0], ks.live2);
        }
#pragma unroll
        for (int f = 0; f < St::F; ++f) {
            ks.get_k(tid, f);
            ks.get_v(f);
        }
        __syncthreads();
        s1 = s2 = da_bias(Kb[0], lh);
        const T *K0 = Ks[0] + l31 * LD, *V0 = Vs[0] + l31 * LD;
#pragma unroll
        for (int i = 0; i < KC; ++i) {
            const Frag fa = M::row(K0 + 16 * i, lh), fb = M::row(K0 + D + 16 * i, lh);
            const Frag fc = M::row(V0 + 32 * i, lh), fd = M::row(V0 + 32 * i + 16, lh);
#pragma unroll
            for (int e = 0; e < M::STEPS; ++e) {
                M::step(s1, fa, q1[i], e);
                M::step(dp, fc, go[2 * i], e);
                M::step(s2, fb, q2[i], e);
                M::step(dp, fd, go[2 * i + 1], e);
            }
        }
#pragma unroll
        for (int f = 0; f < St::F; ++f) {
            ks.put_k(tid, f, Ks[1], Kb[1]);
            ks.put_v(tid, f, Vs[1], ks.live2);
            ks.get_k(tid, f);
            ks.get_v(f);
        }
        __syncthreads();
        ready(1, 1);
        int t = 0;
        if (M::ONE_LOOP) {
            for (; t < ntiles; ++t) {
                body(DA_BOOL(true), DA_BOOL(true), t, s1, s2, dp, n1, n2, np);
                s1 = n1;
                s2 = n2;
                dp = np;
            }
        } else {
            for (; t + 1 < min(nplain, ntiles - 1); t += 2) {
                body(DA_BOOL(true), DA_BOOL(false), t, s1, s2, dp, n1, n2, np);
                body(DA_BOOL(true), DA_BOOL(false), t + 1, n1, n2, np, s1, s2, dp);
            }
            for (; t + 1 < ntiles; ++t) {
                body(DA_BOOL(true), DA_BOOL(true), t, s1, s2, dp, n1, n2, np);
                s1 = n1;
                s2 = n2;
                dp = np;
            }
            body(DA_BOOL(false), DA_BOOL(true), t, s1, s2, dp, n1, n2, np);
        }
    }
    if (!ro.live) return;
    const float f2 = -da_lambda(a, ro.head) * a.scale;
    const bool alone = a.alone[ro.bi] != 0;  // the softmax of one key is constant: exactly no gradient
#pragma unroll
    for (int j = 0; j < DB; ++j)
#pragma unroll
        for (int g4 = 0; g4 < 4; ++g4) {
            const int ch = 32 * j + 8 * g4 + 4 * lh;
            f32x4 x = quad(g1[j], g4) * a.scale, y = quad(g2[j], g4) * f2;
            if (alone) x = y = f32x4{0.f, 0.f, 0.f, 0.f};
            // D = 16: map 1 sits in channels 0..15 of its product, map 2 in channels 16..31 of its own
            const bool ok1 = D >= 32 || ch < D, ok2 = D >= 32 || ch >= D;
            if (nparts > 1) {
                float* p = a.part + (size_t)ro.part * a.b * a.nq * a.h * W + o;
                if (ok1) *reinterpret_cast<f32x4*>(p + ch) = x;
                if (ok2) *reinterpret_cast<f32x4*>(p + C2 + ch) = y;
            } else {
                T* p = reinterpret_cast<T*>(a.dq) + o;
                if (ok1) M::store4(p + ch, x);
                if (ok2) M::store4(p + C2 + ch, y);
            }
        }
}

// dk, dv: a wave owns 32 keys and streams row tiles; the rows' constants come from LDS, four at a time.  Same pipeline as dq, with
// q and dO read along rows in A (tile t + 1) and along columns in B (tile t): four buffers each.
// Measured (16 D operations): fp32, 2 x 18000 rows and keys, D = 64: 5.46 ms, 121 TFLOP/s; bf16, the 2 x 4 frames below: 206 us,
// 368 TFLOP/s and the second terms of P and dS.
template <typename T, int D>
__global__ __launch_bounds__(256, 1) void da_dkv_kernel(const DaArgs a) {
    typedef Mx<T> M;
    typedef typename M::Frag Frag;
    typedef Stager<T, D, 256> St;
    constexpr int W = 2 * D, LD = St::LD, KC = D / 16, DB = (D + 31) / 32, CB = W / 32, C2 = D < 32 ? 0 : D;
    __shared__ __attribute__((aligned(16))) T Qs[4][DA_TILE * LD];
    __shared__ __attribute__((aligned(16))) T Gs[4][DA_TILE * LD];
    __shared__ __attribute__((aligned(16))) float Rs[4][6][DA_TILE];  // lse 1, lse 2, D_1, D_2, lambda, key limit (int)

    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, l31 = lane & 31, lh = lane >> 5;
    int tile, part, bh;
    da_place(a, true, tile, part, bh);
    const int bi = bh / a.hk, kh = bh % a.hk;
    const int block0 = tile * 128;
    const int part0 = da_key_parts(a, block0);
    if (part < part0) return;
    const int key = block0 + wave * 32 + l31;
    const bool live = key < a.nk && (!a.mask || a.mask[(size_t)bi * a.nk + min(key, a.nk - 1)]);
    const size_t n = (size_t)a.b * a.hk * a.rows;

    Frag k1[KC], k2[KC], v[2 * KC];
    {
        const int kc = min(key, a.nk - 1);
        const T* kp = reinterpret_cast<const T*>(a.k) + bi * a.k_sb + kh * a.k_sh + kc * a.k_sn;
        const T* vp = reinterpret_cast<const T*>(a.v) + bi * a.v_sb + kh * a.v_sh + kc * a.v_sn;
#pragma unroll
        for (int i = 0; i < KC; ++i) {
            k1[i] = live ? M::row(kp + 16 * i, lh) : M::zero();
            k2[i] = live ? M::row(kp + a.k_sm + 16 * i, lh) : M::zero();
            v[2 * i] = live ? M::row(vp + 32 * i, lh) : M::zero();
            v[2 * i + 1] = live ? M::row(vp + 32 * i + 16, lh) : M::zero();
        }
    }
    int row_begin = part * a.span;
    const int row_end = min(a.rows, row_begin + a.span);
    int nedge = 0;   // leading tiles with rows that do not see all of the workgroup's keys (rows see more and more of them)
    if (a.frame) {
        const int last = min(block0 + 128, a.nk) - 1;
        const long long q1 = (long long)(last / a.frame) * a.frame - a.nk + a.nq;
        const long long r0 = da_first_row(a, block0);  // the first row that sees the first key
        if (r0 > row_begin) row_begin = r0 < row_end ? (int)r0 : row_end;
        const long long r1 = q1 * a.g - row_begin;  // the first row that sees the last key
        nedge = r1 > 0 ? (int)min((r1 + DA_TILE - 1) / DA_TILE, (long long)INT_MAX) : 0;
    }
    const int ntiles = row_end > row_begin ? (row_end - row_begin + DA_TILE - 1) / DA_TILE : 0;
    const char* qb = reinterpret_cast<const char*>(reinterpret_cast<const T*>(a.q) + bi * a.q_sb + kh * a.g * a.q_sh);
    const char* gb = reinterpret_cast<const char*>(reinterpret_cast<const T*>(a.go) + ((size_t)bi * a.nq * a.h + kh * a.g) * W);
    constexpr int E = (int)sizeof(T);
    const unsigned q_sn = (unsigned)a.q_sn * E, q_sh = (unsigned)a.q_sh * E, g_sn = a.h * W * E, g_sh = W * E;
    const unsigned gcol = St::col(tid) * E, qcol = (St::col(tid) >= D ? (unsigned)a.q_sm + St::col(tid) - D : St::col(tid)) * E;

    St sq, sg;
    float rs = 0.f;
    int stile = 0, srows = 0;  // first row of the tile in flight; how many rows the tile being put has
    auto get = [&](int f, int t) {  // tiles past the end read the last row again
        const int r0 = min(row_begin + t * DA_TILE, a.rows - 1), qi0 = da_div(a, r0);
        const int row = min(r0 + St::row(tid, f), a.rows - 1), qi = da_div(a, row), g = row - qi * a.g;
        sq.get(f, qb + qi0 * a.q_sn * E, (qi - qi0) * q_sn + g * q_sh + qcol);
        sg.get(f, gb + (size_t)qi0 * a.h * W * E, (qi - qi0) * g_sn + g * g_sh + gcol);
        if (f == 0) {
            stile = row_begin + t * DA_TILE;
            rs = a.stat[min(tid / DA_TILE, 5) * n + (size_t)bh * a.rows + min(stile + tid % DA_TILE, a.rows - 1)];
        }
    };
    auto put = [&](int f, int buf) {
        if (f == 0) {
            srows = row_end - stile;  // rows past the end: weight 0
            Rs[buf][min(tid / DA_TILE, 5)][tid % DA_TILE] = (tid % DA_TILE >= srows) & (tid < 2 * DA_TILE) ? DA_INF : rs;
        }
        sq.put(tid, f, Qs[buf], St::row(tid, f) < srows);
        sg.put(tid, f, Gs[buf], St::row(tid, f) < srows);
    };
    f32x16 gk1[DB], gk2[DB], gv[CB], s1 = zero16(), s2 = zero16(), dp = zero16(), n1, n2, np;
#pragma unroll
    for (int j = 0; j < DB; ++j) gk1[j] = gk2[j] = zero16();
#pragma unroll
    for (int j = 0; j < CB; ++j) gv[j] = zero16();
    Frag ga, gb_, gc, gd;  // the first operands of the next A

    auto ready = [&](int buf) {
        ga = M::row(Qs[buf] + l31 * LD, lh);
        gb_ = M::row(Qs[buf] + l31 * LD + D, lh);
        gc = M::row(Gs[buf] + l31 * LD, lh);
        gd = M::row(Gs[buf] + l31 * LD + 16, lh);
    };
    auto body = [&](auto next, auto edge, int t, f32x16& s1, f32x16& s2, f32x16& dp, f32x16& n1, f32x16& n2, f32x16& np) {
        constexpr bool NEXT = decltype(next)::value;
        const int b0 = t & 3, b1 = (t + 1) & 3, b2 = (t + 2) & 3;
        const T *Qn = Qs[b1] + l31 * LD, *Gn = Gs[b1] + l31 * LD;
        f32x16 mix;
        f32x4 e1, e2, d1, d2, lam;
        constexpr int SL = KC * M::STEPS;
#pragma unroll
        for (int i = 0; i < KC; ++i) {
            const Frag fa = ga, fb = gb_, fc = gc, fd = gd;
            if (NEXT && i + 1 < KC) {
                ga = M::row(Qn + 16 * (i + 1), lh);
                gb_ = M::row(Qn + D + 16 * (i + 1), lh);
                gc = M::row(Gn + 32 * (i + 1), lh);
                gd = M::row(Gn + 32 * (i + 1) + 16, lh);
            }
#pragma unroll
            for (int e = 0; e < M::STEPS; ++e) {
                if (NEXT && i + e == 0) {
                    n1 = M::first(fa, k1[0], zero16());
                    np = M::first(fc, v[0], zero16());
                    n2 = M::first(fb, k2[0], zero16());
                    M::step(np, fd, v[1], 0);
                } else if (NEXT) {
                    M::step(n1, fa, k1[i], e);
                    M::step(np, fc, v[2 * i], e);
                    M::step(n2, fb, k2[i], e);
                    M::step(np, fd, v[2 * i + 1], e);
                }
                const int slot = i * M::STEPS + e;
#pragma unroll
                for (int r = slot * 16 / SL; r < (slot + 1) * 16 / SL; ++r) {
                    const int o = 8 * (r >> 2) + 4 * lh, x = r & 3;
                    if (x == 0) {
                        e1 = *reinterpret_cast<const f32x4*>(&Rs[b0][0][o]);
                        e2 = *reinterpret_cast<const f32x4*>(&Rs[b0][1][o]);
                        d1 = *reinterpret_cast<const f32x4*>(&Rs[b0][2][o]);
                        d2 = *reinterpret_cast<const f32x4*>(&Rs[b0][3][o]);
                        lam = *reinterpret_cast<const f32x4*>(&Rs[b0][4][o]);
                    }
                    float p1 = __builtin_amdgcn_exp2f(fmaf(s1[r], a.c, -e1[x])), p2 = __builtin_amdgcn_exp2f(fmaf(s2[r], a.c, -e2[x]));
                    if (decltype(edge)::value) {
                        const bool hide = key >= __float_as_int(Rs[b0][5][o + x]);
                        p1 = hide ? 0.f : p1;
                        p2 = hide ? 0.f : p2;
                    }
                    p2 *= lam[x];
                    mix[r] = p1 - p2;
                    s1[r] = p1 * (dp[r] - d1[x]);
                    s2[r] = p2 * (d2[x] - dp[r]);
                }
                if (NEXT) {
#pragma unroll
                    for (int f = slot * St::F / SL; f < (slot + 1) * St::F / SL; ++f) {
                        put(f, b2);
                        get(f, t + 3);
                    }
                }
                da_pin();
            }
        }
        Frag nx = M::col(Gs[b0], LD, 0, 0, lane);
        __syncthreads();
        da_pin();
#pragma unroll
        for (int t2 = 0; t2 < 2; ++t2) {
            const typename M::RegFrag pm = M::reg(mix, t2), p1 = M::reg(s1, t2), p2 = M::reg(s2, t2);
#pragma unroll
            for (int j = 0; j < CB + 2 * DB; ++j) {  // dO's CB blocks, then the DB blocks of q_1 and of q_2
                const Frag c = nx;
                const int j1 = (j + 1) % (CB + 2 * DB), k0 = 16 * (t2 + (j + 1) / (CB + 2 * DB));
                if (k0 < 32) {
                    if (j1 < CB)
                        nx = M::col(Gs[b0], LD, k0, 32 * j1, lane);
                    else if (j1 < CB + DB)
                        nx = M::col(Qs[b0], LD, k0, 32 * (j1 - CB), lane);
                    else
                        nx = M::col(Qs[b0], LD, k0, C2 + 32 * (j1 - CB - DB), lane);
                }
#pragma unroll
                for (int e = 0; e < M::RSTEPS; ++e) {
                    if (j < CB)
                        M::rstep(gv[j < CB ? j : 0], c, pm, e);
                    else if (j < CB + DB)
                        M::rstep(gk1[j < CB + DB && j >= CB ? j - CB : 0], c, p1, e);
                    else
                        M::rstep(gk2[j >= CB + DB ? j - CB - DB : 0], c, p2, e);
                }
                da_pin();
            }
        }
        if (NEXT) ready(b2);
    };

    if (ntiles > 0) {
#pragma unroll
        for (int f = 0; f < St::F; ++f) get(f, 0);
#pragma unroll
        for (int f = 0; f < St::F; ++f) put(f, 0);
#pragma unroll
        for (int f = 0; f < St::F; ++f) get(f, 1);
        __syncthreads();
        const T *Q0 = Qs[0] + l31 * LD, *G0 = Gs[0] + l31 * LD;
#pragma unroll
        for (int i = 0; i < KC; ++i) {
            const Frag fa = M::row(Q0 + 16 * i, lh), fb = M::row(Q0 + D + 16 * i, lh);
            const Frag fc = M::row(G0 + 32 * i, lh), fd = M::row(G0 + 32 * i + 16, lh);
#pragma unroll
            for (int e = 0; e < M::STEPS; ++e) {
                M::step(s1, fa, k1[i], e);
                M::step(dp, fc, v[2 * i], e);
                M::step(s2, fb, k2[i], e);
                M::step(dp, fd, v[2 * i + 1], e);
            }
        }
#pragma unroll
        for (int f = 0; f < St::F; ++f) {
            put(f, 1);
        }
#pragma unroll
        for (int f = 0; f < St::F; ++f) get(f, 2);
        __syncthreads();
        ready(1);
        int t = 0;
        if (M::ONE_LOOP) {
            for (; t < ntiles; ++t) {
                body(DA_BOOL(true), DA_BOOL(true), t, s1, s2, dp, n1, n2, np);
                s1 = n1;
                s2 = n2;
                dp = np;
            }
        } else {
            for (; t < min(nedge, ntiles - 1); ++t) {
                body(DA_BOOL(true), DA_BOOL(true), t, s1, s2, dp, n1, n2, np);
                s1 = n1;
                s2 = n2;
                dp = np;
            }
            for (; t + 2 < ntiles; t += 2) {
                body(DA_BOOL(true), DA_BOOL(false), t, s1, s2, dp, n1, n2, np);
                body(DA_BOOL(true), DA_BOOL(false), t + 1, n1, n2, np, s1, s2, dp);
            }
            if (t + 1 < ntiles) {
                body(DA_BOOL(true), DA_BOOL(true), t, s1, s2, dp, n1, n2, np);
                s1 = n1;
                s2 = n2;
                dp = np;
                ++t;
            }
            body(DA_BOOL(false), DA_BOOL(true), t, s1, s2, dp, n1, n2, np);
        }
    }
    if (key >= a.nk) return;
    const size_t o = (((size_t)bi * a.nk + key) * a.hk + kh) * W;
    const size_t all = (size_t)a.b * a.nk * a.hk * W;
    const bool alone = a.alone[bi] != 0;  // the softmax of one key is constant: exactly no gradient
    auto out = [&](int which, int ch, f32x4 x) {
        if (!live || (alone && which == 0)) x = f32x4{0.f, 0.f, 0.f, 0.f};  // whatever a hidden key's column holds, it never left this lane
        if (part0 + 1 < a.parts)
            *reinterpret_cast<f32x4*>(a.part + ((size_t)part * 2 + which) * all + o + ch) = x;
        else
            M::store4(reinterpret_cast<T*>(which == 0 ? a.dk : a.dv) + o + ch, x);
    };
#pragma unroll
    for (int g4 = 0; g4 < 4; ++g4) {
        const int c4 = 8 * g4 + 4 * lh;
#pragma unroll
        for (int j = 0; j < CB; ++j) out(1, 32 * j + c4, quad(gv[j], g4));
#pragma unroll
        for (int j = 0; j < DB; ++j) {
            const int ch = 32 * j + c4;
            if (D >= 32 || ch < D) out(0, ch, quad(gk1[j], g4) * a.scale);
            if (D >= 32 || ch >= D) out(0, C2 + ch, quad(gk2[j], g4) * a.scale);
        }
    }
}

// out = sum over the parts that were written, part[p * stride + i], rounded once.  KEYS: dk or dv [b][nk][hk][w], else dq
// [b][nq][h][w].
template <typename T, bool KEYS>
__global__ __launch_bounds__(256) void da_sum_kernel(const DaArgs a, const float* __restrict__ part, T* __restrict__ out,
                                                     long long n4, long long stride, int w4) {
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < n4; i += (long long)gridDim.x * 256) {
        int p0 = 0, p1 = a.parts;
        if (a.frame) {
            const long long x = i / w4;
            if (KEYS) {
                p0 = da_key_parts(a, (int)(x / a.hk % a.nk) / 128 * 128);
            } else {
                const int row = (int)(x / a.h % a.nq) * a.g + (int)(x % a.h) % a.g;
                p1 = da_row_parts(a, min(row / 128 * 128 + 128, a.rows) - 1);
            }
            if (p0 + 1 >= p1) continue;
        }
        f32x4 s = *reinterpret_cast<const f32x4*>(part + p0 * stride + 4 * i);
        for (int p = p0 + 1; p < p1; ++p) s += *reinterpret_cast<const f32x4*>(part + p * stride + 4 * i);
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
// well filled; a part costs about `extra` tiles of prologue, epilogue and joining, and each `join` more.
static int da_parts(long long nb, int nt, int slots, int extra, double join, int most) {
    int best = 1;
    double cost = 1e300;
    for (int p = 1, len = nt; p <= most; len = vspw_cdiv(nt, p)) {  // the fewest parts for each length
        const long long rounds = (nb * p + slots - 1) / slots;
        const double c = (double)rounds * (len + (p > 1 ? extra : 0)) + (p > 1 ? join * p : 0.0);
        if (c < cost * 0.98) {
            cost = c;
            best = p;
        }
        if (len == 1) break;
        p = vspw_cdiv(nt, len - 1);
    }
    return best;
}
// The same with frames, where the tiles of rows or keys stream different lengths (up to 8 of them are looked at) and the
// longest begin first: the end of that schedule, and `join` tiles for reading a piece again.  bf16, 2 x 4 frames of 961, 4 heads
// on 2 of 64: forward 192 us in one part, 163 + 13 in two, 152 + 19 in three (taken), 171 + 27 in five; dk and dv 263 us in two
// (as without frames), 202 + 12 in three.
#define DA_LENGTHS 8
static int da_parts_frames(const int* len, int n, double each, int nt, int slots, int extra, double join, int most) {
    int best = 1, span = 0;
    double cost = 1e300;
    const double rounds = 4.0 * slots / (n * each) + 4.0;  // more pieces than that no longer even anything out
    if (rounds < most) most = (int)rounds;
    for (int p = 1; p <= most && p <= nt; ++p) {
        if (vspw_cdiv(nt, p) == span) continue;
        span = vspw_cdiv(nt, p);
        double at[DA_LENGTHS * 2 + 2], count[DA_LENGTHS * 2 + 2];  // slots by the time they become free, in order
        int groups = 1;
        double split = 0.0;  // pieces to be joined
        at[0] = 0.0;
        count[0] = slots;
        for (int s = -1; s < n; ++s) {  // whole pieces first; lengths come in falling order
            double items = 0.0, size = 0.0;
            if (s >= 0 && len[s] > span) split += each * vspw_cdiv(len[s], span);
            if (s < 0) {
                for (int i = 0; i < n; ++i) items += each * (len[i] / span);
                size = span + (p > 1 ? extra : 0);
            } else if (len[s] % span) {
                items = each;
                size = len[s] % span + (len[s] > span ? extra : 0);
            }
            if (s < 0 && items > slots) {  // whole rounds
                at[0] = floor(items / slots) * size;
                items -= floor(items / slots) * slots;
            }
            while (items > 1e-6) {
                const double take = items < count[0] ? items : count[0], t = at[0] + size;
                items -= take;
                count[0] -= take;
                if (count[0] <= 1e-6) {
                    --groups;
                    for (int i = 0; i < groups; ++i) at[i] = at[i + 1], count[i] = count[i + 1];
                }
                int i = groups;
                while (i > 0 && at[i - 1] > t) --i;
                if (i > 0 && t - at[i - 1] < 0.5) {
                    count[i - 1] += take;
                    continue;
                }
                if (groups == (int)(sizeof(at) / sizeof(at[0]))) break;
                for (int k = groups; k > i; --k) at[k] = at[k - 1], count[k] = count[k - 1];
                at[i] = t;
                count[i] = take;
                ++groups;
            }
        }
        const double c = at[groups - 1] + (split > 0.0 ? 1.0 + join * split / slots : 0.0);
        if (c < cost * 0.98) {
            cost = c;
            best = p;
        }
    }
    return best;
}
static int da_span(int n, int parts) { return vspw_cdiv(vspw_cdiv(n, DA_TILE), parts) * DA_TILE; }

#define DA_NEAR (1LL << 24)  // elements: 32 rows of a tile times 4 bytes stay below 2^31

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
    if (rows > INT_MAX - 65536 || d->nk > INT_MAX - 65536 || p.bhk * rows > (1LL << 40) || (long long)d->b * d->nk * d->hk > (1LL << 40))
        return false;
    p.rows = (int)rows;
    const int W = 2 * d->d, nt = vspw_cdiv(d->nk, DA_TILE);
    if ((long long)d->h * W >= DA_NEAR) return false;  // a row of the output and of its gradient
    // up to 32 rows: single-wave workgroups, many parts of the key axis; else four waves share a key tile
    p.wn = p.rows <= 32 ? 1 : 4;
    p.tiles = vspw_cdiv(p.rows, 32 * p.wn);
    const int slots = 256;
    p.qt = vspw_cdiv(p.rows, 128);
    p.kt = vspw_cdiv(d->nk, 128);
    const int rt = vspw_cdiv(p.rows, DA_TILE), fslots = d->d == 64 ? 256 : 512;
    if (p.wn == 1) {
        p.parts = da_parts(p.tiles * p.bhk, nt, 1024, 1, 0.002, DA_ROW_PARTS);
    } else {
        p.parts = da_parts(p.tiles * p.bhk, nt, fslots, 4, 0.02, 32);
    }
    p.qparts = da_parts(p.qt * p.bhk, nt, slots, 4, 0.02, 16);
    p.kparts = da_parts(p.kt * p.bhk, rt, slots, 4, 0.02, 16);
    if (d->frame > 0 && p.wn == 4) {
        const double join = d->dtype == VSPW_F32 ? 0.8 : 2.5;  // reading a piece again, in tiles: bytes and fast products
        int len[DA_LENGTHS];
        bool even = true;
        const long long shift = (long long)d->nk - d->nq;
        int n = p.qt < DA_LENGTHS ? p.qt : DA_LENGTHS;
        for (int s = 0; s < n; ++s) {
            const long long tile = p.qt - 1 - (long long)(2 * s + 1) * p.qt / (2 * n), last = tile * 128 + 127;
            const long long pos = (last < rows ? last : rows - 1) / p.g + shift;
            const long long lim = pos < 0 ? 0 : (pos / d->frame + 1) * d->frame;
            len[s] = vspw_cdiv(lim < d->nk ? lim : d->nk, DA_TILE);
            even = even && len[s] == nt;
        }
        if (!even) {
            p.parts = da_parts_frames(len, n, (double)p.qt * p.bhk / n, nt, fslots, 4, join, 32);
            p.qparts = fslots == slots ? (p.parts < 16 ? p.parts : 16) : da_parts_frames(len, n, (double)p.qt * p.bhk / n, nt, slots, 4, join, 16);
        }
        even = true;
        n = p.kt < DA_LENGTHS ? p.kt : DA_LENGTHS;
        for (int s = 0; s < n; ++s) {
            const long long key = (long long)(2 * s + 1) * p.kt / (2 * n) * 128, q0 = key / d->frame * d->frame - shift;
            const long long r0 = q0 > 0 ? q0 * p.g / DA_TILE : 0;
            len[s] = r0 < rt ? (int)(rt - r0) : 0;
            even = even && len[s] == rt;
        }
        if (!even) p.kparts = da_parts_frames(len, n, (double)p.kt * p.bhk / n, rt, slots, 4, join, 16);
    }
    p.span = da_span(d->nk, p.parts);
    p.parts = vspw_cdiv(d->nk, p.span);
    p.fwd_bytes = p.parts > 1 ? (size_t)p.parts * p.bhk * p.rows * (2 * W + 4) * sizeof(float) : 0;
    p.qspan = da_span(d->nk, p.qparts);
    p.qparts = vspw_cdiv(d->nk, p.qspan);
    p.kspan = da_span(p.rows, p.kparts);
    p.kparts = vspw_cdiv(p.rows, p.kspan);
    const long long bh = (long long)d->b * d->h;
    long long lc = 2048 / bh;
    const long long most = vspw_cdiv(d->nq, 4 * (256 / (W / 4)));
    if (lc > most) lc = most;
    if (lc < 1) lc = 1;
    p.lchunks = (int)lc;
    if (p.tiles * p.bhk * p.parts > INT_MAX || p.qt * p.bhk * p.qparts > INT_MAX || p.kt * p.bhk * p.kparts > INT_MAX ||
        bh * p.lchunks > INT_MAX || p.bhk * p.rows > INT_MAX || (p.parts > DA_JOIN_PARTS && p.bhk * p.rows * (W / 8) > INT_MAX))
        return false;
    size_t parts = 0;  // dq and dk/dv run one after the other and share the partial sums' memory
    if (p.qparts > 1) parts = (size_t)p.qparts * p.bhk * p.rows * W;
    if (p.kparts > 1 && (size_t)p.kparts * 2 * p.bhk * d->nk * W > parts) parts = (size_t)p.kparts * 2 * p.bhk * d->nk * W;
    p.bwd_bytes = (size_t)bh * p.lchunks * sizeof(double) + ((size_t)6 * p.bhk * p.rows + parts) * sizeof(float);
    p.bwd_bytes += (size_t)d->b * sizeof(int) + 48;  // alone; alignment of the pieces
    return true;
}
static bool da_strides_ok(const vspw_dattn_desc* d, const DaPlan& p, const void* q, const void* k, const void* v) {
    const long long ve = d->dtype == VSPW_F32 ? 4 : 8;
    const long long s[] = {d->q_sb, d->q_sn, d->q_sh, d->q_sm, d->k_sb, d->k_sn, d->k_sh, d->k_sm, d->v_sb, d->v_sn, d->v_sh};
    for (long long x : s)
        if (x % ve) return false;
    const long long near[] = {d->q_sn, d->q_sm, d->k_sn, d->k_sm, d->v_sn, p.g > 1 ? p.g * d->q_sh : 0};  // inside a tile: 32 bits
    for (long long x : near)
        if (x < 0 || x >= DA_NEAR) return false;
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
    unsigned l = 0;  // 2^l >= g: gm = ceil(2^(31 + l) / g) is off by less than 2^l / g, exact for 31-bit x
    while ((1ull << l) < (unsigned)p.g) ++l;
    a.gs = 31 + l;
    a.gm = (unsigned)(((1ull << a.gs) + p.g - 1) / p.g);
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
    const long long rows = p.bhk * p.rows;
    if (p.parts > DA_JOIN_PARTS)
        hipLaunchKernelGGL((da_join_row_kernel<T, D>), dim3((unsigned)(rows * (2 * D / 8))), dim3(256), 0, st, a);
    else
        hipLaunchKernelGGL((da_join_kernel<T, D>), dim3((unsigned)vspw_cdiv(rows, 256 / (D / 2))), dim3(256), 0, st, a);
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
            hipLaunchKernelGGL((da_sum_kernel<T, false>), dim3(vspw_stream_grid(n / 4, 256)), dim3(256), 0, st, a,
                               (const float*)a.part, reinterpret_cast<T*>(a.dq), n / 4, n, D / 2);
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
            hipLaunchKernelGGL((da_sum_kernel<T, true>), dim3(vspw_stream_grid(n / 4, 256)), dim3(256), 0, st, a,
                               (const float*)a.part, reinterpret_cast<T*>(a.dk), n / 4, 2 * n, D / 2);
            rc = vspw_launch_status();
            if (rc == VSPW_OK)
                hipLaunchKernelGGL((da_sum_kernel<T, true>), dim3(vspw_stream_grid(n / 4, 256)), dim3(256), 0, st, a,
                                   (const float*)(a.part + n), reinterpret_cast<T*>(a.dv), n / 4, 2 * n, D / 2);
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
                                  const unsigned char* key_mask, void* out, float* maps, float* lse, void* ws, size_t ws_bytes,
                                  void* stream) {
    DaPlan p;
    if (!q || !k || !v || !lam || !out || !da_plan(d, p) || !da_strides_ok(d, p, q, k, v)) return VSPW_EINVAL;
    if ((((uintptr_t)out | (uintptr_t)maps | (uintptr_t)ws) & 15) || ws_bytes < p.fwd_bytes || (p.fwd_bytes && !ws)) return VSPW_EINVAL;
    DaArgs a;
    da_fill(a, d, p, q, k, v, lam, key_mask);
    a.out = out;
    a.maps = maps;
    a.lse = lse;
    a.tiles = p.tiles;
    a.parts = p.parts;
    a.span = p.span;
    a.part = reinterpret_cast<float*>(ws);
    if (p.parts > 1) a.ml = a.part + (size_t)p.parts * p.bhk * p.rows * 4 * d->d;
    return DA_DISPATCH(da_fwd_launch, a, p, vspw_stream(stream));
}

extern "C" int vspw_diff_attn_bwd(const vspw_dattn_desc* d, const void* q, const void* k, const void* v, const void* lam,
                                  const unsigned char* key_mask, const float* maps, const float* lse, const void* go,
                                  void* dq, void* dk, void* dv, void* dlam, void* ws, size_t ws_bytes,
                                  void* stream) {
    DaPlan p;
    if (!q || !k || !v || !lam || !maps || !lse || !go || !da_plan(d, p) || !da_strides_ok(d, p, q, k, v)) return VSPW_EINVAL;
    if ((dk == nullptr) != (dv == nullptr) || !ws || ws_bytes < p.bwd_bytes) return VSPW_EINVAL;
    if (((uintptr_t)maps | (uintptr_t)go | (uintptr_t)dq | (uintptr_t)dk | (uintptr_t)dv | (uintptr_t)ws) & 15)
        return VSPW_EINVAL;
    DaArgs a;
    da_fill(a, d, p, q, k, v, lam, key_mask);
    a.maps = const_cast<float*>(maps);
    a.lse = const_cast<float*>(lse);
    a.go = go;
    a.dq = dq;
    a.dk = dk;
    a.dv = dv;
    a.dlam = dlam;
    // [lpart doubles][stat][alone][partial sums], every piece on 16 bytes
    a.lpart = reinterpret_cast<double*>(ws);
    size_t off = ((size_t)d->b * d->h * p.lchunks * sizeof(double) + 15) / 16 * 16;
    a.stat = reinterpret_cast<float*>(reinterpret_cast<char*>(ws) + off);
    off += ((size_t)6 * p.bhk * p.rows * sizeof(float) + 15) / 16 * 16;
    a.alone = reinterpret_cast<int*>(reinterpret_cast<char*>(ws) + off);
    off += ((size_t)d->b * sizeof(int) + 15) / 16 * 16;
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
