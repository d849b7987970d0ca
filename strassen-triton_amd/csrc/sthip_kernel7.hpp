// Products with an epilogue, C = r + act(A B + b), on tiles whose edges may lie anywhere.
//
// One workgroup computes a BM x BN tile of C from operand tiles of 128 bytes of k.  Operands in whole 16-byte chunks
// go global -> LDS by direct loads (sthip_prims.hpp), two k-steps in flight; rows and columns beyond the edge of the
// operand are not skipped but clamped to its last row or chunk, so that every load is whole and in bounds, and what they
// contribute is never stored.  A k-range that is no multiple of a k-step ends in one step whose tile is written to LDS
// through registers with zeros beyond the end (zeros on BOTH operands: a clamped infinity times zero would be NaN).
// Operands that are not made of aligned 16-byte chunks take that register form for every step.
//
// Layouts: an operand is contiguous along k (KC; an input row, a weight row) or along its own index (the transposed
// operands of the gradients).  The LDS images, swizzles and fragment reads are those of the 256 x 256 kernel
// (sthip_kernel4.hpp), written for other tile widths.
//
// Bound by the matrix instructions on the largest tiles, by LDS reads and the operands' way on smaller ones, by one load latency a
// k-step in the register form.  MI355X: dx and dW of 8192 x 2048 -> 8192 bf16 400 us = 1375 TFLOP/s, matrix cores 72 % busy; the forward
// with gelu and the pre-activation kept 309 us = 890 TFLOP/s, its epilogue on top; 1999 x 4096 -> 4096 bf16 58.8 us = 1140 TFLOP/s.
#pragma once
#include "sthip_kernel4.hpp"

namespace sthip {

enum { ACT_NONE = 0, ACT_RELU = 1, ACT_GELU = 2, ACT_GELU_TANH = 3, ACT_SILU = 4 };

struct Gemm7Params {
    const void* A; const void* B;      // A[m][k], B[k][n]; KC: k contiguous, ld = distance of m (n); else ld = distance of k
    int64_t a_ld, b_ld;                // elements
    int M, N, K;
    int tiles_m, tiles_n;
    int splits, k_split;               // k range of one workgroup (a multiple of a k-step) and how many there are
    // epilogue: v = A B + bias; pre = v; C = residual + act(v).  With more than one split the sums go to part instead.
    const void* bias; const void* res; void* C; void* pre;
    int64_t c_ld, res_ld, pre_ld;
    float* part;                       // [splits][M][N]
    int act;
    int far;                           // register form: the lanes' 32-bit offsets do not reach over a tile
    int stream;                        // outputs larger than the caches: streaming stores
};

// ------------------------------------------------------------------ elements
template <class T> __device__ __forceinline__ float to_f32(const T* p);
template <> __device__ __forceinline__ float to_f32<float>(const float* p) { return *p; }
template <> __device__ __forceinline__ float to_f32<bf16_t>(const bf16_t* p) { return bf16lo(p->v); }
template <> __device__ __forceinline__ float to_f32<f16_t>(const f16_t* p) { return (float)__builtin_bit_cast(_Float16, p->v); }
__device__ __forceinline__ void from_f32(float* p, float v) { *p = v; }
__device__ __forceinline__ void from_f32(bf16_t* p, float v) { p->v = (uint16_t)pack_bf16(v, 0.f); }
__device__ __forceinline__ void from_f32(f16_t* p, float v) { p->v = (uint16_t)pack_f16(v, 0.f); }

template <class T> __device__ __forceinline__ void unpack2(uint32_t w, float& lo, float& hi) {
    if constexpr (__is_same(T, bf16_t)) { lo = bf16lo(w); hi = bf16hi(w); }
    else { const f16x2 h = as_f16x2(w); lo = (float)h[0]; hi = (float)h[1]; }
}
template <class T> __device__ __forceinline__ uint32_t pack2(float lo, float hi) {
    if constexpr (__is_same(T, bf16_t)) return pack_bf16(lo, hi);
    else return pack_f16(lo, hi);
}
// 16- and 8-byte pieces of rows that start anywhere an element may: global memory takes such accesses whole, those that
// cross a line in two.
typedef uint32_t any_u32x4 __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t any_u32x2 __attribute__((ext_vector_type(2), aligned(2)));
typedef float any_f32x4 __attribute__((ext_vector_type(4), aligned(4)));

// The 16-byte chunk at p as bits, its first n elements where fewer than a chunk exist, zeros behind them.
template <class T> __device__ __forceinline__ u32x4 load_chunk(const T* p, int n) {
    constexpr int N = 16 / (int)sizeof(T);
    if (n >= N) return *reinterpret_cast<const any_u32x4*>(p);
    u32x4 w = {0u, 0u, 0u, 0u};
#pragma unroll
    for (int e = 0; e < N - 1; ++e) if (e < n) {
        if constexpr (sizeof(T) == 4) w[e] = reinterpret_cast<const uint32_t*>(p)[e];
        else w[e >> 1] |= (uint32_t)reinterpret_cast<const uint16_t*>(p)[e] << (16 * (e & 1));
    }
    return w;
}
template <class T> __device__ __forceinline__ void store_chunk(T* p, const u32x4& w, int n) {
    constexpr int N = 16 / (int)sizeof(T);
    if (n >= N) {
        *reinterpret_cast<any_u32x4*>(p) = w;
        return;
    }
#pragma unroll
    for (int e = 0; e < N - 1; ++e) if (e < n) {
        if constexpr (sizeof(T) == 4) reinterpret_cast<uint32_t*>(p)[e] = w[e];
        else reinterpret_cast<uint16_t*>(p)[e] = (uint16_t)(w[e >> 1] >> (16 * (e & 1)));
    }
}

// Four consecutive elements, or the first n of them.
template <class T> __device__ __forceinline__ f32x4 load4(const T* p, int n) {
    f32x4 r = {0.f, 0.f, 0.f, 0.f};
    if (n >= 4) {
        if constexpr (sizeof(T) == 4) r = *reinterpret_cast<const any_f32x4*>(p);
        else {
            const u32x2 w = *reinterpret_cast<const any_u32x2*>(p);
            float a, b, c, d;
            unpack2<T>(w[0], a, b); unpack2<T>(w[1], c, d);
            r = f32x4{a, b, c, d};
        }
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) if (e < n) r[e] = to_f32<T>(p + e);
    }
    return r;
}
template <class T> __device__ __forceinline__ void store4(T* p, const f32x4& v, int n) {
    if (n >= 4) {
        if constexpr (sizeof(T) == 4) *reinterpret_cast<any_f32x4*>(p) = v;
        else { u32x2 w = {pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3])}; *reinterpret_cast<any_u32x2*>(p) = w; }
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) if (e < n) from_f32(p + e, v[e]);
    }
}
// The same in LDS, at 16- (fp32) or 8-byte places.
template <class T> __device__ __forceinline__ f32x4 lds_load4(const char* p) {
    if constexpr (sizeof(T) == 4) return *reinterpret_cast<const f32x4*>(p);
    else {
        const u32x2 w = *reinterpret_cast<const u32x2*>(p);
        float a, b, c, d;
        unpack2<T>(w[0], a, b); unpack2<T>(w[1], c, d);
        return f32x4{a, b, c, d};
    }
}
template <class T> __device__ __forceinline__ void lds_store4(char* p, const f32x4& v) {
    if constexpr (sizeof(T) == 4) *reinterpret_cast<f32x4*>(p) = v;
    else { u32x2 w = {pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3])}; *reinterpret_cast<u32x2*>(p) = w; }
}

// ------------------------------------------------------------------ activations
// exp by the hardware's exp2 (relative error about 1e-6 at the arguments that matter here), reciprocal by v_rcp_f32 (one ulp).
__device__ __forceinline__ float fast_exp(float x) { return __builtin_amdgcn_exp2f(x * 1.4426950408889634f); }
__device__ __forceinline__ float sigmoid(float z) { return __builtin_amdgcn_rcpf(1.f + fast_exp(-z)); }
// P(Z <= z) of the normal distribution: erfc by formula 7.1.26 of Abramowitz and Stegun (absolute error below 1.5e-7), from
// the side on which nothing cancels; e receives exp(-z^2 / 2), which the slope needs as well.
__device__ __forceinline__ float normal_cdf(float z, float& e) {
    const float a = __builtin_fabsf(z) * 0.70710678118654752f;
    const float t = __builtin_amdgcn_rcpf(1.f + 0.3275911f * a);
    e = fast_exp(-a * a);
    const float q = 0.5f * e * t * (0.254829592f + t * (-0.284496736f + t * (1.421413741f + t * (-1.453152027f + t * 1.061405429f))));
    return z < 0.f ? q : 1.f - q;
}
constexpr float kTanhC = 0.79788456080286536f, kTanhA = 0.044715f;   // sqrt(2 / pi); 0.5 (1 + tanh u) = sigmoid(2 u)

template <int ACT> __device__ __forceinline__ float activate(float z) {
    if constexpr (ACT == ACT_RELU) return z < 0.f ? 0.f : z;                       // NaN stays NaN
    else if constexpr (ACT == ACT_GELU) { float e; return z * normal_cdf(z, e); }
    else if constexpr (ACT == ACT_GELU_TANH) return z * sigmoid(2.f * kTanhC * (z + kTanhA * z * z * z));
    else if constexpr (ACT == ACT_SILU) return z * sigmoid(z);
    else return z;
}
// f<ACT>() for the activation that a call asks for: the choice is made once, not at every element.
template <class F> __host__ __device__ __forceinline__ void with_activation(int act, F&& f) {
    switch (act) {
        case ACT_RELU: f.template operator()<ACT_RELU>(); break;
        case ACT_GELU: f.template operator()<ACT_GELU>(); break;
        case ACT_GELU_TANH: f.template operator()<ACT_GELU_TANH>(); break;
        case ACT_SILU: f.template operator()<ACT_SILU>(); break;
        default: f.template operator()<ACT_NONE>();
    }
}
// The derivative.  Beyond |z| = 100 every activation here is its asymptote to the last bit; stopping z there keeps
// infinity times zero out of the products below.
template <int ACT> __device__ __forceinline__ float activation_slope(float z) {
    z = z > 100.f ? 100.f : z < -100.f ? -100.f : z;
    if constexpr (ACT == ACT_RELU) return z > 0.f ? 1.f : z != z ? z : 0.f;
    else if constexpr (ACT == ACT_GELU) { float e; const float p = normal_cdf(z, e); return p + z * e * 0.39894228040143268f; }
    else if constexpr (ACT == ACT_GELU_TANH) {
        const float s = sigmoid(2.f * kTanhC * (z + kTanhA * z * z * z));
        return s + z * s * (1.f - s) * 2.f * kTanhC * (1.f + 3.f * kTanhA * z * z);
    } else if constexpr (ACT == ACT_SILU) { const float s = sigmoid(z); return s * (1.f + z * (1.f - s)); }
    else return 1.f;
}
// The pre-activation that is kept for the gradient, rounded to the operand type.  fp16 alone can overflow here while the
// activation's value does not (silu, gelu of a large negative number): it stops at the largest finite value.
template <class T> __device__ __forceinline__ float keepable(float z) {
    if constexpr (__is_same(T, f16_t)) return z > 65504.f ? 65504.f : z < -65504.f ? -65504.f : z;
    else return z;
}

struct Activate4 {
    f32x4 v;
    template <int ACT> __device__ __forceinline__ void operator()() {
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = activate<ACT>(v[e]);
    }
};

// v (four consecutive n of one m, `n` of them inside) through the epilogue.
template <class T> __device__ __forceinline__ void finish4(const Gemm7Params& P, int64_t m, int n0, f32x4 v, int n) {
    if (P.bias) v += load4<T>(reinterpret_cast<const T*>(P.bias) + n0, n);
    if (P.pre) {
        f32x4 z;
#pragma unroll
        for (int e = 0; e < 4; ++e) z[e] = keepable<T>(v[e]);
        store4<T>(reinterpret_cast<T*>(P.pre) + m * P.pre_ld + n0, z, n);
    }
    Activate4 apply = {v};
    with_activation(P.act, apply);
    v = apply.v;
    if (P.res) v += load4<T>(reinterpret_cast<const T*>(P.res) + m * P.res_ld + n0, n);
    store4<T>(reinterpret_cast<T*>(P.C) + m * P.c_ld + n0, v, n);
}

// ------------------------------------------------------------------ operand tiles
// Image of one operand tile (W rows or columns, one k-step) in LDS: `kRows` rows of `kRowBytes`, 16-byte chunk c of
// row r in slot c ^ swizzle(r).
template <class T, int W, bool KC>
struct Tile7 {
    static constexpr int ES = (int)sizeof(T), EPC = 16 / ES, BK = 128 / ES;
    static constexpr int kRowBytes = KC ? 128 : W * ES;
    static constexpr int kBytes = W * 128;
    static constexpr int kChunks = kRowBytes / 16;

    static __device__ __forceinline__ int swizzle(int r) {
        if constexpr (KC) return (r >> 1) & 7;                                 // 16 rows of one chunk column: all banks once
        else if constexpr (ES == 4 && W == 32) return ((r >> 2) & 1) << 2;    // rows of 128 bytes: two of the four spread, the others share
        else if constexpr (ES == 4) return ((r >> 2) & 3) << 2;                // four k-rows 4 apart, 64 bytes of each
        else if constexpr (W >= 128) return ((r & 3) << 2) ^ (((r >> 3) & 1) << 1);   // eight k-rows, 32 bytes of each
        else return (((r >> 1) & 1) << 2) ^ (((r >> 3) & 1) << 1);            // rows of 128 bytes: r & 1 picks the half of the banks
    }
    // Row and chunk whose place in LDS is byte 16 * lane of the tile's KiB number q.
    static __device__ __forceinline__ void place(int q, int lane, int& row, int& chunk) {
        const int b = q * 64 + lane;
        row = b / kChunks;
        chunk = (b % kChunks) ^ swizzle(row);
    }
    // Fragment of the 16-wide block at `sub`: lane L holds index L % 16, k = 8 (L / 16) .. + 7 of a group of 32
    // (fp32: 4 (L / 16) .. + 3 of 16).
    static __device__ __forceinline__ u32x4 fragment(const char* tile, int sub, int kg) {
        const int lane = threadIdx.x & 63, l16 = lane & 15, g = lane >> 4;
        if constexpr (KC) {
            const int row = sub + l16;
            return *reinterpret_cast<const u32x4*>(tile + row * 128 + (((kg * 4 + g) ^ swizzle(row)) * 16));
        } else if constexpr (ES == 4) {
            const int e = sub + l16, k0 = kg * 16 + g * 4;
            const char* p = tile + k0 * kRowBytes + (((e >> 2) ^ swizzle(k0)) * 16) + (e & 3) * 4;
            u32x4 r;
#pragma unroll
            for (int c = 0; c < 4; ++c) r[c] = *reinterpret_cast<const uint32_t*>(p + c * kRowBytes);
            return r;
        } else {
            // two transposing reads of four k-rows each (see read_frag16_mc); the second starts four rows on, where
            // the swizzle is the same
            const int k = kg * 32 + g * 8 + (l16 >> 2);
            const int chunk = (sub >> 3) + ((l16 & 3) >> 1);
            const char* p = tile + k * kRowBytes + ((chunk ^ swizzle(k)) * 16) + (l16 & 1) * 8;
            const u32x2 a = __builtin_bit_cast(u32x2, lds_read_tr16_b64(p)), b = __builtin_bit_cast(u32x2, lds_read_tr16_b64(p + 4 * kRowBytes));
            u32x4 r = {a[0], a[1], b[0], b[1]};
            return r;
        }
    }
};

// One operand of one workgroup: where its tile comes from.
template <class T, int W, bool KC, int WAVES>
struct Operand7 {
    typedef Tile7<T, W, KC> Tile;
    static constexpr int kLoads = W / 8 / WAVES;   // loads of 1 KiB a wave and k-step
    const T* base;       // tile's first row / column, k = 0 (uniform)
    int64_t ld;
    int extent;          // rows / columns of the operand from the tile's first on
    int last;            // the operand's last k
    uint32_t voff[kLoads];

    __device__ __forceinline__ void point(const void* p, int64_t ld_, int tile, int limit, int K, int wave) {
        ld = ld_;
        extent = limit - tile;
        last = K - 1;
        base = reinterpret_cast<const T*>(p) + (KC ? (int64_t)tile * ld : tile);
        const int lane = threadIdx.x & 63;
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            int row, chunk;
            Tile::place(wave * kLoads + i, lane, row, chunk);
            int64_t e;
            if constexpr (KC) e = (int64_t)min(row, extent - 1) * ld + chunk * Tile::EPC;
            else e = (int64_t)row * ld + min(chunk * Tile::EPC, (extent - 1) / Tile::EPC * Tile::EPC);
            voff[i] = (uint32_t)(e * Tile::ES);
        }
    }
    __device__ __forceinline__ const char* at_k(int k) const {
        return reinterpret_cast<const char*>(base + (KC ? (int64_t)k : (int64_t)k * ld));
    }
    // A step takes whole chunks at the lane offsets without asking where it lies inside the k range.  A chunk that straddles the
    // end of the operand's own index then reads on into the next row, which is memory of the same matrix (if its rows lie a
    // chunk apart) and decides nothing that is stored; the matrix's last row has no next one.
    __device__ __forceinline__ bool whole(int k, int kend, bool far) const {
        return k + Tile::BK <= (KC || W <= extent ? kend : min(kend, last)) && (KC || W <= extent || ld >= Tile::EPC) && !far;
    }
    __device__ __forceinline__ void fetch(u32x4 (&r)[kLoads], int k) const {
        const char* p = at_k(k);
#pragma unroll
        for (int i = 0; i < kLoads; ++i) r[i] = *reinterpret_cast<const any_u32x4*>(p + voff[i]);
    }
    __device__ __forceinline__ void put(const u32x4& r, int i, char* lds, int wave) const {
        *reinterpret_cast<u32x4*>(lds + (wave * kLoads + i) * 1024 + (threadIdx.x & 63) * 16) = r;
    }
    __device__ __forceinline__ void put(const u32x4 (&r)[kLoads], char* lds, int wave) const {
#pragma unroll
        for (int i = 0; i < kLoads; ++i) put(r[i], i, lds, wave);
    }
    // The wave's part of the tile at k .. kend straight into LDS, zeros from kend on (and where the operand has no row).  Whole
    // loads again, cut to what exists afterwards; element by element only where a chunk would leave the matrix.
    __device__ __forceinline__ void put_edge(char* lds, int k, int kend, int wave) const {
        const int lane = opaque_lane4();
        const int64_t end = KC ? (int64_t)(extent - 1) * ld + last + 1 : (int64_t)last * ld + extent;   // of the matrix, from base
        u32x4 r[kLoads];
        int n[kLoads];
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            int row, chunk;
            Tile::place(wave * kLoads + i, lane, row, chunk);
            const int c0 = chunk * Tile::EPC;
            const bool live = KC ? row < extent : k + row < kend;
            n[i] = live ? (KC ? kend - k : extent) - c0 : 0;
            r[i] = u32x4{0u, 0u, 0u, 0u};
            const int64_t at = KC ? (int64_t)row * ld + (k + c0) : (int64_t)(k + row) * ld + c0;
            if (n[i] > 0 && at + Tile::EPC <= end) r[i] = *reinterpret_cast<const any_u32x4*>(base + at);
            else if (n[i] > 0) r[i] = load_chunk(base + at, n[i]);
        }
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            if constexpr (KC) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    if constexpr (sizeof(T) == 4) r[i][e] = e < n[i] ? r[i][e] : 0u;
                    else r[i][e] = 2 * e + 1 < n[i] ? r[i][e] : 2 * e < n[i] ? r[i][e] & 0xffffu : 0u;
                }
            }
            put(r[i], i, lds, wave);
        }
    }
};

// Tile number `id`: contiguous runs of tiles per XCD (workgroup x, x + 8, ... run on XCD x), walked four tile rows at a
// time so that the run's panels stay in that XCD's L2; the splits of a tile follow one another.
__device__ __forceinline__ void map_tile7(const Gemm7Params& P, int id, int& tm, int& tn, int& split) {
    const int total = P.tiles_m * P.tiles_n * P.splits, per = total / 8;
    int t = id < per * 8 ? (id & 7) * per + (id >> 3) : id;
    split = t % P.splits;
    t /= P.splits;
    const int width = 4 * P.tiles_n, grp = t / width, rows = min(4, P.tiles_m - grp * 4), in = t - grp * width;
    // (uniform divisions are done by the vector unit: back to scalars, which everything below is derived from)
    tm = __builtin_amdgcn_readfirstlane(grp * 4 + in % rows);
    tn = __builtin_amdgcn_readfirstlane(in / rows);
    split = __builtin_amdgcn_readfirstlane(split);
}

template <class T, int WM, int WN, int NWM, int NWN, int NS, bool A_KC, bool B_KC>
struct Pipe7 {   // NS: stages of operand tiles in LDS
    static constexpr int TM = WM / 16, TN = WN / 16, BM = WM * NWM, BN = WN * NWN, WAVES = NWM * NWN;
    static_assert(sizeof(T) == 4 || TN >= 2, "a row of blocks is where the 16-bit loop places its loads");
    typedef Operand7<T, BM, A_KC, WAVES> OpA;
    typedef Operand7<T, BN, B_KC, WAVES> OpB;
    static constexpr int ES = (int)sizeof(T), BK = 128 / ES;
    static constexpr int kA = BM * 128, kStage = (BM + BN) * 128, kSmem = NS * kStage;
    static constexpr int LOADS = OpA::kLoads + OpB::kLoads;

    OpA a; OpB b;
    char* smem; uint32_t smem_addr;
    int wave, wm, wn;
    f32x4 acc[TM][TN];
    u32x4 fa[2][TM], fb[2][TN];

    // fp32: the four instructions of a row's blocks, component-major, so that those on one accumulator are TN apart; with
    // fewer than four of them the compiler's own form, which knows how long a result takes.
    __device__ __forceinline__ void mma_row_f32(int buf, int i) {
#pragma unroll
        for (int c = 0; c < 4; ++c)
#pragma unroll
            for (int j = 0; j < TN; ++j) {
                if constexpr (TN >= 4) mfma16_step_f32(acc[i][j], fa[buf][i][c], fb[buf][j][c]);
                else {
                    // through scalars: a bit cast of a vector element expression reads element 0
                    const uint32_t ua = fa[buf][i][c], ub = fb[buf][j][c];
                    acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(__builtin_bit_cast(float, ub), __builtin_bit_cast(float, ua), acc[i][j], 0, 0, 0);
                }
            }
    }
    __device__ __forceinline__ void read_a(int buf, int slot, int kg, int i) { fa[buf][i] = OpA::Tile::fragment(smem + slot * kStage, wm + i * 16, kg); }
    __device__ __forceinline__ void read_b(int buf, int slot, int kg, int j) { fb[buf][j] = OpB::Tile::fragment(smem + slot * kStage + kA, wn + j * 16, kg); }
    __device__ __forceinline__ void read_all(int buf, int slot, int kg) {
#pragma unroll
        for (int j = 0; j < TN; ++j) read_b(buf, slot, kg, j);
#pragma unroll
        for (int i = 0; i < TM; ++i) read_a(buf, slot, kg, i);
    }
    // Load q of the wave (A's first, then B's) of the k-step at ap / bp.
    __device__ __forceinline__ void load(const char* ap, const char* bp, int slot, int q) {
        const uint32_t s = smem_addr + slot * kStage;
        if (q < OpA::kLoads) lds_dma16_k(ap, a.voff[q], s + wave * OpA::kLoads * 1024, q * 1024);
        else lds_dma16_k(bp, b.voff[q - OpA::kLoads], s + wave * OpB::kLoads * 1024, kA + (q - OpA::kLoads) * 1024);
    }
    // The same where `live` holds.  With two stages, the large tiles' form, without a branch between the matrix instructions: under a
    // lane mask that is all ones or none (see Pipe4::run16).
    __device__ __forceinline__ void load_if(bool live, uint32_t mask, const char* ap, const char* bp, int slot, int q) {
        if constexpr (NS == 2) {
            const uint32_t s = smem_addr + slot * kStage;
            if (q < OpA::kLoads) lds_dma16_km(ap, a.voff[q], s + wave * OpA::kLoads * 1024, q * 1024, mask);
            else lds_dma16_km(bp, b.voff[q - OpA::kLoads], s + wave * OpB::kLoads * 1024, kA + (q - OpA::kLoads) * 1024, mask);
        } else if (live) load(ap, bp, slot, q);
    }

    // Waits until the first of `left` k-steps in flight has landed (no more than NS - 1 are).
    __device__ __forceinline__ void wait_first(int left) {
        if (NS > 3 && left >= 3) wait_vmcnt_imm<2 * LOADS>();
        else if (NS > 2 && left >= 2) wait_vmcnt_imm<LOADS>();
        else wait_vmcnt_imm<0>();
    }

    // Whole k-steps k0, k0 + BK, ...: the order of one step is that of Pipe4::run16.
    __device__ __forceinline__ void run(int k0, int steps) {
        static_assert(NS >= 2 && NS <= 4, "wait_first");
        const int64_t a_step = A_KC ? 128 : (int64_t)BK * a.ld * ES, b_step = B_KC ? 128 : (int64_t)BK * b.ld * ES;
        const char* ap = a.at_k(k0);
        const char* bp = b.at_k(k0);
#pragma unroll
        for (int st = 0; st < NS; ++st) {
            if (st < steps) {
#pragma unroll
                for (int q = 0; q < LOADS; ++q) load(ap, bp, st, q);
            }
            ap += a_step; bp += b_step;
        }
        if (steps >= NS) wait_vmcnt_imm<(NS - 1) * LOADS>(); else wait_vmcnt_imm<0>();
        __syncthreads();
        read_all(0, 0, 0);
        int slot = 0;
        for (int left = steps; left > 0; --left) {   // k-steps to multiply, this one among them
            const uint32_t live = (uint32_t)__builtin_amdgcn_readfirstlane(left > NS ? -1 : 0);
            const int after = slot + 1 == NS ? 0 : slot + 1;
#pragma unroll
            for (int kg = 0; kg < 2; ++kg) {
                if (kg == 1) {
                    // every wave holds the fragments of this step, and the next one has landed (those behind it may be on their
                    // way): its stage may be read and this one refilled with the step NS ahead
                    wait_first(left - 1);
                    __syncthreads();
                }
                const int next = kg == 0 ? slot : after;
#pragma unroll
                for (int i = 0; i < TM; ++i) {
                    if constexpr (ES == 4) {
                        read_a(kg ^ 1, next, kg ^ 1, i);
#pragma unroll
                        for (int r = i * TN / TM; r < (i + 1) * TN / TM; ++r) read_b(kg ^ 1, next, kg ^ 1, r);
                        if (kg == 1) {
#pragma unroll
                            for (int q = i * LOADS / TM; q < (i + 1) * LOADS / TM; ++q) load_if(left > NS, live, ap, bp, slot, q);
                        }
                        mma_row_f32(kg, i);
                        __builtin_amdgcn_sched_barrier(0);
                        continue;
                    }
#pragma unroll
                    for (int jj = 0; jj < TN; ++jj) {
                        const int j = (i & 1) ? TN - 1 - jj : jj;
                        mfma16_step<T>(acc[i][j], fa[kg][i], fb[kg][j]);
                        __builtin_amdgcn_sched_barrier(0);
                        if (jj == 0) read_a(kg ^ 1, next, kg ^ 1, i);
                        if (jj == (TN - 1) / 2) {
#pragma unroll
                            for (int r = i * TN / TM; r < (i + 1) * TN / TM; ++r) read_b(kg ^ 1, next, kg ^ 1, r);
                        }
                        if (kg == 1 && jj == TN - 2) {
#pragma unroll
                            for (int q = i * LOADS / TM; q < (i + 1) * LOADS / TM; ++q) load_if(left > NS, live, ap, bp, slot, q);
                        }
                        __builtin_amdgcn_sched_barrier(0);
                    }
                }
            }
            ap += a_step; bp += b_step;
            slot = after;
        }
    }
    __device__ __forceinline__ void multiply_stage() {
#pragma unroll
        for (int kg = 0; kg < 2; ++kg) {
            read_all(kg, 0, kg);
#pragma unroll
            for (int i = 0; i < TM; ++i) {
                if constexpr (ES == 4) mma_row_f32(kg, i);
                else {
#pragma unroll
                    for (int j = 0; j < TN; ++j) mfma16_step<T>(acc[i][j], fa[kg][i], fb[kg][j]);
                }
            }
        }
    }
    // The k-steps from k to kend through registers: the next step's chunks are on their way while this one is multiplied.
    __device__ __forceinline__ void run_regs(int k, int kend, bool far) {
        u32x4 ra[OpA::kLoads], rb[OpB::kLoads];
        bool wa = a.whole(k, kend, far), wb = b.whole(k, kend, far);
        if (wa) a.fetch(ra, k);
        if (wb) b.fetch(rb, k);
        for (; k < kend; k += BK) {
            __syncthreads();   // every wave has read the fragments of the step before
            if (wa) a.put(ra, smem, wave); else a.put_edge(smem, k, kend, wave);
            if (wb) b.put(rb, smem + kA, wave); else b.put_edge(smem + kA, k, kend, wave);
            __syncthreads();
            wa = a.whole(k + BK, kend, far);
            wb = b.whole(k + BK, kend, far);
            if (wa) a.fetch(ra, k + BK);
            if (wb) b.fetch(rb, k + BK);
            multiply_stage();
        }
    }
    // The one step that is left when the k range is no multiple of a step.
    __device__ __forceinline__ void run_tail(int k, int kend) {
        __syncthreads();
        a.put_edge(smem, k, kend, wave);
        b.put_edge(smem + kA, k, kend, wave);
        __syncthreads();
        multiply_stage();
    }
    // The matrix instructions are opaque to the compiler's hazard checks: the last ones retire before anything reads the
    // accumulators (the empty statements keep the reads behind the wait).
    // Row i of the accumulators is read from here on and not before: reads that two ways of storing have in common would
    // otherwise be made ahead of both, into registers that do not exist.
    __device__ __forceinline__ void refresh(int i) {
#pragma unroll
        for (int j = 0; j < TN; ++j) asm volatile("" : "+a"(acc[i][j]));
    }
    __device__ __forceinline__ void settle() {
        asm volatile("s_nop 15\n\ts_nop 15");
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
            for (int j = 0; j < TN; ++j) asm volatile("" : "+a"(acc[i][j]));
    }
};

// The epilogue of a wave's tile.  Lane l of block (i, j) holds m = 16 i + l % 16 and n = 16 j + 4 (l / 16) + 0..3; stored from
// there an instruction would write sixteen pieces of 32 bytes.  The results go through LDS instead, each wave its own part of the
// idle stage buffers, and leave as whole rows of the wave's tile in 16-byte chunks; the residual comes in the same way.  Row r
// of a pass lies at r * RB, its 16-byte chunk c in slot c ^ flip(r), which spreads the sixteen rows that are written
// at once over the banks.
template <class Pipe, class O>
struct Rows7 {
    static constexpr int ES = (int)sizeof(O), EPC = 16 / ES, WM = Pipe::TM * 16, WN = Pipe::TN * 16;
    static constexpr int RB = WN * ES, CPR = RB / 16, PER = 64 / CPR;      // bytes and chunks of a row, rows an instruction
    static constexpr int kRegion = Pipe::kSmem / Pipe::WAVES, PR = kRegion / RB < WM ? kRegion / RB : WM;   // rows a pass
    static __device__ __forceinline__ int flip(int r) { return (r / (256 / RB)) & (CPR - 1); }
    static __device__ __forceinline__ char* quad_at(char* w, int r, int c4) {   // four elements: number c4 of row r
        if constexpr (ES == 4) return w + r * RB + ((c4 ^ flip(r)) * 16);
        else return w + r * RB + (((c4 >> 1) ^ flip(r)) * 16) + (c4 & 1) * 8;
    }
    // Rows of the pass between LDS and a matrix whose element (0, 0) of the pass is at (m0, n0).
    template <int PR> static __device__ __forceinline__ void out(const char* w, O* base, int64_t ld, int m0, int n0, const Gemm7Params& P) {
        const int lane = opaque_lane4(), r0 = lane / CPR, c = lane % CPR, n = n0 + c * EPC;
        O* p = base + (int64_t)(m0 + r0) * ld + n;
        if (m0 + PR <= P.M && n0 + WN <= P.N) {
#pragma unroll 4
            for (int k = 0; k < PR / PER; ++k, p += PER * ld) {
                const u32x4 v = *reinterpret_cast<const u32x4*>(w + (k * PER + r0) * RB + ((c ^ flip(k * PER + r0)) * 16));
                any_u32x4* q = reinterpret_cast<any_u32x4*>(p);
                if (P.stream) __builtin_nontemporal_store((any_u32x4)v, q); else *q = v;
            }
            return;
        }
#pragma unroll 1
        for (int k = 0; k < PR / PER; ++k, p += PER * ld) {
            const int r = k * PER + r0;
            if (m0 + r < P.M) store_chunk(p, *reinterpret_cast<const u32x4*>(w + r * RB + ((c ^ flip(r)) * 16)), P.N - n);
        }
    }
    template <int PR> static __device__ __forceinline__ void in(char* w, const O* base, int64_t ld, int m0, int n0, const Gemm7Params& P) {
        const int lane = opaque_lane4(), r0 = lane / CPR, c = lane % CPR, n = n0 + c * EPC;
        const O* p = base + (int64_t)(m0 + r0) * ld + n;
        if (m0 + PR <= P.M && n0 + WN <= P.N) {
#pragma unroll 4
            for (int k = 0; k < PR / PER; ++k, p += PER * ld)
                *reinterpret_cast<u32x4*>(w + (k * PER + r0) * RB + ((c ^ flip(k * PER + r0)) * 16)) = *reinterpret_cast<const any_u32x4*>(p);
            return;
        }
#pragma unroll 1
        for (int k = 0; k < PR / PER; ++k, p += PER * ld) {
            const int r = k * PER + r0;
            *reinterpret_cast<u32x4*>(w + r * RB + ((c ^ flip(r)) * 16)) = load_chunk(p, m0 + r < P.M ? P.N - n : 0);
        }
    }
    // Passes of FR rows, each value formed once: the residual comes into the second half of the wave's LDS, the pre-activation
    // goes into the first, the result into the second, both leave.  One copy of the code for each activation: a choice at
    // every element, or values that are needed twice, make the compiler spill the accumulators.
    static constexpr int FR = kRegion / 2 / RB < WM ? kRegion / 2 / RB : WM;
    template <int ACT> static __device__ __forceinline__ void finish(Pipe& p, const Gemm7Params& P, int row0, int col0) {
        const int lane = opaque_lane4(), l16 = lane & 15, q = lane >> 4;
        char* kept = p.smem + p.wave * kRegion;
        char* w = kept + FR * RB;
        const int n0 = col0 + p.wn;
        f32x4 bias[Pipe::TN];
#pragma unroll
        for (int j = 0; j < Pipe::TN; ++j) {
            const int n = n0 + 16 * j + 4 * q;
            bias[j] = P.bias ? load4<O>(reinterpret_cast<const O*>(P.bias) + n, P.N - n) : f32x4{0.f, 0.f, 0.f, 0.f};
        }
#pragma unroll
        for (int h = 0; h < WM / FR; ++h) {
            const int m0 = row0 + p.wm + h * FR;
            if (P.res) {
                in<FR>(w, reinterpret_cast<const O*>(P.res), P.res_ld, m0, n0, P);
                wave_exchange_point();
            }
#pragma unroll
            for (int i = 0; i < FR / 16; ++i) {
                p.refresh(h * (FR / 16) + i);
#pragma unroll
                for (int j = 0; j < Pipe::TN; ++j) {
                    char* at = quad_at(w, 16 * i + l16, 4 * j + q);
                    f32x4 v = p.acc[h * (FR / 16) + i][j] + bias[j];
                    if (P.pre) {
                        f32x4 z;
#pragma unroll
                        for (int e = 0; e < 4; ++e) z[e] = keepable<O>(v[e]);
                        lds_store4<O>(at - FR * RB, z);
                    }
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[e] = activate<ACT>(v[e]);
                    if (P.res) v += lds_load4<O>(at);
                    lds_store4<O>(at, v);
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
            wave_exchange_point();
            if (P.pre) out<FR>(kept, reinterpret_cast<O*>(P.pre), P.pre_ld, m0, n0, P);
            out<FR>(w, reinterpret_cast<O*>(P.C), P.c_ld, m0, n0, P);
            wave_exchange_point();
        }
    }
    struct Finish {
        Pipe& p; const Gemm7Params& P; int row0, col0;
        template <int ACT> __device__ __forceinline__ void operator()() { finish<ACT>(p, P, row0, col0); }
    };
    // The sums alone.
    static __device__ __forceinline__ void store(Pipe& p, const Gemm7Params& P, O* C, int64_t ld, int row0, int col0) {
        const int lane = opaque_lane4(), l16 = lane & 15, q = lane >> 4;
        char* w = p.smem + p.wave * kRegion;
#pragma unroll
        for (int h = 0; h < WM / PR; ++h) {
#pragma unroll
            for (int i = 0; i < PR / 16; ++i) {
                p.refresh(h * (PR / 16) + i);
#pragma unroll
                for (int j = 0; j < Pipe::TN; ++j) lds_store4<O>(quad_at(w, 16 * i + l16, 4 * j + q), p.acc[h * (PR / 16) + i][j]);
                __builtin_amdgcn_sched_barrier(0);
            }
            wave_exchange_point();
            out<PR>(w, C, ld, row0 + p.wm + h * PR, col0 + p.wn, P);
            wave_exchange_point();
        }
    }
};

// Tile `id` of one product.
template <class T, int WM, int WN, int NWM, int NWN, int NS, bool A_KC, bool B_KC, bool DMA>
__device__ __forceinline__ void gemm7_tile(const Gemm7Params& P, int id, char* smem) {
    typedef Pipe7<T, WM, WN, NWM, NWN, NS, A_KC, B_KC> Pipe;
    Pipe p;
    int tm, tn, split;
    map_tile7(P, id, tm, tn, split);
    p.smem = smem;
    p.smem_addr = (uint32_t)(uintptr_t)(lptr_t)smem;
    p.wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    p.wm = (p.wave / NWN) * WM;
    p.wn = (p.wave % NWN) * WN;
    const int row0 = tm * Pipe::BM, col0 = tn * Pipe::BN;
    p.a.point(P.A, P.a_ld, row0, P.M, P.K, p.wave);
    p.b.point(P.B, P.b_ld, col0, P.N, P.K, p.wave);
#pragma unroll
    for (int i = 0; i < Pipe::TM; ++i)
#pragma unroll
        for (int j = 0; j < Pipe::TN; ++j) p.acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

    const int k0 = split * P.k_split, kend = min(P.K, k0 + P.k_split);
    int k = k0;
    if constexpr (DMA) {
        const int steps = (kend - k0) / Pipe::BK;
        if (steps > 0) p.run(k0, steps);
        k += steps * Pipe::BK;
        if (k < kend) p.run_tail(k, kend);
    } else if (k < kend) p.run_regs(k, kend, P.far != 0);
    p.settle();

    __syncthreads();   // every wave has read its last fragments: the stage buffers are free
    if (P.splits > 1) Rows7<Pipe, float>::store(p, P, P.part + (int64_t)split * P.M * P.N, P.N, row0, col0);
    else if constexpr (A_KC && B_KC) {
        typename Rows7<Pipe, T>::Finish finish = {p, P, row0, col0};
        with_activation(P.act, finish);
    } else Rows7<Pipe, T>::store(p, P, reinterpret_cast<T*>(P.C), P.c_ld, row0, col0);   // the gradients' products have no epilogue
}

template <class T, int WM, int WN, int NWM, int NWN, int NS, bool A_KC, bool B_KC, bool DMA>
__global__ void __launch_bounds__(NWM * NWN * 64) gemm7_kernel(const Gemm7Params P) {
    extern __shared__ __attribute__((aligned(1024))) char smem[];
    gemm7_tile<T, WM, WN, NWM, NWN, NS, A_KC, B_KC, DMA>(P, __builtin_amdgcn_readfirstlane((int)blockIdx.x), smem);
}

// The two products of a layer's gradient, dx = dz W and dW = dz^T x, as one launch: neither waits for the other, so their
// tiles fill the chip together, and a small layer pays one launch instead of two.
struct Gemm7Pair { Gemm7Params dx, dw; int dx_tiles; };
template <class T, int WM, int WN, int NWM, int NWN, int NS, bool DMA>
__global__ void __launch_bounds__(NWM * NWN * 64) gemm7_pair_kernel(const Gemm7Pair P) {
    extern __shared__ __attribute__((aligned(1024))) char smem[];
    const int id = __builtin_amdgcn_readfirstlane((int)blockIdx.x);
    if (id < P.dx_tiles) gemm7_tile<T, WM, WN, NWM, NWN, NS, true, false, DMA>(P.dx, id, smem);
    else gemm7_tile<T, WM, WN, NWM, NWN, NS, false, false, DMA>(P.dw, id - P.dx_tiles, smem);
}

// ------------------------------------------------------------------ few rows
// C = r + act(x W^T + b) for up to 16 rows: what has to be moved is W, once.  A workgroup takes 16 columns, its eight waves
// share the k range 32 (fp32: 16) at a time, and W goes from memory straight into the matrix instruction's operand, four chunks
// of a lane on their way at once; x's rows come from the caches.  The waves' sums meet in LDS and the first wave does the
// epilogue: one launch.  MI355X, 4096 -> 16384 bf16, 1 row: 26.0 us = 5.2 TB/s of W; 768 -> 2304: 6.0 us
// (64 x 64 tiles with the k range split: 29.8 and 9.7).  Each workgroup reads all of x, so that with 16 rows x costs as
// many bytes from L2 as W does: two or four column blocks a workgroup halve that and lose more to fewer waves.  Where the columns
// make few workgroups and the k range is long, it is split over blockIdx.y and joined in a second launch.
constexpr int kWavesF = 8, kTurnF = kWavesF * 4 * 64;   // bytes of a row of W that a workgroup's waves take in a turn
template <class T>
__global__ void __launch_bounds__(kWavesF * 64) few_rows_kernel(const Gemm7Params P) {
    constexpr int ES = (int)sizeof(T), EPC = 16 / ES, STEP = 4 * EPC, U = kTurnF / 64 / kWavesF;
    __shared__ f32x4 sums[kWavesF][64];
    const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6)), lane = threadIdx.x & 63, l16 = lane & 15, g = lane >> 4;
    const int n0 = blockIdx.x * 16;
    const bool live = l16 < P.M;
    const T* w = reinterpret_cast<const T*>(P.B) + (int64_t)min(n0 + l16, P.N - 1) * P.b_ld + g * EPC;
    const T* x = reinterpret_cast<const T*>(P.A) + (int64_t)(live ? l16 : 0) * P.a_ld + g * EPC;
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    auto multiply = [&](const u32x4& a, const u32x4& b) {
        if constexpr (ES == 4) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const uint32_t ua = a[e], ub = b[e];   // through scalars: a bit cast of a vector element expression reads element 0
                acc = __builtin_amdgcn_mfma_f32_16x16x4f32(__builtin_bit_cast(float, ub), __builtin_bit_cast(float, ua), acc, 0, 0, 0);
            }
        } else if constexpr (__is_same(T, bf16_t)) acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, b), __builtin_bit_cast(bf16x8, a), acc, 0, 0, 0);
        else acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, b), __builtin_bit_cast(f16x8, a), acc, 0, 0, 0);
    };
    // wave v takes the steps U v .. U v + U - 1 of every U kWavesF; a split but the last has whole turns
    const int split = blockIdx.y, end = P.splits > 1 ? min(P.K, (split + 1) * P.k_split) : P.K;
    int k = split * P.k_split + wave * U * STEP;
    for (; k + U * STEP <= end; k += kWavesF * U * STEP) {
        u32x4 wf[U], xf[U];
#pragma unroll
        for (int u = 0; u < U; ++u) wf[u] = *reinterpret_cast<const any_u32x4*>(w + k + u * STEP);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            xf[u] = u32x4{0u, 0u, 0u, 0u};
            if (live) xf[u] = *reinterpret_cast<const any_u32x4*>(x + k + u * STEP);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) multiply(xf[u], wf[u]);
    }
    for (int u = 0; u < U && k < end; ++u, k += STEP) {   // what is left of the k range: at most one turn of one wave
        const int n = end - k - g * EPC;
        const u32x4 wf = load_chunk(w + k, n);
        multiply(load_chunk(x + k, live ? n : 0), wf);
    }
    sums[wave][lane] = acc;
    __syncthreads();
    if (wave > 0) return;
    f32x4 v = sums[0][lane];
#pragma unroll
    for (int s = 1; s < kWavesF; ++s) v += sums[s][lane];
    const int n = n0 + 4 * g;
    if (!live || n >= P.N) return;
    if (P.splits > 1) store4<float>(P.part + ((int64_t)split * P.M + l16) * P.N + n, v, P.N - n);
    else finish4<T>(P, l16, n, v, P.N - n);
}

// The partial sums of the splits joined in their order, then the epilogue: four consecutive n a thread, `t` its number.
template <class T> __device__ __forceinline__ void join7(const Gemm7Params& P, int64_t t) {
    const int per_row = (P.N + 3) / 4;
    if (t >= (int64_t)P.M * per_row) return;
    const int m = (int)(t / per_row), n = (int)(t % per_row) * 4;
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
    for (int s = 0; s < P.splits; ++s) v += load4<float>(P.part + ((int64_t)s * P.M + m) * P.N + n, P.N - n);
    finish4<T>(P, m, n, v, P.N - n);
}
template <class T>
__global__ void __launch_bounds__(256) gemm7_join_kernel(const Gemm7Params P) {
    join7<T>(P, (int64_t)blockIdx.x * 256 + threadIdx.x);
}
template <class T>
__global__ void __launch_bounds__(256) gemm7_join_pair_kernel(const Gemm7Pair P, int64_t dx_blocks) {
    const int64_t b = blockIdx.x;
    if (b < dx_blocks) join7<T>(P.dx, b * 256 + threadIdx.x);
    else join7<T>(P.dw, (b - dx_blocks) * 256 + threadIdx.x);
}

}  // namespace sthip
