// Kernels that go over rows: layer norm, the activation's gradient with the bias gradient, column sums.  All of them are
// bound by memory; values are held in fp32 between one load and one store of each element.
#pragma once
#include "sthip_kernel7.hpp"

namespace sthip {

// One 16-byte chunk (8 or 4 elements) as fp32.
template <class T> struct Chunk {
    static constexpr int N = 16 / (int)sizeof(T);
    float v[N];
    __device__ __forceinline__ void unpack(const u32x4& w) {
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int e = 0; e < 4; ++e) { const uint32_t u = w[e]; v[e] = __builtin_bit_cast(float, u); }
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) unpack2<T>(w[e], v[2 * e], v[2 * e + 1]);
        }
    }
    __device__ __forceinline__ u32x4 pack() const {
        u32x4 w;
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int e = 0; e < 4; ++e) w[e] = __builtin_bit_cast(uint32_t, v[e]);
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) w[e] = pack2<T>(v[2 * e], v[2 * e + 1]);
        }
        return w;
    }
    __device__ __forceinline__ void load(const T* p, int n) { unpack(load_chunk(p, n)); }
    __device__ __forceinline__ void store(T* p, int n) const { store_chunk(p, pack(), n); }
};
// N parameters of type P from p on, n of them there (a chunk of T has N elements, one of P may have half as many).
template <class P, int N> __device__ __forceinline__ void load_params(const P* p, int n, float (&v)[N]) {
    constexpr int C = Chunk<P>::N < N ? Chunk<P>::N : N;
    static_assert(Chunk<P>::N <= N, "parameters are as wide as the input or wider");
#pragma unroll
    for (int h = 0; h < N / C; ++h) {
        Chunk<P> c;
        c.load(p + h * C, n - h * C);
#pragma unroll
        for (int e = 0; e < C; ++e) v[h * C + e] = c.v[e];
    }
}

struct NormParams {
    const void* x; const void* w; const void* b; void* y;   // w, b may be null: one and zero
    const void* dy; void* dx;                               // gradient
    float* mean; float* rstd;                               // forward writes them where given, the gradient reads them
    float* part;                                            // [parts][2][cols]: the workgroups' shares of dw and db
    int64_t x_rs, y_rs, dy_rs, dx_rs;
    int rows, cols, parts;
    float eps;
};

// Sums over the TPR threads that share a row.  `red` has room for two sums of every wave, twice: calls alternate between the
// halves, so that one barrier a call is enough (a half is written again only after the barrier of the call between).  Every
// thread of the workgroup calls.
struct RowSum {
    float* red;
    int waves, half;
    template <int TPR> __device__ __forceinline__ void operator()(float& x, float& y) {
        x = wave_sum(x);
        y = wave_sum(y);
        if constexpr (TPR > 64) {
            constexpr int W = TPR / 64;
            const int wave = threadIdx.x >> 6, first = wave / W * W;
            float* r = red + half * 2 * waves;
            half ^= 1;
            if ((threadIdx.x & 63) == 0) { r[wave] = x; r[waves + wave] = y; }
            __syncthreads();
            x = r[first]; y = r[waves + first];
#pragma unroll
            for (int i = 1; i < W; ++i) { x += r[first + i]; y += r[waves + first + i]; }
        }
    }
    template <int TPR> __device__ __forceinline__ float one(float x) {
        x = wave_sum(x);
        if constexpr (TPR > 64) {
            constexpr int W = TPR / 64;
            const int wave = threadIdx.x >> 6, first = wave / W * W;
            float* r = red + half * 2 * waves;
            half ^= 1;
            if ((threadIdx.x & 63) == 0) r[wave] = x;
            __syncthreads();
            x = r[first];
#pragma unroll
            for (int i = 1; i < W; ++i) x += r[first + i];
        }
        return x;
    }
};

// y = (x - mean) rstd w + b.  A row is held in registers by TPR threads, EPT elements each, so that it is read once and the
// variance is the mean of squared distances from the mean (nothing cancels where the mean is large).  RPB groups of TPR
// threads a workgroup, each walks rows: the next one's chunks are on their way while this one is summed, and w and b, which
// in fp32 are twice a 16-bit row, are read once a workgroup instead of once a row.  Bound by memory: MI355X, 8192 x 4096 bf16 with
// fp32 parameters 27 us = 5.0 TB/s (one row a workgroup, nothing ahead: 37.5); 4999 x 1537 fp32, whose rows start
// anywhere, 13.6 us = 4.5 TB/s; one row of 768 is a launch, 3.3 us.
template <class T, class P, int TPR, int EPT, int RPB>
__global__ void __launch_bounds__(TPR * RPB) norm_forward_kernel(const NormParams p) {
    constexpr int N = Chunk<T>::N, NV = EPT / N, WAVES = TPR * RPB / 64;
    __shared__ float red[4 * WAVES];
    RowSum sum = {red, WAVES, 0};
    const int t = threadIdx.x % TPR, sub = threadIdx.x / TPR;
    float w[NV][N], b[NV][N];
    u32x4 next[NV];
    auto fetch = [&](int row) {
        const T* x = reinterpret_cast<const T*>(p.x) + (int64_t)(row < p.rows ? row : 0) * p.x_rs;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int at = (i * TPR + t) * N;
            next[i] = load_chunk(x + at, row < p.rows ? p.cols - at : 0);
        }
    };
    const int step = (int)gridDim.x * RPB;
    fetch(blockIdx.x * RPB + sub);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int at = (i * TPR + t) * N;
        if (p.w) load_params<P, N>(reinterpret_cast<const P*>(p.w) + at, p.cols - at, w[i]);
        if (p.b) load_params<P, N>(reinterpret_cast<const P*>(p.b) + at, p.cols - at, b[i]);
#pragma unroll
        for (int e = 0; e < N; ++e) { if (!p.w) w[i][e] = 1.f; if (!p.b) b[i][e] = 0.f; }
    }
    // all groups of a workgroup make the same number of turns: the sums hold barriers
    for (int row0 = blockIdx.x * RPB; row0 < p.rows; row0 += step) {
        const int row = row0 + sub;
        Chunk<T> c[NV];
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            c[i].unpack(next[i]);
#pragma unroll
            for (int e = 0; e < N; ++e) s += c[i].v[e];
        }
        fetch(row + step);
        const float mean = sum.one<TPR>(s) / (float)p.cols;
        s = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int n = p.cols - (i * TPR + t) * N;
#pragma unroll
            for (int e = 0; e < N; ++e) { c[i].v[e] -= mean; if (e < n) s += c[i].v[e] * c[i].v[e]; }
        }
        const float rstd = 1.f / __builtin_sqrtf(sum.one<TPR>(s) / (float)p.cols + p.eps);
        if (row >= p.rows) continue;   // the last turn: no barrier follows
        if (p.mean && t == 0) { p.mean[row] = mean; p.rstd[row] = rstd; }
        T* y = reinterpret_cast<T*>(p.y) + (int64_t)row * p.y_rs;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int at = (i * TPR + t) * N;
#pragma unroll
            for (int e = 0; e < N; ++e) c[i].v[e] = c[i].v[e] * rstd * w[i][e] + b[i][e];
            c[i].store(y + at, p.cols - at);
        }
    }
}

// Rows too long for registers: the same three sweeps over the row, the second and third out of the caches.  A workgroup a row: MI355X,
// 4096 x 20000 bf16 111 us against 64 of bytes, 1024 x 65536 fp32 211 against 105, 16 x 131072 bf16 33 (16 workgroups).
template <class T, class P>
__global__ void __launch_bounds__(512) norm_forward_long_kernel(const NormParams p) {
    constexpr int N = Chunk<T>::N, TPR = 512;
    __shared__ float red[4 * (TPR / 64)];
    RowSum sum = {red, TPR / 64, 0};
    const int row = blockIdx.x, t = threadIdx.x;
    const T* x = reinterpret_cast<const T*>(p.x) + (int64_t)row * p.x_rs;
    T* y = reinterpret_cast<T*>(p.y) + (int64_t)row * p.y_rs;
    Chunk<T> c;
    float s = 0.f;
    for (int at = t * N; at < p.cols; at += TPR * N) {
        c.load(x + at, p.cols - at);
#pragma unroll
        for (int e = 0; e < N; ++e) s += c.v[e];
    }
    const float mean = sum.one<TPR>(s) / (float)p.cols;
    s = 0.f;
    for (int at = t * N; at < p.cols; at += TPR * N) {
        c.load(x + at, p.cols - at);
#pragma unroll
        for (int e = 0; e < N; ++e) if (e < p.cols - at) { const float d = c.v[e] - mean; s += d * d; }
    }
    const float rstd = 1.f / __builtin_sqrtf(sum.one<TPR>(s) / (float)p.cols + p.eps);
    if (p.mean && t == 0) { p.mean[row] = mean; p.rstd[row] = rstd; }
    for (int at = t * N; at < p.cols; at += TPR * N) {
        const int n = p.cols - at;
        c.load(x + at, n);
        float w[N], b[N];
        if (p.w) load_params<P, N>(reinterpret_cast<const P*>(p.w) + at, n, w);
        if (p.b) load_params<P, N>(reinterpret_cast<const P*>(p.b) + at, n, b);
#pragma unroll
        for (int e = 0; e < N; ++e) {
            float v = (c.v[e] - mean) * rstd;
            if (p.w) v *= w[e];
            if (p.b) v += b[e];
            c.v[e] = v;
        }
        c.store(y + at, n);
    }
}

// dx = rstd (g - mean(g) - h mean(g h)) with h = (x - mean) rstd, g = dy w; dw = sum dy h, db = sum dy over the rows.
// RPB groups of TPR threads a workgroup, each walks the rows group, group + groups, ...: x and dy are read once, the next row's
// chunks while this row is summed, and a group's share of dw and db stays in registers until its last row.  The groups of a
// workgroup join theirs in LDS, the workgroups' shares are joined by column_sum_kernel: fp32 sums in a fixed order.  Bound by
// memory: MI355X, 8192 x 4096 bf16 47 us = 4.3 TB/s and 4 us of joining; 4999 x 1537 fp32 26.7 us = 3.5 TB/s (a quarter of the threads'
// 2048 places is empty, and of the three turns that 512 workgroups of four rows make the last one is 44 % full).
template <class T, class P, int TPR, int EPT, int RPB>
__global__ void __launch_bounds__(TPR * RPB) norm_backward_kernel(const NormParams p) {
    constexpr int N = Chunk<T>::N, NV = EPT / N, WAVES = TPR * RPB / 64;
    __shared__ float red[4 * WAVES];
    __shared__ float join[RPB > 1 ? TPR * EPT : 1];
    RowSum sum = {red, WAVES, 0};
    const int t = threadIdx.x % TPR, sub = threadIdx.x / TPR;
    float dw[NV][N], db[NV][N], w[NV][N];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int at = (i * TPR + t) * N;
        if (p.w) load_params<P, N>(reinterpret_cast<const P*>(p.w) + at, p.cols - at, w[i]);
#pragma unroll
        for (int e = 0; e < N; ++e) { dw[i][e] = db[i][e] = 0.f; if (!p.w) w[i][e] = 1.f; }
    }
    u32x4 nx[NV], ng[NV];
    float nmean = 0.f, nrstd = 0.f;
    auto fetch = [&](int row) {
        const bool live = row < p.rows;
        const T* x = reinterpret_cast<const T*>(p.x) + (int64_t)(live ? row : 0) * p.x_rs;
        const T* dy = reinterpret_cast<const T*>(p.dy) + (int64_t)(live ? row : 0) * p.dy_rs;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int at = (i * TPR + t) * N, n = live ? p.cols - at : 0;
            nx[i] = load_chunk(x + at, n);
            ng[i] = load_chunk(dy + at, n);
        }
        nmean = live ? p.mean[row] : 0.f;
        nrstd = live ? p.rstd[row] : 0.f;
    };
    const int step = (int)gridDim.x * RPB;
    fetch(blockIdx.x * RPB + sub);
    // all groups of a workgroup make the same number of turns: the sums hold barriers
    for (int row0 = blockIdx.x * RPB; row0 < p.rows; row0 += step) {
        const int row = row0 + sub;
        Chunk<T> h[NV], g[NV];
        const float mean = nmean, rstd = nrstd;
        float s1 = 0.f, s2 = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i) { h[i].unpack(nx[i]); g[i].unpack(ng[i]); }
        fetch(row + step);
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int n = p.cols - (i * TPR + t) * N;
#pragma unroll
            for (int e = 0; e < N; ++e) {
                const float d = g[i].v[e];
                h[i].v[e] = e < n ? (h[i].v[e] - mean) * rstd : 0.f;
                dw[i][e] += d * h[i].v[e];
                db[i][e] += d;
                g[i].v[e] = d * w[i][e];
                s1 += g[i].v[e];
                s2 += g[i].v[e] * h[i].v[e];
            }
        }
        sum.operator()<TPR>(s1, s2);
        const float m1 = s1 / (float)p.cols, m2 = s2 / (float)p.cols;
        if (row < p.rows && p.dx) {
            T* dx = reinterpret_cast<T*>(p.dx) + (int64_t)row * p.dx_rs;
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int at = (i * TPR + t) * N;
#pragma unroll
                for (int e = 0; e < N; ++e) g[i].v[e] = rstd * (g[i].v[e] - m1 - h[i].v[e] * m2);
                g[i].store(dx + at, p.cols - at);
            }
        }
    }
    if (!p.part) return;
    float* out = p.part + (int64_t)blockIdx.x * 2 * p.cols;
    for (int which = 0; which < 2; ++which, out += p.cols) {
        auto& mine = which == 0 ? dw : db;
#pragma unroll
        for (int r = 1; r < RPB; ++r) {
            if (sub == r) {
#pragma unroll
                for (int i = 0; i < NV; ++i)
#pragma unroll
                    for (int e = 0; e < N; ++e) join[(i * N + e) * TPR + t] = mine[i][e];
            }
            __syncthreads();
            if (sub == 0) {
#pragma unroll
                for (int i = 0; i < NV; ++i)
#pragma unroll
                    for (int e = 0; e < N; ++e) mine[i][e] += join[(i * N + e) * TPR + t];
            }
            __syncthreads();
        }
        if (sub == 0) {
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int at = (i * TPR + t) * N;
#pragma unroll
                for (int e = 0; e < N; e += 4) store4<float>(out + at + e, f32x4{mine[i][e], mine[i][e + 1], mine[i][e + 2], mine[i][e + 3]}, p.cols - at - e);
            }
        }
    }
}

// Rows too long for registers: dx alone, a workgroup a row, two sweeps (with dw and db: 4096 x 20000 bf16 241 us against 96 of bytes,
// 1024 x 65536 fp32 364 against 157), ...
template <class T, class P>
__global__ void __launch_bounds__(512) norm_backward_long_kernel(const NormParams p) {
    constexpr int N = Chunk<T>::N, TPR = 512;
    __shared__ float red[4 * (TPR / 64)];
    RowSum sum = {red, TPR / 64, 0};
    const int row = blockIdx.x, t = threadIdx.x;
    const T* x = reinterpret_cast<const T*>(p.x) + (int64_t)row * p.x_rs;
    const T* dy = reinterpret_cast<const T*>(p.dy) + (int64_t)row * p.dy_rs;
    T* dx = reinterpret_cast<T*>(p.dx) + (int64_t)row * p.dx_rs;
    const float mean = p.mean[row], rstd = p.rstd[row];
    float s1 = 0.f, s2 = 0.f, m1 = 0.f, m2 = 0.f;
    for (int pass = 0; pass < 2; ++pass) {
        for (int at = t * N; at < p.cols; at += TPR * N) {
            const int n = p.cols - at;
            Chunk<T> h, g;
            h.load(x + at, n);
            g.load(dy + at, n);
            float w[N];
            if (p.w) load_params<P, N>(reinterpret_cast<const P*>(p.w) + at, n, w);
#pragma unroll
            for (int e = 0; e < N; ++e) {
                if (e < n) {
                    const float hv = (h.v[e] - mean) * rstd, gv = p.w ? g.v[e] * w[e] : g.v[e];
                    if (pass == 0) { s1 += gv; s2 += gv * hv; }
                    else g.v[e] = rstd * (gv - m1 - hv * m2);
                }
            }
            if (pass == 1) g.store(dx + at, n);
        }
        if (pass == 0) { sum.operator()<TPR>(s1, s2); m1 = s1 / (float)p.cols; m2 = s2 / (float)p.cols; }
    }
}
// ... and dw, db by columns: 256 columns a workgroup, the rows part, part + parts, ...
template <class T>
__global__ void __launch_bounds__(256) norm_params_long_kernel(const NormParams p) {
    const int col = blockIdx.x * 256 + threadIdx.x, part = blockIdx.y;
    if (col >= p.cols) return;
    float dw = 0.f, db = 0.f;
    for (int row = part; row < p.rows; row += p.parts) {
        const float d = to_f32<T>(reinterpret_cast<const T*>(p.dy) + (int64_t)row * p.dy_rs + col);
        dw += d * (to_f32<T>(reinterpret_cast<const T*>(p.x) + (int64_t)row * p.x_rs + col) - p.mean[row]) * p.rstd[row];
        db += d;
    }
    p.part[(int64_t)part * 2 * p.cols + col] = dw;
    p.part[(int64_t)part * 2 * p.cols + p.cols + col] = db;
}

// out[c] = sum over the parts, rounded once.  `stride` floats lie between two parts; blockIdx.y picks the array (dw, db).  A
// workgroup takes 32 columns: 8 threads of four columns side by side, 32 of them over the parts, whose sums meet in LDS.
struct ColumnSumParams { const float* part; void* out[2]; int64_t stride, second; int parts, cols; };
template <class P>
__global__ void __launch_bounds__(256) column_sum_kernel(const ColumnSumParams p) {
    __shared__ float s[32][32];
    const int c4 = threadIdx.x & 7, r = threadIdx.x >> 3, col = blockIdx.x * 32 + c4 * 4;
    P* out = reinterpret_cast<P*>(p.out[blockIdx.y]);
    if (!out) return;
    const float* part = p.part + blockIdx.y * p.second + col;
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 8
    for (int i = r; i < p.parts; i += 32) v += load4<float>(part + i * p.stride, p.cols - col);
#pragma unroll
    for (int e = 0; e < 4; ++e) s[r][c4 * 4 + e] = v[e];
    __syncthreads();
    if (threadIdx.x < 32 && blockIdx.x * 32 + (int)threadIdx.x < p.cols) {
        float f = s[0][threadIdx.x];
#pragma unroll
        for (int i = 1; i < 32; ++i) f += s[i][threadIdx.x];
        from_f32(out + blockIdx.x * 32 + threadIdx.x, f);
    }
}

// dz = dy act'(pre), and the column sums of dz (the bias gradient) from the values before they are rounded.  A workgroup
// takes 32 chunks of columns and a strip of rows, eight rows at a time, the next eight on their way meanwhile.
// dz leaves in the operand type, since the matrix cores read it twice: with bf16 that is 1.66e-3 of dx and dW, as much as their own
// rounding; pre, rounded as well, adds 0.55e-3 (together 2.41e-3 against 1.66e-3).  In two terms of 16 bits dz would cost both
// products twice, and pre in fp32 alone, at twice its bytes, would gain 3 % of the error.  Bound by memory:
// MI355X, 8192 x 8192 bf16 gelu 84 us = 4.8 TB/s (without the next rows ahead 93).
struct ActParams {
    const void* dy; const void* pre; void* dz;   // without an activation the sums alone: dz = dy
    void* dbias;                                 // one strip: its sums, rounded
    float* part;                                 // several: [strips][cols]
    int64_t dy_rs;
    int rows, cols, strip;
};
template <class T, int ACT>
__global__ void __launch_bounds__(256) act_backward_kernel(const ActParams p) {
    constexpr int N = Chunk<T>::N;
    __shared__ float s[8][32 * N];
    const int ct = threadIdx.x & 31, rt = threadIdx.x >> 5;
    const int at = (blockIdx.x * 32 + ct) * N, n = p.cols - at;
    const int row_end = min(p.rows, ((int)blockIdx.y + 1) * p.strip);
    float sum[N];
#pragma unroll
    for (int e = 0; e < N; ++e) sum[e] = 0.f;
    if (n > 0) {
        int row = blockIdx.y * p.strip + rt;
        const T* dy = reinterpret_cast<const T*>(p.dy) + (int64_t)row * p.dy_rs + at;
        const T* pre = reinterpret_cast<const T*>(p.pre) + (int64_t)row * p.cols + at;
        T* dz = reinterpret_cast<T*>(p.dz) + (int64_t)row * p.cols + at;
        u32x4 ng = {0u, 0u, 0u, 0u}, nz = {0u, 0u, 0u, 0u};
        auto fetch = [&](int r) {
            if (r >= row_end) return;
            ng = load_chunk(dy, n);
            if constexpr (ACT != ACT_NONE) nz = load_chunk(pre, n);
        };
        fetch(row);
        while (row < row_end) {
            Chunk<T> g, z;
            g.unpack(ng);
            z.unpack(nz);
            dy += 8 * p.dy_rs;
            pre += (int64_t)8 * p.cols;
            fetch(row + 8);
            if constexpr (ACT != ACT_NONE) {
#pragma unroll
                for (int e = 0; e < N; ++e) g.v[e] *= activation_slope<ACT>(z.v[e]);
                g.store(dz, n);
                dz += (int64_t)8 * p.cols;
            }
#pragma unroll
            for (int e = 0; e < N; ++e) sum[e] += g.v[e];
            row += 8;
        }
    }
    if (!p.part && !p.dbias) return;
#pragma unroll
    for (int e = 0; e < N; ++e) s[rt][ct * N + e] = sum[e];
    __syncthreads();
    for (int c = threadIdx.x; c < 32 * N; c += 256) {
        const int col = blockIdx.x * 32 * N + c;
        float v = s[0][c];
#pragma unroll
        for (int i = 1; i < 8; ++i) v += s[i][c];
        if (col < p.cols) {
            if (p.part) p.part[(int64_t)blockIdx.y * p.cols + col] = v;
            else from_f32(reinterpret_cast<T*>(p.dbias) + col, v);
        }
    }
}

}  // namespace sthip
