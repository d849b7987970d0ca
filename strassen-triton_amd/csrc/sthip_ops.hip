// C-ABI front end of the operators around the Linear layers: the product with its epilogue and gradients, layer norm,
// rotary positions.  Argument checks, the choice of tiles and splits, launches.  See include/strassen_hip.h.
#include <hip/hip_runtime.h>
#include <algorithm>

#include "../../include/strassen_hip.h"
#include "sthip_launch7.hpp"
#include "sthip_rotary.hpp"

namespace sthip {
namespace {

inline int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
inline size_t align256(size_t x) { return (x + 255) & ~(size_t)255; }
inline int elem_size(int dt) { return dt == STHIP_F32 ? 4 : 2; }
inline bool aligned_to(const void* p, size_t a) { return (reinterpret_cast<uintptr_t>(p) % a) == 0; }
constexpr int64_t kMaxSize = (int64_t)1 << 30;   // tile and chunk numbers are 32-bit

int launched(hipError_t e, const char* what) {
    return e == hipSuccess ? STHIP_OK : fail(STHIP_ERR_HIP, "%s launch failed: %s", what, hipGetErrorString(e));
}

// ------------------------------------------------------------------ products
struct Plan7 { int tile, splits, k_split; };

// Time of a product in microseconds by the tile it runs on, from sweeps on MI355X (bf16 and fp32, K = 1024 and 4096, 16 to 2048
// tiles): a launch costs `fixed`, a k-step of 128 bytes costs a CU rate[q - 1] while it runs q workgroups of that tile, at most
// `held` at once.  16-bit: what a step waits for is its operands' way (two stages of 128 x 128: 0.62 us with one workgroup a
// CU, four stages 0.48; four stages of 64 x 64: 0.18), with the CU full the LDS (128 x 128 0.86 for two, 256 x 128 0.78,
// 256 x 256 1.44 for twice that area); fp32: the matrix instructions (0.6 us a 64 x 64 tile and
// step).  Operands that come through registers have one stage and pay its latency at every step: `through`.
struct TileCost { int tile, held; double fixed, rate[6], through; };
const TileCost kCost16[] = {{TILE7_256, 1, 11, {1.44}, 0}, {TILE7_128, 2, 7, {0.62, 0.86}, 1.5}, {TILE7_128_DEEP, 1, 8.5, {0.48}, 0},
                             {TILE7_256_128, 1, 9.5, {0.78}, 0}, {TILE7_64, 2, 5, {0.18, 0.36}, 2}};
const TileCost kCost32[] = {{TILE7_256, 1, 12, {7.2}, 0}, {TILE7_128, 2, 8, {2.0, 3.7}, 1.15}, {TILE7_64, 2, 5, {0.56, 1.02}, 1.2}, {TILE7_32, 5, 3.6, {0.18, 0.32, 0.45, 0.585, 0.75}, 1.35}};
constexpr int kCus = 256;
struct Tiles { const TileCost* begin_; const TileCost* end_; const TileCost* begin() const { return begin_; } const TileCost* end() const { return end_; } };
Tiles tiles_for(int dt) { return dt == STHIP_F32 ? Tiles{kCost32, kCost32 + 4} : Tiles{kCost16, kCost16 + 5}; }
bool usable(int tile, int dt, bool dma) { return dma || tile == TILE7_128 || tile == TILE7_64 || tile == TILE7_32; }   // the register form exists on these
// Whether the debug switch asks for another tile that this product could take.
bool passed_over(int tile, int dt, bool dma, int forced) {
    if (forced < 0 || forced == tile) return false;
    for (const TileCost& c : tiles_for(dt)) if (c.tile == forced) return usable(forced, dt, dma);
    return false;
}
// Microseconds of a k-step on a CU with q workgroups of the tile.
double step_time(const TileCost& c, int dt, bool dma, int64_t q, int64_t workgroups) {
    if (c.tile == TILE7_256 && dt != STHIP_F32 && workgroups < kCus) return 1.0 + 0.44 * (double)workgroups / kCus;   // a chip half idle runs faster
    return c.rate[q - 1] * (dma ? 1.0 : c.through);
}

// Tile and splits of the k range by the sizes alone, so that the workspace query and the call agree: the cheapest by the table of
// those whose workgroups one launch holds; tile -1 where there is none.  A split costs the joining launch (3 us) and its sums' way to
// memory and back.
Plan7 plan7(int64_t M, int64_t N, int64_t K, int dt, bool dma) {
    const int bk = 128 / elem_size(dt), forced = debug_tile7();
    const int64_t steps = std::max<int64_t>(1, ceil_div(K, bk));
    Plan7 best = {-1, 1, (int)(steps * bk)};
    double least = 1e300;
    for (const TileCost& c : tiles_for(dt)) {
        if (!usable(c.tile, dt, dma) || passed_over(c.tile, dt, dma, forced)) continue;
        const int64_t tiles = ceil_div(M, tile7_rows(c.tile)) * ceil_div(N, tile7_cols(c.tile));
        if (!launchable(tiles, tile7_threads(c.tile))) continue;   // splits are made of few tiles only
        for (int64_t s = 1; s <= 16; ++s) {
            if (s > 1 && (steps < 4 * s || tiles * (s - 1) >= kCus * c.held)) break;
            const int64_t per = ceil_div(steps, s), splits = ceil_div(steps, per), wgs = tiles * splits;
            const int64_t q = ceil_div(wgs, kCus), rest = q % c.held;
            double t = c.fixed * (double)ceil_div(q, c.held) + (double)per * (double)(q / c.held) * step_time(c, dt, dma, c.held, wgs);
            if (rest) t += (double)per * step_time(c, dt, dma, rest, wgs);
            if (splits > 1) t += 3.0 + (double)splits * M * N * 8 / 4e6;
            if (t < least) { least = t; best = {c.tile, (int)splits, (int)(per * bk)}; }
        }
    }
    return best;
}
// Whether the forward product runs on few_rows_kernel.  Up to 4096 columns are a workgroup a CU; beyond, a second round begins, in
// which each workgroup reads all of x again: with 9 to 16 rows the tiles are faster there.  Microseconds, few rows against the
// best tile at k = 1024 / 4096 / 16384:
//   16 rows, bf16:  N = 4096 4.4, 9.7, 37.9 against 6.4, 11.0, 33.1;  N = 16384 at k = 4096 33.7 against 30.4
//   16 rows, fp32:  N = 4096 6.7, 19.3, 64.6 against 9.1, 18.9, 61.1;  N = 16384 18.9, 67.0, 256 against 13.4, 57.4, 191
//    8 rows, bf16:  N = 4096 4.4, 8.7, 35.8 against 6.3, 10.7, 32.6;  N = 16384 8.3, 28.7, 113.5 against 7.6, 30.5, 113.9
//    1 row,  fp32:  N = 4096 6.0, 18.0, 58.8 against 10.5, 18.1, 60.5;  N = 16384 16.9, 55.5, 206 against 13.2, 58.9, 190
// Its launch takes 32 threads a column, of which there are less than 2^32.
bool few_rows(int64_t M, int64_t N) { return debug_tile7() < 0 && N < (1 << 26) && (M <= 8 || (M <= 16 && N <= 4096)); }
// Its k range is split where that saves four turns of the eight waves, of 0.8 (16 bits, one row) to 1.4 us (fp32) each, against the
// joining launch's 3 us; a workgroup a CU at most.  One range / split: 12 rows, 12224 -> 64 fp32 39.4 / 10.5 us, bf16 20.9 / 8.2; 1
// row, 6144 -> 64 bf16 8.5 / 5.9; 16384 -> 2048 fp32 51.3 / 34.8, bf16 21.4 / 20.8.
Plan7 plan_few(int64_t N, int64_t K, int dt) {
    const int turn = kTurnF / elem_size(dt);
    const int64_t turns = std::max<int64_t>(1, ceil_div(K, turn)), s = std::max<int64_t>(1, std::min({(int64_t)16, turns / 2, kCus / ceil_div(N, 16)}));
    const int64_t per = ceil_div(turns, s);
    return turns - per < 4 ? Plan7{TILE7_FEW_ROWS, 1, 0} : Plan7{TILE7_FEW_ROWS, (int)ceil_div(turns, per), (int)(per * turn)};
}
size_t product_workspace(int64_t M, int64_t N, int64_t K, int dt, bool forward) {
    size_t most = 0;
    if (forward && few_rows(M, N)) {
        const Plan7 p = plan_few(N, K, dt);
        return p.splits > 1 ? align256((size_t)p.splits * M * N * sizeof(float)) : 0;
    }
    for (int dma = 0; dma < 2; ++dma) {
        const Plan7 p = plan7(M, N, K, dt, dma != 0);
        if (p.splits > 1) most = std::max(most, (size_t)p.splits * M * N * sizeof(float));
    }
    return align256(most);
}

// The two products of a gradient as one launch: the same table over the tiles of both; dx takes sx splits, dW sw.  Tile -1 where no
// launch holds both.  With few rows, whose dW has less than a whole k-step, the table is off by up to a third: its choice against the
// best tile, bias gradient included, 8 x 4096 -> 16384 bf16 76.5 / 75.0 us, fp32 201 / 175; 16 x 4096 -> 4096 bf16 32.8 / 32.3, fp32
// 65.5 / 51.7; 13 x 5198 -> 12799 fp32 225 / 166; 13 x 1024 -> 4096 fp32 24.4 / 24.4.
struct PlanPair { int tile; Plan7 dx, dw; };
PlanPair plan_pair(int64_t rows, int64_t in, int64_t out, int dt, bool dma) {
    const int bk = 128 / elem_size(dt), forced = debug_tile7();
    const int64_t steps_x = std::max<int64_t>(1, ceil_div(out, bk)), steps_w = std::max<int64_t>(1, ceil_div(rows, bk));
    PlanPair best = {-1, {-1, 1, 0}, {-1, 1, 0}};
    double least = 1e300;
    for (const TileCost& c : tiles_for(dt)) {
        if (!usable(c.tile, dt, dma) || passed_over(c.tile, dt, dma, forced)) continue;
        const int bm = tile7_rows(c.tile), bn = tile7_cols(c.tile);
        const int64_t tx = ceil_div(rows, bm) * ceil_div(in, bn), tw = ceil_div(out, bm) * ceil_div(in, bn), slots = (int64_t)kCus * c.held;
        for (int64_t sx = 1; sx <= 16; sx *= 2) {
            if (sx > 1 && (steps_x < 4 * sx || tx * (sx / 2) >= slots)) break;
            for (int64_t sw = 1; sw <= 16; sw *= 2) {
                if (sw > 1 && (steps_w < 4 * sw || tw * (sw / 2) >= slots)) break;
                const int64_t px = ceil_div(steps_x, sx), pw = ceil_div(steps_w, sw), nx = ceil_div(steps_x, px), nw = ceil_div(steps_w, pw);
                const int64_t wgs = tx * nx + tw * nw, most = std::max(px, pw);
                if (!launchable(wgs, tile7_threads(c.tile))) continue;
                double t;
                if (wgs <= slots) t = c.fixed + (double)most * step_time(c, dt, dma, std::max<int64_t>(1, ceil_div(wgs, kCus)), wgs);
                else t = c.fixed * (double)ceil_div(wgs, slots) + step_time(c, dt, dma, c.held, wgs) * ((double)(tx * nx * px + tw * nw * pw) / slots + (wgs % slots ? 0.5 * (double)most : 0.0));
                if (nx > 1 || nw > 1) t += 3.0 + 8.0 / 4e6 * ((nx > 1 ? (double)nx * rows * in : 0.0) + (nw > 1 ? (double)nw * out * in : 0.0));
                if (t < least) { least = t; best = {c.tile, {c.tile, (int)nx, (int)(px * bk)}, {c.tile, (int)nw, (int)(pw * bk)}}; }
            }
        }
    }
    return best;
}
size_t part_bytes(const Plan7& p, int64_t M, int64_t N) { return p.splits > 1 ? align256((size_t)p.splits * M * N * sizeof(float)) : 0; }
size_t pair_workspace(int64_t rows, int64_t in, int64_t out, int dt) {
    size_t most = 0;
    for (int dma = 0; dma < 2; ++dma) {
        const PlanPair p = plan_pair(rows, in, out, dt, dma != 0);
        most = std::max(most, part_bytes(p.dx, rows, in) + part_bytes(p.dw, out, in));
    }
    return most;
}

struct Operand { const void* p; int64_t ld; bool kc; };
struct Epilogue { const void* bias; const void* res; int64_t res_ld; void* pre; int act; };

// Outputs that exceed the L2s (eight of 4 MiB) by a multiple go past them: a round of tiles would push the operands' panels out
// that the next round reads again.  8192 x 2048 x 8192 bf16 with gelu and its pre-activation kept: 355 -> 309 us.
int streamed(size_t bytes) { return bytes > ((size_t)128 << 20) ? 1 : 0; }

// Direct loads: aligned chunks, whole along the contiguous direction where that is not k (the k tail has a form of its own),
// and 32-bit lane offsets over the tile's 256 rows.
bool direct_loads(const Operand& o, int64_t extent, int es) {
    const int epc = 16 / es;
    return aligned_to(o.p, 16) && o.ld % epc == 0 && (o.kc || extent % epc == 0) && o.ld * es < ((int64_t)1 << 23);
}
Gemm7Params product_params(const Operand& a, const Operand& b, void* C, int64_t c_ld, int64_t M, int64_t N, int64_t K, int dt, const Epilogue& ep, const Plan7& pl, void* ws) {
    Gemm7Params P = {};
    P.A = a.p; P.B = b.p; P.a_ld = a.ld; P.b_ld = b.ld;
    P.M = (int)M; P.N = (int)N; P.K = (int)K;
    P.tiles_m = (int)ceil_div(M, tile7_rows(pl.tile)); P.tiles_n = (int)ceil_div(N, tile7_cols(pl.tile));
    P.splits = pl.splits; P.k_split = pl.k_split;
    P.bias = ep.bias; P.res = ep.res; P.res_ld = ep.res_ld; P.pre = ep.pre; P.pre_ld = N; P.act = ep.act;
    P.C = C; P.c_ld = c_ld;
    P.far = std::max(a.ld, b.ld) * elem_size(dt) >= ((int64_t)1 << 23);
    P.stream = streamed((size_t)M * N * elem_size(dt) * (ep.pre ? 2 : 1));
    P.part = reinterpret_cast<float*>(ws);
    return P;
}
int refuse_size(int64_t M, int64_t N, int64_t K) { return fail(STHIP_ERR_SHAPE, "product of %lld x %lld x %lld is too large", (long long)M, (long long)N, (long long)K); }

bool product_direct(const Operand& a, const Operand& b, int64_t M, int64_t N, int dt) { return direct_loads(a, M, elem_size(dt)) && direct_loads(b, N, elem_size(dt)); }
Plan7 plan_product(const Operand& a, const Operand& b, int64_t M, int64_t N, int64_t K, int dt) {
    return a.kc && b.kc && few_rows(M, N) ? plan_few(N, K, dt) : plan7(M, N, K, dt, product_direct(a, b, M, N, dt));
}
int product(const Plan7& pl, const Operand& a, const Operand& b, void* C, int64_t c_ld, int64_t M, int64_t N, int64_t K, int dt, const Epilogue& ep, void* ws, hipStream_t stream) {
    const int layout = a.kc ? (b.kc ? LAYOUT_NT : LAYOUT_NN) : LAYOUT_TN;
    const LaunchFn7 fn = layout == LAYOUT_NT ? (dt == STHIP_F32 ? kForward7_0 : dt == STHIP_F16 ? kForward7_1 : kForward7_2)
                                             : (dt == STHIP_F32 ? kGradient7_0 : dt == STHIP_F16 ? kGradient7_1 : kGradient7_2);
    return launched(fn(product_params(a, b, C, c_ld, M, N, K, dt, ep, pl, ws), pl.tile, layout, product_direct(a, b, M, N, dt), stream), "linear_act product");
}

int check_linear(int64_t rows, int64_t in, int64_t out, int dtype, int act) {
    if (rows < 0 || in < 0 || out < 0) return fail(STHIP_ERR_SHAPE, "negative size: rows=%lld in=%lld out=%lld", (long long)rows, (long long)in, (long long)out);
    if (rows >= kMaxSize || in >= kMaxSize || out >= kMaxSize) return fail(STHIP_ERR_SHAPE, "a size of 2^30 or more: rows=%lld in=%lld out=%lld", (long long)rows, (long long)in, (long long)out);
    if (dtype < STHIP_F32 || dtype > STHIP_BF16) return fail(STHIP_ERR_DTYPE, "unknown dtype %d", dtype);
    if (act < STHIP_ACT_NONE || act > STHIP_ACT_SILU) return fail(STHIP_ERR_ARG, "unknown activation %d", act);
    return STHIP_OK;
}
int check_stride(const char* what, int64_t rs, int64_t width, int64_t rows) {
    if (rows > 1 && rs < width) return fail(STHIP_ERR_LAYOUT, "%s: row stride %lld is less than its %lld columns", what, (long long)rs, (long long)width);
    if (rs < 0) return fail(STHIP_ERR_LAYOUT, "%s: negative row stride", what);
    return STHIP_OK;
}
int check_workspace(const void* ws, size_t have, size_t need) {
    if (need && (!ws || have < need)) return fail(STHIP_ERR_WORKSPACE, "workspace too small: %zu < %zu bytes", ws ? have : (size_t)0, need);
    if (need && !aligned_to(ws, 256)) return fail(STHIP_ERR_WORKSPACE, "the workspace must be 256-byte aligned");
    return STHIP_OK;
}

// The activation's gradient and the bias gradient: strips of rows such that a few thousand workgroups run, at least 64 rows each
// (eight turns of a thread; up to 128 rows are one strip, whose sums need no second launch).
struct ActPlan { int col_blocks, strip, strips; };
ActPlan act_plan(int64_t rows, int64_t cols, int dt) {
    ActPlan p;
    p.col_blocks = (int)std::max<int64_t>(1, ceil_div(cols, 32 * (16 / elem_size(dt))));
    const int64_t strips = std::max<int64_t>(1, std::min<int64_t>(rows <= 128 ? 1 : ceil_div(rows, 64), ceil_div(2048, p.col_blocks)));
    p.strip = (int)std::max<int64_t>(8, ceil_div(ceil_div(rows, strips), 8) * 8);
    p.strips = (int)std::max<int64_t>(1, ceil_div(rows, p.strip));
    return p;
}
size_t act_part_bytes(int64_t rows, int64_t cols, int dt) {
    const ActPlan p = act_plan(rows, cols, dt);
    return p.strips > 1 ? align256((size_t)p.strips * cols * sizeof(float)) : 0;
}

struct LaunchAct {
    const ActParams& a; int dt; dim3 grid; hipStream_t s;
    template <int ACT> void operator()() {
        if (dt == STHIP_F32) hipLaunchKernelGGL((act_backward_kernel<float, ACT>), grid, dim3(256), 0, s, a);
        else if (dt == STHIP_F16) hipLaunchKernelGGL((act_backward_kernel<f16_t, ACT>), grid, dim3(256), 0, s, a);
        else hipLaunchKernelGGL((act_backward_kernel<bf16_t, ACT>), grid, dim3(256), 0, s, a);
    }
};
// Eight threads a column, in launches of 2^24 columns (at 2^29 a launch would hold too many threads).
template <class P> int column_sum(ColumnSumParams c, int arrays, hipStream_t s) {
    const int64_t most = 1 << 24;
    for (int64_t left = c.cols; left > 0; left -= most) {
        c.cols = (int)std::min(left, most);
        hipLaunchKernelGGL((column_sum_kernel<P>), dim3((unsigned)ceil_div(c.cols, 32), (unsigned)arrays), dim3(256), 0, s, c);
        c.part += most;
        for (void*& out : c.out) if (out) out = reinterpret_cast<P*>(out) + most;
    }
    return launched(hipGetLastError(), "column_sum");
}
int column_sum(const ColumnSumParams& c, int arrays, int dt, hipStream_t s) {
    return dt == STHIP_F32 ? column_sum<float>(c, arrays, s) : dt == STHIP_F16 ? column_sum<f16_t>(c, arrays, s) : column_sum<bf16_t>(c, arrays, s);
}

// ------------------------------------------------------------------ layer norm
template <class T, class P, int TPR, int EPT, int RPB> void norm_forward(const NormParams& p, hipStream_t s) {
    const int64_t blocks = std::min<int64_t>(ceil_div(p.rows, RPB), kCus * (2048 / (TPR * RPB)));   // 2048 threads a CU
    hipLaunchKernelGGL((norm_forward_kernel<T, P, TPR, EPT, RPB>), dim3((unsigned)blocks), dim3(TPR * RPB), 0, s, p);
}
// Rows of 512 threads each, in launches of 2^16 rows (at 2^23 a launch would hold too many threads; 2 GiB of rows hide a launch).
template <class T, class F> void long_rows(NormParams p, F&& launch) {
    const int64_t most = 1 << 16;
    for (int64_t left = p.rows; left > 0; left -= most) {
        p.rows = (int)std::min(left, most);
        launch(p);
        auto on = [&](auto*& q, int64_t rs) { if (q) q = (T*)q + most * rs; };
        on(p.x, p.x_rs), on(p.y, p.y_rs), on(p.dy, p.dy_rs), on(p.dx, p.dx_rs);
        if (p.mean) p.mean += most, p.rstd += most;
    }
}
template <class T, class P> void norm_forward_any(const NormParams& p, hipStream_t s) {
    if (p.cols <= 512) norm_forward<T, P, 64, 8, 4>(p, s);
    else if (p.cols <= 1024) norm_forward<T, P, 64, 16, 4>(p, s);
    else if (p.cols <= 2048) norm_forward<T, P, 128, 16, 2>(p, s);
    else if (p.cols <= 4096) norm_forward<T, P, 256, 16, 1>(p, s);
    else if (p.cols <= 8192) norm_forward<T, P, 512, 16, 1>(p, s);
    else if (p.cols <= 16384) norm_forward<T, P, 512, 32, 1>(p, s);
    else long_rows<T>(p, [&](const NormParams& r) { hipLaunchKernelGGL((norm_forward_long_kernel<T, P>), dim3((unsigned)r.rows), dim3(512), 0, s, r); });
}
constexpr int64_t kNormHeld = 16384;   // columns of the longest row that is held in registers
// Threads a row and rows a workgroup of the gradient: 16 elements a thread up to 8192 columns (8 for short rows).
struct NormBack { int tpr, rpb; };
NormBack norm_back(int64_t cols) {
    if (cols <= 1024) return {64, 8};
    if (cols <= 2048) return {128, 4};
    if (cols <= 4096) return {256, 2};
    return {512, 1};
}
template <class T, class P, int TPR, int EPT, int RPB> void norm_backward(const NormParams& p, hipStream_t s) {
    hipLaunchKernelGGL((norm_backward_kernel<T, P, TPR, EPT, RPB>), dim3((unsigned)p.parts), dim3(TPR * RPB), 0, s, p);
}
template <class T, class P> void norm_backward_any(const NormParams& p, hipStream_t s) {
    if (p.cols <= 512) norm_backward<T, P, 64, 8, 8>(p, s);
    else if (p.cols <= 1024) norm_backward<T, P, 64, 16, 8>(p, s);
    else if (p.cols <= 2048) norm_backward<T, P, 128, 16, 4>(p, s);
    else if (p.cols <= 4096) norm_backward<T, P, 256, 16, 2>(p, s);
    else if (p.cols <= 8192) norm_backward<T, P, 512, 16, 1>(p, s);
    else if (p.cols <= kNormHeld) norm_backward<T, P, 512, 32, 1>(p, s);
    else {
        if (p.dx) long_rows<T>(p, [&](const NormParams& r) { hipLaunchKernelGGL((norm_backward_long_kernel<T, P>), dim3((unsigned)r.rows), dim3(512), 0, s, r); });
        if (p.part) hipLaunchKernelGGL((norm_params_long_kernel<T>), dim3((unsigned)ceil_div(p.cols, 256), (unsigned)p.parts), dim3(256), 0, s, p);
    }
}
template <class F> void by_types(int dt, int pdt, F&& f) {
    if (dt == STHIP_F32) f((float*)nullptr, (float*)nullptr);
    else if (dt == STHIP_F16) { if (pdt == STHIP_F32) f((f16_t*)nullptr, (float*)nullptr); else f((f16_t*)nullptr, (f16_t*)nullptr); }
    else { if (pdt == STHIP_F32) f((bf16_t*)nullptr, (float*)nullptr); else f((bf16_t*)nullptr, (bf16_t*)nullptr); }
}
// Workgroups that share the rows of the gradient: enough to fill the chip, few enough that their shares of dw and db (two
// floats a column and workgroup) stay small next to x and dy.
int norm_parts(int64_t rows, int64_t cols) {
    if (cols > kNormHeld) return (int)std::max<int64_t>(1, std::min<int64_t>(64, rows));
    return (int)std::max<int64_t>(1, std::min<int64_t>(512, ceil_div(rows, norm_back(cols).rpb)));
}
int check_norm(int64_t rows, int64_t cols, int dtype, int param_dtype) {
    if (rows < 0 || cols < 0) return fail(STHIP_ERR_SHAPE, "negative size: rows=%lld cols=%lld", (long long)rows, (long long)cols);
    if (rows >= kMaxSize || cols >= kMaxSize) return fail(STHIP_ERR_SHAPE, "a size of 2^30 or more: rows=%lld cols=%lld", (long long)rows, (long long)cols);
    if (dtype < STHIP_F32 || dtype > STHIP_BF16) return fail(STHIP_ERR_DTYPE, "unknown dtype %d", dtype);
    if (param_dtype != dtype && param_dtype != STHIP_F32) return fail(STHIP_ERR_DTYPE, "parameters must have the input's type or fp32, got %d", param_dtype);
    return STHIP_OK;
}

template <class T> void launch_rotary(const RotaryParams& p, int v, unsigned blocks, hipStream_t s) {
    if constexpr (sizeof(T) == 2) if (v == 8) { hipLaunchKernelGGL((rotary_kernel<T, 8>), dim3(blocks), dim3(256), 0, s, p); return; }
    if (v == 4) hipLaunchKernelGGL((rotary_kernel<T, 4>), dim3(blocks), dim3(256), 0, s, p);
    else if (v == 2) hipLaunchKernelGGL((rotary_kernel<T, 2>), dim3(blocks), dim3(256), 0, s, p);
    else hipLaunchKernelGGL((rotary_kernel<T, 1>), dim3(blocks), dim3(256), 0, s, p);
}

}  // namespace
}  // namespace sthip

using namespace sthip;

extern "C" {

size_t sthip_linear_act_workspace_bytes(int64_t rows, int64_t in_features, int64_t out_features, int dtype) {
    if (rows <= 0 || in_features < 0 || out_features <= 0 || dtype < STHIP_F32 || dtype > STHIP_BF16) return 0;
    return product_workspace(rows, out_features, in_features, dtype, true);
}

int sthip_linear_act_forward(const void* x, const void* W, const void* bias, const void* residual, void* y, void* pre,
                             int64_t rows, int64_t in_features, int64_t out_features,
                             int64_t x_row_stride, int64_t w_row_stride, int64_t residual_row_stride, int64_t y_row_stride,
                             int dtype, int activation, void* workspace, size_t workspace_bytes, void* stream) {
    clear_error();
    int rc = check_linear(rows, in_features, out_features, dtype, activation);
    if (rc) return rc;
    if (rows == 0 || out_features == 0) return STHIP_OK;
    if (!y || (in_features > 0 && (!x || !W))) return fail(STHIP_ERR_ARG, "null pointer");
    if ((rc = check_stride("x", x_row_stride, in_features, rows)) || (rc = check_stride("W", w_row_stride, in_features, out_features)) ||
        (rc = check_stride("y", y_row_stride, out_features, rows)) || (residual && (rc = check_stride("residual", residual_row_stride, out_features, rows)))) return rc;
    if ((rc = check_workspace(workspace, workspace_bytes, sthip_linear_act_workspace_bytes(rows, in_features, out_features, dtype)))) return rc;
    const Epilogue ep = {bias, residual, residual ? residual_row_stride : 0, pre, activation};
    const Operand a = {x, x_row_stride, true}, b = {W, w_row_stride, true};
    const Plan7 pl = plan_product(a, b, rows, out_features, in_features, dtype);
    if (pl.tile < 0) return refuse_size(rows, out_features, in_features);
    return product(pl, a, b, y, y_row_stride, rows, out_features, in_features, dtype, ep, workspace, reinterpret_cast<hipStream_t>(stream));
}

size_t sthip_linear_act_backward_workspace_bytes(int64_t rows, int64_t in_features, int64_t out_features, int dtype, int activation) {
    if (rows < 0 || in_features < 0 || out_features <= 0 || dtype < STHIP_F32 || dtype > STHIP_BF16) return 0;
    const size_t dz = activation == STHIP_ACT_NONE ? 0 : align256((size_t)rows * out_features * elem_size(dtype));
    const size_t products = std::max({product_workspace(rows, in_features, out_features, dtype, false), product_workspace(out_features, in_features, rows, dtype, false),
                                      pair_workspace(rows, in_features, out_features, dtype)});
    return dz + std::max(products, act_part_bytes(rows, out_features, dtype));
}

int sthip_linear_act_backward(const void* dy, const void* x, const void* W, const void* pre, void* dx, void* dW, void* dbias,
                              int64_t rows, int64_t in_features, int64_t out_features,
                              int64_t dy_row_stride, int64_t x_row_stride, int64_t w_row_stride,
                              int dtype, int activation, void* workspace, size_t workspace_bytes, void* stream) {
    clear_error();
    int rc = check_linear(rows, in_features, out_features, dtype, activation);
    if (rc) return rc;
    const int64_t M = rows, K = in_features, N = out_features;
    if ((!dx && !dW && !dbias) || (N == 0 && (!dx || M == 0 || K == 0))) return STHIP_OK;
    if (N > 0 && M > 0 && (!dy || (activation != STHIP_ACT_NONE && !pre) || (dx && K > 0 && !W) || (dW && K > 0 && !x))) return fail(STHIP_ERR_ARG, "null pointer");
    if ((rc = check_stride("dy", dy_row_stride, N, M)) || (dW && (rc = check_stride("x", x_row_stride, K, M))) || (dx && (rc = check_stride("W", w_row_stride, K, N)))) return rc;
    if ((rc = check_workspace(workspace, workspace_bytes, sthip_linear_act_backward_workspace_bytes(M, K, N, dtype, activation)))) return rc;
    const hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    const int es = elem_size(dtype);
    char* ws = reinterpret_cast<char*>(workspace);
    const void* dz = dy;
    int64_t dz_ld = dy_row_stride;
    const bool act = activation != STHIP_ACT_NONE;
    if (act) { dz = ws; dz_ld = N; ws += align256((size_t)M * N * es); }
    // dx = dz W: W's rows are the k index; dW = dz^T x: both operands' rows are
    const Operand rows_dz = {dz, dz_ld, true}, cols_dz = {dz, dz_ld, false}, w = {W, w_row_stride, false}, xo = {x, x_row_stride, false};
    const bool has_dx = dx && M > 0 && K > 0, has_dw = dW && N > 0 && K > 0;
    const bool dma = has_dx && has_dw && product_direct(rows_dz, w, M, K, dtype) && product_direct(cols_dz, xo, N, K, dtype);
    const PlanPair pair = has_dx && has_dw ? plan_pair(M, K, N, dtype, dma) : PlanPair{-1, {}, {}};
    Plan7 plan_x = {}, plan_w = {};
    if (pair.tile < 0) {   // one by one; refused, if at all, before anything is launched
        if (has_dx && (plan_x = plan_product(rows_dz, w, M, K, N, dtype)).tile < 0) return refuse_size(M, K, N);
        if (has_dw && (plan_w = plan_product(cols_dz, xo, N, K, M, dtype)).tile < 0) return refuse_size(N, K, M);
    }
    if (N > 0 && (dbias || (act && M > 0))) {
        const ActPlan pl = act_plan(M, N, dtype);
        ActParams a = {};
        a.dy = dy; a.dy_rs = dy_row_stride; a.rows = (int)M; a.cols = (int)N; a.strip = pl.strip;
        if (act) { a.pre = pre; a.dz = const_cast<void*>(dz); }
        if (dbias && pl.strips > 1) a.part = reinterpret_cast<float*>(ws);
        else a.dbias = dbias;
        const dim3 grid((unsigned)pl.col_blocks, (unsigned)pl.strips);
        LaunchAct launch = {a, dtype, grid, s};
        with_activation(activation, launch);
        if ((rc = launched(hipGetLastError(), "act_backward"))) return rc;
        if (a.part) {
            const ColumnSumParams c = {a.part, {dbias, nullptr}, N, 0, pl.strips, (int)N};
            if ((rc = column_sum(c, 1, dtype, s))) return rc;
        }
    }
    const Epilogue none = {nullptr, nullptr, 0, nullptr, ACT_NONE};
    if (pair.tile >= 0) {
        Gemm7Pair P;
        P.dx = product_params(rows_dz, w, dx, K, M, K, N, dtype, none, pair.dx, ws);
        P.dw = product_params(cols_dz, xo, dW, K, N, K, M, dtype, none, pair.dw, ws + part_bytes(pair.dx, M, K));
        P.dx_tiles = P.dx.tiles_m * P.dx.tiles_n * P.dx.splits;
        const LaunchPair7 fn = dtype == STHIP_F32 ? kPair7_0 : dtype == STHIP_F16 ? kPair7_1 : kPair7_2;
        return launched(fn(P, pair.tile, dma, s), "linear_act gradient");
    }
    if (has_dx && (rc = product(plan_x, rows_dz, w, dx, K, M, K, N, dtype, none, ws, s))) return rc;
    if (has_dw && (rc = product(plan_w, cols_dz, xo, dW, K, N, K, M, dtype, none, ws, s))) return rc;
    return STHIP_OK;
}

int sthip_layer_norm_forward(const void* x, const void* weight, const void* bias, void* y, float* mean, float* rstd,
                             int64_t rows, int64_t cols, int64_t x_row_stride, int64_t y_row_stride,
                             int dtype, int param_dtype, double eps, void* stream) {
    clear_error();
    int rc = check_norm(rows, cols, dtype, param_dtype);
    if (rc) return rc;
    if (rows == 0 || cols == 0) return STHIP_OK;
    if (!x || !y || (!mean != !rstd)) return fail(STHIP_ERR_ARG, "null pointer");
    if (!(eps >= 0.0)) return fail(STHIP_ERR_ARG, "eps must not be negative, got %g", eps);
    if ((rc = check_stride("x", x_row_stride, cols, rows)) || (rc = check_stride("y", y_row_stride, cols, rows))) return rc;
    NormParams p = {};
    p.x = x; p.w = weight; p.b = bias; p.y = y; p.mean = mean; p.rstd = rstd; p.x_rs = x_row_stride; p.y_rs = y_row_stride;
    p.rows = (int)rows; p.cols = (int)cols; p.eps = (float)eps;
    const hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    by_types(dtype, param_dtype, [&](auto* t, auto* q) { norm_forward_any<std::remove_pointer_t<decltype(t)>, std::remove_pointer_t<decltype(q)>>(p, s); });
    return launched(hipGetLastError(), "layer_norm_forward");
}

size_t sthip_layer_norm_backward_workspace_bytes(int64_t rows, int64_t cols) {
    if (rows < 0 || cols <= 0) return 0;
    return align256((size_t)norm_parts(rows, cols) * 2 * cols * sizeof(float));
}

int sthip_layer_norm_backward(const void* dy, const void* x, const void* weight, const float* mean, const float* rstd,
                              void* dx, void* dweight, void* dbias, int64_t rows, int64_t cols,
                              int64_t dy_row_stride, int64_t x_row_stride, int64_t dx_row_stride,
                              int dtype, int param_dtype, void* workspace, size_t workspace_bytes, void* stream) {
    clear_error();
    int rc = check_norm(rows, cols, dtype, param_dtype);
    if (rc) return rc;
    if (cols == 0 || (!dx && !dweight && !dbias)) return STHIP_OK;
    if (rows > 0 && (!dy || !x || !mean || !rstd)) return fail(STHIP_ERR_ARG, "null pointer");
    if ((rc = check_stride("dy", dy_row_stride, cols, rows)) || (rc = check_stride("x", x_row_stride, cols, rows)) || (dx && (rc = check_stride("dx", dx_row_stride, cols, rows)))) return rc;
    const bool sums = dweight || dbias;
    if (sums && (rc = check_workspace(workspace, workspace_bytes, sthip_layer_norm_backward_workspace_bytes(rows, cols)))) return rc;
    NormParams p = {};
    p.x = x; p.w = weight; p.dy = dy; p.dx = dx; p.mean = const_cast<float*>(mean); p.rstd = const_cast<float*>(rstd);
    p.x_rs = x_row_stride; p.dy_rs = dy_row_stride; p.dx_rs = dx_row_stride;
    p.rows = (int)rows; p.cols = (int)cols; p.parts = norm_parts(rows, cols);
    p.part = sums ? reinterpret_cast<float*>(workspace) : nullptr;
    const hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    if (rows > 0 || sums)
        by_types(dtype, param_dtype, [&](auto* t, auto* q) { norm_backward_any<std::remove_pointer_t<decltype(t)>, std::remove_pointer_t<decltype(q)>>(p, s); });
    if ((rc = launched(hipGetLastError(), "layer_norm_backward"))) return rc;
    if (!sums) return STHIP_OK;
    const ColumnSumParams c = {p.part, {dweight, dbias}, 2 * cols, cols, p.parts, (int)cols};
    return column_sum(c, 2, param_dtype, s);
}

int sthip_rotary(const void* q, const void* k, void* q_out, void* k_out,
                 int64_t batch, int64_t tokens, int64_t q_heads, int64_t k_heads, int64_t head_dim, int64_t rotary_dim,
                 const int64_t q_strides[3], const int64_t k_strides[3], const int64_t q_out_strides[3], const int64_t k_out_strides[3],
                 const double* frequencies, const void* positions, int positions_bits, int64_t positions_batch_stride,
                 int64_t positions_token_stride, int64_t first_position, double gain, int interleaved, int inverse,
                 int dtype, void* stream) {
    clear_error();
    if (batch < 0 || tokens < 0 || q_heads < 0 || k_heads < 0 || head_dim < 0)
        return fail(STHIP_ERR_SHAPE, "negative size");
    if (dtype < STHIP_F32 || dtype > STHIP_BF16) return fail(STHIP_ERR_DTYPE, "unknown dtype %d", dtype);
    if (rotary_dim < 2 || rotary_dim % 2 || rotary_dim > head_dim)
        return fail(STHIP_ERR_SHAPE, "rotary_dim must be even, at least 2 and at most the head's %lld, got %lld", (long long)head_dim, (long long)rotary_dim);
    if (positions && positions_bits != 32 && positions_bits != 64) return fail(STHIP_ERR_ARG, "positions are 32- or 64-bit integers, got %d", positions_bits);
    if (!k) k_heads = 0;
    if (batch >= kMaxSize || tokens >= kMaxSize || q_heads >= (1 << 20) || k_heads >= (1 << 20) || head_dim >= (1 << 20) || batch * tokens >= kMaxSize)
        return fail(STHIP_ERR_SHAPE, "too many tokens, heads or elements of a head");
    const int64_t rows = batch * tokens, heads = q_heads + k_heads;
    if (rows == 0 || heads == 0) return STHIP_OK;
    if (!frequencies || (q_heads > 0 && (!q || !q_out || !q_strides || !q_out_strides)) || (k_heads > 0 && (!k_out || !k_strides || !k_out_strides)))
        return fail(STHIP_ERR_ARG, "null pointer");
    // in place with other strides a head would be written where another one is still to be read
    auto moved = [&](const void* from, const void* to, const int64_t* a, const int64_t* b, int64_t n) {
        return from == to && ((batch > 1 && a[0] != b[0]) || (tokens > 1 && a[1] != b[1]) || (n > 1 && a[2] != b[2]));
    };
    if ((q_heads > 0 && moved(q, q_out, q_strides, q_out_strides, q_heads)) || (k_heads > 0 && moved(k, k_out, k_strides, k_out_strides, k_heads)))
        return fail(STHIP_ERR_LAYOUT, "rotary in place needs the same strides on both sides");
    RotaryParams p = {};
    p.q = q; p.k = k; p.qo = q_out; p.ko = k_out;
    p.freq = frequencies; p.pos = positions; p.pos64 = positions_bits == 64; p.pos_bs = positions_batch_stride; p.pos_ts = positions_token_stride; p.first = first_position;
    p.tokens = (int)tokens; p.rows = (int)rows; p.heads_q = (int)q_heads; p.heads = (int)heads;
    p.rot = (int)rotary_dim; p.interleaved = interleaved != 0;
    p.gain = (float)gain; p.sign = inverse ? -1.f : 1.f;
    const int es = elem_size(dtype), n = 16 / es;
    auto take = [&](int64_t (&to)[3], const int64_t* from) { for (int i = 0; i < 3; ++i) to[i] = from[i]; };
    if (q_heads > 0) { take(p.qs, q_strides); take(p.qos, q_out_strides); }
    if (k_heads > 0) { take(p.ks, k_strides); take(p.kos, k_out_strides); }
    // turned in place: nothing to do behind the rotated part
    const bool copy = (q_heads > 0 && q != q_out) || (k_heads > 0 && k != k_out);
    // pairs a thread: the longest pieces that divide the pairs and what is copied
    int v = n;
    while (v > 1 && (rotary_dim / 2 % v || (copy && (head_dim - rotary_dim) % v))) v /= 2;
    p.turn_items = (int)(rotary_dim / 2 / v);
    p.items = p.turn_items + (copy ? (int)((head_dim - rotary_dim) / v) : 0);
    // a thread keeps its cosines for several heads where there are threads enough without
    const int64_t wanted = ceil_div((int64_t)256 * 2048, rows * p.items);
    p.groups = (int)std::max<int64_t>(1, std::min<int64_t>(heads, std::max<int64_t>(wanted, ceil_div(heads, 8))));
    const int64_t blocks = ceil_div(rows * p.items * p.groups, 256), most = (int64_t)1 << 23;
    const hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    for (p.first_block = 0; p.first_block < blocks; p.first_block += most) {
        const unsigned n = (unsigned)std::min(most, blocks - p.first_block);
        if (dtype == STHIP_F32) launch_rotary<float>(p, v, n, s);
        else if (dtype == STHIP_F16) launch_rotary<f16_t>(p, v, n, s);
        else launch_rotary<bf16_t>(p, v, n, s);
        if (const int rc = launched(hipGetLastError(), "rotary")) return rc;
    }
    return STHIP_OK;
}

}  // extern "C"
