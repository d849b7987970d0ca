// Launch side of the edge-capable GEMM kernel (sthip_kernel7.hpp).
#pragma once
#include "sthip_launch.hpp"
#include "sthip_kernel7.hpp"

namespace sthip {

// 128_DEEP: 16-bit, four stages of LDS instead of two, one workgroup a CU; 256_128: 16-bit, three stages; 32: fp32 alone; the last is no
// tile but few_rows_kernel.
enum { TILE7_256 = 0, TILE7_128 = 1, TILE7_64 = 2, TILE7_32 = 3, TILE7_128_DEEP = 4, TILE7_256_128 = 5, TILE7_FEW_ROWS = 6 };
inline int tile7_rows(int tile) { return tile == TILE7_256 || tile == TILE7_256_128 ? 256 : tile == TILE7_64 ? 64 : tile == TILE7_32 ? 32 : 128; }
inline int tile7_cols(int tile) { return tile == TILE7_256 ? 256 : tile == TILE7_64 ? 64 : tile == TILE7_32 ? 32 : 128; }
constexpr int tile7_threads(int tile) { return tile == TILE7_256 || tile == TILE7_256_128 ? 512 : 256; }
// A launch holds less than 2^32 threads.
constexpr bool launchable(int64_t workgroups, int threads) { return workgroups < ((int64_t)1 << 32) / threads; }
// The tile that the debug switch (sthip_debug_force_tile) asks for, -1 if none.
int debug_tile7();
enum { LAYOUT_NT = 0, LAYOUT_NN = 1, LAYOUT_TN = 2 };   // both k-contiguous; B by its index; both by their index

// One function per element type and part of sthip_inst7.hip: the forward product, the gradients' one by one, the two of a
// gradient together.  p.splits > 1: the joining launch follows.
typedef hipError_t (*LaunchFn7)(const Gemm7Params& p, int tile, int layout, bool dma, hipStream_t stream);
typedef hipError_t (*LaunchPair7)(const Gemm7Pair& p, int tile, bool dma, hipStream_t stream);
extern const LaunchFn7 kForward7_0, kForward7_1, kForward7_2, kGradient7_0, kGradient7_1, kGradient7_2;
extern const LaunchPair7 kPair7_0, kPair7_1, kPair7_2;

// Whether the tile grid covers C and no tile lies outside of it, which the loaders' clamps rely on, and one launch holds it.
inline bool covers(const Gemm7Params& p, int bm, int bn, int threads) {
    return launchable((int64_t)p.tiles_m * p.tiles_n * p.splits, threads) && p.M > 0 && p.N > 0 && p.tiles_m == (p.M + bm - 1) / bm && p.tiles_n == (p.N + bn - 1) / bn && p.splits >= 1 && p.k_split > 0 &&
           (int64_t)p.k_split * p.splits >= p.K;
}

template <class T, int WM, int WN, int NWM, int NWN, int NS, bool A_KC, bool B_KC, bool DMA>
hipError_t launch_gemm7_one(const Gemm7Params& p, hipStream_t stream) {
    if (!covers(p, WM * NWM, WN * NWN, NWM * NWN * 64)) return hipErrorInvalidValue;
    auto kern = gemm7_kernel<T, WM, WN, NWM, NWN, NS, A_KC, B_KC, DMA>;
    constexpr int smem_bytes = Pipe7<T, WM, WN, NWM, NWN, NS, A_KC, B_KC>::kSmem;
    static OptIn opted;
    hipError_t e = opt_in_lds(opted, reinterpret_cast<const void*>(kern), smem_bytes);
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL(kern, dim3((unsigned)(p.tiles_m * p.tiles_n * p.splits)), dim3(NWM * NWN * 64), smem_bytes, stream, p);
    return hipGetLastError();
}

template <bool FORWARD, class T, int WM, int WN, int NWM, int NWN, int NS, bool DMA>
hipError_t launch_gemm7_layout(const Gemm7Params& p, int layout, hipStream_t stream) {
    if constexpr (FORWARD) {
        if (layout == LAYOUT_NT) return launch_gemm7_one<T, WM, WN, NWM, NWN, NS, true, true, DMA>(p, stream);
    } else {
        if (layout == LAYOUT_NN) return launch_gemm7_one<T, WM, WN, NWM, NWN, NS, true, false, DMA>(p, stream);
        if (layout == LAYOUT_TN) return launch_gemm7_one<T, WM, WN, NWM, NWN, NS, false, false, DMA>(p, stream);
    }
    return hipErrorInvalidValue;
}

template <class T, int WM, int WN, int NWM, int NWN, int NS, bool DMA>
hipError_t launch_gemm7_pair_one(const Gemm7Pair& p, hipStream_t stream) {
    constexpr int threads = NWM * NWN * 64;
    if (!covers(p.dx, WM * NWM, WN * NWN, threads) || !covers(p.dw, WM * NWM, WN * NWN, threads)) return hipErrorInvalidValue;
    const int tiles = p.dx_tiles + p.dw.tiles_m * p.dw.tiles_n * p.dw.splits;
    if (!launchable(tiles, threads)) return hipErrorInvalidValue;
    auto kern = gemm7_pair_kernel<T, WM, WN, NWM, NWN, NS, DMA>;
    constexpr int smem_bytes = Pipe7<T, WM, WN, NWM, NWN, NS, true, false>::kSmem;
    static OptIn opted;
    hipError_t e = opt_in_lds(opted, reinterpret_cast<const void*>(kern), smem_bytes);
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL(kern, dim3((unsigned)tiles), dim3(threads), smem_bytes, stream, p);
    return hipGetLastError();
}

template <class T>
hipError_t launch_gemm7_pair(const Gemm7Pair& p, int tile, bool dma, hipStream_t stream) {
    hipError_t e = hipErrorInvalidValue;
    switch (tile) {
        case TILE7_256: if (dma) e = launch_gemm7_pair_one<T, 128, 64, 2, 4, 2, true>(p, stream); break;
        case TILE7_128: e = dma ? launch_gemm7_pair_one<T, 64, 64, 2, 2, 2, true>(p, stream) : launch_gemm7_pair_one<T, 64, 64, 2, 2, 2, false>(p, stream); break;
        case TILE7_64: e = dma ? launch_gemm7_pair_one<T, 32, 32, 2, 2, 4, true>(p, stream) : launch_gemm7_pair_one<T, 32, 32, 2, 2, 2, false>(p, stream); break;
        case TILE7_256_128: if constexpr (sizeof(T) == 2) if (dma) e = launch_gemm7_pair_one<T, 64, 64, 4, 2, 3, true>(p, stream); break;
        case TILE7_128_DEEP: if constexpr (sizeof(T) == 2) if (dma) e = launch_gemm7_pair_one<T, 64, 64, 2, 2, 4, true>(p, stream); break;
        case TILE7_32: if constexpr (sizeof(T) == 4) e = dma ? launch_gemm7_pair_one<T, 16, 16, 2, 2, 4, true>(p, stream) : launch_gemm7_pair_one<T, 16, 16, 2, 2, 2, false>(p, stream); break;
    }
    if (e != hipSuccess || (p.dx.splits <= 1 && p.dw.splits <= 1)) return e;
    auto blocks = [](const Gemm7Params& q) { return q.splits > 1 ? ((int64_t)q.M * ((q.N + 3) / 4) + 255) / 256 : (int64_t)0; };
    hipLaunchKernelGGL((gemm7_join_pair_kernel<T>), dim3((unsigned)(blocks(p.dx) + blocks(p.dw))), dim3(256), 0, stream, p, blocks(p.dx));
    return hipGetLastError();
}

template <class T>
hipError_t launch_few_rows(const Gemm7Params& p, hipStream_t stream) {
    if (p.M > 16 || p.splits < 1 || (p.splits > 1 && (!p.part || p.k_split % (kTurnF / (int)sizeof(T)) || (int64_t)p.k_split * p.splits < p.K))) return hipErrorInvalidValue;
    hipLaunchKernelGGL((few_rows_kernel<T>), dim3((unsigned)((p.N + 15) / 16), (unsigned)p.splits), dim3(kWavesF * 64), 0, stream, p);
    return hipGetLastError();
}

template <bool FORWARD, class T>
hipError_t launch_gemm7(const Gemm7Params& p, int tile, int layout, bool dma, hipStream_t stream) {
    hipError_t e = hipErrorInvalidValue;
    switch (tile) {
        case TILE7_FEW_ROWS: if constexpr (FORWARD) e = launch_few_rows<T>(p, stream); break;
        case TILE7_256: if (dma) e = launch_gemm7_layout<FORWARD, T, 128, 64, 2, 4, 2, true>(p, layout, stream); break;
        case TILE7_128: e = dma ? launch_gemm7_layout<FORWARD, T, 64, 64, 2, 2, 2, true>(p, layout, stream) : launch_gemm7_layout<FORWARD, T, 64, 64, 2, 2, 2, false>(p, layout, stream); break;
        case TILE7_64: e = dma ? launch_gemm7_layout<FORWARD, T, 32, 32, 2, 2, 4, true>(p, layout, stream) : launch_gemm7_layout<FORWARD, T, 32, 32, 2, 2, 2, false>(p, layout, stream); break;
        case TILE7_256_128: if constexpr (sizeof(T) == 2) if (dma) e = launch_gemm7_layout<FORWARD, T, 64, 64, 4, 2, 3, true>(p, layout, stream); break;
        case TILE7_128_DEEP: if constexpr (sizeof(T) == 2) if (dma) e = launch_gemm7_layout<FORWARD, T, 64, 64, 2, 2, 4, true>(p, layout, stream); break;
        case TILE7_32: if constexpr (sizeof(T) == 4) e = dma ? launch_gemm7_layout<FORWARD, T, 16, 16, 2, 2, 4, true>(p, layout, stream) : launch_gemm7_layout<FORWARD, T, 16, 16, 2, 2, 2, false>(p, layout, stream); break;
    }
    if (e != hipSuccess || p.splits <= 1) return e;
    const int64_t threads = (int64_t)p.M * ((p.N + 3) / 4);
    hipLaunchKernelGGL((gemm7_join_kernel<T>), dim3((unsigned)((threads + 255) / 256)), dim3(256), 0, stream, p);
    return hipGetLastError();
}

}  // namespace sthip
