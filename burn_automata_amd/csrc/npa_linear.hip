// npa_linear.hip - the linear layer y = act(x W^T + b) + residual and its adjoint.
//
// Adjoint: dz = dy act'(z), dx = dz W, dW = dz^T x, db = sum over rows of dz. All three products are
// C[m][n] = sum_k A(m, k) B(n, k) with operands of which either index runs through memory.
#include "npa_tiles.hpp"

namespace npa {
namespace {

// Measured: f32 8,192, 1,024 -> 1,024 99 us, 174 TFLOP/s (the f32 matrix cores reach 153), the matrix cores busy
// for 53 % of the time beside the splitting of operands; 65,536, 66 -> 128 f32 with z kept 23 us, 3.7 TB/s. f32's
// 64 x 64 tiles keep to the registers of four blocks a CU (65,536, 128 -> 18: 14.7 us, 17.0 with three).
template <class T, int BM, int BN, int WM, int WN, int DEPTH>
__global__ __launch_bounds__(256, sizeof(T) == 4 && BM == 64 ? 4 : 2) void k_forward(ProductArgs g) {
    using X = Tile<T, BM, BN, WM, WN, DEPTH, true, true, false>;
    __shared__ __align__(16) char lds[X::LDS];
    product_block<X, T, BM, BN, WN>(g, blockIdx.x, lds);
}

// Both products of the adjoint in one launch, the one with the longer blocks first (`dx_last`: dW's): short ones
// fill what the long ones leave. Measured: f16 3,001, 777 -> 1,111 33 us (dW first with blocks of a third of dx's
// length 50); f32 65,536, 66 -> 128 through relu 49 us, where dy and z pass twice.
template <class T, int BM, int BN, int WM, int WN, int DEPTH, bool SLOPE>
__global__ __launch_bounds__(256, sizeof(T) == 4 && BM == 64 ? 3 : 2) void k_adjoint(ProductArgs dw, ProductArgs dx, uint32_t first_blocks, bool dx_last) {
    using W = Tile<T, BM, BN, WM, WN, DEPTH, false, false, SLOPE>;
    using X = Tile<T, BM, BN, WM, WN, DEPTH, true, false, SLOPE>;
    __shared__ __align__(16) char lds[W::LDS];
    const bool first = blockIdx.x < first_blocks;
    const uint32_t block = first ? blockIdx.x : blockIdx.x - first_blocks;
    if (first == dx_last)
        product_block<W, T, BM, BN, WN>(dw, block, lds);
    else
        product_block<X, T, BM, BN, WN>(dx, block, lds);
}

// 256 x 256 in steps of 64, two buffers, waves of 128 x 64. Measured at 16,384 x 8,192 -> 8,192 bf16: 1,280
// TFLOP/s; steps of 32 in four buffers 1,150; 256 x 128 tiles of four waves, two blocks a CU, 960 (the tiles'
// way through L2 grows by half); four waves of 128 x 128 990. Over a launch of 16,384, 2,048 -> 8,192 the matrix cores
// are busy for 54 % of the CUs' cycles, over the adjoint's, which store less, for 63 and 66 %, and bank conflicts take 1
// to 4 % of the LDS reads' cycles; the loads' arrival and the stores at the end bound it. Results are stored past the
// caches (16,384, 2,048 -> 8,192: 459 us, 504 through them; 4,096, 2,048 -> 2,048 47 us, 48), which a layer that reads them at
// once pays for where they would have stayed there (two layers of 4,096, 2,048 -> 2,048: 104 us, 99 through the caches; of
// 8,192 rows 125 both ways). f32 tiles lose 4 % by it and do not.
template <class T, int BM, int BN, int BK, int WM, int WN, int STAGES, bool AF, bool BF>
__global__ __launch_bounds__(WM * WN * 64, 2) void k_direct(ProductArgs g) {
    using X = Direct<T, BM, BN, BK, WM, WN, STAGES, AF, BF>;
    extern __shared__ __align__(16) char lds[];
    direct_block<X, T, BM, BN, WN, AF, BF>(g, lds);
}

template <class T, int RT>
__global__ __launch_bounds__(kFewWaves * 64) void k_few(ProductArgs g) {
    __shared__ float red[kFewWaves][RT * 16][17];
    few_block<T, RT>(g, 0, g.M, blockIdx.x * 16, red);
}

template <class T, int ACT>
__global__ __launch_bounds__(256) void k_slope(SlopeArgs g) {
    __shared__ float shared[256][9];
    slope_block<T, ACT>(g, g.rows * blockIdx.y / gridDim.y, g.rows * (blockIdx.y + 1) / gridDim.y,
                        g.partials ? g.partials + (uint64_t)blockIdx.y * g.cols : nullptr, shared);
}

template <class T, bool AF, bool BF>
bool direct_applies(const ProductArgs& g, int cus) {
    if (sizeof(T) != 2 || g.M < 256 || g.N < 256 || g.K < 256 || g.K % 64) return false;
    if (!direct_operand<AF>(g.a, g.M) || !direct_operand<BF>(g.b, g.N)) return false;
    // Half a tile a CU or more, with splits of 1,024 columns at least: fewer leave more of the chip idle
    // than smaller tiles lose (16,384, 8,192 -> 8,192 bf16: 1.69 ms, 2.81 in smaller tiles; at the limit 4,096, 512 -> 2,048 18 us, 21,
    // and 1,024, 2,048 -> 4,096 42 us, 42).
    return (uint64_t)((g.M + 255) / 256) * ((g.N + 255) / 256) * std::max<uint64_t>(1, g.K / 1024) >= (uint64_t)cus / 2;
}

template <class T, int BM, int BN, int BK, int WM, int WN, int STAGES, bool AF, bool BF>
hipError_t direct_of(ProductArgs g, LayerWorkspace& ws, int cus, hipStream_t stream) {
    using X = Direct<T, BM, BN, BK, WM, WN, STAGES, AF, BF>;
    const auto kernel = k_direct<T, BM, BN, BK, WM, WN, STAGES, AF, BF>;
    static LdsLimitFlags flags;
    hipError_t e = raise_lds_limit((const void*)kernel, flags);
    if (e != hipSuccess) return e;
    const uint64_t steps = g.K / BK;
    set_plan(g, plan(kDirect, false, false, g.M, g.N, steps, cus, (uint32_t)std::max<uint64_t>(1, steps * BK / 1024)), kDirect, BK);
    if (part_floats(g)) {
        if ((e = ws.reserve(ws.partials, part_floats(g) * 4, stream)) != hipSuccess) return e;
        g.partials = ws.partials.as<float>();
    }
    hipLaunchKernelGGL(kernel, dim3(block_count(g)), dim3(X::WAVES * 64), X::LDS, stream, g);
    if ((e = hipGetLastError()) != hipSuccess) return e;
    return join<T>(&g, nullptr, BiasArgs(), stream);
}

template <class T, bool AF, bool BF>
hipError_t direct(const ProductArgs& g, LayerWorkspace& ws, int cus, hipStream_t stream) {
    if constexpr (sizeof(T) == 2) return direct_of<T, 256, 256, 64, 2, 4, 2, AF, BF>(g, ws, cus, stream);
    return hipErrorInvalidValue;
}

template <class T>
hipError_t few_rows(const ProductArgs& g, hipStream_t stream) {
    // four runs a wave or more, up to sixteen waves
    const uint32_t runs = (uint32_t)((g.K + 31) / 32);
    uint32_t waves = 1;
    while (waves < kFewWaves && waves * 4 < runs) waves *= 2;
    const dim3 grid((g.N + 15) / 16), block(waves * 64);
    if (g.M <= 16)
        hipLaunchKernelGGL((k_few<T, 1>), grid, block, 0, stream, g);
    else
        hipLaunchKernelGGL((k_few<T, 2>), grid, block, 0, stream, g);
    return hipGetLastError();
}

template <class T>
hipError_t linear_of(const LinearArgs& a, LayerWorkspace& ws, int cus, hipStream_t stream) {
    constexpr bool F32 = sizeof(T) == 4;
    constexpr uint64_t BK = F32 ? 32 : 64;
    ProductArgs g;
    g.M = (uint32_t)a.rows;
    g.N = a.out_dims;
    g.K = a.in_dims;
    g.a = {a.x, a.x_stride, a.rows};
    g.b = {a.w, a.w_stride, a.out_dims};
    Epilogue& e = g.e;
    e.out = a.out;
    e.out_stride = a.out_stride;
    e.bias = a.bias;
    e.bias_f32 = a.bias_f32;
    e.residual = a.residual;
    e.residual_stride = a.residual_stride;
    e.z = a.z;
    e.z_stride = a.z_stride;
    e.act = a.activation;
    e.out_f32 = F32;
    if (direct_applies<T, true, true>(g, cus)) return direct<T, true, true>(g, ws, cus, stream);
    const uint64_t steps = (g.K + BK - 1) / BK;
    int best = 0;
    Plan p;
    for (int k = 0; k < 3; ++k) {
        // (the largest tiles never are too many: their results would not fit the memory)
        if ((k == 2 && g.N > 32) || (k && tile_count(kShapes[k], g.M, g.N) >= kTooManyTiles)) continue;
        const Plan q = plan(kShapes[k], F32, false, g.M, g.N, steps, cus, kMostSplits);
        if (k == 0 || q.us < p.us) {
            p = q;
            best = k;
        }
    }
    if (g.M <= 32 && g.N <= (1u << 25)) {  // more outputs could be 2^32 threads
        // Measured: what a CU's blocks read of weights and x comes at 60 GB/s, at most 4.6 TB/s for all of them;
        // 1 x 4,096 -> 4,096 bf16 10 us, 14 in split tiles; 30 x 4,000 -> 1,000 f32 24 us, 14 in split tiles.
        const double block = 16.0 * g.K * sizeof(T) * (g.M <= 16 ? 2 : 3), blocks = (g.N + 15) / 16;
        if (3.0 + std::max(std::ceil(blocks / cus) * block / 60e3, blocks * 16.0 * g.K * sizeof(T) / 4.6e6) < p.us)
            return few_rows<T>(g, stream);
    }
    set_plan(g, p, kShapes[best], BK);
    hipError_t err = hipSuccess;
    if (part_floats(g)) {
        if ((err = ws.reserve(ws.partials, part_floats(g) * 4, stream)) != hipSuccess) return err;
        g.partials = ws.partials.as<float>();
    }
    const dim3 grid(block_count(g)), block(256);
    switch (best) {
        case 0: hipLaunchKernelGGL((k_forward<T, 128, 128, 2, 2, 2>), grid, block, 0, stream, g); break;
        case 1: hipLaunchKernelGGL((k_forward<T, 64, 64, 2, 2, 3>), grid, block, 0, stream, g); break;
        default: hipLaunchKernelGGL((k_forward<T, 128, 32, 4, 1, 3>), grid, block, 0, stream, g);
    }
    if ((err = hipGetLastError()) != hipSuccess) return err;
    return join<T>(&g, nullptr, BiasArgs(), stream);
}

// Rows of dz in the workspace: whole units.
uint64_t dz_stride(const LinearArgs& a) { return (a.out_dims + 7) & ~7ull; }

// dz and the bias gradient's partial sums by a kernel of their own.
template <class T>
hipError_t slope_of(const LinearArgs& a, LayerWorkspace& ws, int cus, BiasArgs& bias, hipStream_t stream) {
    const bool slope = a.activation != NPA_ACT_IDENTITY;
    SlopeArgs g;
    g.dy = a.dy;
    g.z = a.z;
    g.dy_stride = a.dy_stride;
    g.z_stride = a.z_stride;
    g.rows = a.rows;
    g.cols = a.out_dims;
    const uint32_t units = (g.cols + 7) / 8;
    for (g.lanes = 1; g.lanes < 32 && g.lanes < units;) g.lanes *= 2;
    const uint32_t across = (units + g.lanes - 1) / g.lanes;
    // about eight blocks a CU, each with at least two rows a thread, and no more than 512 rows of partial sums
    const uint64_t down = std::max<uint64_t>(1, std::min({(uint64_t)(8 * cus + across - 1) / across, (uint64_t)512,
                                                          a.rows * g.lanes / 512}));
    hipError_t e = hipSuccess;
    if (slope && (a.dx || a.dw)) {
        g.dz_stride = dz_stride(a);
        if ((e = ws.reserve(ws.dz, a.rows * g.dz_stride * sizeof(T), stream)) != hipSuccess) return e;
        g.dz = ws.dz.ptr;
    }
    if (a.db) {
        if ((e = ws.reserve(ws.columns, down * g.cols * 4, stream)) != hipSuccess) return e;
        g.partials = ws.columns.as<float>();
        bias.partials = g.partials;
        bias.parts = (uint32_t)down;
    }
    const dim3 grid(across, (uint32_t)down);
    switch (a.activation) {
        case NPA_ACT_IDENTITY: hipLaunchKernelGGL((k_slope<T, NPA_ACT_IDENTITY>), grid, dim3(256), 0, stream, g); break;
        case NPA_ACT_RELU: hipLaunchKernelGGL((k_slope<T, NPA_ACT_RELU>), grid, dim3(256), 0, stream, g); break;
        case NPA_ACT_GELU: hipLaunchKernelGGL((k_slope<T, NPA_ACT_GELU>), grid, dim3(256), 0, stream, g); break;
        default: hipLaunchKernelGGL((k_slope<T, NPA_ACT_SILU>), grid, dim3(256), 0, stream, g);
    }
    return hipGetLastError();
}

template <class T, int BM, int BN, int WM, int WN, int DEPTH>
hipError_t launch_adjoint(const ProductArgs& dw, const ProductArgs& dx, uint32_t dw_blocks, uint32_t dx_blocks, bool slope,
                          hipStream_t stream) {
    const dim3 grid(dw_blocks + dx_blocks), block(256);
    const bool dx_last = !dx_blocks || (dw_blocks && dw.split_len >= dx.split_len);
    const uint32_t first = dx_last ? dw_blocks : dx_blocks;
    if (slope)
        hipLaunchKernelGGL((k_adjoint<T, BM, BN, WM, WN, DEPTH, true>), grid, block, 0, stream, dw, dx, first, dx_last);
    else
        hipLaunchKernelGGL((k_adjoint<T, BM, BN, WM, WN, DEPTH, false>), grid, block, 0, stream, dw, dx, first, dx_last);
    return hipGetLastError();
}

template <class T>
hipError_t linear_adjoint_of(const LinearArgs& a, LayerWorkspace& ws, int cus, hipStream_t stream) {
    constexpr bool F32 = sizeof(T) == 4;
    constexpr uint64_t BK = F32 ? 32 : 64;
    const bool active = a.activation != NPA_ACT_IDENTITY;
    hipError_t err = hipSuccess;
    ProductArgs dw, dx;
    dw.M = a.out_dims;
    dw.N = a.in_dims;
    dw.K = a.rows;
    dw.a = {a.dy, a.dy_stride, a.rows};
    dw.b = {a.x, a.x_stride, a.rows};
    dw.e.out = a.dw;
    dw.e.out_stride = a.in_dims;
    dw.e.out_f32 = a.grad_f32;
    dw.e.accumulate = a.accumulate;
    dx.M = (uint32_t)a.rows;
    dx.N = a.in_dims;
    dx.K = a.out_dims;
    dx.a = {a.dy, a.dy_stride, a.rows};
    dx.b = {a.w, a.w_stride, a.out_dims};
    dx.e.out = a.dx;
    dx.e.out_stride = a.dx_stride;
    dx.e.out_f32 = F32;
    BiasArgs bias;
    bias.db = a.db;
    bias.cols = a.out_dims;
    bias.f32 = a.grad_f32;
    bias.accumulate = a.accumulate;
    const bool want_dx = a.dx && a.rows, want_dw = a.dw;
    // Large aligned products straight from memory: dz has to be there.
    if (active) dw.a = dx.a = {nullptr, dz_stride(a), a.rows};
    const bool direct_dx = want_dx && direct_applies<T, true, false>(dx, cus);
    const bool direct_dw = want_dw && direct_applies<T, false, false>(dw, cus);
    // Few elements: the slope in the products themselves, as often as a tile stages an element, without a
    // launch and dz in memory (8,391 rows, 45 -> 50: 15 us, 18 with them; 3,001 rows, 777 -> 1,111: 89 us, 47
    // with them). relu's slope costs nothing where each element is staged once (65,536 rows, 66 -> 128 f32: 51 us, 59).
    // The bias gradient of the identity is always theirs.
    const uint64_t again = (a.in_dims + 127) / 128;
    const bool staged = !direct_dx && !direct_dw && want_dw && (!active || a.rows * a.out_dims * again <= (1u << 19) ||
                         (a.activation == NPA_ACT_RELU && again == 1));
    if (!staged && (active || a.db)) {
        if ((err = slope_of<T>(a, ws, cus, bias, stream)) != hipSuccess) return err;
    }
    if (active) dw.a = dx.a = staged ? Operand{a.dy, a.dy_stride, a.rows} : Operand{ws.dz.ptr, dz_stride(a), a.rows};
    if (direct_dx && (err = direct<T, true, false>(dx, ws, cus, stream)) != hipSuccess) return err;
    if (direct_dw && (err = direct<T, false, false>(dw, ws, cus, stream)) != hipSuccess) return err;

    const bool tiled_dx = want_dx && !direct_dx, tiled_dw = want_dw && !direct_dw;
    uint32_t dw_blocks = 0, dx_blocks = 0;
    if (tiled_dx || tiled_dw) {
        int best = 0;
        double least = 0.0;
        Plan pw, px;
        for (int k = 0; k < 3; ++k) {
            const uint64_t tiles = (tiled_dw ? tile_count(kShapes[k], dw.M, dw.N) : 0) +
                                   (tiled_dx ? tile_count(kShapes[k], dx.M, dx.N) : 0);
            if ((k == 2 && a.in_dims > 32) || (k && tiles >= kTooManyTiles)) continue;
            Plan w, x;
            double us;
            if (tiled_dw && tiled_dx)
                us = plan(kShapes[k], F32, dw, dx, BK, cus, w, x);
            else if (tiled_dw)
                us = (w = plan(kShapes[k], F32, true, dw.M, dw.N, (dw.K + BK - 1) / BK, cus, kMostSplits)).us;
            else
                us = (x = plan(kShapes[k], F32, true, dx.M, dx.N, (dx.K + BK - 1) / BK, cus, kMostSplits)).us;
            if (k == 0 || us < least) {
                least = us;
                pw = w;
                px = x;
                best = k;
            }
        }
        if (tiled_dw) {
            set_plan(dw, pw, kShapes[best], BK);
            dw_blocks = block_count(dw);
        }
        if (tiled_dx) {
            set_plan(dx, px, kShapes[best], BK);
            dx_blocks = block_count(dx);
        }
        const uint64_t floats = (tiled_dw ? part_floats(dw) : 0) + (tiled_dx ? part_floats(dx) : 0);
        if (floats) {
            if ((err = ws.reserve(ws.partials, floats * 4, stream)) != hipSuccess) return err;
            dw.partials = ws.partials.as<float>();
            dx.partials = dw.partials + (tiled_dw ? part_floats(dw) : 0);
        }
        if (staged && active) {
            dw.a.z = dx.a.z = a.z;
            dw.a.z_stride = dx.a.z_stride = a.z_stride;
            dw.a.act = dx.a.act = a.activation;
        }
        if (staged && a.db && dw.splits == 1) {
            dw.db = a.db;
            dw.db_f32 = a.grad_f32;
            dw.db_accumulate = a.accumulate;
            bias.db = nullptr;  // no parts to join
        } else if (staged && a.db) {
            if ((err = ws.reserve(ws.columns, (uint64_t)dw.splits * dw.M * 4, stream)) != hipSuccess) return err;
            dw.columns = ws.columns.as<float>();
            bias.partials = dw.columns;
            bias.parts = dw.splits;
        }
        const bool slope = staged && active;
        if (best == 0)
            err = launch_adjoint<T, 128, 128, 2, 2, 1>(dw, dx, dw_blocks, dx_blocks, slope, stream);
        else if (best == 1)
            err = launch_adjoint<T, 64, 64, 2, 2, 3>(dw, dx, dw_blocks, dx_blocks, slope, stream);
        else
            err = launch_adjoint<T, 128, 32, 4, 1, 2>(dw, dx, dw_blocks, dx_blocks, slope, stream);
        if (err != hipSuccess) return err;
    }
    return join<T>(dw_blocks ? &dw : nullptr, dx_blocks ? &dx : nullptr, bias, stream);
}

}  // namespace

// One object for each element type (all in one without NPA_PART).
#if !defined(NPA_PART) || NPA_PART == 0
hipError_t linear_f32(const LinearArgs& a, LayerWorkspace& ws, int cus, hipStream_t stream) { return linear_of<float>(a, ws, cus, stream); }
hipError_t linear_adjoint_f32(const LinearArgs& a, LayerWorkspace& ws, int cus, hipStream_t stream) { return linear_adjoint_of<float>(a, ws, cus, stream); }

hipError_t launch_linear(const LinearArgs& a, LayerWorkspace& ws, int cus, hipStream_t stream) {
    if (!a.rows) return hipSuccess;
    if (a.type == NPA_TYPE_F32) return linear_f32(a, ws, cus, stream);
    return a.type == NPA_TYPE_BF16 ? linear_bf16(a, ws, cus, stream) : linear_f16(a, ws, cus, stream);
}

hipError_t launch_linear_adjoint(const LinearArgs& a, LayerWorkspace& ws, int cus, hipStream_t stream) {
    if (a.type == NPA_TYPE_F32) return linear_adjoint_f32(a, ws, cus, stream);
    return a.type == NPA_TYPE_BF16 ? linear_adjoint_bf16(a, ws, cus, stream) : linear_adjoint_f16(a, ws, cus, stream);
}
#endif
#if !defined(NPA_PART) || NPA_PART == 1
hipError_t linear_bf16(const LinearArgs& a, LayerWorkspace& ws, int cus, hipStream_t stream) { return linear_of<__bf16>(a, ws, cus, stream); }
hipError_t linear_adjoint_bf16(const LinearArgs& a, LayerWorkspace& ws, int cus, hipStream_t stream) { return linear_adjoint_of<__bf16>(a, ws, cus, stream); }
#endif
#if !defined(NPA_PART) || NPA_PART == 2
hipError_t linear_f16(const LinearArgs& a, LayerWorkspace& ws, int cus, hipStream_t stream) { return linear_of<_Float16>(a, ws, cus, stream); }
hipError_t linear_adjoint_f16(const LinearArgs& a, LayerWorkspace& ws, int cus, hipStream_t stream) { return linear_adjoint_of<_Float16>(a, ws, cus, stream); }
#endif

}  // namespace npa
