// npa_linear.hip - the linear layer y = act(x W^T + b) + residual and its adjoint.
//
// Adjoint: dz = dy act'(z), dx = dz W, dW = dz^T x, db = sum over rows of dz. All three products are
// C[m][n] = sum_k A(m, k) B(n, k) with operands of which either index runs through memory.
#include "npa_layers.hpp"

#include <algorithm>

namespace npa {
namespace {

struct Operand {
    const void* p = nullptr;
    uint64_t stride = 0;  // of the slow index
    bool k_fast = true;   // [m][k], else [k][m]
};

// What becomes of a finished sum.
struct Epilogue {
    void* out = nullptr;
    uint64_t out_stride = 0;
    const void* bias = nullptr;
    const void* residual = nullptr;
    uint64_t residual_stride = 0;
    void* z = nullptr;
    uint64_t z_stride = 0;
    uint32_t act = NPA_ACT_IDENTITY;
    bool bias_f32 = false, out_f32 = false, accumulate = false;
};

__device__ inline float activate_any(uint32_t act, float z) {
    switch (act) {
        case NPA_ACT_RELU: return activate<NPA_ACT_RELU>(z);
        case NPA_ACT_GELU: return activate<NPA_ACT_GELU>(z);
        case NPA_ACT_SILU: return activate<NPA_ACT_SILU>(z);
    }
    return z;
}

__device__ inline float activate_adjoint_any(uint32_t act, float dy, float z) {
    switch (act) {
        case NPA_ACT_RELU: return activate_adjoint<NPA_ACT_RELU>(dy, z);
        case NPA_ACT_GELU: return activate_adjoint<NPA_ACT_GELU>(dy, z);
        case NPA_ACT_SILU: return activate_adjoint<NPA_ACT_SILU>(dy, z);
    }
    return dy;
}

template <class T>
__device__ inline void finish(const Epilogue& e, uint64_t m, uint64_t n, float v) {
    if (e.bias) v += load_param<T>(e.bias, e.bias_f32, n);
    if (e.z) ((T*)e.z)[m * e.z_stride + n] = (T)v;
    v = activate_any(e.act, v);
    if (e.residual) v += (float)((const T*)e.residual)[m * e.residual_stride + n];
    store_param<T>(e.out, e.out_f32, e.accumulate, m * e.out_stride + n, v);
}

// A 64 x 64 tile of C a block, 4 x 4 sums a thread, operands staged through LDS 16 columns at a time.
template <class T>
__global__ __launch_bounds__(256) void k_product(Operand a, Operand b, uint32_t M, uint32_t N, uint64_t K, Epilogue e) {
    __shared__ float sa[16][65], sb[16][65];
    const uint32_t tiles = (N + 63) / 64;
    const uint64_t m0 = (uint64_t)(blockIdx.x / tiles) * 64, n0 = (uint64_t)(blockIdx.x % tiles) * 64;
    const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
    float acc[4][4] = {};
    auto stage = [&](const Operand& o, uint64_t first, uint64_t count, uint64_t k0, float (*to)[65]) {
        for (int i = threadIdx.x; i < 64 * 16; i += 256) {
            const int m = o.k_fast ? i / 16 : i % 64, k = o.k_fast ? i % 16 : i / 64;
            float v = 0.0f;
            if (first + m < count && k0 + k < K) {
                const uint64_t slow = o.k_fast ? first + m : k0 + k, fast = o.k_fast ? k0 + k : first + m;
                v = (float)((const T*)o.p)[slow * o.stride + fast];
            }
            to[k][m] = v;
        }
    };
    for (uint64_t k0 = 0; k0 < K; k0 += 16) {
        __syncthreads();
        stage(a, m0, M, k0, sa);
        stage(b, n0, N, k0, sb);
        __syncthreads();
#pragma unroll
        for (int k = 0; k < 16; ++k)
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(sa[k][ty * 4 + i], sb[k][tx + j * 16], acc[i][j]);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (m0 + ty * 4 + i < M && n0 + tx + j * 16 < N) finish<T>(e, m0 + ty * 4 + i, n0 + tx + j * 16, acc[i][j]);
}

// dz = dy act'(z), rounded to the layer's type: the operand of both products of the adjoint.
template <class T>
__global__ __launch_bounds__(256) void k_slope(const T* dy, uint64_t dy_stride, const T* z, uint64_t z_stride, T* dz,
                                               uint64_t rows, uint32_t cols, uint32_t act) {
    const uint64_t total = rows * cols, step = (uint64_t)gridDim.x * 256;
    for (uint64_t i = (uint64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += step) {
        const uint64_t r = i / cols, c = i % cols;
        dz[i] = (T)activate_adjoint_any(act, (float)dy[r * dy_stride + c], (float)z[r * z_stride + c]);
    }
}

// db, from dz before its rounding: a block sums 16 columns over all rows, 16 threads a column.
template <class T>
__global__ __launch_bounds__(256) void k_column_sums(const T* dy, uint64_t dy_stride, const T* z, uint64_t z_stride,
                                                     uint32_t act, uint64_t rows, uint32_t cols, void* db, bool f32,
                                                     bool accumulate) {
    __shared__ float shared[16][17];
    const uint32_t c = threadIdx.x % 16, q = threadIdx.x / 16, col = blockIdx.x * 16 + c;
    float s = 0.0f;
    if (col < cols)
        for (uint64_t r = q; r < rows; r += 16)
            s += activate_adjoint_any(act, (float)dy[r * dy_stride + col], z ? (float)z[r * z_stride + col] : 0.0f);
    shared[q][c] = s;
    __syncthreads();
    if (q || col >= cols) return;
    s = 0.0f;
    for (int k = 0; k < 16; ++k) s += shared[k][c];
    store_param<T>(db, f32, accumulate, col, s);
}

template <class T>
hipError_t product(const Operand& a, const Operand& b, uint32_t M, uint32_t N, uint64_t K, const Epilogue& e,
                   hipStream_t stream) {
    if (!M || !N) return hipSuccess;
    const uint64_t blocks = (uint64_t)((M + 63) / 64) * ((N + 63) / 64);
    hipLaunchKernelGGL(k_product<T>, dim3((uint32_t)blocks), dim3(256), 0, stream, a, b, M, N, K, e);
    return hipGetLastError();
}

template <class T>
hipError_t linear_of(const LinearArgs& a, LayerWorkspace& ws, int cus, hipStream_t stream) {
    Epilogue e;
    e.out = a.out;
    e.out_stride = a.out_stride;
    e.bias = a.bias;
    e.bias_f32 = a.bias_f32;
    e.residual = a.residual;
    e.residual_stride = a.residual_stride;
    e.z = a.z;
    e.z_stride = a.z_stride;
    e.act = a.activation;
    e.out_f32 = sizeof(T) == 4;
    return product<T>({a.x, a.x_stride, true}, {a.w, a.w_stride, true}, (uint32_t)a.rows, a.out_dims, a.in_dims, e,
                      stream);
}

template <class T>
hipError_t linear_adjoint_of(const LinearArgs& a, LayerWorkspace& ws, int cus, hipStream_t stream) {
    const uint32_t K = a.in_dims, N = a.out_dims;
    const T* dz = (const T*)a.dy;
    uint64_t dz_stride = a.dy_stride;
    hipError_t err = hipSuccess;
    if (a.activation != NPA_ACT_IDENTITY && a.rows) {
        if ((err = ws.dz.reserve(a.rows * N * sizeof(T))) != hipSuccess) return err;
        const uint32_t blocks = (uint32_t)std::min<uint64_t>((a.rows * N + 255) / 256, (uint64_t)cus * 16);
        hipLaunchKernelGGL(k_slope<T>, dim3(blocks), dim3(256), 0, stream, dz, dz_stride, (const T*)a.z, a.z_stride,
                           ws.dz.as<T>(), a.rows, N, a.activation);
        if ((err = hipGetLastError()) != hipSuccess) return err;
        dz = ws.dz.as<T>();
        dz_stride = N;
    }
    if (a.dx) {
        Epilogue e;
        e.out = a.dx;
        e.out_stride = a.dx_stride;
        e.out_f32 = sizeof(T) == 4;
        err = product<T>({dz, dz_stride, true}, {a.w, a.w_stride, false}, (uint32_t)a.rows, K, N, e, stream);
        if (err != hipSuccess) return err;
    }
    if (a.dw) {
        Epilogue e;
        e.out = a.dw;
        e.out_stride = K;
        e.out_f32 = a.grad_f32;
        e.accumulate = a.accumulate;
        err = product<T>({dz, dz_stride, false}, {a.x, a.x_stride, false}, N, K, a.rows, e, stream);
        if (err != hipSuccess) return err;
    }
    if (a.db) {
        hipLaunchKernelGGL(k_column_sums<T>, dim3((N + 15) / 16), dim3(256), 0, stream, (const T*)a.dy, a.dy_stride,
                           (const T*)a.z, a.z_stride, a.activation, a.rows, N, a.db, a.grad_f32, a.accumulate);
        err = hipGetLastError();
    }
    return err;
}

}  // namespace

hipError_t launch_linear(const LinearArgs& a, LayerWorkspace& ws, int cus, hipStream_t stream) {
    if (!a.rows) return hipSuccess;
    if (a.type == NPA_TYPE_F32) return linear_of<float>(a, ws, cus, stream);
    if (a.type == NPA_TYPE_BF16) return linear_of<__bf16>(a, ws, cus, stream);
    return linear_of<_Float16>(a, ws, cus, stream);
}

hipError_t launch_linear_adjoint(const LinearArgs& a, LayerWorkspace& ws, int cus, hipStream_t stream) {
    if (a.type == NPA_TYPE_F32) return linear_adjoint_of<float>(a, ws, cus, stream);
    if (a.type == NPA_TYPE_BF16) return linear_adjoint_of<__bf16>(a, ws, cus, stream);
    return linear_adjoint_of<_Float16>(a, ws, cus, stream);
}

}  // namespace npa
