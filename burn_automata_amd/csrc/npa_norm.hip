// npa_norm.hip - layer norm over the rows' last axis and its adjoint.
//
// Forward: mu = mean_k x, v = mean_k (x - mu)^2, r = 1 / sqrt(v + eps), y = (x - mu) r gamma + beta.
// Adjoint, with xh = (x - mu) r and g = dy gamma: dx = r (g - mean_k g - xh mean_k(g xh)),
// dgamma = sum over rows of dy xh, dbeta = sum over rows of dy.
//
// Both are bound by memory: about 10 operations an element against 4 to 12 bytes. A group of L lanes
// holds one row in registers (at most 16 elements a lane), so each row is read once and the variance is
// the two-pass one. Sums and statistics are f32.
#include "npa_layers.hpp"

#include <algorithm>

namespace npa {
namespace {

constexpr int kPerLane = 16;             // elements of a row that one lane holds
constexpr uint32_t kRowCap = 1024 * 16;  // wider rows are read from memory again for each pass
constexpr uint64_t kMostBlocks = 1u << 20;  // of one launch; the blocks take further rows in turn

template <class T, int V>
__device__ inline void load_cols(const T* row, uint32_t col, uint32_t width, float (&o)[V]) {
    if (col + V <= width) {
        const typename VecOf<T, V>::type v = *(const typename VecOf<T, V>::type*)(row + col);
#pragma unroll
        for (int j = 0; j < V; ++j) o[j] = (float)v[j];
    } else {
#pragma unroll
        for (int j = 0; j < V; ++j) o[j] = col + j < width ? (float)row[col + j] : 0.0f;
    }
}

template <class T, int V>
__device__ inline void store_cols(T* row, uint32_t col, uint32_t width, const float (&o)[V]) {
    if (col + V <= width) {
        typename VecOf<T, V>::type v;
#pragma unroll
        for (int j = 0; j < V; ++j) v[j] = (T)o[j];
        *(typename VecOf<T, V>::type*)(row + col) = v;
    } else {
#pragma unroll
        for (int j = 0; j < V; ++j)
            if (col + j < width) row[col + j] = (T)o[j];
    }
}

template <class T, int V>
__device__ inline void load_params(const void* p, bool f32, uint32_t col, uint32_t width, float other, float (&o)[V]) {
    if (!p) {
#pragma unroll
        for (int j = 0; j < V; ++j) o[j] = other;
    } else if (f32) {
        load_cols<float, V>((const float*)p, col, width, o);
    } else {
        load_cols<T, V>((const T*)p, col, width, o);
    }
}

// Sum of two values over a group of L lanes, the same bits in each of them. Groups wider than a wave
// meet in `shared` (two floats a wave); every thread of the block calls it then.
template <int L>
__device__ inline void group_sum(float& a, float& b, float* shared) {
#pragma unroll
    for (int m = (L < 64 ? L : 64) / 2; m; m >>= 1) {
        a += __shfl_xor(a, m);
        b += __shfl_xor(b, m);
    }
    if (L > 64) {
        constexpr int W = L > 64 ? L / 64 : 1;
        const int wave = threadIdx.x / 64;
        __syncthreads();
        if ((threadIdx.x & 63) == 0) {
            shared[2 * wave] = a;
            shared[2 * wave + 1] = b;
        }
        __syncthreads();
        const int first = wave / W * W;
        a = 0.0f;
        b = 0.0f;
#pragma unroll
        for (int k = 0; k < W; ++k) {
            a += shared[2 * (first + k)];
            b += shared[2 * (first + k) + 1];
        }
    }
}

template <class T, int L, int NV>
__global__ __launch_bounds__(L < 256 ? 256 : L) void k_norm(NormArgs a) {
    constexpr int V = 16 / sizeof(T), G = (L < 256 ? 256 : L) / L;
    __shared__ float shared[32];
    const uint32_t lane = threadIdx.x % L;
    const float inv = 1.0f / (float)a.width;
    for (uint64_t base = (uint64_t)blockIdx.x * G; base < a.rows; base += (uint64_t)gridDim.x * G) {
        const uint64_t row = base + threadIdx.x / L;
        const bool live = row < a.rows;
        const T* x = (const T*)a.x + (live ? row : 0) * a.x_stride;
        float v[NV][V];
        float sum = 0.0f, none = 0.0f;
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            load_cols<T, V>(x, (lane + k * L) * V, a.width, v[k]);
#pragma unroll
            for (int j = 0; j < V; ++j) sum += v[k][j];
        }
        group_sum<L>(sum, none, shared);
        const float mean = sum * inv;
        float var = 0.0f;
#pragma unroll
        for (int k = 0; k < NV; ++k)
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const float d = v[k][j] - mean;
                var += (lane + k * L) * V + j < a.width ? d * d : 0.0f;
            }
        group_sum<L>(var, none, shared);
        const float rstd = 1.0f / sqrtf(var * inv + a.eps);
        if (!live) continue;
        if (lane == 0) {
            if (a.mean) a.mean[row] = mean;
            if (a.rstd) a.rstd[row] = rstd;
        }
        T* out = (T*)a.out + row * a.out_stride;
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const uint32_t col = (lane + k * L) * V;
            if (col >= a.width) continue;
            float g[V], b[V];
            load_params<T, V>(a.gamma, a.param_f32, col, a.width, 1.0f, g);
            load_params<T, V>(a.beta, a.param_f32, col, a.width, 0.0f, b);
#pragma unroll
            for (int j = 0; j < V; ++j) g[j] = (v[k][j] - mean) * rstd * g[j] + b[j];
            store_cols<T, V>(out, col, a.width, g);
        }
    }
}

// The adjoint: each block takes every gridDim-th group of rows and keeps its columns' sums in
// registers; `partials` [gridDim][2][width] receives them (dgamma, then dbeta).
template <class T, int L, int NV>
__global__ __launch_bounds__(L < 256 ? 256 : L) void k_norm_adjoint(NormArgs a, float* partials) {
    constexpr int V = 16 / sizeof(T), G = (L < 256 ? 256 : L) / L;
    __shared__ float shared[32];
    __shared__ float sums[G > 1 ? 256 * V : 1];
    const uint32_t lane = threadIdx.x % L, group = threadIdx.x / L;
    const float inv = 1.0f / (float)a.width;
    float dgamma[NV][V], dbeta[NV][V];
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
        for (int j = 0; j < V; ++j) dgamma[k][j] = dbeta[k][j] = 0.0f;
    for (uint64_t base = (uint64_t)blockIdx.x * G; base < a.rows; base += (uint64_t)gridDim.x * G) {
        const uint64_t row = base + group;
        const bool live = row < a.rows;
        const T* x = (const T*)a.x + (live ? row : 0) * a.x_stride;
        const T* dy = (const T*)a.dy + (live ? row : 0) * a.dy_stride;
        const float mean = a.mean[live ? row : 0], rstd = a.rstd[live ? row : 0];
        float xh[NV][V], d[NV][V];
        float s1 = 0.0f, s2 = 0.0f;
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const uint32_t col = (lane + k * L) * V;
            float g[V];
            load_cols<T, V>(x, col, a.width, xh[k]);
            load_cols<T, V>(dy, col, live ? a.width : 0u, d[k]);
            load_params<T, V>(a.gamma, a.param_f32, col, a.width, 1.0f, g);
#pragma unroll
            for (int j = 0; j < V; ++j) {
                xh[k][j] = col + j < a.width ? (xh[k][j] - mean) * rstd : 0.0f;
                if (live) {
                    dgamma[k][j] += d[k][j] * xh[k][j];
                    dbeta[k][j] += d[k][j];
                }
                d[k][j] *= g[j];
                s1 += d[k][j];
                s2 += d[k][j] * xh[k][j];
            }
        }
        group_sum<L>(s1, s2, shared);
        s1 *= inv;
        s2 *= inv;
        if (live && a.dx) {
            T* dx = (T*)a.dx + row * a.dx_stride;
#pragma unroll
            for (int k = 0; k < NV; ++k) {
                const uint32_t col = (lane + k * L) * V;
                if (col >= a.width) continue;
#pragma unroll
                for (int j = 0; j < V; ++j) d[k][j] = rstd * (d[k][j] - s1 - xh[k][j] * s2);
                store_cols<T, V>(dx, col, a.width, d[k]);
            }
        }
    }
    if (!partials) return;
    float* to = partials + (uint64_t)blockIdx.x * 2 * a.width;
#pragma unroll
    for (int which = 0; which < 2; ++which, to += a.width)
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            float s[V];
#pragma unroll
            for (int j = 0; j < V; ++j) s[j] = which ? dbeta[k][j] : dgamma[k][j];
            if (G > 1) {  // the block's groups meet in LDS
                __syncthreads();
#pragma unroll
                for (int j = 0; j < V; ++j) sums[(j * G + group) * L + lane] = s[j];
                __syncthreads();
                if (group == 0) {
#pragma unroll
                    for (int j = 0; j < V; ++j) {
                        s[j] = 0.0f;
                        for (int q = 0; q < G; ++q) s[j] += sums[(j * G + q) * L + lane];
                    }
                }
            }
            if (group == 0) store_cols<float, V>(to, (lane + k * L) * V, a.width, s);
        }
}

// dgamma and dbeta from `parts` rows of partial sums: a block sums 16 columns, 16 threads a column.
template <class T>
__global__ __launch_bounds__(256) void k_norm_params(const float* partials, uint32_t parts, NormArgs a) {
    __shared__ float shared[16][17];
    const uint32_t c = threadIdx.x % 16, q = threadIdx.x / 16;
    const uint64_t col = (uint64_t)blockIdx.x * 16 + c, cols = 2ull * a.width;
    float s = 0.0f;
    if (col < cols)
        for (uint32_t p = q; p < parts; p += 16) s += partials[p * cols + col];
    shared[q][c] = s;
    __syncthreads();
    if (q || col >= cols) return;
    s = 0.0f;
    for (int k = 0; k < 16; ++k) s += shared[k][c];
    void* to = col < a.width ? a.dgamma : a.dbeta;
    if (to) store_param<T>(to, a.param_f32, a.accumulate, col < a.width ? col : col - a.width, s);
}

// ---------------------------------------------------------------- rows wider than kRowCap
template <class T>
__global__ __launch_bounds__(1024) void k_norm_wide(NormArgs a) {
    constexpr int V = 16 / sizeof(T);
    __shared__ float shared[32];
    for (uint64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const T* x = (const T*)a.x + row * a.x_stride;
        float sum = 0.0f, none = 0.0f, v[V], g[V], b[V];
        for (uint32_t col = threadIdx.x * V; col < a.width; col += 1024 * V) {
            load_cols<T, V>(x, col, a.width, v);
#pragma unroll
            for (int j = 0; j < V; ++j) sum += v[j];
        }
        group_sum<1024>(sum, none, shared);
        const float inv = 1.0f / (float)a.width, mean = sum * inv;
        float var = 0.0f;
        for (uint32_t col = threadIdx.x * V; col < a.width; col += 1024 * V) {
            load_cols<T, V>(x, col, a.width, v);
#pragma unroll
            for (int j = 0; j < V; ++j) var += col + j < a.width ? (v[j] - mean) * (v[j] - mean) : 0.0f;
        }
        group_sum<1024>(var, none, shared);
        const float rstd = 1.0f / sqrtf(var * inv + a.eps);
        if (threadIdx.x == 0) {
            if (a.mean) a.mean[row] = mean;
            if (a.rstd) a.rstd[row] = rstd;
        }
        T* out = (T*)a.out + row * a.out_stride;
        for (uint32_t col = threadIdx.x * V; col < a.width; col += 1024 * V) {
            load_cols<T, V>(x, col, a.width, v);
            load_params<T, V>(a.gamma, a.param_f32, col, a.width, 1.0f, g);
            load_params<T, V>(a.beta, a.param_f32, col, a.width, 0.0f, b);
#pragma unroll
            for (int j = 0; j < V; ++j) v[j] = (v[j] - mean) * rstd * g[j] + b[j];
            store_cols<T, V>(out, col, a.width, v);
        }
    }
}

template <class T>
__global__ __launch_bounds__(1024) void k_norm_wide_adjoint(NormArgs a) {
    constexpr int V = 16 / sizeof(T);
    __shared__ float shared[32];
    for (uint64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const T* x = (const T*)a.x + row * a.x_stride;
        const T* dy = (const T*)a.dy + row * a.dy_stride;
        const float mean = a.mean[row], rstd = a.rstd[row], inv = 1.0f / (float)a.width;
        float s1 = 0.0f, s2 = 0.0f, v[V], d[V], g[V];
        for (uint32_t col = threadIdx.x * V; col < a.width; col += 1024 * V) {
            load_cols<T, V>(x, col, a.width, v);
            load_cols<T, V>(dy, col, a.width, d);
            load_params<T, V>(a.gamma, a.param_f32, col, a.width, 1.0f, g);
#pragma unroll
            for (int j = 0; j < V; ++j) {
                s1 += d[j] * g[j];
                s2 += d[j] * g[j] * ((v[j] - mean) * rstd);
            }
        }
        group_sum<1024>(s1, s2, shared);
        s1 *= inv;
        s2 *= inv;
        T* dx = (T*)a.dx + row * a.dx_stride;
        for (uint32_t col = threadIdx.x * V; col < a.width; col += 1024 * V) {
            load_cols<T, V>(x, col, a.width, v);
            load_cols<T, V>(dy, col, a.width, d);
            load_params<T, V>(a.gamma, a.param_f32, col, a.width, 1.0f, g);
#pragma unroll
            for (int j = 0; j < V; ++j) d[j] = rstd * (d[j] * g[j] - s1 - (v[j] - mean) * rstd * s2);
            store_cols<T, V>(dx, col, a.width, d);
        }
    }
}

// Column sums of wide rows: block (x, y) sums 256 * V columns over every gridDim.y-th row.
template <class T>
__global__ __launch_bounds__(256) void k_norm_wide_columns(NormArgs a, float* partials) {
    constexpr int V = 16 / sizeof(T);
    const uint32_t col = (blockIdx.x * 256 + threadIdx.x) * V;
    if (col >= a.width) return;
    float dgamma[V], dbeta[V], v[V], d[V];
#pragma unroll
    for (int j = 0; j < V; ++j) dgamma[j] = dbeta[j] = 0.0f;
    for (uint64_t row = blockIdx.y; row < a.rows; row += gridDim.y) {
        load_cols<T, V>((const T*)a.x + row * a.x_stride, col, a.width, v);
        load_cols<T, V>((const T*)a.dy + row * a.dy_stride, col, a.width, d);
        const float mean = a.mean[row], rstd = a.rstd[row];
#pragma unroll
        for (int j = 0; j < V; ++j) {
            dgamma[j] += d[j] * ((v[j] - mean) * rstd);
            dbeta[j] += d[j];
        }
    }
    float* to = partials + (uint64_t)blockIdx.y * 2 * a.width;
    store_cols<float, V>(to, col, a.width, dgamma);
    store_cols<float, V>(to + a.width, col, a.width, dbeta);
}

// The instantiation for a row width: the fewest lanes that hold the row at NV vectors a lane.
template <class T, class F>
hipError_t with_row_shape(uint32_t width, F f) {
    constexpr uint32_t V = 16 / sizeof(T), most = kPerLane / V;
    const uint32_t vecs = (width + V - 1) / V;
#define NPA_LANES(L)                                                             \
    if (vecs <= L * most) {                                                      \
        const uint32_t nv = (vecs + L - 1) / L;                                  \
        if (nv <= 1) return f(std::integral_constant<int, L>(), std::integral_constant<int, 1>()); \
        if (nv == 2 || most == 2) return f(std::integral_constant<int, L>(), std::integral_constant<int, 2>()); \
        if (nv == 3) return f(std::integral_constant<int, L>(), std::integral_constant<int, most == 2 ? 2 : 3>()); \
        return f(std::integral_constant<int, L>(), std::integral_constant<int, most == 2 ? 2 : 4>()); \
    }
    NPA_LANES(8)
    NPA_LANES(16)
    NPA_LANES(32)
    NPA_LANES(64)
    NPA_LANES(128)
    NPA_LANES(256)
    NPA_LANES(512)
    NPA_LANES(1024)
#undef NPA_LANES
    return hipErrorInvalidValue;
}

template <class T>
hipError_t norm_of(const NormArgs& a, hipStream_t stream) {
    if (a.width > kRowCap) {
        hipLaunchKernelGGL(k_norm_wide<T>, dim3((uint32_t)std::min<uint64_t>(a.rows, kMostBlocks)), dim3(1024), 0, stream, a);
        return hipGetLastError();
    }
    return with_row_shape<T>(a.width, [&](auto lanes, auto nv) {
        constexpr int L = decltype(lanes)::value, NV = decltype(nv)::value, threads = L < 256 ? 256 : L;
        const uint32_t blocks = (uint32_t)std::min<uint64_t>((a.rows + threads / L - 1) / (threads / L), kMostBlocks);
        hipLaunchKernelGGL((k_norm<T, L, NV>), dim3(blocks), dim3(threads), 0, stream, a);
        return hipGetLastError();
    });
}

template <class T>
hipError_t norm_adjoint_of(const NormArgs& a, LayerWorkspace& ws, int cus, hipStream_t stream) {
    constexpr uint32_t V = 16 / sizeof(T);
    const bool params = a.dgamma || a.dbeta;
    uint32_t parts = 0;
    hipError_t e = hipSuccess;
    auto reserve = [&] { return params ? ws.partials.reserve((uint64_t)parts * 2 * a.width * 4) : hipSuccess; };
    if (a.width > kRowCap) {
        if (a.dx && a.rows) {
            hipLaunchKernelGGL(k_norm_wide_adjoint<T>, dim3((uint32_t)std::min<uint64_t>(a.rows, kMostBlocks)), dim3(1024), 0, stream, a);
            if ((e = hipGetLastError()) != hipSuccess) return e;
        }
        if (!params) return hipSuccess;
        parts = (uint32_t)std::min<uint64_t>(a.rows, 64);
        if ((e = reserve()) != hipSuccess) return e;
        if (a.rows) {
            const uint32_t blocks = (a.width + 256 * V - 1) / (256 * V);
            hipLaunchKernelGGL(k_norm_wide_columns<T>, dim3(blocks, parts), dim3(256), 0, stream, a,
                               ws.partials.as<float>());
        }
        e = hipGetLastError();
    } else if (a.rows) {
        e = with_row_shape<T>(a.width, [&](auto lanes, auto nv) {
            constexpr int L = decltype(lanes)::value, NV = decltype(nv)::value, threads = L < 256 ? 256 : L;
            constexpr uint32_t G = threads / L;
            // about 2,048 threads a CU; each block leaves one row of partial sums
            const uint64_t most = (uint64_t)cus * (2048 / threads);
            parts = (uint32_t)std::min<uint64_t>((a.rows + G - 1) / G, most);
            hipError_t r = reserve();
            if (r != hipSuccess) return r;
            hipLaunchKernelGGL((k_norm_adjoint<T, L, NV>), dim3(parts), dim3(threads), 0, stream, a,
                               params ? ws.partials.as<float>() : (float*)nullptr);
            return hipGetLastError();
        });
    }
    if (e != hipSuccess || !params) return e;
    hipLaunchKernelGGL(k_norm_params<T>, dim3((uint32_t)((2ull * a.width + 15) / 16)), dim3(256), 0, stream,
                       ws.partials.as<float>(), parts, a);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_layer_norm(const NormArgs& a, int cus, hipStream_t stream) {
    if (!a.rows) return hipSuccess;
    if (a.type == NPA_TYPE_F32) return norm_of<float>(a, stream);
    if (a.type == NPA_TYPE_BF16) return norm_of<__bf16>(a, stream);
    return norm_of<_Float16>(a, stream);
}

hipError_t launch_layer_norm_adjoint(const NormArgs& a, LayerWorkspace& ws, int cus, hipStream_t stream) {
    if (a.type == NPA_TYPE_F32) return norm_adjoint_of<float>(a, ws, cus, stream);
    if (a.type == NPA_TYPE_BF16) return norm_adjoint_of<__bf16>(a, ws, cus, stream);
    return norm_adjoint_of<_Float16>(a, ws, cus, stream);
}

}  // namespace npa
