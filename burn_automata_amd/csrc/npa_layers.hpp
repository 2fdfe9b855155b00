// npa_layers.hpp - the dense layers of a trained update rule: element types, activations and the
// host interfaces of npa_norm.hip and npa_linear.hip.
#pragma once

#include <new>
#include <vector>

#include "npa_internal.hpp"

namespace npa {

inline uint32_t type_bytes(uint32_t type) { return type == NPA_TYPE_F32 ? 4u : 2u; }

// N consecutive elements at any element-aligned address (gfx950's vector memory takes them unaligned).
template <class T, int N>
struct VecOf {
    typedef T type __attribute__((ext_vector_type(N), aligned(sizeof(T))));
};

// A parameter or gradient array held in f32 or in the layer's own 16-bit type.
template <class T>
__device__ inline float load_param(const void* p, bool f32, uint64_t i) {
    return f32 ? ((const float*)p)[i] : (float)((const T*)p)[i];
}
template <class T>
__device__ inline void store_param(void* p, bool f32, bool accumulate, uint64_t i, float v) {
    if (accumulate) v += load_param<T>(p, f32, i);
    if (f32)
        ((float*)p)[i] = v;
    else
        ((T*)p)[i] = (T)v;
}

// The sums of the columns of `partials` [parts][cols] in blocks of THREADS: 16 columns a block, THREADS / 16
// threads a column, four rows in flight; `put` takes each column's. Block `block` of `blocks` takes every
// blocks-th 16 columns, as a launch has to stay below 2^32 threads.
template <int THREADS, class F>
__device__ inline void column_sums(const float* partials, uint32_t parts, uint64_t cols, uint32_t block, uint32_t blocks,
                                   F put) {
    constexpr int Q = THREADS / 16;
    __shared__ float shared[Q][17];
    const uint32_t c = threadIdx.x % 16, q = threadIdx.x / 16;
    for (uint64_t first = block * 16ull; first < cols; first += blocks * 16ull) {
        const uint64_t col = first + c;
        float s[4] = {};
        if (col < cols)
            for (uint32_t p = q; p < parts; p += 4 * Q)
#pragma unroll
                for (int j = 0; j < 4; ++j) s[j] += p + j * Q < parts ? partials[(uint64_t)(p + j * Q) * cols + col] : 0.0f;
        if (first != block * 16ull) __syncthreads();
        shared[q][c] = (s[0] + s[1]) + (s[2] + s[3]);
        __syncthreads();
        if (q >= 16 || first + q >= cols) continue;
        float t = 0.0f;  // sixteen lanes a column now
#pragma unroll
        for (int k = 0; k < Q; k += 16) t += shared[c + k][q];
#pragma unroll
        for (int m = 8; m; m >>= 1) t += __shfl_xor(t, m);
        if (c == 0) put(first + q, t);
    }
}

// ------------------------------------------------------------------ layer norm (npa_norm.hip)
struct NormArgs {
    const void* x = nullptr;
    const void* gamma = nullptr;
    const void* beta = nullptr;
    void* out = nullptr;
    float* mean = nullptr;   // forward: written unless null; adjoint: read
    float* rstd = nullptr;
    const void* dy = nullptr;
    void* dx = nullptr;
    void* dgamma = nullptr;
    void* dbeta = nullptr;
    uint64_t rows = 0;
    uint64_t x_stride = 0, out_stride = 0, dy_stride = 0, dx_stride = 0;
    uint32_t width = 0;
    uint32_t type = 0;
    uint32_t param_f32 = 0;
    uint32_t accumulate = 0;
    float eps = 0.0f;
};

// Device memory of the layers' calls, kept by the context. A graph that has captured a call holds its buffers'
// addresses: a buffer that such a call used stays as it is until the context's release, also where a larger call
// takes another in its place.
struct LayerWorkspace {
    struct Buffer : DevBuf {
        bool captured = false;  // a captured call uses it
    };
    Buffer partials;  // column sums of the norm's adjoint, split products
    Buffer columns;   // column sums of dz
    Buffer dz;        // out_adjoint times the activation's slope
    DevBuf tickets;   // blocks of the norm's adjoint that have left their sums, by their number: 0 between calls
    std::vector<Buffer> outgrown;

    // For a call on `stream`. While it captures, allocations happen at once, beside the graph, and nothing is freed.
    hipError_t reserve(Buffer& b, uint64_t bytes, hipStream_t stream) {
        hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
        hipError_t e = stream ? hipStreamIsCapturing(stream, &status) : hipSuccess;  // the default stream never does
        if (e != hipSuccess) return e;
        const bool capturing = status != hipStreamCaptureStatusNone;
        if (!b.ptr || bytes > b.bytes) {
            AllocationsInCapture allowed;
            if (b.ptr && (b.captured || capturing)) {
                try {
                    outgrown.push_back(b);
                } catch (const std::bad_alloc&) {
                    return hipErrorOutOfMemory;
                }
                b = Buffer();
            }
            if ((e = b.DevBuf::reserve(bytes)) != hipSuccess) return e;
        }
        b.captured |= capturing;
        return hipSuccess;
    }
    // The tickets, cleared before any stream of the context uses them, on a stream that captures nothing.
    hipError_t reserve_tickets(size_t bytes) {
        if (tickets.ptr) return hipSuccess;
        AllocationsInCapture allowed;
        hipStream_t own = nullptr;
        hipError_t e = hipStreamCreateWithFlags(&own, hipStreamNonBlocking);
        if (e != hipSuccess) return e;
        e = tickets.reserve(bytes);
        if (e == hipSuccess) e = hipMemsetAsync(tickets.ptr, 0, bytes, own);
        if (e == hipSuccess) e = hipStreamSynchronize(own);
        if (e != hipSuccess) tickets.release();
        (void)hipStreamDestroy(own);
        return e;
    }
    void release() {
        partials.release();
        columns.release();
        dz.release();
        tickets.release();
        for (Buffer& b : outgrown) b.release();
        outgrown.clear();
    }
};

hipError_t launch_layer_norm(const NormArgs& a, int cus, hipStream_t stream);
hipError_t launch_layer_norm_adjoint(const NormArgs& a, LayerWorkspace& ws, int cus, hipStream_t stream);

// ------------------------------------------------------------------ linear layer (npa_linear.hip)
struct LinearArgs {
    const void* x = nullptr;
    const void* w = nullptr;
    const void* bias = nullptr;
    const void* residual = nullptr;
    void* out = nullptr;
    void* z = nullptr;        // forward: written unless null; adjoint: read (activations other than identity)
    const void* dy = nullptr;
    void* dx = nullptr;
    void* dw = nullptr;
    void* db = nullptr;
    uint64_t rows = 0;
    uint64_t x_stride = 0, w_stride = 0, residual_stride = 0, out_stride = 0, z_stride = 0, dy_stride = 0,
             dx_stride = 0;
    uint32_t in_dims = 0, out_dims = 0;
    uint32_t type = 0;
    uint32_t activation = 0;
    uint32_t bias_f32 = 0;   // the bias, and
    uint32_t grad_f32 = 0;   // the gradients of weights and bias, are f32 (else of `type`)
    uint32_t accumulate = 0;
};

// of each element type (an object each)
hipError_t linear_f32(const LinearArgs& a, LayerWorkspace& ws, int cus, hipStream_t stream);
hipError_t linear_bf16(const LinearArgs& a, LayerWorkspace& ws, int cus, hipStream_t stream);
hipError_t linear_f16(const LinearArgs& a, LayerWorkspace& ws, int cus, hipStream_t stream);
hipError_t linear_adjoint_f32(const LinearArgs& a, LayerWorkspace& ws, int cus, hipStream_t stream);
hipError_t linear_adjoint_bf16(const LinearArgs& a, LayerWorkspace& ws, int cus, hipStream_t stream);
hipError_t linear_adjoint_f16(const LinearArgs& a, LayerWorkspace& ws, int cus, hipStream_t stream);
hipError_t launch_linear(const LinearArgs& a, LayerWorkspace& ws, int cus, hipStream_t stream);
hipError_t launch_linear_adjoint(const LinearArgs& a, LayerWorkspace& ws, int cus, hipStream_t stream);

// ------------------------------------------------------------------ activations
// 1 / (1 + exp(-v)): silu(z) = z sigma(z), and the tanh form of gelu is z sigma(2u) with
// u = sqrt(2 / pi) (z + 0.044715 z^3), as (1 + tanh(u)) / 2 = sigma(2u).
// The hardware's exp2 and reciprocal (1 ulp each): the product by log2(e) is off by |v| 2^-24, so sigma
// is within (2 + |v|) ulp, relative; where |v| is large that is of a sigma near 0, or of its distance
// from 1. The IEEE forms cost the wide forward layer 100 us of 650.
__device__ inline float sigma(float v) {
    return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-1.4426950408889634f * v));
}

constexpr float kGelu2A = 1.5957691216057308f;  // 2 sqrt(2 / pi)
constexpr float kGeluB = 0.044715f;

template <int ACT>
__device__ inline float activate(float z) {
    if (ACT == NPA_ACT_RELU) return z < 0.0f ? 0.0f : z;  // a NaN stays one
    if (ACT == NPA_ACT_GELU) return z * sigma(kGelu2A * (z + kGeluB * z * z * z));
    if (ACT == NPA_ACT_SILU) return z * sigma(z);
    return z;
}

// dy times the activation's slope at z (relu's is 0 at a NaN). The slope's polynomial factors take z clamped to +-100, where
// the sigmoid's factor is 0 in f32, so that no 0 * inf arises at large z.
template <int ACT>
__device__ inline float activate_adjoint(float dy, float z) {
    if (ACT == NPA_ACT_RELU) return z > 0.0f ? dy : 0.0f;
    if (ACT == NPA_ACT_GELU) {
        const float c = fminf(fmaxf(z, -100.0f), 100.0f);
        const float s = sigma(kGelu2A * (z + kGeluB * z * z * z));
        return dy * (s + c * (s * (1.0f - s)) * (kGelu2A * (1.0f + 3.0f * kGeluB * c * c)));
    }
    if (ACT == NPA_ACT_SILU) {
        const float c = fminf(fmaxf(z, -100.0f), 100.0f);
        const float s = sigma(z);
        return dy * (s * (1.0f + c * (1.0f - s)));
    }
    return dy;
}

}  // namespace npa
