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

// ------------------------------------------------------------------ matrix-core tiles
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned int u32x2 __attribute__((ext_vector_type(2)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

// One step of 16 of a 32 x 32 tile: lane l holds row (or column) l % 32 and steps 8 (l / 32) .. + 7 of
// both operands; sum i of lane l is row 8 (i / 4) + 4 (l / 32) + i % 4, column l % 32.
template <class T>
__device__ inline f32x16 mma(u32x4 a, u32x4 b, f32x16 c) {
    if (sizeof(T) == 2 && __is_same(T, _Float16))
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// Two bf16 in one word, rounded to nearest even.
__device__ inline uint32_t pack_bf16(float a, float b) {
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, bf16x2{(__bf16)a, (__bf16)b});
}

// Eight elements as they come from memory: one 16-byte load, or two for f32.
template <class T>
struct Unit {
    u32x4 v[sizeof(T) / 2];
    __device__ void clear() {
        for (auto& x : v) x = u32x4{0, 0, 0, 0};
    }
    // The first n of eight elements, zeros after them.
    __device__ void load(const T* p, int n) {
        if (n >= 8) {
            load_all(p);
            return;
        }
        typedef const __attribute__((address_space(1))) T global;
        T e[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            e[j] = (T)0.0f;
            if (j < n) e[j] = ((global*)p)[j];
        }
        __builtin_memcpy(v, e, sizeof v);
    }
    __device__ void load_all(const T* p) {
        typedef const __attribute__((address_space(1))) typename VecOf<T, 16 / sizeof(T)>::type loose;
#pragma unroll
        for (int j = 0; j < (int)sizeof(T) / 2; ++j) v[j] = __builtin_bit_cast(u32x4, ((loose*)p)[j]);
    }
};

// A product's tile of BM x BN sums a block of four waves, WM x WN of them, in steps of BK.
//
// 16-bit operands go to LDS as they are. f32 operands are split into three bf16 parts that sum to them
// (h: the upper 16 bits; m and l: the rest, rounded to nearest), and six of the nine products of parts are
// summed: h h', h m', m h', m m', h l', l h'. The three left out are below 2^-22 of the product and of
// either sign, about as much as f32's own rounding of it. That is 2.67 times the f32 matrix rate at
// most. An infinity has no such parts (inf - inf, inf * 0): sums that are not finite are computed again on
// the f32 matrix cores.
template <class T, int BM, int BN, int WM, int WN, bool AF, bool BF>
struct Tile {
    static constexpr bool F32 = sizeof(T) == 4;
    static constexpr int BK = F32 ? 32 : 64, PLANES = F32 ? 3 : 1;
    static constexpr int TM = BM / WM, TN = BN / WN, MI = TM / 32, NI = TN / 32;
    static constexpr int UA = (BM * BK / 8 + 255) / 256, UB = (BN * BK / 8 + 255) / 256;  // units a thread stages
    static constexpr int LDS_A = BM * BK * 2, LDS_B = BN * BK * 2;       // bytes a plane
    static constexpr int OUT_STRIDE = TN + 4;                            // floats a row of the epilogue's stage
    static constexpr int LDS_TILES = PLANES * (LDS_A + LDS_B), LDS_OUT = 4 * 32 * OUT_STRIDE * 4;
    static constexpr int LDS = LDS_TILES > LDS_OUT ? LDS_TILES : LDS_OUT;
    static_assert(WM * WN == 4, "four waves");

    // Byte offset of 16-byte chunk c of row r in an operand's plane. [row][BK]: rows of BK / 8 chunks,
    // permuted so that the eight lanes of a read's phase, at eight rows, meet different banks.
    // [BK][row]: a transposing read takes 32 bytes of four rows at a time; their chunks are moved apart.
    template <bool FAST, int ROWS>
    static __device__ inline int at(int r, int c) {
        if (FAST) return BK == 64 ? r * 128 + ((c ^ (r & 7)) << 4) : r * 64 + ((c ^ ((r >> 1) & 3)) << 4);
        const int s = ROWS >= 128 ? (r & 1) * 6 ^ (r & 2) * 5 : ROWS == 64 ? (r & 3) * 2 : (r & 2);
        return r * ROWS * 2 + ((c ^ s) << 4);
    }

    // The operand's units of one step, from memory.
    template <bool FAST, int ROWS, int U>
    static __device__ inline void fetch(const Operand& o, uint64_t first, uint64_t count, uint64_t k0, uint64_t K,
                                        Unit<T> (&u)[U]) {
        const bool inside = k0 + BK <= K && (FAST || first + ROWS <= count);
#pragma unroll
        for (int i = 0; i < U; ++i) {
            const int id = i * 256 + threadIdx.x;
            if (U * 256 > ROWS * BK / 8 && id >= ROWS * BK / 8) break;
            if (FAST) {
                const int c = id % (BK / 8), r = id / (BK / 8);
                const uint64_t row = first + r < count ? first + r : count - 1;  // rows past the end: not stored
                const T* p = (const T*)o.p + row * o.stride + k0 + c * 8;
                if (inside)
                    u[i].load_all(p);
                else
                    u[i].load(p, k0 + c * 8 < K ? (int)(K - k0 - c * 8 < 8 ? K - k0 - c * 8 : 8) : 0);
            } else {
                const int c = id % (ROWS / 8), r = id / (ROWS / 8);
                const uint64_t col = first + c * 8;
                const T* p = (const T*)o.p + (k0 + r) * o.stride + col;
                if (inside)
                    u[i].load_all(p);
                else
                    u[i].load(p, k0 + r < K && col < count ? (int)(count - col < 8 ? count - col : 8) : 0);
            }
        }
    }

    // Units to LDS.
    template <bool FAST, int ROWS, int U>
    static __device__ inline void stage(char* lds, const Unit<T> (&u)[U]) {
        constexpr int PLANE = ROWS * BK * 2;
#pragma unroll
        for (int i = 0; i < U; ++i) {
            const int id = i * 256 + threadIdx.x, per = FAST ? BK / 8 : ROWS / 8;
            if (U * 256 > ROWS * BK / 8 && id >= ROWS * BK / 8) break;
            char* to = lds + at<FAST, ROWS>(id / per, id % per);
            if constexpr (!F32) {
                *(u32x4*)to = u[i].v[0];
            } else {
                u32x4 h, m, l;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const uint32_t w0 = u[i].v[j / 2][j % 2 * 2], w1 = u[i].v[j / 2][j % 2 * 2 + 1];
                    const uint32_t t0 = w0 & 0xffff0000u, t1 = w1 & 0xffff0000u;
                    const float x0 = __uint_as_float(w0), x1 = __uint_as_float(w1);
                    const float r0 = x0 - __uint_as_float(t0), r1 = x1 - __uint_as_float(t1);
                    h[j] = (t0 >> 16) | t1;
                    const uint32_t mm = pack_bf16(r0, r1);
                    m[j] = mm;
                    l[j] = pack_bf16(r0 - __uint_as_float(mm << 16), r1 - __uint_as_float(mm & 0xffff0000u));
                }
                *(u32x4*)to = h;
                *(u32x4*)(to + PLANE) = m;
                *(u32x4*)(to + 2 * PLANE) = l;
            }
        }
    }

    // A lane's eight steps of row `row` + lane % 32 at step ks * 16.
    template <bool FAST, int ROWS>
    static __device__ inline u32x4 fragment(const char* lds, int row, int ks) {
        const int lane = threadIdx.x & 63;
        if (FAST) return *(const u32x4*)(lds + at<true, ROWS>(row + (lane & 31), ks * 2 + (lane >> 5)));
        const int i = lane & 15, k = ks * 16 + (lane >> 5) * 8 + (i >> 2), col = row + (lane & 16) + (i & 3) * 4;
        const char* p = lds + at<false, ROWS>(k, col >> 3) + (col & 4) * 2;
        const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)p);
        const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(p + 4 * ROWS * 2));
        const u32x2 a = __builtin_bit_cast(u32x2, lo), b = __builtin_bit_cast(u32x2, hi);
        return u32x4{a[0], a[1], b[0], b[1]};
    }

    static __device__ void sum(const Operand& a, const Operand& b, uint64_t m0, uint64_t n0, uint64_t M, uint64_t N,
                               uint64_t k0, uint64_t k1, char* lds, f32x16 (&acc)[MI][NI]) {
        const int wave = threadIdx.x / 64, wm = wave / WN * TM, wn = wave % WN * TN;
        Unit<T> ua[UA], ub[UB];
        fetch<AF, BM>(a, m0, M, k0, k1, ua);
        fetch<BF, BN>(b, n0, N, k0, k1, ub);
        for (uint64_t k = k0; k < k1; k += BK) {
            __syncthreads();
            stage<AF, BM>(lds, ua);
            stage<BF, BN>(lds + PLANES * LDS_A, ub);
            __syncthreads();
            if (k + BK < k1) {
                fetch<AF, BM>(a, m0, M, k + BK, k1, ua);
                fetch<BF, BN>(b, n0, N, k + BK, k1, ub);
            }
            const int steps = k1 - k >= BK ? BK / 16 : (int)((k1 - k + 15) / 16);
#pragma unroll
            for (int ks = 0; ks < BK / 16; ++ks) {
                if (ks >= steps) continue;
                u32x4 fa[PLANES][MI], fb[PLANES][NI];
#pragma unroll
                for (int p = 0; p < PLANES; ++p) {
#pragma unroll
                    for (int i = 0; i < MI; ++i) fa[p][i] = fragment<AF, BM>(lds + p * LDS_A, wm + i * 32, ks);
#pragma unroll
                    for (int j = 0; j < NI; ++j)
                        fb[p][j] = fragment<BF, BN>(lds + PLANES * LDS_A + p * LDS_B, wn + j * 32, ks);
                }
#pragma unroll
                for (int i = 0; i < MI; ++i)
#pragma unroll
                    for (int j = 0; j < NI; ++j) {
                        if constexpr (F32) {
                            acc[i][j] = mma<T>(fa[2][i], fb[0][j], acc[i][j]);
                            acc[i][j] = mma<T>(fa[0][i], fb[2][j], acc[i][j]);
                            acc[i][j] = mma<T>(fa[1][i], fb[1][j], acc[i][j]);
                            acc[i][j] = mma<T>(fa[1][i], fb[0][j], acc[i][j]);
                            acc[i][j] = mma<T>(fa[0][i], fb[1][j], acc[i][j]);
                        }
                        acc[i][j] = mma<T>(fa[0][i], fb[0][j], acc[i][j]);
                    }
            }
        }
        if constexpr (F32) {
#pragma unroll
            for (int i = 0; i < MI; ++i)
#pragma unroll
                for (int j = 0; j < NI; ++j) mend(a, b, m0 + wm + i * 32, n0 + wn + j * 32, M, N, k0, k1, acc[i][j]);
        }
    }

    // Sums that are not finite, again on the f32 matrix cores, straight from memory: f32's own result
    // where an operand is an infinity or a NaN, or where the sum overflows.
    static __device__ inline void mend(const Operand& a, const Operand& b, uint64_t m, uint64_t n, uint64_t M, uint64_t N,
                                       uint64_t k0, uint64_t k1, f32x16& acc) {
        float odd = 0.0f;
#pragma unroll
        for (int q = 0; q < 16; ++q) odd = fmaf(acc[q], 0.0f, odd);
        if (!__any(odd != 0.0f)) return;
        const int lane = threadIdx.x & 63;
        m = m + (lane & 31) < M ? m + (lane & 31) : M - 1;
        n = n + (lane & 31) < N ? n + (lane & 31) : N - 1;
        const float* pa = (const float*)a.p + (AF ? m * a.stride : m);
        const float* pb = (const float*)b.p + (BF ? n * b.stride : n);
        f32x16 again = {};
        for (uint64_t k = k0 + (lane >> 5); k < k1 + (lane >> 5); k += 2) {
            const float x = k < k1 ? pa[AF ? k : k * a.stride] : 0.0f, y = k < k1 ? pb[BF ? k : k * b.stride] : 0.0f;
            again = __builtin_amdgcn_mfma_f32_32x32x2f32(x, y, again, 0, 0, 0);
        }
#pragma unroll
        for (int q = 0; q < 16; ++q) acc[q] = acc[q] - acc[q] == 0.0f ? acc[q] : again[q];
    }
};

// Eight sums of one row, columns n .. n + 7 (fewer at the matrix's edge).
template <class T>
__device__ inline void finish8(const Epilogue& e, uint64_t m, uint32_t n, uint32_t N, float (&v)[8]) {
    typedef typename VecOf<T, 8>::type vec;
    typedef VecOf<float, 8>::type vec32;
    const int count = N - n < 8 ? (int)(N - n) : 8;
    if (count < 8 || e.accumulate) {
        for (int j = 0; j < 8; ++j)
            if (j < count) finish<T>(e, m, n + j, v[j]);
        return;
    }
    if (e.bias) {
        if (e.bias_f32) {
            const vec32 b = *(const vec32*)((const float*)e.bias + n);
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] += b[j];
        } else {
            const vec b = *(const vec*)((const T*)e.bias + n);
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] += (float)b[j];
        }
    }
    if (e.z) {
        vec z;
#pragma unroll
        for (int j = 0; j < 8; ++j) z[j] = (T)v[j];
        *(vec*)((T*)e.z + m * e.z_stride + n) = z;
    }
    if (e.act != NPA_ACT_IDENTITY) {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = activate_any(e.act, v[j]);
    }
    if (e.residual) {
        const vec r = *(const vec*)((const T*)e.residual + m * e.residual_stride + n);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] += (float)r[j];
    }
    if (e.out_f32) {
        vec32 o;
#pragma unroll
        for (int j = 0; j < 8; ++j) o[j] = v[j];
        *(vec32*)((float*)e.out + m * e.out_stride + n) = o;
    } else {
        vec o;
#pragma unroll
        for (int j = 0; j < 8; ++j) o[j] = (T)v[j];
        *(vec*)((T*)e.out + m * e.out_stride + n) = o;
    }
}

struct ProductArgs {
    Operand a, b;
    Epilogue e;
    uint32_t M = 0, N = 0;
    uint64_t K = 0;
    uint32_t splits = 1;       // of K
    uint64_t split_len = 0;    // steps a split, a multiple of the tile's
    float* partials = nullptr; // [splits][M][N]
    uint32_t tiles_m = 0, tiles_n = 0;
};

// Tiles are taken so that the blocks of one XCD (block index modulo 8) share operands in its L2: each XCD
// has a run of tiles, in strips of 8 tile rows.
__device__ inline void tile_of(const ProductArgs& g, uint32_t& tm, uint32_t& tn) {
    const uint32_t tiles = g.tiles_m * g.tiles_n, id = blockIdx.x, per = tiles / 8, whole = per * 8;
    const uint32_t t = id < whole ? id % 8 * per + id / 8 : id;
    const uint32_t strip = t / (8 * g.tiles_n), in = t % (8 * g.tiles_n);
    const uint32_t height = g.tiles_m - strip * 8 < 8 ? g.tiles_m - strip * 8 : 8;
    tm = strip * 8 + in % height;
    tn = in / height;
}

template <class T, int BM, int BN, int WM, int WN, bool AF, bool BF>
__global__ __launch_bounds__(256, 2) void k_tiles(ProductArgs g) {
    using X = Tile<T, BM, BN, WM, WN, AF, BF>;
    __shared__ __align__(16) char lds[X::LDS];
    uint32_t tm, tn;
    tile_of(g, tm, tn);
    const uint64_t m0 = (uint64_t)tm * BM, n0 = (uint64_t)tn * BN;
    const uint64_t k0 = blockIdx.y * g.split_len, k1 = g.K - k0 < g.split_len ? g.K : k0 + g.split_len;
    f32x16 acc[X::MI][X::NI];
#pragma unroll
    for (int i = 0; i < X::MI; ++i)
#pragma unroll
        for (int j = 0; j < X::NI; ++j) acc[i][j] = f32x16{};
    X::sum(g.a, g.b, m0, n0, g.M, g.N, k0, k1, lds, acc);

    Epilogue part;  // a split's sums go to memory as they are
    if (g.splits > 1) {
        part.out = g.partials + (uint64_t)blockIdx.y * g.M * g.N;
        part.out_stride = g.N;
        part.out_f32 = true;
    }
    const Epilogue& e = g.splits > 1 ? part : g.e;
    // through LDS, 32 rows of a wave at a time, so that a lane has eight columns of one row
    const int wave = threadIdx.x / 64, lane = threadIdx.x & 63;
    float* out = (float*)lds + wave * 32 * X::OUT_STRIDE;
    constexpr int PER_ROW = X::TN / 8, ROWS = 64 / PER_ROW;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < X::MI; ++i) {
#pragma unroll
        for (int j = 0; j < X::NI; ++j)
#pragma unroll
            for (int q = 0; q < 16; ++q)
                out[(8 * (q / 4) + 4 * (lane >> 5) + q % 4) * X::OUT_STRIDE + j * 32 + (lane & 31)] = acc[i][j][q];
        __builtin_amdgcn_wave_barrier();
        const uint64_t m = m0 + wave / WN * X::TM + i * 32;
        const uint32_t n = (uint32_t)n0 + wave % WN * X::TN + lane % PER_ROW * 8;
#pragma unroll
        for (int s = 0; s < 32 / ROWS; ++s) {
            const int r = s * ROWS + lane / PER_ROW;
            float v[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = out[r * X::OUT_STRIDE + lane % PER_ROW * 8 + j];
            if (m + r < g.M && n < g.N) finish8<T>(e, m + r, n, g.N, v);
        }
        __builtin_amdgcn_wave_barrier();
    }
}

// The splits of a product, added in order.
template <class T>
__global__ __launch_bounds__(256) void k_join(ProductArgs g) {
    const uint32_t per_row = (g.N + 7) / 8;
    const uint64_t units = (uint64_t)g.M * per_row, plane = (uint64_t)g.M * g.N;
    for (uint64_t u = (uint64_t)blockIdx.x * 256 + threadIdx.x; u < units; u += (uint64_t)gridDim.x * 256) {
        const uint64_t m = u / per_row;
        const uint32_t n = (uint32_t)(u % per_row) * 8;
        const float* p = g.partials + m * g.N + n;
        float v[8] = {};
        if (n + 8 <= g.N) {
            for (uint32_t s = 0; s < g.splits; ++s, p += plane) {
                const VecOf<float, 8>::type x = *(const VecOf<float, 8>::type*)p;
#pragma unroll
                for (int j = 0; j < 8; ++j) v[j] += x[j];
            }
        } else {
            for (uint32_t s = 0; s < g.splits; ++s, p += plane)
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (n + j < g.N) v[j] += p[j];
        }
        finish8<T>(g.e, m, n, g.N, v);
    }
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

template <class T, int BM, int BN, int WM, int WN, bool AF, bool BF>
hipError_t tiles_of(ProductArgs g, LayerWorkspace& ws, int cus, hipStream_t stream) {
    using X = Tile<T, BM, BN, WM, WN, AF, BF>;
    g.tiles_m = (g.M + BM - 1) / BM;
    g.tiles_n = (g.N + BN - 1) / BN;
    const uint64_t tiles = (uint64_t)g.tiles_m * g.tiles_n, steps = (g.K + X::BK - 1) / X::BK;
    // few tiles and a long sum: split it, at least eight steps a part, to two blocks a CU
    uint64_t splits = std::max<uint64_t>(1, std::min<uint64_t>(2ull * cus / tiles, steps / 8));
    splits = std::min<uint64_t>(splits, 512);
    const uint64_t len = (steps + splits - 1) / splits;
    splits = steps ? (steps + len - 1) / len : 1;
    g.splits = (uint32_t)splits;
    g.split_len = len * X::BK;
    if (splits > 1) {
        hipError_t e = ws.partials.reserve(splits * g.M * g.N * 4);
        if (e != hipSuccess) return e;
        g.partials = ws.partials.as<float>();
    }
    hipLaunchKernelGGL((k_tiles<T, BM, BN, WM, WN, AF, BF>), dim3((uint32_t)tiles, g.splits), dim3(256), 0, stream, g);
    if (splits > 1) {
        const uint64_t units = (uint64_t)g.M * ((g.N + 7) / 8);
        hipLaunchKernelGGL(k_join<T>, dim3((uint32_t)std::min<uint64_t>((units + 255) / 256, 4096)), dim3(256), 0, stream, g);
    }
    return hipGetLastError();
}

template <class T, bool AF, bool BF>
hipError_t product(const Operand& a, const Operand& b, uint32_t M, uint32_t N, uint64_t K, const Epilogue& e,
                   LayerWorkspace& ws, int cus, hipStream_t stream) {
    if (!M || !N) return hipSuccess;
    ProductArgs g;
    g.a = a;
    g.b = b;
    g.e = e;
    g.M = M;
    g.N = N;
    g.K = K;
    if (N <= 32) return tiles_of<T, 128, 32, 4, 1, AF, BF>(g, ws, cus, stream);
    if (M <= 32) return tiles_of<T, 32, 128, 1, 4, AF, BF>(g, ws, cus, stream);
    const uint64_t big = (uint64_t)((M + 127) / 128) * ((N + 127) / 128);
    if (big * 2 < (uint64_t)cus && K < 4096) return tiles_of<T, 64, 64, 2, 2, AF, BF>(g, ws, cus, stream);
    return tiles_of<T, 128, 128, 2, 2, AF, BF>(g, ws, cus, stream);
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
    return product<T, true, true>({a.x, a.x_stride}, {a.w, a.w_stride}, (uint32_t)a.rows, a.out_dims, a.in_dims, e, ws,
                                  cus, stream);
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
        err = product<T, true, false>({dz, dz_stride}, {a.w, a.w_stride}, (uint32_t)a.rows, K, N, e, ws, cus, stream);
        if (err != hipSuccess) return err;
    }
    if (a.dw) {
        Epilogue e;
        e.out = a.dw;
        e.out_stride = K;
        e.out_f32 = a.grad_f32;
        e.accumulate = a.accumulate;
        err = product<T, false, false>({dz, dz_stride}, {a.x, a.x_stride}, N, K, a.rows, e, ws, cus, stream);
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
