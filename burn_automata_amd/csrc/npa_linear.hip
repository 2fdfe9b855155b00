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

// Byte offset of 16-byte chunk c of row r of an operand in LDS. [row][BK]: rows of BK / 8 chunks,
// permuted so that the eight lanes of a read's phase, at eight rows, meet different banks.
// [BK][row]: a transposing read takes 32 bytes of four rows at a time; their chunks are moved apart.
template <bool FAST, int BK, int ROWS>
__device__ inline int chunk_at(int r, int c) {
    if (FAST) return BK == 64 ? r * 128 + ((c ^ (r & 7)) << 4) : r * 64 + ((c ^ ((r >> 1) & 3)) << 4);
    const int s = ROWS >= 128 ? (r & 1) * 6 ^ (r & 2) * 5 : ROWS == 64 ? (r & 3) * 2 : (r & 2);
    return r * ROWS * 2 + ((c ^ s) << 4);
}

// A lane's eight steps of row `row` + lane % 32 at step ks * 16.
template <bool FAST, int BK, int ROWS>
__device__ inline u32x4 fragment(const char* lds, int row, int ks) {
    const int lane = threadIdx.x & 63;
    if (FAST) return *(const u32x4*)(lds + chunk_at<true, BK, ROWS>(row + (lane & 31), ks * 2 + (lane >> 5)));
    // a group of 16 lanes gives the addresses of four steps of 16 rows; lane i gets row i's four steps
    const int i = lane & 15, k = ks * 16 + (lane >> 5) * 8 + (i >> 2), col = row + (lane & 16) + (i & 3) * 4;
    const char* p = lds + chunk_at<false, BK, ROWS>(k, col >> 3) + (col & 4) * 2;
    const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)p);
    const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(p + 4 * ROWS * 2));
    const u32x2 a = __builtin_bit_cast(u32x2, lo), b = __builtin_bit_cast(u32x2, hi);
    return u32x4{a[0], a[1], b[0], b[1]};
}

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
    static constexpr int LDS_TILES = PLANES * (LDS_A + LDS_B), LDS_OUT = 4 * 32 * (TN + 4) * 4;
    static constexpr int LDS = LDS_TILES > LDS_OUT ? LDS_TILES : LDS_OUT;
    static_assert(WM * WN == 4, "four waves");

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
            char* to = lds + chunk_at<FAST, BK, ROWS>(id / per, id % per);
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
                    for (int i = 0; i < MI; ++i) fa[p][i] = fragment<AF, BK, BM>(lds + p * LDS_A, wm + i * 32, ks);
#pragma unroll
                    for (int j = 0; j < NI; ++j)
                        fb[p][j] = fragment<BF, BK, BN>(lds + PLANES * LDS_A + p * LDS_B, wn + j * 32, ks);
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

// A wave's sums through LDS (a stage of 32 rows for each wave), so that a lane has eight columns of one
// row, to the epilogue or, of a split product, to memory as they are.
template <int NI>
constexpr int kOutStride = NI * 32 + 4;  // floats a row of the stage

template <class T, int MI, int NI>
__device__ inline void store_tile(const ProductArgs& g, uint64_t m, uint32_t n, float* lds, const f32x16 (&acc)[MI][NI]) {
    Epilogue part;
    if (g.splits > 1) {
        part.out = g.partials + (uint64_t)blockIdx.y * g.M * g.N;
        part.out_stride = g.N;
        part.out_f32 = true;
    }
    const Epilogue& e = g.splits > 1 ? part : g.e;
    constexpr int PER_ROW = NI * 4, ROWS = 64 / PER_ROW, STRIDE = kOutStride<NI>;
    const int lane = threadIdx.x & 63;
    float* out = lds + threadIdx.x / 64 * 32 * STRIDE;
    n += lane % PER_ROW * 8;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < MI; ++i) {
#pragma unroll
        for (int j = 0; j < NI; ++j)
#pragma unroll
            for (int q = 0; q < 16; ++q)
                out[(8 * (q / 4) + 4 * (lane >> 5) + q % 4) * STRIDE + j * 32 + (lane & 31)] = acc[i][j][q];
        __builtin_amdgcn_wave_barrier();
        for (int r = lane / PER_ROW; r < 32; r += ROWS) {
            float v[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = out[r * STRIDE + lane % PER_ROW * 8 + j];
            if (m + i * 32 + r < g.M && n < g.N) finish8<T>(e, m + i * 32 + r, n, g.N, v);
        }
        __builtin_amdgcn_wave_barrier();
    }
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

    store_tile<T, X::MI, X::NI>(g, m0 + threadIdx.x / 64 / WN * X::TM, (uint32_t)n0 + threadIdx.x / 64 % WN * X::TN,
                                (float*)lds, acc);
}

// ------------------------------------------------------------------ large aligned 16-bit products
// A tile of 256 x 256 a block, operands from memory to LDS without registers in between, two buffers:
// the next step's 64 KiB arrive while this step's are multiplied.
typedef __attribute__((address_space(3))) unsigned int lds_u32;

template <class T, int WM, int WN, bool AF, bool BF>
struct Direct {
    static constexpr int B = 256, BK = 64, WAVES = WM * WN, TM = B / WM, TN = B / WN, MI = TM / 32, NI = TN / 32;
    static constexpr int OPERAND = B * BK * 2, BUFFER = 2 * OPERAND, LOADS = OPERAND / 1024 / WAVES;
    static constexpr int LDS = 2 * BUFFER;

    // Byte offsets from the tile's first element of the 16 bytes that this lane brings with each load.
    template <bool FAST>
    static __device__ inline void offsets(uint64_t stride, uint64_t first, uint64_t count, uint32_t (&off)[LOADS]) {
        const int lane = threadIdx.x & 63, wave = threadIdx.x / 64;
#pragma unroll
        for (int i = 0; i < LOADS; ++i) {
            const int q = wave * LOADS + i;
            if (FAST) {
                int r = q * 8 + lane / 8;
                const int c = (lane & 7) ^ (r & 7);
                if (first + r >= count) r = (int)(count - 1 - first);  // not stored
                off[i] = (uint32_t)(r * stride + c * 8) * 2;
            } else {
                const int r = q * 2 + lane / 32;
                int c = (lane & 31) ^ ((r & 1) * 6 ^ (r & 2) * 5);
                if (first + c * 8 >= count) c = (int)((count - 8 - first) / 8);  // not stored
                off[i] = (uint32_t)(r * stride + c * 8) * 2;
            }
        }
    }

    // Buffer loads, not flat ones: they leave the order of LDS reads' completion known, and take a
    // scalar base. Offsets are within the tile, so the range is not used as a bound.
    static __device__ inline void load(const char* from, const uint32_t (&off)[LOADS], char* __restrict to) {
        const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
        const __amdgpu_buffer_rsrc_t base = __builtin_amdgcn_make_buffer_rsrc((void*)from, 0, 0xffffffff, 0x00020000);
#pragma unroll
        for (int i = 0; i < LOADS; ++i)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(base, (lds_u32*)(to + (wave * LOADS + i) * 1024), 16, off[i], 0, 0, 0);
    }

    struct Fragments {
        u32x4 a[MI], b[NI];
    };
    static __device__ __forceinline__ void read(const char* __restrict lds, int ks, Fragments& f) {
        const int wave = threadIdx.x / 64, wm = wave / WN * TM, wn = wave % WN * TN;
#pragma unroll
        for (int j = 0; j < NI; ++j) f.b[j] = fragment<BF, BK, B>(lds + OPERAND, wn + j * 32, ks);
#pragma unroll
        for (int i = 0; i < MI; ++i) f.a[i] = fragment<AF, BK, B>(lds, wm + i * 32, ks);
    }
    static __device__ __forceinline__ void multiply(const Fragments& f, f32x16 (&acc)[MI][NI]) {
#pragma unroll
        for (int i = 0; i < MI; ++i)
#pragma unroll
            for (int j = 0; j < NI; ++j) acc[i][j] = mma<T>(f.a[i], f.b[j], acc[i][j]);
    }
    // The order of a stretch: reads between the first products, so that neither waits for the other.
    static __device__ __forceinline__ void interleave() {
        constexpr int READS = MI * (AF ? 1 : 2) + NI * (BF ? 1 : 2);
#pragma unroll
        for (int i = 0; i < READS / 2; ++i) {
            __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);  // LDS reads
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);  // matrix products
        }
        __builtin_amdgcn_sched_group_barrier(0x008, MI * NI - READS / 2, 0);
        __builtin_amdgcn_sched_barrier(0);
    }

    // One step: each 16 columns' products run while the next fragments are read. The barrier stands
    // before the last products: by then every wave has read the last of `now`, which takes the loads
    // of the step after the next, and `next` has arrived.
    static __device__ __forceinline__ void step(const char* a, const char* b, bool more, const uint32_t (&oa)[LOADS],
                                                const uint32_t (&ob)[LOADS], char* __restrict now,
                                                const char* __restrict next, Fragments& f, f32x16 (&acc)[MI][NI]) {
        Fragments g;
        read(now, 1, g);
        multiply(f, acc);
        interleave();
        read(now, 2, f);
        multiply(g, acc);
        interleave();
        read(now, 3, g);
        multiply(f, acc);
        interleave();
        __builtin_amdgcn_s_waitcnt(0x0070);  // this wave's reads, and its loads to LDS (vmcnt 0, lgkmcnt 0)
        __builtin_amdgcn_s_barrier();
        if (more) {
            load(a, oa, now);
            load(b, ob, now + OPERAND);
        }
        read(next, 0, f);
        multiply(g, acc);
        interleave();
    }
};

template <class T, int WM, int WN, bool AF, bool BF>
__global__ __launch_bounds__(WM * WN * 64, WM * WN / 4) void k_direct(ProductArgs g) {
    using X = Direct<T, WM, WN, AF, BF>;
    extern __shared__ __align__(16) char lds[];
    uint32_t tm, tn;
    tile_of(g, tm, tn);
    const uint64_t m0 = (uint64_t)tm * X::B, n0 = (uint64_t)tn * X::B;
    const uint64_t k0 = blockIdx.y * g.split_len, k1 = g.K - k0 < g.split_len ? g.K : k0 + g.split_len;
    uint32_t oa[X::LOADS], ob[X::LOADS];
    X::template offsets<AF>(g.a.stride, m0, g.M, oa);
    X::template offsets<BF>(g.b.stride, n0, g.N, ob);
    const char* a = (const char*)g.a.p + (AF ? m0 * g.a.stride + k0 : k0 * g.a.stride + m0) * 2;
    const char* b = (const char*)g.b.p + (BF ? n0 * g.b.stride + k0 : k0 * g.b.stride + n0) * 2;
    const uint64_t da = (AF ? 1 : g.a.stride) * X::BK * 2, db = (BF ? 1 : g.b.stride) * X::BK * 2;
    f32x16 acc[X::MI][X::NI];
#pragma unroll
    for (int i = 0; i < X::MI; ++i)
#pragma unroll
        for (int j = 0; j < X::NI; ++j) acc[i][j] = f32x16{};
    int steps = (int)((k1 - k0) / X::BK), now = 0;
    X::load(a, oa, lds);
    X::load(b, ob, lds + X::OPERAND);
    if (steps > 1) {
        X::load(a + da, oa, lds + X::BUFFER);
        X::load(b + db, ob, lds + X::BUFFER + X::OPERAND);
    }
    __builtin_amdgcn_s_waitcnt(0x0070);
    __builtin_amdgcn_s_barrier();
    typename X::Fragments f;
    X::read(lds, 0, f);
    a += 2 * da;
    b += 2 * db;
    while (steps--) {
        X::step(a, b, steps > 1, oa, ob, lds + now, lds + (now ^ X::BUFFER), f, acc);
        a += da;
        b += db;
        now ^= X::BUFFER;
    }
    store_tile<T, X::MI, X::NI>(g, m0 + threadIdx.x / 64 / WN * X::TM, (uint32_t)n0 + threadIdx.x / 64 % WN * X::TN,
                                (float*)lds, acc);
}

// The splits of a product, added up: G threads for eight columns of a row, each with every G-th split.
template <class T, int G>
__global__ __launch_bounds__(256) void k_join(ProductArgs g) {
    constexpr int UNITS = 256 / G;
    __shared__ float shared[G > 1 ? 256 : 1][9];
    const uint32_t per_row = (g.N + 7) / 8, unit = threadIdx.x % UNITS, part = threadIdx.x / UNITS;
    const uint64_t units = (uint64_t)g.M * per_row, plane = (uint64_t)g.M * g.N;
    for (uint64_t base = (uint64_t)blockIdx.x * UNITS; base < units; base += (uint64_t)gridDim.x * UNITS) {
        const uint64_t u = base + unit, m = u / per_row;
        const uint32_t n = (uint32_t)(u % per_row) * 8;
        const float* p = g.partials + m * g.N + n + part * plane;
        float v[8] = {};
        if (u < units && n + 8 <= g.N) {
#pragma unroll 4
            for (uint32_t s = part; s < g.splits; s += G, p += G * plane) {
                const VecOf<float, 8>::type x = *(const VecOf<float, 8>::type*)p;
#pragma unroll
                for (int j = 0; j < 8; ++j) v[j] += x[j];
            }
        } else if (u < units) {
            for (uint32_t s = part; s < g.splits; s += G, p += G * plane)
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (n + j < g.N) v[j] += p[j];
        }
        if (G > 1) {
            __syncthreads();
#pragma unroll
            for (int j = 0; j < 8; ++j) shared[threadIdx.x][j] = v[j];
            __syncthreads();
            if (part == 0) {
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    for (int q = 1; q < G; ++q) v[j] += shared[q * UNITS + unit][j];
            }
        }
        if (part == 0 && u < units) finish8<T>(g.e, m, n, g.N, v);
    }
}

// ------------------------------------------------------------------ dz and its column sums
template <class T, int N>
__device__ inline void load_some(const T* p, int n, float (&o)[N]) {
    if (n >= N) {
        const typename VecOf<T, N>::type v = *(const typename VecOf<T, N>::type*)p;
#pragma unroll
        for (int j = 0; j < N; ++j) o[j] = (float)v[j];
    } else {
#pragma unroll
        for (int j = 0; j < N; ++j) o[j] = j < n ? (float)p[j] : 0.0f;
    }
}

struct SlopeArgs {
    const void* dy = nullptr;
    const void* z = nullptr;
    void* dz = nullptr;         // written unless null
    float* partials = nullptr;  // [gridDim.y][cols], written unless null
    uint64_t dy_stride = 0, z_stride = 0, rows = 0;
    uint32_t cols = 0;
    uint32_t lanes = 0;  // of a block across the columns, eight each; the others are further rows
};

// dz = dy act'(z), rounded to the layer's type: the operand of both products of the adjoint; and its
// column sums before that rounding. A block takes 8 * lanes columns of one of gridDim.y parts of the rows.
template <class T, int ACT>
__global__ __launch_bounds__(256) void k_slope(SlopeArgs g) {
    __shared__ float shared[256][9];
    const uint32_t lane = threadIdx.x % g.lanes, group = threadIdx.x / g.lanes, groups = 256 / g.lanes;
    const uint32_t col = (blockIdx.x * g.lanes + lane) * 8;
    const int n = col < g.cols ? (g.cols - col < 8 ? (int)(g.cols - col) : 8) : 0;
    float sum[8] = {};
    const uint64_t first = g.rows * blockIdx.y / gridDim.y, last = g.rows * (blockIdx.y + 1) / gridDim.y;
    if (n)
        for (uint64_t r = first + group; r < last; r += groups) {
            float d[8], z[8];
            load_some<T, 8>((const T*)g.dy + r * g.dy_stride + col, n, d);
            if (ACT != NPA_ACT_IDENTITY) {
                load_some<T, 8>((const T*)g.z + r * g.z_stride + col, n, z);
#pragma unroll
                for (int j = 0; j < 8; ++j) d[j] = activate_adjoint<ACT>(d[j], z[j]);
                T* to = (T*)g.dz + r * g.cols + col;
                if (g.dz && n == 8) {
                    typename VecOf<T, 8>::type v;
#pragma unroll
                    for (int j = 0; j < 8; ++j) v[j] = (T)d[j];
                    *(typename VecOf<T, 8>::type*)to = v;
                } else if (g.dz) {
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        if (j < n) to[j] = (T)d[j];
                }
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) sum[j] += j < n ? d[j] : 0.0f;
        }
    if (!g.partials) return;
#pragma unroll
    for (int j = 0; j < 8; ++j) shared[threadIdx.x][j] = sum[j];
    __syncthreads();
    for (uint32_t c = threadIdx.x; c < g.lanes * 8; c += 256) {
        const uint32_t at = blockIdx.x * g.lanes * 8 + c;
        if (at >= g.cols) continue;
        float s = 0.0f;
        for (uint32_t q = 0; q < groups; ++q) s += shared[q * g.lanes + c / 8][c % 8];
        g.partials[(uint64_t)blockIdx.y * g.cols + at] = s;
    }
}

// db from `parts` rows of partial sums.
template <class T>
__global__ __launch_bounds__(1024) void k_bias(const float* partials, uint32_t parts, uint32_t cols, void* db, bool f32,
                                               bool accumulate) {
    column_sums(partials, parts, cols, [&](uint64_t col, float s) { store_param<T>(db, f32, accumulate, col, s); });
}

template <class T>
hipError_t join(const ProductArgs& g, hipStream_t stream) {
    const uint64_t units = (uint64_t)g.M * ((g.N + 7) / 8);
    auto blocks = [&](uint64_t per) { return dim3((uint32_t)std::min<uint64_t>((units + per - 1) / per, 4096)); };
    if (g.splits >= 32)
        hipLaunchKernelGGL((k_join<T, 16>), blocks(16), dim3(256), 0, stream, g);
    else
        hipLaunchKernelGGL((k_join<T, 1>), blocks(256), dim3(256), 0, stream, g);
    return hipGetLastError();
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
    return splits > 1 ? join<T>(g, stream) : hipGetLastError();
}

// Whether the direct loads can serve an operand: whole 16-byte chunks at aligned addresses, offsets
// inside a tile below 2^32 bytes.
template <bool FAST>
bool direct_operand(const Operand& o, uint64_t count) {
    return reinterpret_cast<uintptr_t>(o.p) % 16 == 0 && o.stride % 8 == 0 && o.stride < (1u << 22) &&
           (FAST || count % 8 == 0);
}

template <class T, bool AF, bool BF>
hipError_t direct_of(ProductArgs g, LayerWorkspace& ws, int cus, hipStream_t stream) {
    constexpr int WM = 2, WN = 4;  // waves of 128 x 64: 1,127 TFLOP/s where 2 x 2 waves of 128 x 128 reached 880
    using X = Direct<T, WM, WN, AF, BF>;
    static LdsLimitFlags flags;
    hipError_t e = raise_lds_limit((const void*)k_direct<T, WM, WN, AF, BF>, flags);
    if (e != hipSuccess) return e;
    g.tiles_m = (g.M + X::B - 1) / X::B;
    g.tiles_n = (g.N + X::B - 1) / X::B;
    const uint64_t tiles = (uint64_t)g.tiles_m * g.tiles_n, steps = g.K / X::BK;
    uint64_t splits = std::max<uint64_t>(1, std::min<uint64_t>((uint64_t)cus / tiles, steps / 16));
    const uint64_t len = (steps + splits - 1) / splits;
    splits = (steps + len - 1) / len;
    g.splits = (uint32_t)splits;
    g.split_len = len * X::BK;
    if (splits > 1) {
        if ((e = ws.partials.reserve(splits * g.M * g.N * 4)) != hipSuccess) return e;
        g.partials = ws.partials.as<float>();
    }
    hipLaunchKernelGGL((k_direct<T, WM, WN, AF, BF>), dim3((uint32_t)tiles, g.splits), dim3(X::WAVES * 64), X::LDS, stream, g);
    return splits > 1 ? join<T>(g, stream) : hipGetLastError();
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
    if constexpr (sizeof(T) == 2) {
        if (M >= 256 && N >= 256 && K >= 256 && K % 64 == 0 && direct_operand<AF>(a, M) && direct_operand<BF>(b, N) &&
            (uint64_t)((M + 255) / 256) * ((N + 255) / 256) * std::max<uint64_t>(1, K / 1024) >= (uint64_t)cus / 2)
            return direct_of<T, AF, BF>(g, ws, cus, stream);
    }
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
hipError_t slope_of(const LinearArgs& a, LayerWorkspace& ws, int cus, hipStream_t stream) {
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
        if ((e = ws.dz.reserve(a.rows * g.cols * sizeof(T))) != hipSuccess) return e;
        g.dz = ws.dz.ptr;
    }
    if (a.db) {
        if ((e = ws.columns.reserve(down * g.cols * 4)) != hipSuccess) return e;
        g.partials = ws.columns.as<float>();
    }
    const dim3 grid(across, (uint32_t)down);
    switch (a.activation) {
        case NPA_ACT_IDENTITY: hipLaunchKernelGGL((k_slope<T, NPA_ACT_IDENTITY>), grid, dim3(256), 0, stream, g); break;
        case NPA_ACT_RELU: hipLaunchKernelGGL((k_slope<T, NPA_ACT_RELU>), grid, dim3(256), 0, stream, g); break;
        case NPA_ACT_GELU: hipLaunchKernelGGL((k_slope<T, NPA_ACT_GELU>), grid, dim3(256), 0, stream, g); break;
        default: hipLaunchKernelGGL((k_slope<T, NPA_ACT_SILU>), grid, dim3(256), 0, stream, g);
    }
    if (a.db)
        hipLaunchKernelGGL(k_bias<T>, dim3((g.cols + 15) / 16), dim3(1024), 0, stream, g.partials, (uint32_t)down, g.cols,
                           a.db, a.grad_f32, a.accumulate);
    return hipGetLastError();
}

template <class T>
hipError_t linear_adjoint_of(const LinearArgs& a, LayerWorkspace& ws, int cus, hipStream_t stream) {
    const uint32_t K = a.in_dims, N = a.out_dims;
    const void* dz = a.dy;
    uint64_t dz_stride = a.dy_stride;
    const bool slope = a.activation != NPA_ACT_IDENTITY && a.rows;
    hipError_t err = hipSuccess;
    if (slope || a.db) {
        if ((err = slope_of<T>(a, ws, cus, stream)) != hipSuccess) return err;
        if (slope) {
            dz = ws.dz.ptr;
            dz_stride = N;
        }
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
