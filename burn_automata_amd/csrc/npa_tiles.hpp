// npa_tiles.hpp - matrix-core tiles of the products C[m][n] = sum_k A(m, k) B(n, k), operands of which either index
// runs through memory: their staging, epilogues, split sums, and the model by which calls choose tiles and splits.
// npa_linear.hip and npa_experts.hip build their kernels of them.
#pragma once

#include <algorithm>
#include <cmath>
#include <type_traits>

#include "npa_layers.hpp"

namespace npa {
namespace {

struct Operand {
    const void* p = nullptr;
    uint64_t stride = 0;        // of the slow index
    uint64_t slow = 0;          // how many of it there are
    const void* z = nullptr;    // the operand is p act'(z), evaluated as it is staged
    uint64_t z_stride = 0;
    uint32_t act = NPA_ACT_IDENTITY;
    // gathered: row i of the operand is row order[i] / per of p
    const uint32_t* order = nullptr;
    uint32_t per = 1;
    __device__ inline uint64_t gathered(uint64_t i) const {
        const uint64_t r = order[i] / per;
        return r < slow ? r : slow - 1;
    }
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

__device__ inline float activate_adjoint_any(uint32_t act, float dy, float z) {
    switch (act) {
        case NPA_ACT_RELU: return activate_adjoint<NPA_ACT_RELU>(dy, z);
        case NPA_ACT_GELU: return activate_adjoint<NPA_ACT_GELU>(dy, z);
        case NPA_ACT_SILU: return activate_adjoint<NPA_ACT_SILU>(dy, z);
    }
    return dy;
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
    // The first n of eight elements, what follows them unset until keep(n): the loads stay under way.
    // `over`: the memory past the elements is the caller's, too.
    __device__ inline void load(const T* p, int n, bool over) {
#pragma unroll
        for (int j = 0; j < (int)sizeof(T) / 2; ++j) v[j] = u32x4{0, 0, 0, 0};
        const bool whole = n >= 8 || (over && n > 0);
        if (!whole && n > 0) {  // one by one, all under way at once: elements past the n-th are the n-th
            typedef const __attribute__((address_space(1))) T global;
            float e[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) e[j] = (float)((global*)p)[j < n ? j : n - 1];
            set(e);
        }
        if (whole) load_all(p);
    }
    // Zeros after the first n.
    __device__ inline void keep(int n) {
        if (sizeof(T) == 2) {
#pragma unroll
            for (int j = 0; j < 4; ++j) v[0][j] &= n >= 2 * j + 2 ? 0xffffffffu : n == 2 * j + 1 ? 0xffffu : 0u;
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j / 4 % (sizeof(T) / 2)][j % 4] = j < n ? v[j / 4 % (sizeof(T) / 2)][j % 4] : 0u;
        }
    }
    __device__ inline void load_all(const T* p) {
        typedef const __attribute__((address_space(1))) typename VecOf<T, 16 / sizeof(T)>::type loose;
#pragma unroll
        for (int j = 0; j < (int)sizeof(T) / 2; ++j) v[j] = __builtin_bit_cast(u32x4, ((loose*)p)[j]);
    }
    __device__ inline void get(float (&o)[8]) const {
        T e[8];
        __builtin_memcpy(e, v, sizeof v);
#pragma unroll
        for (int j = 0; j < 8; ++j) o[j] = (float)e[j];
    }
    __device__ inline void set(const float (&o)[8]) {
        T e[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) e[j] = (T)o[j];
        __builtin_memcpy(v, e, sizeof v);
    }
};

// Eight f32 elements as three bf16 parts that sum to them: the upper 16 bits, and what is left of them, rounded twice.
// The lower half of `lost` stays 0 while they do.
__device__ inline void split_parts(const Unit<float>& u, u32x4 (&part)[3], uint32_t& lost) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const uint32_t w0 = u.v[j / 2][j % 2 * 2], w1 = u.v[j / 2][j % 2 * 2 + 1];
        const uint32_t t0 = w0 & 0xffff0000u, t1 = w1 & 0xffff0000u;
        const float x0 = __uint_as_float(w0), x1 = __uint_as_float(w1);
        const float r0 = x0 - __uint_as_float(t0), r1 = x1 - __uint_as_float(t1);
        part[0][j] = (t0 >> 16) | t1;
        const uint32_t mm = pack_bf16(r0, r1);
        part[1][j] = mm;
        const float d0 = r0 - __uint_as_float(mm << 16), d1 = r1 - __uint_as_float(mm & 0xffff0000u);
        part[2][j] = pack_bf16(d0, d1);
        lost |= __float_as_uint(d0) | __float_as_uint(d1);  // bits that the last part has no room for
    }
}

// Byte offset of 16-byte chunk c of row r of an operand in LDS. [row][BK]: rows of BK / 8 chunks,
// permuted so that sixteen lanes of a read, at sixteen rows, meet different ones of the 64 banks.
// [BK][row]: a transposing read takes 32 bytes of four rows at a time; their chunks are moved apart.
template <bool FAST, int BK, int ROWS>
__device__ inline int chunk_at(int r, int c) {
    if (FAST) return BK == 64 ? r * 128 + ((c ^ ((r >> 1) & 7)) << 4) : r * 64 + ((c ^ ((r >> 2) & 3)) << 4);
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
// the f32 matrix cores. So are sums that operands below 2^-110 could matter to, whose l, and in the end m and h, have
// bits below bf16's smallest subnormal number (the matrix cores keep subnormal ones, of operands and sums): a tile that
// meets such operands reads its own again for the size that its sums have to have. 8,192, 1,024 -> 1,024: 100 us,
// 148 with a value of 1e-36 in each tile, 1,012 with only such values of x; the test costs ordinary tiles up to 7 %.
//
// DEPTH steps' units are on their way in registers, as a step that waits for memory takes 1 to 3 us. GATHER: an operand's
// slow index is gathered: A's, whose rows are the same in all steps, or, where A's slow index is k, B's, whose rows' numbers
// are loaded a step ahead of their use.
template <class T, int BM, int BN, int WM, int WN, int DEPTH, bool AF, bool BF, bool SLOPE, bool GATHER = false>
struct Tile {
    static constexpr bool F32 = sizeof(T) == 4;
    static constexpr int BK = F32 ? 32 : 64, PLANES = F32 ? 3 : 1;
    static constexpr int TM = BM / WM, TN = BN / WN, MI = TM / 32, NI = TN / 32;
    static constexpr int UA = (BM * BK / 8 + 255) / 256, UB = (BN * BK / 8 + 255) / 256;  // units a thread stages
    static constexpr int LDS_A = BM * BK * 2, LDS_B = BN * BK * 2;       // bytes a plane
    static constexpr int LDS_TILES = PLANES * (LDS_A + LDS_B), LDS_OUT = 4 * 32 * (TN + 4) * 4;
    static constexpr int LDS_FLAGS = LDS_TILES > LDS_OUT ? LDS_TILES : LDS_OUT;  // of f32: a word a wave
    static constexpr int LDS = LDS_FLAGS + (F32 ? 16 : 0);
    static_assert(WM * WN == 4, "four waves");
    static constexpr bool GATHER_A = GATHER && AF, GATHER_B = GATHER && !AF;
    static_assert(!GATHER_A || !SLOPE, "a gathered A has no slope");
    static_assert(!GATHER_B || !BF, "a gathered B's rows are steps");

    // How many of unit `id`'s eight elements the operand has.
    template <bool FAST, int ROWS>
    static __device__ inline int valid(int id, uint64_t first, uint64_t count, uint64_t k0, uint64_t K) {
        const uint64_t slow = FAST ? 0 : k0 + id / (ROWS / 8);
        const uint64_t at = FAST ? k0 + id % (BK / 8) * 8 : first + id % (ROWS / 8) * 8, end = FAST ? K : count;
        if ((!FAST && slow >= K) || at >= end) return 0;
        return end - at < 8 ? (int)(end - at) : 8;
    }
    // Whether a step's units can be loaded whole and used as they are. Rows past the end are not stored and may
    // hold anything; a unit that ends past its row's end reads on into the next row, which all but the last have.
    // Of gathered steps the next row may be any, so a unit that ends past its row's end is checked by itself.
    template <bool FAST, int ROWS, bool GATHERED>
    static __device__ inline bool inside(uint64_t slow, uint64_t first, uint64_t count, uint64_t k0, uint64_t K) {
        return k0 + BK <= K && (FAST || first + ROWS <= count || (!GATHERED && count >= 7 && k0 + BK < slow));
    }

    // The rows of a thread's units of the A operand.
    struct Rows {
        uint64_t at[GATHER_A ? UA : 1];
        __device__ inline Rows(const Operand& a, uint64_t m0, uint64_t M) {
            if constexpr (GATHER_A) {
#pragma unroll
                for (int i = 0; i < UA; ++i) {
                    const uint64_t row = m0 + (i * 256 + threadIdx.x) / (BK / 8);
                    at[i] = a.gathered(row < M ? row : M - 1);  // rows past the end: not stored
                }
            }
        }
        __device__ inline uint64_t operator()(int i, uint64_t row) const { return GATHER_A ? at[GATHER_A ? i : 0] : row; }
    };
    // The rows of a thread's units of the B operand in one step.
    struct Steps {
        uint32_t entry[GATHER_B ? UB : 1], per;
        __device__ inline void load(const Operand& b, uint64_t k, uint64_t K) {
            if constexpr (GATHER_B) {
                per = b.per;
#pragma unroll
                for (int i = 0; i < UB; ++i) {
                    const uint64_t row = k + (i * 256 + threadIdx.x) / (BN / 8);
                    entry[i] = b.order[row < K ? row : K - 1];
                }
            }
        }
        __device__ inline uint64_t operator()(int i, uint64_t row) const { return GATHER_B ? entry[GATHER_B ? i : 0] / per : row; }
    };
    // The operand's units of one step, from memory.
    template <bool FAST, int ROWS, bool GATHERED = false, int U, class At>
    static __device__ inline void fetch(const void* base, uint64_t stride, uint64_t slow, uint64_t first, uint64_t count,
                                        uint64_t k0, uint64_t K, uint64_t all_k, Unit<T> (&u)[U], const At& at) {
        const bool whole = inside<FAST, ROWS, GATHERED>(slow, first, count, k0, K);
        const bool wide = (FAST ? all_k : count) >= 7;
#pragma unroll
        for (int i = 0; i < U; ++i) {
            const int id = i * 256 + threadIdx.x;
            if (U * 256 > ROWS * BK / 8 && id >= ROWS * BK / 8) break;
            uint64_t row, col;
            if (FAST) {
                row = first + id / (BK / 8);
                row = at(i, row < count ? row : count - 1);  // rows past the end: not stored
                col = k0 + id % (BK / 8) * 8;
            } else {
                row = k0 + id / (ROWS / 8);
                if (GATHERED) row = at(i, row) < slow ? at(i, row) : slow - 1;
                col = first + id % (ROWS / 8) * 8;
                col = col < count ? col : count < 8 ? 0 : count - 8;
            }
            const T* p = (const T*)base + row * stride + col;
            if (whole)
                u[i].load_all(p);
            else
                u[i].load(p, valid<FAST, ROWS>(id, first, count, k0, K), wide && row + 1 < slow);
        }
    }
    template <bool FAST, int ROWS, bool GATHERED = false, int U>
    static __device__ inline void settle(uint64_t slow, uint64_t first, uint64_t count, uint64_t k0, uint64_t K,
                                         Unit<T> (&u)[U]) {
        if (!inside<FAST, ROWS, GATHERED>(slow, first, count, k0, K)) cut<FAST, ROWS>(first, count, k0, K, u);
    }
    template <bool FAST, int ROWS, int U>
    static __device__ inline void cut(uint64_t first, uint64_t count, uint64_t k0, uint64_t K, Unit<T> (&u)[U]) {
#pragma unroll
        for (int i = 0; i < U; ++i) u[i].keep(valid<FAST, ROWS>(i * 256 + threadIdx.x, first, count, k0, K));
    }

    // Units to LDS. The lower half of `lost` stays 0 while the elements are the sums of their parts.
    template <bool FAST, int ROWS, int U>
    static __device__ inline void stage(char* lds, const Unit<T> (&u)[U], uint32_t& lost) {
        constexpr int PLANE = ROWS * BK * 2;
#pragma unroll
        for (int i = 0; i < U; ++i) {
            const int id = i * 256 + threadIdx.x, per = FAST ? BK / 8 : ROWS / 8;
            if (U * 256 > ROWS * BK / 8 && id >= ROWS * BK / 8) break;
            char* to = lds + chunk_at<FAST, BK, ROWS>(id / per, id % per);
            if constexpr (!F32) {
                *(u32x4*)to = u[i].v[0];
            } else {
                u32x4 part[3];
                split_parts(u[i], part, lost);
#pragma unroll
                for (int p = 0; p < 3; ++p) *(u32x4*)(to + p * PLANE) = part[p];
            }
        }
    }

    // The A operand's units times the slope, and their sums over the steps (of [k][m] units, whose eight
    // columns are the same in every step), before the units' rounding.
    static __device__ inline void slope(const Operand& a, bool sums, Unit<T> (&u)[UA], const Unit<T> (&z)[SLOPE ? UA : 1],
                                        float (&columns)[8]) {
        if (!SLOPE && !sums) return;
#pragma unroll
        for (int i = 0; i < UA; ++i) {
            if (UA * 256 > BM * BK / 8 && i * 256 + threadIdx.x >= BM * BK / 8) break;
            float d[8], s[8];
            u[i].get(d);
            if constexpr (SLOPE) {
                z[i].get(s);
                auto each = [&](auto act) {
#pragma unroll
                    for (int j = 0; j < 8; ++j) d[j] = activate_adjoint<decltype(act)::value>(d[j], s[j]);
                };
                switch (a.act) {
                    case NPA_ACT_RELU: each(std::integral_constant<int, NPA_ACT_RELU>()); break;
                    case NPA_ACT_GELU: each(std::integral_constant<int, NPA_ACT_GELU>()); break;
                    case NPA_ACT_SILU: each(std::integral_constant<int, NPA_ACT_SILU>());
                }
                u[i].set(d);
            }
            if (sums) {
#pragma unroll
                for (int j = 0; j < 8; ++j) columns[j] += d[j];
            }
        }
    }

    static __device__ inline void multiply(const char* lds, int steps, f32x16 (&acc)[MI][NI]) {
        const int wave = threadIdx.x / 64, wm = wave / WN * TM, wn = wave % WN * TN;
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

    // The tile's sums over steps k0 .. k1 - 1 of K; with `sums`, the A operand's over the same steps.
    static __device__ inline void sum(const Operand& a, const Operand& b, uint64_t m0, uint64_t n0, uint64_t M, uint64_t N,
                                      uint64_t k0, uint64_t k1, uint64_t K, bool sums, char* lds, f32x16 (&acc)[MI][NI],
                                      float (&columns)[8]) {
        Unit<T> ua[DEPTH][UA], ub[DEPTH][UB], uz[SLOPE ? DEPTH : 1][SLOPE ? UA : 1];
        uint32_t lost = 0;
        const Rows rows(a, m0, M);
        Steps ahead;
        if (k0 < k1) ahead.load(b, k0, k1);
        auto get = [&](uint64_t k, int s) {
            const Steps now = ahead;
            if (k + BK < k1) ahead.load(b, k + BK, k1);
            fetch<AF, BM>(a.p, a.stride, a.slow, m0, M, k, k1, K, ua[s], rows);
            if constexpr (SLOPE) fetch<AF, BM>(a.z, a.z_stride, a.slow, m0, M, k, k1, K, uz[s], rows);
            fetch<BF, BN, GATHER_B>(b.p, b.stride, b.slow, n0, N, k, k1, K, ub[s], now);
        };
#pragma unroll
        for (int s = 0; s < DEPTH; ++s)
            if (k0 + s * BK < k1) get(k0 + s * BK, s);
        for (uint64_t k = k0; k < k1;) {
#pragma unroll
            for (int s = 0; s < DEPTH; ++s) {
                if (k < k1) {
                    settle<AF, BM>(a.slow, m0, M, k, k1, ua[s]);
                    if constexpr (SLOPE) settle<AF, BM>(a.slow, m0, M, k, k1, uz[s]);
                    settle<BF, BN, GATHER_B>(b.slow, n0, N, k, k1, ub[s]);
                    slope(a, sums, ua[s], uz[SLOPE ? s : 0], columns);
                    __syncthreads();
                    stage<AF, BM>(lds, ua[s], lost);
                    stage<BF, BN>(lds + PLANES * LDS_A, ub[s], lost);
                    if constexpr (F32) {
                        if (k + BK >= k1) wave_flag(lds + LDS_FLAGS, lost & 0xffffu);
                    }
                    __syncthreads();
                    if (k + DEPTH * BK < k1) get(k + DEPTH * BK, s);
                    multiply(lds, k1 - k >= BK ? BK / 16 : (int)((k1 - k + 15) / 16), acc);
                }
                k += BK;
            }
        }
        if constexpr (F32) {
            const int wave = threadIdx.x / 64, wm = wave / WN * TM, wn = wave % WN * TN;
            float enough = 0.0f;
            if (__builtin_expect(k0 < k1 && any_flag(lds + LDS_FLAGS), 0)) enough = enough_of(a, b, m0, n0, M, N, k0, k1, K, lds, ua[0], ub[0], uz[0]);
#pragma unroll
            for (int i = 0; i < MI; ++i)
#pragma unroll
                for (int j = 0; j < NI; ++j)
                    mend(a, b, m0 + wm + i * 32, n0 + wn + j * 32, M, N, k0, k1, enough, acc[i][j]);
        }
    }

    // Whether any thread of the block has a flag: a word a wave before a barrier, all of them after it.
    static __device__ inline void wave_flag(char* flags, bool own) {
        const uint32_t any = __any(own);
        if ((threadIdx.x & 63) == 0) ((uint32_t*)flags)[threadIdx.x / 64] = any;
    }
    static __device__ inline bool any_flag(const char* flags) {
        const u32x4 f = *(const u32x4*)flags;
        return __any(f[0] | f[1] | f[2] | f[3]);
    }

    // How large a sum of the tile has to be for what the parts lose of its operands to be below its own rounding: at
    // most 2^-134 of an element, so 2^-134 len (max |a| + max |b|) of a sum, against 2^-24 of it. 0 where nothing is lost
    // (what made the block ask lies past the matrix's columns, so that results do not depend on it).
    static __device__ inline float enough_of(const Operand& a, const Operand& b, uint64_t m0, uint64_t n0, uint64_t M,
                                             uint64_t N, uint64_t k0, uint64_t k1, uint64_t K, char* lds, Unit<T> (&ua)[UA],
                                             Unit<T> (&ub)[UB], Unit<T> (&uz)[SLOPE ? UA : 1]) {
        uint32_t lost = 0;
        float most_a = 0.0f, most_b = 0.0f, none[8];
        asm volatile("" : "+s"(m0), "+s"(n0), "+s"(k0));  // addresses of its own: the steps' registers are not kept for it
        const Rows rows(a, m0, M);
        auto look = [&](const auto& u, int units, float& most) {
#pragma unroll
            for (int i = 0; i < (int)(sizeof(u) / sizeof(u[0])); ++i) {
                if (i * 256 + (int)threadIdx.x >= units) break;
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const uint32_t w = u[i].v[j / 4][j % 4];
                    const float r = __uint_as_float(w) - __uint_as_float(w & 0xffff0000u);
                    lost |= __float_as_uint(r - __uint_as_float(pack_bf16(r, r) & 0xffff0000u));
                    most = fmaxf(most, fabsf(__uint_as_float(w)));
                }
            }
        };
        for (uint64_t k = k0; k < k1; k += BK) {
            fetch<AF, BM>(a.p, a.stride, a.slow, m0, M, k, k1, K, ua, rows);
            if constexpr (SLOPE) fetch<AF, BM>(a.z, a.z_stride, a.slow, m0, M, k, k1, K, uz, rows);
            Steps now;
            now.load(b, k, k1);
            fetch<BF, BN, GATHER_B>(b.p, b.stride, b.slow, n0, N, k, k1, K, ub, now);
            cut<AF, BM>(m0, M, k, k1, ua);
            if constexpr (SLOPE) cut<AF, BM>(m0, M, k, k1, uz);
            cut<BF, BN>(n0, N, k, k1, ub);
            slope(a, false, ua, uz, none);
            look(ua, BM * BK / 8, most_a);
            look(ub, BN * BK / 8, most_b);
        }
        // the largest of the threads' sums is at least half of the sum of the largest
        float most = most_a + most_b;
#pragma unroll
        for (int m = 1; m < 64; m *= 2) most = fmaxf(most, __shfl_xor(most, m));
        __syncthreads();  // every wave has read its operands, and the flags
        float* red = (float*)lds;
        if ((threadIdx.x & 63) == 0) red[threadIdx.x / 64] = most;
        wave_flag(lds + LDS_FLAGS, lost & 0xffffu);
        __syncthreads();
        if (!any_flag(lds + LDS_FLAGS)) return 0.0f;
        return 0x1p-109f * (float)(k1 - k0) * fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
    }

    // Sums that are not finite, or not `enough`, again on the f32 matrix cores, straight from memory: f32's own result
    // where an operand is an infinity, a NaN or very small, or where the sum overflows.
    static __device__ inline void mend(const Operand& a, const Operand& b, uint64_t m, uint64_t n, uint64_t M, uint64_t N,
                                       uint64_t k0, uint64_t k1, float enough, f32x16& acc) {
        const int lane = threadIdx.x & 63;
        auto good = [&](float v) { return v - v == 0.0f && fabsf(v) >= enough; };
        bool odd = false;
#pragma unroll
        for (int q = 0; q < 16; ++q) {
            const bool stored = m + 8 * (q / 4) + 4 * (lane >> 5) + q % 4 < M && n + (lane & 31) < N;
            odd |= stored && !good(acc[q]);
        }
        if (!__any(odd)) return;
        m = m + (lane & 31) < M ? m + (lane & 31) : M - 1;
        if constexpr (GATHER_A) m = a.gathered(m);
        n = n + (lane & 31) < N ? n + (lane & 31) : N - 1;
        const float* pa = (const float*)a.p + (AF ? m * a.stride : m);
        const float* pz = (const float*)a.z + (AF ? m * a.z_stride : m);
        const float* pb = (const float*)b.p + (BF ? n * b.stride : n);
        f32x16 again = {};
        constexpr int STEPS = 8;  // under way at once
        for (uint64_t k = k0; k < k1; k += 2 * STEPS) {
            float x[STEPS], y[STEPS], z[STEPS];
#pragma unroll
            for (int s = 0; s < STEPS; ++s) {
                const uint64_t own = k + 2 * s + (lane >> 5), at = own < k1 ? own : k1 - 1;
                x[s] = pa[AF ? at : at * a.stride];
                y[s] = pb[BF ? at : (GATHER_B ? b.gathered(at) : at) * b.stride];
                if constexpr (SLOPE) z[s] = pz[AF ? at : at * a.z_stride];
            }
#pragma unroll
            for (int s = 0; s < STEPS; ++s) {
                const bool in = k + 2 * s + (lane >> 5) < k1;
                if constexpr (SLOPE) x[s] = activate_adjoint_any(a.act, x[s], z[s]);
                again = __builtin_amdgcn_mfma_f32_32x32x2f32(in ? x[s] : 0.0f, in ? y[s] : 0.0f, again, 0, 0, 0);
            }
        }
#pragma unroll
        for (int q = 0; q < 16; ++q) acc[q] = good(acc[q]) ? acc[q] : again[q];
    }
};

// The eight columns of a matrix of N that a lane finishes: n .. n + 3 and n + gap .. n + gap + 3. An f32 store
// instruction fills whole lines where lanes take their quads side by side (65,536 rows, 66 -> 128, z kept: 24
// us, 26 with eight columns in a run).
struct Columns {
    uint32_t n, gap;
    int first, second;  // of each quad's four, how many the matrix has
    __device__ Columns(uint32_t n_, uint32_t gap_, uint32_t N) : n(n_), gap(gap_) {
        first = n >= N ? 0 : N - n < 4 ? (int)(N - n) : 4;
        second = n + gap >= N ? 0 : N - n - gap < 4 ? (int)(N - n - gap) : 4;
    }
};

// Eight elements of a row of f32 or T, what the matrix does not have unset.
template <class T>
__device__ inline void load8(const void* p, bool f32, uint64_t row, const Columns& c, bool over, float (&o)[8]) {
    if constexpr (sizeof(T) == 4) {
        const float* q = (const float*)p + row + c.n;
        typedef typename VecOf<float, 4>::type quad;
        auto get = [&](const float* from, int count, float* to) {
            if (count == 4 || (over && count > 0)) {
                const quad v = *(const quad*)from;
#pragma unroll
                for (int j = 0; j < 4; ++j) to[j] = v[j];
            } else if (count > 0) {
#pragma unroll
                for (int j = 0; j < 4; ++j) to[j] = from[j < count ? j : count - 1];
            }
        };
        get(q, c.first, o);
        get(q + c.gap, c.second, o + 4);
    } else if (f32) {
        Unit<float> u;
        u.load((const float*)p + row + c.n, c.first + c.second, over);
        u.get(o);
    } else {
        Unit<T> u;
        u.load((const T*)p + row + c.n, c.first + c.second, over);
        u.get(o);
    }
}
template <class E, int W, bool STREAM>
__device__ inline void store_some(E* p, int n, const float* v) {
    if (n >= W) {
        typename VecOf<E, W>::type o;
#pragma unroll
        for (int j = 0; j < W; ++j) o[j] = (E)v[j];
        if (STREAM)
            __builtin_nontemporal_store(o, (typename VecOf<E, W>::type*)p);
        else
            *(typename VecOf<E, W>::type*)p = o;
    } else {
#pragma unroll
        for (int j = 0; j < W; ++j)
            if (j < n) p[j] = (E)v[j];
    }
}
template <class T, bool STREAM>
__device__ inline void store8(void* p, bool f32, uint64_t row, const Columns& c, const float (&v)[8]) {
    if constexpr (sizeof(T) == 4) {
        store_some<float, 4, STREAM>((float*)p + row + c.n, c.first, v);
        store_some<float, 4, STREAM>((float*)p + row + c.n + c.gap, c.second, v + 4);
    } else if (f32) {
        store_some<float, 8, false>((float*)p + row + c.n, c.first + c.second, v);
    } else {
        store_some<T, 8, STREAM>((T*)p + row + c.n, c.first + c.second, v);
    }
}

// P rows' sums of a lane's columns, rows m, m + step, ..; what the epilogue adds is loaded for all of them at
// once. `bias` holds the columns' own.
template <class T, int P, bool STREAM = false>
__device__ inline void finish(const Epilogue& e, uint64_t m, int step, uint64_t M, const Columns& c, uint32_t N,
                              const float (&bias)[8], float (&v)[P][8]) {
    if (!c.first) return;
    const bool wide = N >= 7;
    float add[P][8];
#pragma unroll
    for (int p = 0; p < P; ++p) {
        const uint64_t r = m + p * step;
        if (e.residual && r < M)
            load8<T>(e.residual, false, r * e.residual_stride, c, wide && r + 1 < M, add[p]);
        else if (e.accumulate && r < M)
            load8<T>(e.out, e.out_f32, r * e.out_stride, c, wide && r + 1 < M, add[p]);
    }
    if (e.bias) {
#pragma unroll
        for (int p = 0; p < P; ++p)
#pragma unroll
            for (int j = 0; j < 8; ++j) v[p][j] += bias[j];
    }
    if (e.z) {
#pragma unroll
        for (int p = 0; p < P; ++p)
            if (m + p * step < M) store8<T, STREAM>(e.z, false, (m + p * step) * e.z_stride, c, v[p]);
    }
    auto each = [&](auto act) {
#pragma unroll
        for (int p = 0; p < P; ++p)
#pragma unroll
            for (int j = 0; j < 8; ++j) v[p][j] = activate<decltype(act)::value>(v[p][j]);
    };
    switch (e.act) {
        case NPA_ACT_RELU: each(std::integral_constant<int, NPA_ACT_RELU>()); break;
        case NPA_ACT_GELU: each(std::integral_constant<int, NPA_ACT_GELU>()); break;
        case NPA_ACT_SILU: each(std::integral_constant<int, NPA_ACT_SILU>());
    }
#pragma unroll
    for (int p = 0; p < P; ++p) {
        const uint64_t r = m + p * step;
        if (r >= M) break;
        if (e.residual || e.accumulate) {
#pragma unroll
            for (int j = 0; j < 8; ++j) v[p][j] += add[p][j];
        }
        store8<T, STREAM>(e.out, e.out_f32, r * e.out_stride, c, v[p]);
    }
}

template <class T>
__device__ inline void load_bias(const Epilogue& e, const Columns& c, float (&bias)[8]) {
    if (!e.bias || !c.first) return;
    if constexpr (sizeof(T) == 4)
        load8<T>(e.bias, true, 0, c, false, bias);
    else
        load8<T>(e.bias, e.bias_f32, 0, c, false, bias);
}

struct ProductArgs {
    Operand a, b;
    Epilogue e;
    uint32_t M = 0, N = 0;
    uint64_t K = 0;
    uint32_t splits = 1;       // of K
    uint64_t split_len = 0;    // steps a split, a multiple of the tile's
    float* partials = nullptr; // [splits][M][N rounded up to eight]
    // The A operand's sums over its steps: to `db` of a product in one part, else to columns [splits][M].
    float* columns = nullptr;
    void* db = nullptr;
    bool db_f32 = false, db_accumulate = false;
    uint32_t tiles_m = 0, tiles_n = 0;
};

__host__ __device__ inline uint32_t part_cols(const ProductArgs& g) { return (g.N + 7) / 8 * 8; }

// Tiles are taken so that the blocks of one XCD (block index modulo 8) share operands in its L2: each XCD
// has a run of tiles, in strips of 8 tile rows.
__device__ inline void tile_of(const ProductArgs& g, uint32_t id, uint32_t& tm, uint32_t& tn) {
    const uint32_t tiles = g.tiles_m * g.tiles_n, per = tiles / 8, whole = per * 8;
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

template <class T, int MI, int NI, bool STREAM = false>
__device__ inline void store_tile(const ProductArgs& g, uint32_t split, uint64_t m, uint32_t n, float* lds,
                                  const f32x16 (&acc)[MI][NI]) {
    Epilogue part;
    const uint32_t N = g.splits > 1 ? part_cols(g) : g.N;
    if (g.splits > 1) {
        part.out = g.partials + (uint64_t)split * g.M * N;
        part.out_stride = N;
        part.out_f32 = true;
    }
    const Epilogue& e = g.splits > 1 ? part : g.e;
    constexpr int PER_ROW = NI * 4, ROWS = 64 / PER_ROW, STRIDE = kOutStride<NI>;
    constexpr int GAP = sizeof(T) == 4 ? NI * 16 : 4, QUAD = sizeof(T) == 4 ? 4 : 8;
    const int lane = threadIdx.x & 63, col = lane % PER_ROW * QUAD;
    float* out = lds + threadIdx.x / 64 * 32 * STRIDE;
    const Columns c(n + col, GAP, N);
    float bias[8];
    load_bias<T>(e, c, bias);
    __syncthreads();
#pragma unroll
    for (int i = 0; i < MI; ++i) {
#pragma unroll
        for (int j = 0; j < NI; ++j)
#pragma unroll
            for (int q = 0; q < 16; ++q)
                out[(8 * (q / 4) + 4 * (lane >> 5) + q % 4) * STRIDE + j * 32 + (lane & 31)] = acc[i][j][q];
        __builtin_amdgcn_wave_barrier();
        float v[32 / ROWS][8];
#pragma unroll
        for (int p = 0; p < 32 / ROWS; ++p)
#pragma unroll
            for (int j = 0; j < 8; ++j) v[p][j] = out[(p * ROWS + lane / PER_ROW) * STRIDE + col + j % 4 + j / 4 * GAP];
        finish<T, 32 / ROWS, STREAM>(e, m + i * 32 + lane / PER_ROW, ROWS, g.M, c, N, bias, v);
        __builtin_amdgcn_wave_barrier();
    }
}

// Column threadIdx.x's sum of a tile's A operand, of those the threads of the block hold for their units.
template <class X, int BM>
__device__ inline float tile_columns(float (*red)[9], const float (&columns)[8]) {  // 256 rows: 9 KiB of the tiles'
    __syncthreads();
#pragma unroll
    for (int j = 0; j < 8; ++j) red[threadIdx.x][j] = columns[j];
    __syncthreads();
    constexpr int PER = BM / 8 < 256 ? BM / 8 : 256;
    float s = 0.0f;
    if (threadIdx.x < BM)
        for (int q = threadIdx.x / 8; q < 256; q += PER) s += red[q][threadIdx.x % 8];
    return s;
}

// One block's part of a product: tile and split `id`.
template <class X, class T, int BM, int BN, int WN>
__device__ inline void product_block(const ProductArgs& g, uint32_t id, char* lds) {
    uint32_t tm, tn;
    const uint32_t tiles = g.tiles_m * g.tiles_n, split = id / tiles;
    tile_of(g, id % tiles, tm, tn);
    const uint64_t m0 = (uint64_t)tm * BM, n0 = (uint64_t)tn * BN;
    const uint64_t k0 = split * g.split_len, k1 = g.K - k0 < g.split_len ? g.K : k0 + g.split_len;
    const bool sums = (g.columns || g.db) && tn == 0;
    f32x16 acc[X::MI][X::NI];
    float columns[8] = {};
#pragma unroll
    for (int i = 0; i < X::MI; ++i)
#pragma unroll
        for (int j = 0; j < X::NI; ++j) acc[i][j] = f32x16{};
    X::sum(g.a, g.b, m0, n0, g.M, g.N, k0, k1, g.K, sums, lds, acc, columns);
    store_tile<T, X::MI, X::NI>(g, split, m0 + threadIdx.x / 64 / WN * X::TM,
                                (uint32_t)n0 + threadIdx.x / 64 % WN * X::TN, (float*)lds, acc);
    if (!sums) return;
    const float s = tile_columns<X, BM>((float(*)[9])lds, columns);
    if (threadIdx.x >= BM || m0 + threadIdx.x >= g.M) return;
    if (g.db)
        store_param<T>(g.db, g.db_f32, g.db_accumulate, m0 + threadIdx.x, s);
    else
        g.columns[(uint64_t)split * g.M + m0 + threadIdx.x] = s;
}

// ------------------------------------------------------------------ large aligned 16-bit products
// A tile of BM x BN a block, operands from memory to LDS without registers in between, STAGES buffers in
// turn: the loads of STAGES - 1 steps are under way while one step is multiplied.
typedef __attribute__((address_space(3))) unsigned int lds_u32;

template <class T, int BM, int BN, int BK_, int WM, int WN, int STAGES_, bool AF, bool BF, bool BOUND_ = false>
struct Direct {
    static constexpr bool BOUND = BOUND_;
    static constexpr int BK = BK_, STAGES = STAGES_, WAVES = WM * WN;
    static constexpr int TM = BM / WM, TN = BN / WN, MI = TM / 32, NI = TN / 32;
    static constexpr int BYTES_A = BM * BK * 2, BUFFER = (BM + BN) * BK * 2;
    static constexpr int LOADS_A = BYTES_A / 1024 / WAVES, LOADS_B = BN * BK * 2 / 1024 / WAVES, LOADS = LOADS_A + LOADS_B;
    static constexpr int LDS = STAGES * BUFFER;
    static_assert(BK % 32 == 0 && LDS >= WAVES * 32 * (TN + 4) * 4, "an even number of stretches; the epilogue's stage");

    // Byte offsets from the tile's first element of the 16 bytes that this lane brings with each load: the
    // chunks of chunk_at, in LDS order. `at_row`: the operand's row of a row of the tile.
    template <bool FAST, int ROWS, int N, class At>
    static __device__ inline void offsets(uint64_t stride, uint64_t first, uint64_t count, uint32_t (&off)[N], const At& at_row) {
        const int lane = threadIdx.x & 63, wave = threadIdx.x / 64;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            constexpr int PER = FAST ? BK / 8 : ROWS / 8;  // chunks a row
            const int at = (wave * N + i) * 64 + lane;
            int r = at / PER, c = at % PER;
            c = chunk_at<FAST, BK, ROWS>(r, c) / 16 % PER;  // the permutation is its own inverse
            if (FAST && first + r >= count) r = (int)(count - 1 - first);            // not stored
            if (!FAST && first + c * 8 >= count) c = (int)((count - 8 - first) / 8);  // not stored
            off[i] = (uint32_t)(at_row(r) * stride + c * 8) * 2;
        }
    }

    static_assert(!BOUND || (!AF && !BF), "rows past the last one are past the operand's end");

    // An operand's bytes from the step on that is loaded next. BOUND: what follows the last row reads as zeros.
    struct Source {
        const char* p;
        uint64_t step, left;
        __device__ inline void next() {
            p += step;
            if (BOUND) left = left > step ? left - step : 0;
        }
        __device__ inline uint32_t bytes() const { return BOUND && left < 0xffffffffu ? (uint32_t)left : 0xffffffffu; }
    };

    // Buffer loads, not flat ones: they leave the order of LDS reads' completion known, and take a
    // scalar base. Offsets are within the tile, so the range is a bound only where a Source has one.
    static __device__ inline void load_a(const Source& a, const uint32_t (&oa)[LOADS_A], char* __restrict to) {
        const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
        const __amdgpu_buffer_rsrc_t base = __builtin_amdgcn_make_buffer_rsrc((void*)a.p, 0, a.bytes(), 0x00020000);
#pragma unroll
        for (int i = 0; i < LOADS_A; ++i)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(base, (lds_u32*)(to + (wave * LOADS_A + i) * 1024), 16, oa[i], 0, 0, 0);
    }
    static __device__ inline void load_b(const Source& b, const uint32_t (&ob)[LOADS_B], char* __restrict to) {
        const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
        const __amdgpu_buffer_rsrc_t base = __builtin_amdgcn_make_buffer_rsrc((void*)b.p, 0, b.bytes(), 0x00020000);
#pragma unroll
        for (int i = 0; i < LOADS_B; ++i)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(base, (lds_u32*)(to + BYTES_A + (wave * LOADS_B + i) * 1024), 16, ob[i],
                                                     0, 0, 0);
    }

    struct Fragments {
        u32x4 a[MI], b[NI];
    };
    static __device__ __forceinline__ void read(const char* __restrict lds, int ks, Fragments& f) {
        const int wave = threadIdx.x / 64, wm = wave / WN * TM, wn = wave % WN * TN;
#pragma unroll
        for (int j = 0; j < NI; ++j) f.b[j] = fragment<BF, BK, BN>(lds + BYTES_A, wn + j * 32, ks);
#pragma unroll
        for (int i = 0; i < MI; ++i) f.a[i] = fragment<AF, BK, BM>(lds, wm + i * 32, ks);
    }
    static __device__ __forceinline__ void multiply(const Fragments& f, f32x16 (&acc)[MI][NI]) {
#pragma unroll
        for (int i = 0; i < MI; ++i)
#pragma unroll
            for (int j = 0; j < NI; ++j) acc[i][j] = mma<T>(f.a[i], f.b[j], acc[i][j]);
    }
    // The order of a stretch: reads between the first products and loads between the next, so that none
    // holds the others up (a CU takes a load of 64 lanes in 16 cycles, and a wave's products wait behind it).
    template <int N>
    static __device__ __forceinline__ void interleave() {
        constexpr int READS = MI * (AF ? 1 : 2) + NI * (BF ? 1 : 2), REST = MI * NI - READS / 2;
#pragma unroll
        for (int i = 0; i < READS / 2; ++i) {
            __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);  // LDS reads
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);  // matrix products
        }
#pragma unroll
        for (int i = 0; i < N; ++i) {
            __builtin_amdgcn_sched_group_barrier(0x010, 1, 0);  // loads
            if (i < REST) __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        }
        if (REST > N) __builtin_amdgcn_sched_group_barrier(0x008, REST > N ? REST - N : 0, 0);
        __builtin_amdgcn_sched_barrier(0);
    }
    // Waits for this wave's LDS reads and for all but the newest LEFT of its loads, then for every wave.
    template <int LEFT>
    static __device__ __forceinline__ void meet() {
        __builtin_amdgcn_s_waitcnt((LEFT & 15) | 0x70 | (LEFT >> 4) << 14);
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    }

    // One step, LEFT (at most STAGES) steps before the last: each 16 columns' products run while the next
    // fragments are read. The barrier stands before the last products: by then every wave has read the last
    // of `now`, and the next step's operands have arrived in `next`. `now` then takes the A operand of the step
    // STAGES ahead, and `before`, free since the last step, the B operand that belongs to the A there.
    template <int LEFT>
    static __device__ __forceinline__ void step(const Source& a, const Source& b, const uint32_t (&oa)[LOADS_A],
                                                const uint32_t (&ob)[LOADS_B], char* __restrict before, char* __restrict now,
                                                const char* __restrict next, Fragments& f, f32x16 (&acc)[MI][NI]) {
        Fragments g;
#pragma unroll
        for (int ks = 1; ks < BK / 16; ++ks) {
            read(now, ks, ks % 2 ? g : f);
            if (ks == 1 && LEFT >= STAGES - 1) load_b(b, ob, before);
            multiply(ks % 2 ? f : g, acc);
            if (ks == 1 && LEFT >= STAGES - 1)
                interleave<LOADS_B>();
            else
                interleave<0>();
        }
        if constexpr (LEFT > 0) {
            meet<(LEFT < STAGES ? LEFT - 1 : STAGES - 2) * LOADS>();
            read(next, 0, f);
            if (LEFT >= STAGES) load_a(a, oa, now);
        }
        multiply(g, acc);
        if (LEFT >= STAGES)
            interleave<LOADS_A>();
        else
            interleave<0>();
    }
    // The last steps, from LEFT steps before the last on.
    template <int LEFT>
    static __device__ __forceinline__ void drain(const Source& a, const Source& b, const uint32_t (&oa)[LOADS_A],
                                                 const uint32_t (&ob)[LOADS_B], char* lds, int before, int now,
                                                 Fragments& f, f32x16 (&acc)[MI][NI]) {
        const int next = now == LDS - BUFFER ? 0 : now + BUFFER;
        step<LEFT>(a, b, oa, ob, lds + before, lds + now, lds + next, f, acc);
        if constexpr (LEFT > 0) drain<LEFT - 1>(a, b, oa, ob, lds, now, next, f, acc);
    }
};

// The tile at m0, n0 over k0 .. k1 - 1: whole steps, or, BOUND, of operands whose slow index is k. `gather`: A's rows are
// gathered, all of them within 2^32 bytes.
template <class X, class T, int BM, int BN, int WN, bool AF, bool BF>
__device__ __forceinline__ void direct_tile(const ProductArgs& g, uint32_t split, uint64_t m0, uint64_t n0, uint64_t k0,
                                            uint64_t k1, bool gather, char* lds) {
    uint32_t oa[X::LOADS_A], ob[X::LOADS_B];
    const auto in_place = [](int r) { return (uint64_t)r; };
    if (AF && gather)
        X::template offsets<AF, BM>(g.a.stride, m0, g.M, oa, [&](int r) { return g.a.gathered(m0 + r); });
    else
        X::template offsets<AF, BM>(g.a.stride, m0, g.M, oa, in_place);
    X::template offsets<BF, BN>(g.b.stride, n0, g.N, ob, in_place);
    typename X::Source a, b;
    a.p = (const char*)g.a.p + (AF ? (gather ? 0 : m0 * g.a.stride) + k0 : k0 * g.a.stride + m0) * 2;
    b.p = (const char*)g.b.p + (BF ? n0 * g.b.stride + k0 : k0 * g.b.stride + n0) * 2;
    a.step = (AF ? 1 : g.a.stride) * X::BK * 2;
    b.step = (BF ? 1 : g.b.stride) * X::BK * 2;
    a.left = (k1 - k0) * g.a.stride * 2;  // a row's columns end before the next row begins
    b.left = (k1 - k0) * g.b.stride * 2;
    f32x16 acc[X::MI][X::NI];
#pragma unroll
    for (int i = 0; i < X::MI; ++i)
#pragma unroll
        for (int j = 0; j < X::NI; ++j) acc[i][j] = f32x16{};
    int steps = (int)((k1 - k0 + (X::BOUND ? X::BK - 1 : 0)) / X::BK);
    typename X::Fragments f;
    if (steps < X::STAGES) {  // a split's short last part
        while (steps--) {
            X::load_a(a, oa, lds);
            X::load_b(b, ob, lds);
            a.next();
            b.next();
            X::template meet<0>();
#pragma unroll
            for (int ks = 0; ks < X::BK / 16; ++ks) {
                X::read(lds, ks, f);
                X::multiply(f, acc);
            }
            __syncthreads();
        }
    } else {
        int now = 0, before = X::LDS - X::BUFFER;
#pragma unroll
        for (int s = 0; s < X::STAGES; ++s) {
            X::load_a(a, oa, lds + s * X::BUFFER);
            a.next();
            if (s + 1 < X::STAGES) {
                X::load_b(b, ob, lds + s * X::BUFFER);
                b.next();
            }
        }
        X::template meet<(X::STAGES - 2) * X::LOADS + X::LOADS_A>();
        X::read(lds, 0, f);
        for (steps -= X::STAGES; steps; --steps) {
            const int next = now == X::LDS - X::BUFFER ? 0 : now + X::BUFFER;
            X::template step<X::STAGES>(a, b, oa, ob, lds + before, lds + now, lds + next, f, acc);
            a.next();
            b.next();
            before = now;
            now = next;
        }
        X::template drain<X::STAGES - 1>(a, b, oa, ob, lds, before, now, f, acc);
    }
    store_tile<T, X::MI, X::NI, true>(g, split, m0 + threadIdx.x / 64 / WN * X::TM,
                                (uint32_t)n0 + threadIdx.x / 64 % WN * X::TN, (float*)lds, acc);
}

template <class X, class T, int BM, int BN, int WN, bool AF, bool BF>
__device__ __forceinline__ void direct_block(const ProductArgs& g, char* lds) {
    uint32_t tm, tn;
    const uint32_t tiles = g.tiles_m * g.tiles_n, split = blockIdx.x / tiles;
    tile_of(g, blockIdx.x % tiles, tm, tn);
    const uint64_t k0 = split * g.split_len, k1 = g.K - k0 < g.split_len ? g.K : k0 + g.split_len;
    direct_tile<X, T, BM, BN, WN, AF, BF>(g, split, (uint64_t)tm * BM, (uint64_t)tn * BN, k0, k1, false, lds);
}

// ------------------------------------------------------------------ few rows
// Up to 16 * RT rows: the weights' way from memory is all there is. A block takes 16 outputs, its waves every
// W-th run of 32 columns of them, straight from memory to the matrix cores (f32 on the f32 ones, which keep
// up here), DEPTH runs ahead; their sums meet in LDS. 16-bit: 16 x 16 x 32, lane l holds row (or output) l % 16 and columns
// 8 (l / 16) .. + 7; f32: eight products of 16 x 16 x 4 take the same eight columns one each. Measured: one row, 4,096 ->
// 4,096 bf16 9.3 us, 3.6 TB/s over the whole launch.
typedef float f32x4 __attribute__((ext_vector_type(4)));

template <class T>
__device__ inline f32x4 mma16(const Unit<T>& a, const Unit<T>& b, f32x4 c) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int j = 0; j < 8; ++j)
            c = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a.v[j / 4][j % 4]), __uint_as_float(b.v[j / 4][j % 4]), c,
                                                     0, 0, 0);
        return c;
    } else if constexpr (__is_same(T, _Float16)) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a.v[0]), __builtin_bit_cast(f16x8, b.v[0]), c, 0,
                                                      0, 0);
    } else {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a.v[0]), __builtin_bit_cast(bf16x8, b.v[0]),
                                                       c, 0, 0, 0);
    }
}

constexpr int kFewWaves = 16;

// Rows first .. end - 1, at most 16 * RT, and outputs n0 .. n0 + 15.
template <class T, int RT, bool GATHER = false>
__device__ inline void few_block(const ProductArgs& g, uint32_t first, uint32_t end, uint32_t n0, float (*red)[RT * 16][17]) {
    constexpr int DEPTH = sizeof(T) == 4 ? 4 : 8;
    const int lane = threadIdx.x & 63, wave = threadIdx.x / 64, waves = blockDim.x / 64;
    const uint32_t runs = (uint32_t)((g.K + 31) / 32);
    const uint64_t n = n0 + (lane & 15) < g.N ? n0 + (lane & 15) : g.N - 1;  // outputs past the end: not stored
    const T* w = (const T*)g.b.p + n * g.b.stride + (lane >> 4) * 8;
    const T* x[RT];
    bool x_over[RT];
    const bool wide = g.K >= 7, w_over = wide && n + 1 < g.N;
#pragma unroll
    for (int t = 0; t < RT; ++t) {
        const uint32_t own = first + t * 16 + (lane & 15), at = own < end ? own : end - 1;  // rows past the end: not stored
        const uint64_t m = GATHER ? g.a.gathered(at) : at;
        x[t] = (const T*)g.a.p + m * g.a.stride + (lane >> 4) * 8;
        x_over[t] = wide && m + 1 < g.a.slow;
    }
    Unit<T> uw[DEPTH], ux[RT][DEPTH];
    auto left = [&](uint32_t r) {  // of the lane's eight columns of run r
        const int64_t v = (int64_t)g.K - (int64_t)r * 32 - (lane >> 4) * 8;
        return v < 0 ? 0 : v > 8 ? 8 : (int)v;
    };
    auto get = [&](uint32_t r, int d) {
        const uint64_t at = (uint64_t)r * 32;
        if (at + 32 <= g.K) {
            uw[d].load_all(w + at);
#pragma unroll
            for (int t = 0; t < RT; ++t) ux[t][d].load_all(x[t] + at);
        } else {
            uw[d].load(w + at, left(r), w_over);
#pragma unroll
            for (int t = 0; t < RT; ++t) ux[t][d].load(x[t] + at, left(r), x_over[t]);
        }
    };
    f32x4 acc[RT];
#pragma unroll
    for (int t = 0; t < RT; ++t) acc[t] = f32x4{};
#pragma unroll
    for (int d = 0; d < DEPTH; ++d)
        if (wave + d * waves < runs) get(wave + d * waves, d);
    for (uint32_t r = wave; r < runs;) {
#pragma unroll
        for (int d = 0; d < DEPTH; ++d) {
            if (r < runs) {
                if ((uint64_t)r * 32 + 32 > g.K) {
                    uw[d].keep(left(r));
#pragma unroll
                    for (int t = 0; t < RT; ++t) ux[t][d].keep(left(r));
                }
#pragma unroll
                for (int t = 0; t < RT; ++t) acc[t] = mma16<T>(ux[t][d], uw[d], acc[t]);
                if (r + DEPTH * waves < runs) get(r + DEPTH * waves, d);
            }
            r += waves;
        }
    }
#pragma unroll
    for (int t = 0; t < RT; ++t)
#pragma unroll
        for (int j = 0; j < 4; ++j) red[wave][t * 16 + (lane >> 4) * 4 + j][lane & 15] = acc[t][j];
    __syncthreads();
    for (int i = threadIdx.x; i < RT * 256; i += blockDim.x) {
        float s = 0.0f;
        for (int q = 0; q < waves; ++q) s += red[q][i / 16][i % 16];
        red[0][i / 16][i % 16] = s;  // this thread alone reads it
    }
    __syncthreads();
    for (int i = threadIdx.x; i < RT * 32; i += blockDim.x) {
        const uint32_t c = n0 + i % 2 * 8;
        float v[1][8], bias[8];
        const Columns cols(c, 4, g.N);
        load_bias<T>(g.e, cols, bias);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[0][j] = red[0][i / 2][i % 2 * 8 + j];
        if (first + i / 2 < end) finish<T, 1>(g.e, first + i / 2, 1, end, cols, g.N, bias, v);
    }
}

// ------------------------------------------------------------------ what the splits left
// The splits of a product, added up in their order: G threads for eight columns of a row, each with every G-th
// split. 256 parts of 128 x 66 and the bias gradient's: 5.6 us.
template <class T, int G>
__device__ inline void join_product(const ProductArgs& g, uint32_t block, uint32_t blocks, float (*shared)[9]) {
    constexpr int UNITS = 256 / G;
    const uint32_t per_row = part_cols(g) / 8, unit = threadIdx.x % UNITS, part = threadIdx.x / UNITS;
    const uint64_t units = (uint64_t)g.M * per_row, plane = units * 8;
    for (uint64_t base = (uint64_t)block * UNITS; base < units; base += (uint64_t)blocks * UNITS) {
        const uint64_t u = base + unit, m = u / per_row;
        const uint32_t n = (uint32_t)(u % per_row) * 8;
        const float* p = g.partials + u * 8 + part * plane;
        float sums[1][8] = {}, bias[8];
        float(&v)[8] = sums[0];
        if (u < units) {
            typedef float f32x8 __attribute__((ext_vector_type(8)));
#pragma unroll 8
            for (uint32_t s = part; s < g.splits; s += G, p += G * plane) {
                const f32x8 x = *(const f32x8*)p;
#pragma unroll
                for (int j = 0; j < 8; ++j) v[j] += x[j];
            }
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
        if (part == 0 && u < units) {
            const Columns cols(n, 4, g.N);
            load_bias<T>(g.e, cols, bias);
            finish<T, 1>(g.e, m, 1, g.M, cols, g.N, bias, sums);
        }
    }
}

__host__ __device__ inline int join_threads(const ProductArgs& g) { return g.splits >= 32 ? 16 : g.splits >= 8 ? 4 : 1; }

template <class T>
__device__ inline void join_any(const ProductArgs& g, uint32_t block, uint32_t blocks, float (*shared)[9]) {
    switch (join_threads(g)) {
        case 16: join_product<T, 16>(g, block, blocks, shared); break;
        case 4: join_product<T, 4>(g, block, blocks, shared); break;
        default: join_product<T, 1>(g, block, blocks, shared);
    }
}

struct BiasArgs {
    const float* partials = nullptr;  // [parts][cols]
    uint32_t parts = 0, cols = 0;
    void* db = nullptr;
    bool f32 = false, accumulate = false;
};

// One launch for all that a call's kernels left in parts: up to two split products and the bias gradient.
template <class T>
__global__ __launch_bounds__(256) void k_join(ProductArgs p, ProductArgs q, BiasArgs b, uint32_t p_blocks, uint32_t q_blocks) {
    __shared__ float shared[256][9];
    uint32_t block = blockIdx.x;
    if (block < p_blocks) {
        join_any<T>(p, block, p_blocks, shared);
        return;
    }
    block -= p_blocks;
    if (block < q_blocks) {
        join_any<T>(q, block, q_blocks, shared);
        return;
    }
    column_sums<256>(b.partials, b.parts, b.cols, block - q_blocks, gridDim.x - p_blocks - q_blocks,
                     [&](uint64_t col, float s) { store_param<T>(b.db, b.f32, b.accumulate, col, s); });
}

// ------------------------------------------------------------------ dz and its column sums
struct SlopeArgs {
    const void* dy = nullptr;
    const void* z = nullptr;
    void* dz = nullptr;         // written unless null
    float* partials = nullptr;  // [gridDim.y][cols], written unless null
    uint64_t dy_stride = 0, z_stride = 0, dz_stride = 0, rows = 0;
    uint32_t cols = 0;
    uint32_t lanes = 0;  // of a block across the columns, eight each; the others are further rows
};

// dz = dy act'(z), rounded to the layer's type: the operand of both products of the adjoint, of which a 16-bit layer's matrix
// cores take 16 bits (an f32 dz would be two operands, and its products twice the work; the rounding is as large as the results'
// own, and of sums of it: against 64 bits they are off by 2.3e-3 in bf16, 1.7e-3 without it, 2.9e-4 and 2.1e-4 in f16); and its
// column sums before that rounding. A block takes 8 * lanes columns of rows first .. last - 1. Bound by
// memory: 8,192 x 8,192 bf16 75 us, 5.4 TB/s.
template <class T, int ACT>
__device__ inline void slope_block(const SlopeArgs& g, uint64_t first, uint64_t last, float* partials, float (*shared)[9]) {
    const uint32_t lane = threadIdx.x % g.lanes, group = threadIdx.x / g.lanes, groups = 256 / g.lanes;
    const uint32_t col = (blockIdx.x * g.lanes + lane) * 8;
    const int n = col < g.cols ? (g.cols - col < 8 ? (int)(g.cols - col) : 8) : 0;
    float sum[8] = {};
    // the next row is on its way while one is worked on
    Unit<T> dy, z, dy_next, z_next;
    auto get = [&](uint64_t r) {
        const bool over = g.cols >= 8 && r + 1 < g.rows;
        dy_next.load((const T*)g.dy + r * g.dy_stride + col, n, over);
        if (ACT != NPA_ACT_IDENTITY) z_next.load((const T*)g.z + r * g.z_stride + col, n, over);
    };
    uint64_t r = first + group;
    if (n && r < last) get(r);
    for (; n && r < last; r += groups) {
        dy = dy_next;
        z = z_next;
        if (r + groups < last) get(r + groups);
        dy.keep(n);
        float d[8], e[8];
        dy.get(d);
        if (ACT != NPA_ACT_IDENTITY) {
            z.keep(n);
            z.get(e);
#pragma unroll
            for (int j = 0; j < 8; ++j) d[j] = activate_adjoint<ACT>(d[j], e[j]);
            if (g.dz) {  // rows of whole units
                Unit<T> u;
                u.set(d);
                *(Unit<T>*)((T*)g.dz + r * g.dz_stride + col) = u;
            }
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) sum[j] += d[j];
    }
    if (!partials) return;
#pragma unroll
    for (int j = 0; j < 8; ++j) shared[threadIdx.x][j] = sum[j];
    __syncthreads();
    for (uint32_t c = threadIdx.x; c < g.lanes * 8; c += 256) {
        const uint32_t at = blockIdx.x * g.lanes * 8 + c;
        if (at >= g.cols) continue;
        float s = 0.0f;
        for (uint32_t q = 0; q < groups; ++q) s += shared[q * g.lanes + c / 8][c % 8];
        partials[at] = s;
    }
}

// ------------------------------------------------------------------ which tiles, which splits
struct Shape {
    int bm, bn, resident;  // resident: blocks a CU holds
    // Measured, us: a tile's beginning and end; a step of one block alone on its CU; and of a CU's matrix
    // cores and LDS for it, 16-bit types and f32.
    double ends, alone16, alone32, busy16, busy32;
};
constexpr Shape kShapes[] = {{128, 128, 2, 6.0, 0.95, 1.73, 0.62, 1.1},
                             {64, 64, 4, 3.5, 0.55, 0.91, 0.27, 0.38},
                             {128, 32, 3, 4.0, 0.65, 1.04, 0.3, 0.45}};
constexpr Shape kDirect = {256, 256, 1, 12.0, 1.65, 0.0, 1.65, 0.0};

constexpr uint32_t kMostSplits = 512;
constexpr uint64_t kTooManyTiles = 1u << 24;  // blocks of 256 threads: a launch has to stay below 2^32

uint64_t tile_count(const Shape& s, uint64_t M, uint64_t N) {
    return ((M + s.bm - 1) / s.bm) * ((N + s.bn - 1) / s.bn);
}

struct Plan {
    uint32_t splits = 1;
    uint64_t len = 0;  // steps a split
    double us = 0.0;
};

// The time of a launch by a model: a block's steps follow each other, each as long as one block alone takes,
// or as the blocks of a CU keep it busy; rounds of blocks follow each other too. Splitting a sum costs a launch
// and its parts' way through memory, and pays where a product has few tiles. (30 x 4,000 -> 1,000 bf16: 42 us
// in one part, 12 in sixteen; 4,096 x 1,000 -> 1,000: 23 us in one, 35 in two.)
struct Split {
    Plan plan;
    double blocks = 0.0, load = 0.0, join = 0.0;  // steps of all blocks; us to join the parts
};
constexpr int kMostWays = 10;

// The ways to split an M x N product of `steps` steps, and the time that its operands' way from memory takes.
int ways(const Shape& s, uint64_t M, uint64_t N, uint64_t steps, int cus, uint32_t most, Split (&out)[kMostWays], double& memory) {
    const uint64_t tiles = tile_count(s, M, N);
    int n = 0;
    memory = (double)(M + N) * steps * 128.0 / 3e6;
    for (uint64_t splits = 1; splits <= most && n < kMostWays; splits *= 2) {
        Split& p = out[n++];
        p.plan.len = steps ? (steps + splits - 1) / splits : 0;
        p.plan.splits = steps ? (uint32_t)((steps + p.plan.len - 1) / p.plan.len) : 1;
        p.blocks = (double)(tiles * p.plan.splits);
        p.load = (double)(tiles * steps);
        p.join = p.plan.splits > 1 ? p.plan.splits * (double)M * N * 8.0 / 4.2e6 : 0.0;
        if (splits >= steps || p.blocks > 2.0 * cus * s.resident) break;
    }
    return n;
}

// Of one product, or the adjoint's two, that share a launch (`b` null: one). The adjoint's steps are slower
// than the forward's, measured: both operands of dW, and dx's weights, are staged across their rows.
double launch_us(const Shape& s, bool f32, bool adjoint, const Split& a, const Split* b, int cus, double memory) {
    const double blocks = a.blocks + (b ? b->blocks : 0.0), slots = (double)cus * s.resident;
    const double load = a.load + (b ? b->load : 0.0);
    const double longest = (double)std::max(a.plan.len, b ? b->plan.len : 0);
    const double shortest = (double)(b ? std::min(a.plan.len, b->plan.len) : a.plan.len);
    const double resident = std::min<double>(s.resident, std::ceil(blocks / cus));
    const double alone = (f32 ? s.alone32 : s.alone16) * (adjoint ? 1.6 : 1.0);
    const double busy = (f32 ? s.busy32 : s.busy16) * (adjoint ? 1.4 : 1.0), each = std::max(alone, resident * busy);
    double us;
    if (blocks <= slots)  // the busiest CU: the longest block and a share of the others
        us = s.ends + std::max(longest * alone, std::min(resident * longest, load / cus + longest) * busy);
    else  // the last round: half filled, by the shortest
        us = std::max(blocks / slots * s.ends + load / slots * each + (b ? 0.6 : 0.3) * (s.ends + shortest * each),
                      s.ends + longest * each);
    us = std::max(us, s.ends + memory);
    if (a.plan.splits > 1 || (b && b->plan.splits > 1)) us += 3.0 + a.join + (b ? b->join : 0.0);
    return us;
}

Plan plan(const Shape& s, bool f32, bool adjoint, uint64_t M, uint64_t N, uint64_t steps, int cus, uint32_t most) {
    Split a[kMostWays];
    double memory;
    Plan best;
    for (int n = ways(s, M, N, steps, cus, most, a, memory), i = 0; i < n; ++i) {
        a[i].plan.us = launch_us(s, f32, adjoint, a[i], nullptr, cus, memory);
        if (i == 0 || a[i].plan.us < best.us) best = a[i].plan;
    }
    return best;
}

// Both products of the adjoint, whose blocks share the CUs and much of what they read.
double plan(const Shape& s, bool f32, const ProductArgs& w, const ProductArgs& x, uint64_t step, int cus, Plan& pw, Plan& px) {
    Split a[kMostWays], b[kMostWays];
    double memory_w, memory_x, best = 0.0;
    const int nw = ways(s, w.M, w.N, (w.K + step - 1) / step, cus, kMostSplits, a, memory_w);
    const int nx = ways(s, x.M, x.N, (x.K + step - 1) / step, cus, kMostSplits, b, memory_x);
    const double memory = std::max(memory_w, memory_x) + 0.3 * std::min(memory_w, memory_x);
    for (int i = 0; i < nw; ++i)
        for (int j = 0; j < nx; ++j) {
            const double us = launch_us(s, f32, true, a[i], &b[j], cus, memory);
            if (i + j > 0 && us >= best) continue;
            best = us;
            pw = a[i].plan;
            px = b[j].plan;
        }
    return best;
}

void set_plan(ProductArgs& g, const Plan& p, const Shape& s, uint64_t step) {
    g.tiles_m = (g.M + s.bm - 1) / s.bm;
    g.tiles_n = (g.N + s.bn - 1) / s.bn;
    g.splits = p.splits;
    g.split_len = p.len * step;
}
uint64_t part_floats(const ProductArgs& g) { return g.splits > 1 ? (uint64_t)g.splits * g.M * part_cols(g) : 0; }
uint32_t block_count(const ProductArgs& g) { return g.tiles_m * g.tiles_n * g.splits; }

template <class T>
hipError_t join(const ProductArgs* p, const ProductArgs* q, const BiasArgs& b, hipStream_t stream) {
    static const ProductArgs none;
    auto blocks = [](const ProductArgs* g) {
        if (!g || g->splits < 2) return 0u;
        const uint64_t per = 256 / join_threads(*g), units = (uint64_t)g->M * part_cols(*g) / 8;
        return (uint32_t)std::min<uint64_t>((units + per - 1) / per, 4096);
    };
    const uint32_t pb = blocks(p), qb = blocks(q), bb = b.db ? std::min((b.cols + 15) / 16, 1u << 20) : 0;
    if (pb + qb + bb)
        hipLaunchKernelGGL(k_join<T>, dim3(pb + qb + bb), dim3(256), 0, stream, p ? *p : none, q ? *q : none, b, pb, qb);
    return hipGetLastError();
}

// Whether the direct loads can serve an operand: whole 16-byte chunks at aligned addresses, offsets
// inside a tile below 2^32 bytes.
template <bool FAST>
bool direct_operand(const Operand& o, uint64_t count) {
    return reinterpret_cast<uintptr_t>(o.p) % 16 == 0 && o.stride % 8 == 0 && o.stride < (1u << 22) &&
           (FAST || count % 8 == 0);
}

}  // namespace
}  // namespace npa
