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
constexpr uint64_t kJoinLoads = 8, kJoinTurns = 2, kJoinParts = 64;  // of calls whose last block joins the sums
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

// The value of a lane's partner in a sum over 2 * M lanes whose halves are uniform already.
template <int M>
__device__ inline float partner(float v) {
    const int i = __float_as_int(v);
    if (M == 1) return __int_as_float(__builtin_amdgcn_mov_dpp(i, 0xb1, 0xf, 0xf, true));   // quad_perm 1 0 3 2
    if (M == 2) return __int_as_float(__builtin_amdgcn_mov_dpp(i, 0x4e, 0xf, 0xf, true));   // quad_perm 2 3 0 1
    if (M == 4) return __int_as_float(__builtin_amdgcn_mov_dpp(i, 0x141, 0xf, 0xf, true));  // half rows mirrored
    if (M == 8) return __int_as_float(__builtin_amdgcn_mov_dpp(i, 0x140, 0xf, 0xf, true));  // rows mirrored
    return __shfl_xor(v, M);
}

// Sum over a group of L lanes of a wave, the same bits in each of them.
template <int L, int M = 1>
__device__ inline float lane_sum(float v) {
    if constexpr (M < (L < 64 ? L : 64)) return lane_sum<L, M * 2>(v + partner<M>(v));
    return v;
}

// A group of more than one wave meets in LDS: each wave leaves N values, and each lane takes one wave's, lanes
// WAVES apart the same, for lane_sum<WAVES>. (Taking all waves' in each lane held 48 registers at 1,024 lanes.) Two
// slots in turn, so that one barrier is enough; every thread of the block calls it.
template <int L, int N>
struct Meet {
    static constexpr int WAVES = L / 64, ALL = (L < 256 ? 256 : L) / 64;
    float slot[2][ALL][N];
    __device__ inline void operator()(int turn, const float (&own)[N], float (&got)[N]) {
        const int wave = threadIdx.x / 64;
        if ((threadIdx.x & 63) == 0) {
#pragma unroll
            for (int j = 0; j < N; ++j) slot[turn & 1][wave][j] = own[j];
        }
        __syncthreads();
#pragma unroll
        for (int j = 0; j < N; ++j) got[j] = slot[turn & 1][wave / WAVES * WAVES + threadIdx.x % WAVES][j];
    }
};
template <int N>
struct Meet<0, N> {};  // one wave a group

template <int L>
constexpr int kMeetLanes = L > 64 ? L : 0;

// A lane's vectors of a row as they lie in memory; what is past its end is unset until keep, before its use, puts
// zeros there, so that the loads stay under way meanwhile.
template <class T, int L, int NV>
struct Row {
    static constexpr int V = 16 / sizeof(T);
    typename VecOf<T, V>::type v[NV];
    // `over`: the memory past the row's end is the caller's, so a vector that crosses it is read whole.
    __device__ inline void load(const T* row, uint32_t lane, uint32_t width, bool over) {
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const uint32_t col = (lane + k * L) * V;
            const bool whole = col + V <= width || (over && col < width);
            if (!whole && col < width) {
#pragma unroll
                for (int j = 0; j < V; ++j) v[k][j] = row[col + j < width ? col + j : width - 1];
            }
            if (whole) v[k] = *(const typename VecOf<T, V>::type*)(row + col);
        }
    }
    __device__ inline void keep(uint32_t lane, uint32_t width) {
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            if ((uint32_t)((k + 1) * L * V) <= width) continue;
#pragma unroll
            for (int j = 0; j < V; ++j) v[k][j] = (lane + k * L) * V + j < width ? v[k][j] : (T)0.0f;
        }
    }
};

// Whether another row of at least a vector follows row r of a matrix.
template <int V>
__device__ inline bool row_follows(const NormArgs& a, uint64_t r) {
    return r + 1 < a.rows && a.width >= V;
}

// Rows to blocks of 256 threads or one row's lanes, `gridDim.x` groups of rows apart; the next row is
// on its way while one is normed. gamma and beta stay in registers. Measured: 32,768 x 4,096 bf16 102 us, 5.3
// TB/s of the 5.7 that a copy reaches; 10,000 x 4,000 f32 59 us, 5.5 TB/s (inputs in turn; a copy of it 60).
template <class T, int L, int NV>
__global__ __launch_bounds__(L < 256 ? 256 : L) void k_norm(NormArgs a) {
    constexpr int V = 16 / sizeof(T), G = (L < 256 ? 256 : L) / L;
    __shared__ Meet<kMeetLanes<L>, 3> meet;
    const uint32_t lane = threadIdx.x % L, first = lane & ~63u;
    const float inv = 1.0f / (float)a.width;
    // elements that this wave's lanes hold of a row
    float count = 0.0f;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        const uint32_t begin = (first + k * L) * V;
        if (begin < a.width) count += (float)min(a.width - begin, (uint32_t)((L < 64 ? L : 64) * V));
    }
    const float wave_inv = count > 0.0f ? 1.0f / count : 0.0f;
    float gamma[NV][V], beta[NV][V];
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        load_params<T, V>(a.gamma, a.param_f32, (lane + k * L) * V, a.width, 1.0f, gamma[k]);
        load_params<T, V>(a.beta, a.param_f32, (lane + k * L) * V, a.width, 0.0f, beta[k]);
    }
    const uint64_t step = (uint64_t)gridDim.x * G;
    uint64_t row = (uint64_t)blockIdx.x * G + threadIdx.x / L;
    Row<T, L, NV> x, ahead;
    auto fetch = [&](uint64_t r, auto& to) {
        r = r < a.rows ? r : 0;
        to.load((const T*)a.x + r * a.x_stride, lane, a.width, row_follows<V>(a, r));
    };
    fetch(row, x);
    for (int turn = 0; row - threadIdx.x / L < a.rows; ++turn, row += step) {
        if (row - threadIdx.x / L + step < a.rows) fetch(row + step, ahead);
        x.keep(lane, a.width);
        float sum = 0.0f, var = 0.0f;
#pragma unroll
        for (int k = 0; k < NV; ++k)
#pragma unroll
            for (int j = 0; j < V; ++j) sum += (float)x.v[k][j];
        float mean = lane_sum<L>(sum) * wave_inv;
#pragma unroll
        for (int k = 0; k < NV; ++k)
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const float d = (float)x.v[k][j] - mean;
                var += (lane + k * L) * V + j < a.width ? d * d : 0.0f;
            }
        var = lane_sum<L>(var);
        if constexpr (L > 64) {  // the waves' own means and squares about them to the row's
            const float own[3] = {mean * count, var, count};
            float w[3];
            meet(turn, own, w);
            mean = lane_sum<L / 64>(w[0]) * inv;
            const float d = w[2] > 0.0f ? w[0] / w[2] - mean : 0.0f;
            var = lane_sum<L / 64>(w[1] + w[2] * d * d);
        }
        const float rstd = 1.0f / sqrtf(var * inv + a.eps);
        if (row < a.rows) {
            if (lane == 0) {
                if (a.mean) a.mean[row] = mean;
                if (a.rstd) a.rstd[row] = rstd;
            }
            T* out = (T*)a.out + row * a.out_stride;
#pragma unroll
            for (int k = 0; k < NV; ++k) {
                const uint32_t col = (lane + k * L) * V;
                float y[V];
#pragma unroll
                for (int j = 0; j < V; ++j) y[j] = ((float)x.v[k][j] - mean) * rstd * gamma[k][j] + beta[k][j];
                if (col < a.width) store_cols<T, V>(out, col, a.width, y);
            }
        }
        x = ahead;
    }
}

// dgamma and dbeta by the block that leaves its sums last, in the blocks' order whichever it is: `threads` threads
// take two columns of a run of partial sums each, Q threads a pair. Its own launch costs 3.7 us of host time, more
// than all else of a small call. `tickets` has a word for each number of blocks, whose count wraps to 0 with the
// last one: calls that overlap on two streams against the rule spoil their own gradients, but leave every count at 0.
template <class T>
__device__ inline void join_last(const NormArgs& a, const float* partials, uint32_t* tickets, float (*red)[2], uint32_t threads) {
    typedef typename VecOf<float, 2>::type pair;
    __shared__ uint32_t before;
    __threadfence();
    __syncthreads();
    if (threadIdx.x == 0) before = atomicInc(tickets + gridDim.x, gridDim.x - 1);
    __syncthreads();
    if (before != gridDim.x - 1) return;
    __threadfence();
    const uint32_t Q = threads > a.width ? threads / a.width : 1, q = Q > 1 ? threadIdx.x / a.width : 0;
    const uint64_t cols = 2ull * a.width;
    for (uint32_t u = Q > 1 ? threadIdx.x % a.width : threadIdx.x; u < a.width; u += threads) {  // once where Q > 1
        float s0 = 0.0f, s1 = 0.0f;
        if (q < Q) {
#pragma unroll 8
            for (uint32_t p = q; p < gridDim.x; p += Q) {
                const pair v = *(const pair*)(partials + p * cols + 2 * u);
                s0 += v[0];
                s1 += v[1];
            }
        }
        if (Q > 1) {
            red[threadIdx.x][0] = s0;
            red[threadIdx.x][1] = s1;
            __syncthreads();  // every thread comes here once: u < width for all
            if (q) return;
            for (uint32_t k = 1; k < Q; ++k) {
                s0 += red[k * a.width + u][0];
                s1 += red[k * a.width + u][1];
            }
        }
        const float s[2] = {s0, s1};
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const uint32_t col = 2 * u + j;
            void* to = col < a.width ? a.dgamma : a.dbeta;
            if (to) store_param<T>(to, a.param_f32, a.accumulate, col < a.width ? col : col - a.width, s[j]);
        }
    }
}

// The adjoint, rows as in k_norm; a block keeps its columns' sums in registers, and `partials`
// [gridDim][2][width] receives them (dgamma, then dbeta); with `tickets` the last block adds them up. Measured:
// 16,384 x 4,096 bf16 82 us, 4.9 TB/s (and 7 for k_norm_params); 65,536 x 66 f32 15 us: rows of 264 bytes are as
// much latency as memory's rate.
template <class T, int L, int NV>
__global__ __launch_bounds__(L < 256 ? 256 : L) void k_norm_adjoint(NormArgs a, float* partials, uint32_t* tickets) {
    constexpr int V = 16 / sizeof(T), G = (L < 256 ? 256 : L) / L;
    __shared__ Meet<kMeetLanes<L>, 2> meet;
    constexpr int PER = L < 64 ? 64 : L;  // threads that leave one row of sums
    constexpr bool AHEAD = L < 1024 || NV * V < kPerLane;  // else the registers do not hold two rows
    __shared__ float red[L < 256 ? 256 : L][2];
    __shared__ float sums[PER < 256 ? 256 / PER : 1][PER < 256 ? 2 * NV * V * L : 1];
    const uint32_t lane = threadIdx.x % L, group = threadIdx.x / L;
    const float inv = 1.0f / (float)a.width;
    float dgamma[NV][V], dbeta[NV][V], gamma[NV][V];
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        load_params<T, V>(a.gamma, a.param_f32, (lane + k * L) * V, a.width, 1.0f, gamma[k]);
#pragma unroll
        for (int j = 0; j < V; ++j) dgamma[k][j] = dbeta[k][j] = 0.0f;
    }
    const uint64_t step = (uint64_t)gridDim.x * G;
    struct {
        Row<T, L, NV> x, dy;
        float mean, rstd;
    } now, ahead;
    // past the last row: zeros, which add nothing
    auto fetch = [&](uint64_t r, auto& to) {
        const bool live = r < a.rows;
        const bool over = row_follows<V>(a, r);
        to.x.load((const T*)a.x + (live ? r : 0) * a.x_stride, lane, live ? a.width : 0u, over);
        to.dy.load((const T*)a.dy + (live ? r : 0) * a.dy_stride, lane, live ? a.width : 0u, over);
        to.mean = live ? a.mean[r] : 0.0f;
        to.rstd = live ? a.rstd[r] : 0.0f;
    };
    uint64_t row = (uint64_t)blockIdx.x * G + group;
    fetch(row, now);
    for (int turn = 0; row - group < a.rows; ++turn, row += step) {
        const bool more = row - group + step < a.rows;
        if (AHEAD && more) fetch(row + step, ahead);
        now.x.keep(lane, row < a.rows ? a.width : 0u);
        now.dy.keep(lane, row < a.rows ? a.width : 0u);
        float s1 = 0.0f, s2 = 0.0f;
#pragma unroll
        for (int k = 0; k < NV; ++k)
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const float d = (float)now.dy.v[k][j], g = d * gamma[k][j];
                const float xh = ((float)now.x.v[k][j] - now.mean) * now.rstd;
                // lanes past the row's end: x is 0 there, not the mean
                const bool in = (lane + k * L) * V + j < a.width;
                dgamma[k][j] += in ? d * xh : 0.0f;
                dbeta[k][j] += d;
                s1 += in ? g : 0.0f;
                s2 += in ? g * xh : 0.0f;
            }
        s1 = lane_sum<L>(s1);
        s2 = lane_sum<L>(s2);
        if constexpr (L > 64) {
            const float own[2] = {s1, s2};
            float w[2];
            meet(turn, own, w);
            s1 = lane_sum<L / 64>(w[0]);
            s2 = lane_sum<L / 64>(w[1]);
        }
        s1 *= inv;
        s2 *= inv;
        if (row < a.rows && a.dx) {
            T* dx = (T*)a.dx + row * a.dx_stride;
#pragma unroll
            for (int k = 0; k < NV; ++k) {
                const uint32_t col = (lane + k * L) * V;
                float o[V];
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    const float xh = ((float)now.x.v[k][j] - now.mean) * now.rstd;
                    o[j] = now.rstd * ((float)now.dy.v[k][j] * gamma[k][j] - s1 - xh * s2);
                }
                if (col < a.width) store_cols<T, V>(dx, col, a.width, o);
            }
        }
        if (AHEAD)
            now = ahead;
        else if (more)
            fetch(row + step, now);
    }
    if (!partials) return;
    float* to = partials + (uint64_t)blockIdx.x * 2 * a.width;
    if constexpr (PER >= 256) {
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const uint32_t col = (lane + k * L) * V;
            if (col >= a.width) continue;
            store_cols<float, V>(to, col, a.width, dgamma[k]);
            store_cols<float, V>(to + a.width, col, a.width, dbeta[k]);
        }
        if (tickets) join_last<T>(a, partials, tickets, red, blockDim.x);
        return;
    }
    // a wave's groups meet in its lanes, the block's waves (or pairs of them) in LDS
    constexpr int COLS = NV * V * L;
#pragma unroll
    for (int which = 0; which < 2; ++which)
#pragma unroll
        for (int k = 0; k < NV; ++k)
#pragma unroll
            for (int j = 0; j < V; ++j) {
                float s = which ? dbeta[k][j] : dgamma[k][j];
#pragma unroll
                for (int m = L; m < 64; m *= 2) s += __shfl_xor(s, m);
                if (PER < 256 && (L >= 64 || (threadIdx.x & 63) < L))
                    sums[threadIdx.x / PER][which * COLS + (lane + k * L) * V + j] = s;
            }
    __syncthreads();
    for (uint32_t c = threadIdx.x; c < 2 * a.width; c += blockDim.x) {
        const uint32_t at = c < a.width ? c : c - a.width + COLS;
        float s = 0.0f;
#pragma unroll
        for (int q = 0; q < 256 / PER; ++q) s += sums[q][PER < 256 ? at : 0];
        to[c] = s;
    }
    if (tickets) join_last<T>(a, partials, tickets, red, blockDim.x);
}

// The same for larger calls, from `parts` rows of partial sums, in the rows' order: a second launch of 3 to 7 us instead of
// atomics, whose order would change the bits.
template <class T>
__global__ __launch_bounds__(1024) void k_norm_params(const float* partials, uint32_t parts, NormArgs a) {
    const uint64_t cols = 2ull * a.width;
    column_sums<1024>(partials, parts, cols, blockIdx.x, gridDim.x, [&](uint64_t col, float s) {
        void* to = col < a.width ? a.dgamma : a.dbeta;
        if (to) store_param<T>(to, a.param_f32, a.accumulate, col < a.width ? col : col - a.width, s);
    });
}

// Sums of two values over a block of 1,024 threads.
__device__ inline void block_sum(float& a, float& b, float* shared) {
    const int wave = threadIdx.x / 64;
    a = lane_sum<64>(a);
    b = lane_sum<64>(b);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) {
        shared[2 * wave] = a;
        shared[2 * wave + 1] = b;
    }
    __syncthreads();
    a = b = 0.0f;
#pragma unroll
    for (int k = 0; k < 16; ++k) {
        a += shared[2 * k];
        b += shared[2 * k + 1];
    }
}

// ---------------------------------------------------------------- rows wider than kRowCap
// A block reads its row three times (forward) or twice, from L2 after the first.
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
        block_sum(sum, none, shared);
        const float inv = 1.0f / (float)a.width, mean = sum * inv;
        float var = 0.0f;
        for (uint32_t col = threadIdx.x * V; col < a.width; col += 1024 * V) {
            load_cols<T, V>(x, col, a.width, v);
#pragma unroll
            for (int j = 0; j < V; ++j) var += col + j < a.width ? (v[j] - mean) * (v[j] - mean) : 0.0f;
        }
        block_sum(var, none, shared);
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
        block_sum(s1, s2, shared);
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

// The instantiation for a row width: the fewest lanes that hold the row, and of those the fewest vectors a lane; more
// than eight lanes hold more than half of their most.
template <class T, class F>
hipError_t with_row_shape(uint32_t width, F f) {
    constexpr uint32_t V = 16 / sizeof(T);
    constexpr int MOST = kPerLane / V;
    const uint32_t vecs = (width + V - 1) / V;
#define NPA_SHAPE(L, NV) \
    if (vecs <= (uint32_t)(L) * (NV)) return f(std::integral_constant<int, L>(), std::integral_constant<int, NV>())
    NPA_SHAPE(8, 1);
    NPA_SHAPE(8, 2);
#define NPA_LANES(L)                               \
    if constexpr (MOST == 4) NPA_SHAPE(L, 3);      \
    NPA_SHAPE(L, MOST)
    NPA_LANES(8);
    NPA_LANES(16);
    NPA_LANES(32);
    NPA_LANES(64);
    NPA_LANES(128);
    NPA_LANES(256);
    NPA_LANES(512);
    NPA_LANES(1024);
#undef NPA_LANES
#undef NPA_SHAPE
    return hipErrorInvalidValue;
}

template <class T>
hipError_t norm_of(const NormArgs& a, int cus, hipStream_t stream) {
    if (a.width > kRowCap) {
        hipLaunchKernelGGL(k_norm_wide<T>, dim3((uint32_t)std::min<uint64_t>(a.rows, kMostBlocks)), dim3(1024), 0, stream, a);
        return hipGetLastError();
    }
    return with_row_shape<T>(a.width, [&](auto lanes, auto nv) {
        constexpr int L = decltype(lanes)::value, NV = decltype(nv)::value, threads = L < 256 ? 256 : L;
        // about 2,048 threads a CU, each block with further rows
        const uint32_t blocks = (uint32_t)std::min<uint64_t>((a.rows + threads / L - 1) / (threads / L),
                                                             (uint64_t)cus * (2048 / threads));
        hipLaunchKernelGGL((k_norm<T, L, NV>), dim3(blocks), dim3(threads), 0, stream, a);
        return hipGetLastError();
    });
}

template <class T>
hipError_t norm_adjoint_of(const NormArgs& a, LayerWorkspace& ws, int cus, hipStream_t stream) {
    constexpr uint32_t V = 16 / sizeof(T);
    const bool params = a.dgamma || a.dbeta;
    uint32_t parts = 0;
    bool joined = false;
    hipError_t e = hipSuccess;
    auto reserve = [&] { return params ? ws.reserve(ws.partials, (uint64_t)parts * 2 * a.width * 4, stream) : hipSuccess; };
    if (a.width > kRowCap) {
        if (params) {  // before dx, which may take dy's place
            parts = (uint32_t)std::min<uint64_t>(a.rows, 64);
            if ((e = reserve()) != hipSuccess) return e;
            if (a.rows) {
                const uint32_t blocks = (a.width + 256 * V - 1) / (256 * V);
                hipLaunchKernelGGL(k_norm_wide_columns<T>, dim3(blocks, parts), dim3(256), 0, stream, a,
                                   ws.partials.as<float>());
                if ((e = hipGetLastError()) != hipSuccess) return e;
            }
        }
        if (a.dx && a.rows)
            hipLaunchKernelGGL(k_norm_wide_adjoint<T>, dim3((uint32_t)std::min<uint64_t>(a.rows, kMostBlocks)), dim3(1024), 0, stream, a);
        e = hipGetLastError();
    } else if (a.rows) {
        e = with_row_shape<T>(a.width, [&](auto lanes, auto nv) {
            constexpr int L = decltype(lanes)::value, NV = decltype(nv)::value, threads = L < 256 ? 256 : L;
            constexpr uint32_t G = threads / L;
            // a thread has two rows' vectors of two arrays in flight: 512 threads a CU, 2,048 where they have
            // one vector and the block at least four groups of rows. Each block leaves one row of partial
            // sums: at 16,384 x 4,096 bf16 2,048 threads took 12 % longer and 256 took 55 %, and at
            // 1,500,000 x 18 f32 512 took three times as long as 2,048.
            const uint64_t groups = (a.rows + G - 1) / G;
            const uint64_t most = std::max<uint64_t>((uint64_t)cus * std::max(1, 512 / threads),
                                                     std::min<uint64_t>((uint64_t)cus * (2048 / (NV * NV) / threads), groups / 4));
            parts = (uint32_t)std::min<uint64_t>(groups, most);
            // Small calls join in the last block: as many blocks as leave kJoinLoads sums to a thread of it, if
            // that makes no more than kJoinTurns groups of rows a block. Measured, f32, us a call: 800 x 66 11.2, in
            // two launches 14.5; past the limits it turns: 2,304 x 66 with 24 sums a thread 18.3, 96 x 1,023 with
            // 24 and four turns 18.3, 1 x 16,384 with 16 21.9.
            const uint64_t few = std::min<uint64_t>(kJoinParts, a.width < (uint32_t)threads
                                                                    ? kJoinLoads * (threads / a.width)
                                                                    : kJoinLoads / ((a.width + threads - 1) / threads));
            uint32_t* tickets = nullptr;
            if (params && groups <= few * kJoinTurns) {
                parts = (uint32_t)std::min<uint64_t>(parts, few);
                const hipError_t r = ws.reserve_tickets((kJoinParts + 1) * sizeof(uint32_t));
                if (r != hipSuccess) return r;
                tickets = ws.tickets.as<uint32_t>();
                joined = true;
            }
            hipError_t r = reserve();
            if (r != hipSuccess) return r;
            hipLaunchKernelGGL((k_norm_adjoint<T, L, NV>), dim3(parts), dim3(threads), 0, stream, a,
                               params ? ws.partials.as<float>() : (float*)nullptr, tickets);
            return hipGetLastError();
        });
    }
    if (e != hipSuccess || !params || joined) return e;
    hipLaunchKernelGGL(k_norm_params<T>, dim3((uint32_t)std::min<uint64_t>((2ull * a.width + 15) / 16, kMostBlocks)), dim3(1024), 0, stream,
                       ws.partials.as<float>(), parts, a);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_layer_norm(const NormArgs& a, int cus, hipStream_t stream) {
    if (!a.rows) return hipSuccess;
    if (a.type == NPA_TYPE_F32) return norm_of<float>(a, cus, stream);
    if (a.type == NPA_TYPE_BF16) return norm_of<__bf16>(a, cus, stream);
    return norm_of<_Float16>(a, cus, stream);
}

hipError_t launch_layer_norm_adjoint(const NormArgs& a, LayerWorkspace& ws, int cus, hipStream_t stream) {
    if (a.type == NPA_TYPE_F32) return norm_adjoint_of<float>(a, ws, cus, stream);
    if (a.type == NPA_TYPE_BF16) return norm_adjoint_of<__bf16>(a, ws, cus, stream);
    return norm_adjoint_of<_Float16>(a, ws, cus, stream);
}

}  // namespace npa
