// npa_route.hip - rows to experts and back: the router's choice and weights, the plan that sorts rows by expert, the
// weighted sum of the experts' rows, and the adjoints.
//
// Scores s = softmax(l) or sigma(l); the top_k experts by s + b (without a bias by l, of which s is monotone), of the
// best groups where there are groups; weights s, divided by their sum + 1e-20 where they are renormalised.
#include <algorithm>
#include <type_traits>

#include "npa_layers.hpp"

namespace npa {
namespace {

constexpr float kSumEps = 1e-20f;

// LDS that only the lanes of one wave share: its instructions execute in order.
__device__ inline void wave_sync() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_wave_barrier();
}

// Maximum over a group of L lanes of a wave, the same in each of them.
template <int L, int M = 1>
__device__ inline float lane_max(float v) {
    if constexpr (M < L) return lane_max<L, M * 2>(fmaxf(v, partner<M>(v)));
    return v;
}
template <int L, int M = 1>
__device__ inline uint32_t lane_max(uint32_t v) {
    if constexpr (M < L) return lane_max<L, M * 2>(max(v, __float_as_uint(partner<M>(__uint_as_float(v)))));
    return v;
}
template <int L, int M = 1>
__device__ inline uint64_t lane_max(uint64_t v) {
    if constexpr (M < L) return lane_max<L, M * 2>(max(v, (uint64_t)__shfl_xor((unsigned long long)v, M)));
    return v;
}
template <int L, int M = 1>
__device__ inline double lane_sum(double v) {
    if constexpr (M < L) return lane_sum<L, M * 2>(v + __shfl_xor(v, M));
    return v;
}

// The bits of a ballot that belong to this thread's group of L lanes.
template <int L>
__device__ inline uint64_t own_lanes(uint64_t ballot) {
    if (L == 64) return ballot;
    return ballot >> (threadIdx.x & 63 & ~(L - 1)) & ((1ull << (L & 63)) - 1);
}

// Keys as whole numbers of the same order, 0 below all of them; NaN is the largest, as in a sort.
__device__ inline uint32_t ordered(float v) {
    const uint32_t u = __float_as_uint(v + 0.0f);
    return v != v ? 0xffffffffu : u ^ ((uint32_t)((int32_t)u >> 31) | 0x80000000u);
}
__device__ inline uint64_t ordered(double v) {
    const uint64_t u = (uint64_t)__double_as_longlong(v + 0.0);
    return v != v ? ~0ull : u ^ ((uint64_t)((int64_t)u >> 63) | 0x8000000000000000ull);
}
__device__ inline float unordered(uint32_t u) {
    return __uint_as_float(u >> 31 ? u ^ 0x80000000u : ~u);
}
__device__ inline double unordered(uint64_t u) {
    return __longlong_as_double((long long)(u >> 63 ? u ^ 0x8000000000000000ull : ~u));
}
template <class F>
struct KeyOf;
template <>
struct KeyOf<float> {
    typedef uint32_t type;
};
template <>
struct KeyOf<double> {
    typedef uint64_t type;
};

template <class F>
__device__ inline F sigmoid_of(F x) {
    if constexpr (sizeof(F) == 4)
        return 1.0f / (1.0f + expf(-x));
    else
        return 1.0 / (1.0 + exp(-x));
}

// What a row chose, and the runner-up behind it.
struct Choice {
    uint32_t expert;
    float x, b, key;
};

// A row's experts in L lanes, V to a lane one after the other.
template <int L, int V>
struct Router {
    float x[V], b[V];
    uint32_t open;    // bit v: expert v of this lane may be chosen
    float most, inv;  // of the softmax
    // Two f32 keys further apart are in the exact order. A key is off by 2^-24 (33 s + |b| + 1) at most, s the row's largest
    // score: a sum of exponentials (16 in a lane, then six levels), each 2 ulp off, of differences rounded once (x - max is off
    // by 2^-24 |x - max|, which exp(x - max) makes 0.37 2^-24 at most), and the roundings of the quotient and of the key.
    float apart;
};

// The best top_k experts of a row (and the runner-up) to `to`, by keys of type F. Returns how many; `certain` becomes
// false where f32 does not tell the exact order. KEYED: by s + b, and groups; else by the logits themselves.
template <class F, bool KEYED, int L, int V>
__device__ inline uint32_t choose(const RouteArgs& a, const Router<L, V>& r, char* shared, Choice* to, bool& certain) {
    typedef typename KeyOf<F>::type Key;
    const uint32_t lane = threadIdx.x % L, first = lane * V;
    Key key[V];
    if constexpr (KEYED) {
        F f[V];
        double inv = 0.0;
        if (sizeof(F) == 8 && !a.sigmoid) {
            double sum = 0.0;
#pragma unroll
            for (int v = 0; v < V; ++v) {
                f[v] = (F)exp((double)r.x[v] - r.most);
                sum += f[v];
            }
            inv = 1.0 / lane_sum<L>(sum);
        }
#pragma unroll
        for (int v = 0; v < V; ++v) {
            if (a.sigmoid)
                f[v] = sigmoid_of((F)r.x[v]);
            else if (sizeof(F) == 8)
                f[v] *= (F)inv;
            else
                f[v] = expf(r.x[v] - r.most) * r.inv;
            key[v] = r.open >> v & 1 ? ordered(f[v] + (F)r.b[v]) : 0;
        }
        if (a.groups > 1) {
            // a group's score is the sum of its two largest keys; `lanes` lanes look at one group
            const uint32_t size = a.count / a.groups;
            char* own = shared + threadIdx.x / L * (a.count + a.groups) * 8;  // waves of either key have places of their own
            Key* score = (Key*)(own + a.count * 8);
            uint32_t lanes = 1;
            while (lanes * 2 * a.groups <= (uint32_t)L) lanes *= 2;
            wave_sync();
            if constexpr (sizeof(F) == 4) {
                Key* keys = (Key*)own;
#pragma unroll
                for (int v = 0; v < V; ++v)
                    if (first + v < a.count) keys[first + v] = key[v];
                wave_sync();
                for (uint32_t g0 = 0; g0 < a.groups; g0 += L / lanes) {
                    const uint32_t g = g0 + lane / lanes;
                    Key best = 0, second = 0;
                    if (g < a.groups)
                        for (uint32_t i = lane % lanes; i < size; i += lanes) {
                            const Key k = keys[g * size + i];
                            second = max(second, min(best, k));
                            best = max(best, k);
                        }
                    for (uint32_t m = 1; m < lanes; m *= 2) {
                        const Key b2 = __shfl_xor(best, m), s2 = __shfl_xor(second, m);
                        second = max(max(second, s2), min(best, b2));
                        best = max(best, b2);
                    }
                    if (g < a.groups && lane % lanes == 0)
                        score[g] = !best ? 0 : ordered(second ? unordered(best) + unordered(second) : unordered(best));
                }
            } else {  // as (s + s') + (b + b'): groups of the same scores and biases are equal whichever bias goes with which score
                float2* pair = (float2*)own;
#pragma unroll
                for (int v = 0; v < V; ++v)
                    if (first + v < a.count) pair[first + v] = {r.open >> v & 1 ? r.x[v] : -INFINITY, r.b[v]};
                wave_sync();
                struct Best {
                    uint64_t key;
                    double s;
                    float b;
                };
                for (uint32_t g = lane; g < a.groups; g += L) {
                    Best best = {0, 0.0, 0.0f}, second = best;
                    for (uint32_t i = g * size; i < (g + 1) * size; ++i) {
                        const float2 e = pair[i];
                        if (e.x == -INFINITY) continue;
                        const double s = a.sigmoid ? sigmoid_of((double)e.x) : exp((double)e.x - r.most) * inv;
                        const Best k = {ordered(s + (double)e.y), s, e.y};
                        if (k.key > best.key) {
                            second = best;
                            best = k;
                        } else if (k.key > second.key) {
                            second = k;
                        }
                    }
                    score[g] = best.key ? ordered((best.s + second.s) + ((double)best.b + (double)second.b)) : 0;
                }
            }
            wave_sync();
            // a group stays if fewer than top_groups are ahead of it
            Key least = ~(Key)0, next = 0;  // of those that stay, and of the others
            uint64_t kept = 0;
            for (uint32_t g0 = 0; g0 < a.groups; g0 += L) {
                const uint32_t g = g0 + lane;
                uint32_t ahead = 0;
                const Key own = g < a.groups ? score[g] : 0;
                for (uint32_t h = 0; h < a.groups; ++h) {
                    const Key other = score[h];
                    ahead += other > own || (other == own && h < g);
                }
                const bool stays = own && ahead < a.top_groups;
                if (stays)
                    least = min(least, own);
                else
                    next = max(next, own);
                kept |= own_lanes<L>(__ballot(stays)) << g0;
            }
            if constexpr (sizeof(F) == 4) {
                next = lane_max<L>(next);
                least = ~lane_max<L>((Key)~least);
                if (next && !(unordered(least) - unordered(next) > 4.0f * r.apart)) certain = false;
            }
#pragma unroll
            for (int v = 0; v < V; ++v)
                if (first + v < a.count && !(kept >> (first + v) / size & 1)) key[v] = 0;
        }
    } else {
#pragma unroll
        for (int v = 0; v < V; ++v) key[v] = r.open >> v & 1 ? ordered((F)r.x[v]) : 0;
    }
    // the largest key again and again; of equal ones the lowest lane's, and there the lowest
    const uint32_t wanted = KEYED && sizeof(F) == 4 ? a.top_k + 1 : a.top_k;
    uint32_t found = 0;
    wave_sync();
    while (found < wanted) {
        Key own = key[0];
#pragma unroll
        for (int v = 1; v < V; ++v) own = max(own, key[v]);
        const Key best = lane_max<L>(own);
        if (!best) break;
        const uint64_t at = own_lanes<L>(__ballot(own == best));
        if (lane == (uint32_t)__builtin_ctzll(at)) {
            bool done = false;
#pragma unroll
            for (int v = 0; v < V; ++v)
                if (!done && key[v] == best) {
                    done = true;
                    key[v] = 0;
                    to[found] = Choice{first + v, r.x[v], r.b[v], (float)unordered(best)};
                }
        }
        ++found;
    }
    wave_sync();
    if constexpr (KEYED && sizeof(F) == 4) {
        bool near = false;
        for (uint32_t i = lane + 1; i < found; i += L) {
            const Choice p = to[i - 1], q = to[i];
            near |= !(p.key - q.key > r.apart) && !(p.x == q.x && p.b == q.b);  // the same inputs: the lower expert, exactly
        }
        if (own_lanes<L>(__ballot(near))) certain = false;
    }
    return min(found, a.top_k);
}

// Rows to groups of L lanes. The selection is exact: keys in f32, and in f64 for a wave of rows of which one has keys too
// near each other for f32 to tell (0.2 % of rows of 256 sigmoid scores).
template <class T, int L, int V, bool KEYED>
__global__ __launch_bounds__(256) void k_route(RouteArgs a) {
    extern __shared__ __align__(16) char shared[];
    constexpr uint32_t ROWS = 256 / L;
    const uint32_t lane = threadIdx.x % L, first = lane * V, in_block = threadIdx.x / L;
    Choice* to = (Choice*)shared + in_block * (a.top_k + 1);
    char* groups = shared + ROWS * (a.top_k + 1) * sizeof(Choice);
    Router<L, V> r;
    uint32_t exists = 0;
    float bias = 0.0f;
#pragma unroll
    for (int v = 0; v < V; ++v) {
        r.b[v] = 0.0f;
        if (first + v < a.count) {
            if (a.bias) r.b[v] = load_param<T>(a.bias, a.bias_f32, first + v);
            if (r.b[v] != -INFINITY) {
                exists |= 1u << v;
                bias = fmaxf(bias, fabsf(r.b[v]));
            }
        }
    }
    bias = lane_max<L>(bias);
    for (uint64_t base = (uint64_t)blockIdx.x * ROWS; base < a.rows; base += (uint64_t)gridDim.x * ROWS) {
        const uint64_t own = base + in_block, row = own < a.rows ? own : a.rows - 1;
        const T* x = (const T*)a.logits + row * a.stride;
        if (first + V <= a.count) {
            const typename VecOf<T, V>::type w = *(const typename VecOf<T, V>::type*)(x + first);
#pragma unroll
            for (int v = 0; v < V; ++v) r.x[v] = (float)w[v];
        } else {
#pragma unroll
            for (int v = 0; v < V; ++v) r.x[v] = first + v < a.count ? (float)x[first + v] : -INFINITY;
        }
        float most = -INFINITY, sum = 0.0f;
        r.open = exists;
#pragma unroll
        for (int v = 0; v < V; ++v) {
            most = fmaxf(most, r.x[v]);
            if (r.x[v] == -INFINITY) r.open &= ~(1u << v);
        }
        r.inv = 1.0f;
        if (!a.sigmoid) {  // of all logits, a closed one's is 0
            most = lane_max<L>(most);
            r.most = most == -INFINITY ? 0.0f : most;
#pragma unroll
            for (int v = 0; v < V; ++v) sum += expf(r.x[v] - r.most);
            r.inv = 1.0f / lane_sum<L>(sum);
        }
        r.apart = 0x1p-23f * (33.0f * (a.sigmoid ? 1.0f : r.inv) + bias + 1.0f);
        bool certain = true;
        uint32_t found = choose<float, KEYED>(a, r, groups, to, certain);
        if (KEYED && __any(!certain)) found = choose<double, KEYED>(a, r, groups, to, certain);
        // weights: a lane for each choice
        float total = 0.0f;
        auto score = [&](uint32_t j) {
            if (j >= found) return 0.0f;
            return a.sigmoid ? sigmoid_of(to[j].x) : expf(to[j].x - r.most) * r.inv;
        };
        if (a.renormalise) {
            for (uint32_t j = lane; j < a.top_k; j += L) total += score(j);
            total = lane_sum<L>(total) + kSumEps;
        }
        if (own < a.rows)
            for (uint32_t j = lane; j < a.top_k; j += L) {
                const float s = score(j);
                a.experts[own * a.top_k + j] = j < found ? (int32_t)to[j].expert : -1;
                a.weights[own * a.top_k + j] = (a.renormalise ? s / total : s) * a.scale;
            }
    }
}

// The gradient of the logits. With Z = sum s_j + 1e-20 over the choices, ds_j = scale (g_j - sum g s / Z) / Z where
// the weights are renormalised, else scale g_j; dl = s (ds - sum_j ds_j s_j) through the softmax, where that sum is
// scale sum(g s) 1e-20 / Z^2 for renormalised weights (no difference of nearly equal sums); ds s (1 - s) through sigma.
// Bound by memory.
template <class T, int L, int V>
__global__ __launch_bounds__(256) void k_route_adjoint(RouteArgs a) {
    constexpr uint32_t ROWS = 256 / L;
    const uint32_t lane = threadIdx.x % L, first = lane * V, in_block = threadIdx.x / L;
    for (uint64_t base = (uint64_t)blockIdx.x * ROWS; base < a.rows; base += (uint64_t)gridDim.x * ROWS) {
        const uint64_t own = base + in_block, row = own < a.rows ? own : a.rows - 1;
        const T* logits = (const T*)a.logits + row * a.stride;
        float x[V];
        if (first + V <= a.count) {
            const typename VecOf<T, V>::type w = *(const typename VecOf<T, V>::type*)(logits + first);
#pragma unroll
            for (int v = 0; v < V; ++v) x[v] = (float)w[v];
        } else {
#pragma unroll
            for (int v = 0; v < V; ++v) x[v] = first + v < a.count ? (float)logits[first + v] : -INFINITY;
        }
        float most = 0.0f, inv = 1.0f;
        if (!a.sigmoid) {
            most = x[0];
#pragma unroll
            for (int v = 1; v < V; ++v) most = fmaxf(most, x[v]);
            most = lane_max<L>(most);
            most = most == -INFINITY ? 0.0f : most;
            float sum = 0.0f;
#pragma unroll
            for (int v = 0; v < V; ++v) sum += expf(x[v] - most);
            inv = lane_sum<L>(sum);
            inv = inv > 0.0f || inv != inv ? 1.0f / inv : 0.0f;  // a row of closed experts: scores of 0
        }
        auto score = [&](float l) { return a.sigmoid ? sigmoid_of(l) : expf(l - most) * inv; };
        // each choice in all lanes: its expert's logit comes from the cache
        const int32_t* chosen = a.experts + row * a.top_k;
        const float* dw = a.dweights + row * a.top_k;
        float z = kSumEps, gs = 0.0f;
        for (uint32_t j = 0; j < a.top_k; ++j) {
            const uint32_t e = (uint32_t)chosen[j];
            if (e >= a.count) continue;
            const float s = score((float)logits[e]);
            z += s;
            gs += dw[j] * s;
        }
        const float through = a.renormalise ? gs / z : 0.0f, by = a.renormalise ? a.scale / z : a.scale;
        const float all = a.sigmoid ? 0.0f : a.renormalise ? by * gs * (kSumEps / z) : by * gs;
        float ds[V];
#pragma unroll
        for (int v = 0; v < V; ++v) ds[v] = 0.0f;
        for (uint32_t j = 0; j < a.top_k; ++j) {
            const uint32_t at = (uint32_t)chosen[j] - first;
            const float g = by * (dw[j] - through);
#pragma unroll
            for (int v = 0; v < V; ++v) ds[v] += at == (uint32_t)v ? g : 0.0f;
        }
        if (own >= a.rows) continue;
        T* out = (T*)a.dlogits + own * a.dstride;
        typename VecOf<T, V>::type o;
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const float s = score(x[v]);
            o[v] = (T)(a.sigmoid ? ds[v] * s * (1.0f - s) : s * (ds[v] - all));
        }
        if (first + V <= a.count)
            *(typename VecOf<T, V>::type*)(out + first) = o;
        else
#pragma unroll
            for (int v = 0; v < V; ++v)
                if (first + v < a.count) out[first + v] = o[v];
    }
}

// ------------------------------------------------------------------ the plan
// A stable counting sort. A block has a run of kChunk entries, each of its waves an equal part of it, 64 at a time.
constexpr uint32_t kChunk = 2048, kSmallPlan = 16384;

__device__ inline uint32_t plan_key(const PlanArgs& p, uint32_t i) { return min((uint32_t)p.chosen[i], p.experts); }

// Entries begin .. end - 1 by key in `counts`, which is cleared first. Every thread of the block calls it.
__device__ inline void count_keys(const PlanArgs& p, uint32_t begin, uint32_t end, uint32_t step, uint32_t lane, uint32_t* counts) {
    for (uint32_t i = begin + lane; i < end; i += step) atomicAdd(counts + plan_key(p, i), 1u);
}

// Exclusive sums of `n` words in LDS, in place, by all threads of the block; returns their total.
template <int THREADS>
__device__ inline uint32_t exclusive(uint32_t* v, uint32_t n, uint32_t* waves) {
    const uint32_t per = (n + THREADS - 1) / THREADS, begin = min(threadIdx.x * per, n), end = min(begin + per, n);
    uint32_t sum = 0;
    for (uint32_t i = begin; i < end; ++i) sum += v[i];
    uint32_t upto = sum;
#pragma unroll
    for (int m = 1; m < 64; m *= 2) {
        const uint32_t o = __shfl_up(upto, m);
        if ((threadIdx.x & 63) >= (uint32_t)m) upto += o;
    }
    if ((threadIdx.x & 63) == 63) waves[threadIdx.x / 64] = upto;
    __syncthreads();
    uint32_t before = 0, all = 0;
    for (uint32_t w = 0; w < THREADS / 64; ++w) {
        before += w < threadIdx.x / 64 ? waves[w] : 0;
        all += waves[w];
    }
    upto += before - sum;
    for (uint32_t i = begin; i < end; ++i) {
        const uint32_t c = v[i];
        v[i] = upto;
        upto += c;
    }
    __syncthreads();
    return all;
}

// counts[key][block]: a block's entries of each key
__global__ __launch_bounds__(256) void k_plan_count(PlanArgs p, uint32_t* counts) {
    __shared__ uint32_t own[kMostExperts + 1];
    for (uint32_t e = threadIdx.x; e <= p.experts; e += 256) own[e] = 0;
    __syncthreads();
    const uint32_t begin = blockIdx.x * kChunk;
    count_keys(p, begin, min(begin + kChunk, p.entries), 256, threadIdx.x, own);
    __syncthreads();
    for (uint32_t e = threadIdx.x; e <= p.experts; e += 256) counts[(uint64_t)e * gridDim.x + blockIdx.x] = own[e];
}

// A key's counts to their exclusive sums over the blocks, and its total to totals[key]
__global__ __launch_bounds__(256) void k_plan_scan(uint32_t* counts, uint32_t* totals, uint32_t blocks) {
    __shared__ uint32_t waves[4], carry;
    uint32_t* c = counts + (uint64_t)blockIdx.x * blocks;
    uint32_t before = 0;
    for (uint32_t base = 0; base < blocks; base += 256) {
        const uint32_t at = base + threadIdx.x, own = at < blocks ? c[at] : 0;
        uint32_t upto = own;
#pragma unroll
        for (int m = 1; m < 64; m *= 2) {
            const uint32_t o = __shfl_up(upto, m);
            if ((threadIdx.x & 63) >= (uint32_t)m) upto += o;
        }
        __syncthreads();
        if ((threadIdx.x & 63) == 63) waves[threadIdx.x / 64] = upto;
        __syncthreads();
        uint32_t all = 0;
        for (uint32_t w = 0; w < 4; ++w) {
            upto += w < threadIdx.x / 64 ? waves[w] : 0;
            all += waves[w];
        }
        if (at < blocks) c[at] = before + upto - own;
        before += all;
    }
    if (threadIdx.x == 0) totals[blockIdx.x] = before;
}

// Entries to their slots. `counts` null: one block has all entries and counts them itself.
template <int THREADS>
__global__ __launch_bounds__(THREADS) void k_plan_place(PlanArgs p, const uint32_t* counts, const uint32_t* totals) {
    constexpr uint32_t WAVES = THREADS / 64;
    extern __shared__ uint32_t lds[];
    __shared__ uint32_t waves[WAVES];
    const uint32_t keys = p.experts + 1, wave = threadIdx.x / 64, lane = threadIdx.x & 63;
    uint32_t *base = lds, *next = lds + keys + wave * keys;  // next[wave][key]
    const uint32_t chunk = counts ? kChunk : p.entries, first = blockIdx.x * chunk, last = min(first + chunk, p.entries);
    const uint32_t part = (chunk + THREADS - 1) / THREADS * 64, begin = min(first + wave * part, last), end = min(begin + part, last);
    for (uint32_t i = threadIdx.x; i < keys * WAVES; i += THREADS) lds[keys + i] = 0;
    __syncthreads();
    count_keys(p, begin, end, 64, lane, next);
    __syncthreads();
    for (uint32_t e = threadIdx.x; e < keys; e += THREADS) {
        uint32_t sum = 0;
        for (uint32_t w = 0; w < WAVES; ++w) sum += lds[keys + w * keys + e];
        base[e] = totals ? totals[e] : sum;
    }
    __syncthreads();
    exclusive<THREADS>(base, keys, waves);
    if (blockIdx.x == 0)
        for (uint32_t e = threadIdx.x; e < keys; e += THREADS) p.offsets[e] = (int32_t)base[e];
    for (uint32_t e = threadIdx.x; e < keys; e += THREADS) {
        uint32_t at = base[e] + (counts ? counts[(uint64_t)e * gridDim.x + blockIdx.x] : 0);
        for (uint32_t w = 0; w < WAVES; ++w) {
            const uint32_t c = lds[keys + w * keys + e];
            lds[keys + w * keys + e] = at;
            at += c;
        }
    }
    __syncthreads();
    const int bits = 32 - __builtin_clz(p.experts);
    for (uint32_t at = begin; at < end; at += 64) {
        const uint32_t i = at + lane;
        const bool in = i < end;
        const uint32_t key = in ? plan_key(p, i) : 0;
        uint64_t same = __ballot(in);
        for (int b = 0; b < bits; ++b) {
            const uint64_t set = __ballot(key >> b & 1);
            same &= key >> b & 1 ? set : ~set;
        }
        if (in) {
            const uint32_t rank = __popcll(same & ((1ull << lane) - 1)), slot = next[key] + rank;
            wave_sync();
            if (rank == 0) next[key] += __popcll(same);
            p.order[slot] = (int32_t)i;
            p.slots[i] = (int32_t)slot;
        }
        wave_sync();
    }
}

// ------------------------------------------------------------------ rows from slots and back
// The entries past the experts' last slot have no expert: they add nothing, whatever their rows hold.
__device__ inline uint32_t live_slots(const CombineArgs& a) {
    const uint64_t all = a.rows * a.top_k;
    const uint32_t n = a.offsets ? (uint32_t)a.offsets[a.experts] : ~0u;
    return n < all ? n : (uint32_t)all;
}

template <class T, int V>
__device__ inline void load_unit(const T* p, uint32_t n, float (&o)[V]) {
    if (n >= V) {
        const typename VecOf<T, V>::type v = *(const typename VecOf<T, V>::type*)p;
#pragma unroll
        for (int j = 0; j < V; ++j) o[j] = (float)v[j];
    } else {
#pragma unroll
        for (int j = 0; j < V; ++j) o[j] = j < (int)n ? (float)p[j] : 0.0f;
    }
}
template <class T, int V>
__device__ inline void store_unit(T* p, uint32_t n, const float (&o)[V]) {
    if (n >= V) {
        typename VecOf<T, V>::type v;
#pragma unroll
        for (int j = 0; j < V; ++j) v[j] = (T)o[j];
        *(typename VecOf<T, V>::type*)p = v;
    } else {
#pragma unroll
        for (int j = 0; j < V; ++j)
            if (j < (int)n) p[j] = (T)o[j];
    }
}

// out = residual + sum_j w_j y[slot_j], summed in the order of j. `lanes` lanes to a row, V elements each.
template <class Y, class T>
__global__ __launch_bounds__(256) void k_combine(CombineArgs a, uint32_t lanes) {
    constexpr int V = 16 / sizeof(T);
    const uint32_t lane = threadIdx.x % lanes, rows = 256 / lanes, live = live_slots(a);
    for (uint64_t row = (uint64_t)blockIdx.x * rows + threadIdx.x / lanes; row < a.rows; row += (uint64_t)gridDim.x * rows) {
        const int32_t* slots = a.slots + row * a.top_k;
        for (uint32_t col = lane * V; col < a.width; col += lanes * V) {
            const uint32_t n = a.width - col;
            float sum[V];
#pragma unroll
            for (int v = 0; v < V; ++v) sum[v] = 0.0f;
            for (uint32_t j = 0; j < a.top_k; ++j) {
                const uint32_t slot = (uint32_t)slots[j];
                if (slot >= live) continue;
                float y[V];
                load_unit<Y, V>((const Y*)a.y + slot * a.y_stride + col, n, y);
                const float w = a.weights ? a.weights[row * a.top_k + j] : 1.0f;
#pragma unroll
                for (int v = 0; v < V; ++v) sum[v] += w * y[v];
            }
            if (a.residual) {
                float x[V];
                load_unit<T, V>((const T*)a.residual + row * a.residual_stride + col, n, x);
#pragma unroll
                for (int v = 0; v < V; ++v) sum[v] += x[v];
            }
            store_unit<T, V>((T*)a.out + row * a.out_stride + col, n, sum);
        }
    }
}

// dy[slot_j] = w_j dout, dw_j = sum y[slot_j] dout; rows of slots without an expert are 0, and so are their weights'.
template <class T, int L>
__global__ __launch_bounds__(256) void k_combine_adjoint(CombineArgs a) {
    constexpr int V = 16 / sizeof(T);
    constexpr uint32_t ROWS = 256 / L;
    const uint32_t lane = threadIdx.x % L, live = live_slots(a);
    const uint64_t all = a.rows * a.top_k;
    for (uint64_t base = (uint64_t)blockIdx.x * ROWS; base < a.rows; base += (uint64_t)gridDim.x * ROWS) {
        const uint64_t row = base + threadIdx.x / L;
        if (row >= a.rows) continue;
        const T* dout = (const T*)a.dout + row * a.dout_stride;
        for (uint32_t j = 0; j < a.top_k; ++j) {
            const uint64_t entry = row * a.top_k + j;
            const uint32_t slot = (uint32_t)a.slots[entry];
            if (slot >= all) continue;
            const bool has = slot < live;
            const float w = !has ? 0.0f : a.weights ? a.weights[entry] : 1.0f;
            float dot = 0.0f;
            for (uint32_t col = lane * V; col < a.width; col += L * V) {
                const uint32_t n = a.width - col;
                float d[V], y[V];
                load_unit<T, V>(dout + col, n, d);
                if (a.dweights && has) {
                    load_unit<T, V>((const T*)a.y + slot * a.y_stride + col, n, y);
#pragma unroll
                    for (int v = 0; v < V; ++v) dot += y[v] * d[v];
                }
                if (a.dy) {
#pragma unroll
                    for (int v = 0; v < V; ++v) d[v] = has ? w * d[v] : 0.0f;
                    store_unit<T, V>((T*)a.dy + slot * a.dy_stride + col, n, d);
                }
            }
            if (a.dweights) {
                dot = lane_sum<L>(dot);
                if (lane == 0) a.dweights[entry] = dot;
            }
        }
    }
}

// ------------------------------------------------------------------ launches
// The fewest lanes that hold a row's experts, four to a lane where there are more than 16.
template <class F>
hipError_t with_experts(uint32_t count, F f) {
#define NPA_EXPERTS(L, V) \
    if (count <= (L) * (V)) return f(std::integral_constant<int, L>(), std::integral_constant<int, V>())
    NPA_EXPERTS(8, 1);
    NPA_EXPERTS(8, 2);
    NPA_EXPERTS(8, 4);
    NPA_EXPERTS(16, 4);
    NPA_EXPERTS(32, 4);
    NPA_EXPERTS(64, 4);
    NPA_EXPERTS(64, 8);
    NPA_EXPERTS(64, 16);
#undef NPA_EXPERTS
    return hipErrorInvalidValue;
}

template <class T>
hipError_t route_of(const RouteArgs& a, int cus, hipStream_t stream) {
    return with_experts(a.count, [&](auto lanes, auto per) {
        constexpr int L = decltype(lanes)::value, V = decltype(per)::value;
        constexpr uint32_t rows = 256 / L;
        const bool keyed = a.bias || a.groups > 1;
        const uint32_t lds = rows * ((a.top_k + 1) * (uint32_t)sizeof(Choice) + (a.groups > 1 ? (a.count + a.groups) * 8 : 0));
        const dim3 grid((uint32_t)std::min<uint64_t>((a.rows + rows - 1) / rows, (uint64_t)cus * 16)), block(256);
        if (keyed)
            hipLaunchKernelGGL((k_route<T, L, V, true>), grid, block, lds, stream, a);
        else
            hipLaunchKernelGGL((k_route<T, L, V, false>), grid, block, lds, stream, a);
        return hipGetLastError();
    });
}

template <class T>
hipError_t route_adjoint_of(const RouteArgs& a, int cus, hipStream_t stream) {
    return with_experts(a.count, [&](auto lanes, auto per) {
        constexpr int L = decltype(lanes)::value, V = decltype(per)::value;
        constexpr uint32_t rows = 256 / L;
        const dim3 grid((uint32_t)std::min<uint64_t>((a.rows + rows - 1) / rows, (uint64_t)cus * 16));
        hipLaunchKernelGGL((k_route_adjoint<T, L, V>), grid, dim3(256), 0, stream, a);
        return hipGetLastError();
    });
}

template <class Y, class T>
hipError_t combine_of(const CombineArgs& a, int cus, hipStream_t stream) {
    constexpr uint32_t V = 16 / sizeof(T);
    uint32_t lanes = 1;
    while (lanes < 256 && lanes * V < a.width) lanes *= 2;
    const uint64_t blocks = (a.rows + 256 / lanes - 1) / (256 / lanes);
    hipLaunchKernelGGL((k_combine<Y, T>), dim3((uint32_t)std::min<uint64_t>(blocks, (uint64_t)cus * 32)), dim3(256), 0, stream, a, lanes);
    return hipGetLastError();
}

template <class T>
hipError_t combine_adjoint_of(const CombineArgs& a, int cus, hipStream_t stream) {
    constexpr uint32_t V = 16 / sizeof(T);
    auto launch = [&](auto lanes) {
        constexpr int L = decltype(lanes)::value;
        const uint64_t blocks = (a.rows + 256 / L - 1) / (256 / L);
        hipLaunchKernelGGL((k_combine_adjoint<T, L>), dim3((uint32_t)std::min<uint64_t>(blocks, (uint64_t)cus * 32)), dim3(256), 0, stream, a);
        return hipGetLastError();
    };
    if (a.width <= 8 * V) return launch(std::integral_constant<int, 8>());
    if (a.width <= 16 * V) return launch(std::integral_constant<int, 16>());
    return launch(std::integral_constant<int, 64>());
}

}  // namespace

hipError_t launch_route(const RouteArgs& a, int cus, hipStream_t stream) {
    if (!a.rows) return hipSuccess;
    if (a.type == NPA_TYPE_F32) return route_of<float>(a, cus, stream);
    if (a.type == NPA_TYPE_BF16) return route_of<__bf16>(a, cus, stream);
    return route_of<_Float16>(a, cus, stream);
}

hipError_t launch_route_adjoint(const RouteArgs& a, int cus, hipStream_t stream) {
    if (!a.rows) return hipSuccess;
    if (a.type == NPA_TYPE_F32) return route_adjoint_of<float>(a, cus, stream);
    if (a.type == NPA_TYPE_BF16) return route_adjoint_of<__bf16>(a, cus, stream);
    return route_adjoint_of<_Float16>(a, cus, stream);
}

hipError_t launch_plan(const PlanArgs& p, LayerWorkspace& ws, hipStream_t stream) {
    const uint32_t keys = p.experts + 1;
    if (p.entries <= kSmallPlan && keys <= 512) {
        constexpr int THREADS = 1024;
        hipLaunchKernelGGL((k_plan_place<THREADS>), dim3(1), dim3(THREADS), keys * (1 + THREADS / 64) * 4, stream, p,
                           (const uint32_t*)nullptr, (const uint32_t*)nullptr);
        return hipGetLastError();
    }
    const uint32_t blocks = (p.entries + kChunk - 1) / kChunk;
    hipError_t e = ws.reserve(ws.counts, (uint64_t)keys * (blocks + 1) * 4, stream);
    if (e != hipSuccess) return e;
    uint32_t *counts = ws.counts.as<uint32_t>(), *totals = counts + (uint64_t)keys * blocks;
    if (blocks) {
        hipLaunchKernelGGL(k_plan_count, dim3(blocks), dim3(256), 0, stream, p, counts);
        if ((e = hipGetLastError()) != hipSuccess) return e;
    }
    hipLaunchKernelGGL(k_plan_scan, dim3(keys), dim3(256), 0, stream, counts, totals, blocks);
    if ((e = hipGetLastError()) != hipSuccess) return e;
    hipLaunchKernelGGL((k_plan_place<256>), dim3(std::max(blocks, 1u)), dim3(256), keys * 5 * 4, stream, p, (const uint32_t*)counts,
                       (const uint32_t*)totals);
    return hipGetLastError();
}

hipError_t launch_combine(const CombineArgs& a, int cus, hipStream_t stream) {
    if (!a.rows) return hipSuccess;
    if (a.type == NPA_TYPE_F32) return combine_of<float, float>(a, cus, stream);
    if (a.type == NPA_TYPE_BF16)
        return a.y_f32 ? combine_of<float, __bf16>(a, cus, stream) : combine_of<__bf16, __bf16>(a, cus, stream);
    return a.y_f32 ? combine_of<float, _Float16>(a, cus, stream) : combine_of<_Float16, _Float16>(a, cus, stream);
}

hipError_t launch_combine_adjoint(const CombineArgs& a, int cus, hipStream_t stream) {
    if (!a.rows) return hipSuccess;
    if (a.type == NPA_TYPE_F32) return combine_adjoint_of<float>(a, cus, stream);
    if (a.type == NPA_TYPE_BF16) return combine_adjoint_of<__bf16>(a, cus, stream);
    return combine_adjoint_of<_Float16>(a, cus, stream);
}

}  // namespace npa
