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
constexpr uint64_t kMostBlocks = 1u << 23;  // of 256 threads: a launch stays below 2^32

// V elements of which n are there; what is not is 0.
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

// Keys as whole numbers of the same order: 0 is -infinity, and NaN the largest, as in a sort. (A zero is +0.)
constexpr uint32_t kKeyBase = 0x007fffffu;
constexpr uint64_t kKeyBase64 = 0x000fffffffffffffull;
__device__ inline uint32_t ordered(float v) {
    const uint32_t u = __float_as_uint(v);
    return v != v ? 0xffffffffu : (u ^ ((uint32_t)((int32_t)u >> 31) | 0x80000000u)) - kKeyBase;
}
__device__ inline uint64_t ordered(double v) {
    const uint64_t u = (uint64_t)__double_as_longlong(v);
    return v != v ? ~0ull : (u ^ ((uint64_t)((int64_t)u >> 63) | 0x8000000000000000ull)) - kKeyBase64;
}
__device__ inline float unordered(uint32_t k) {
    const uint32_t u = k + kKeyBase;
    return k == 0xffffffffu ? NAN : __uint_as_float(u >> 31 ? u ^ 0x80000000u : ~u);
}

__device__ inline float sigmoid_of(float x) { return 1.0f / (1.0f + expf(-x)); }

// LDS of a block of four waves. By row: the lanes' largest keys, a counter, candidates and choices. Rows done in 64 bits take
// a wave's part of it instead: a key for each expert, a value for each group, and choices.
constexpr uint32_t kCandidates = 128;
struct RouteLds {
    uint32_t row, wave;  // bytes a row's lanes, and a wave, have
    __host__ __device__ RouteLds(uint32_t lanes, uint32_t count, uint32_t top_k) {
        row = (2 * lanes + kMostGroups) * 4 + kCandidates * 8 + (top_k + 2) / 2 * 16;
        const uint32_t rows = 64 / lanes * row, exact = (count + kMostGroups) * 8 + (top_k + 2) / 2 * 16;
        wave = ((rows > exact ? rows : exact) + 15) & ~15u;
    }
};

// One row by a whole wave, its keys in 64 bits: the top_k best, one after the other, to `to`. Without a bias the keys are the
// logits; groups, which are valued by scores, only close some. Returns how many there are.
template <class T>
__device__ inline uint32_t choose_exactly(const RouteArgs& a, const T* x, bool keyed, char* lds, uint64_t* to) {
    const uint32_t lane = threadIdx.x & 63;
    uint64_t *keys = (uint64_t*)lds, *value = keys + a.count;
    auto bias = [&](uint32_t e) { return a.bias ? load_param<T>(a.bias, a.bias_f32, e) : 0.0f; };
    float most = -INFINITY;
    double sum = 0.0, inv = 0.0;
    if (keyed && !a.sigmoid) {
#pragma unroll 1
        for (uint32_t e = lane; e < a.count; e += 64) most = fmaxf(most, (float)x[e]);
        most = lane_max<64>(most);
        if (most == -INFINITY) most = 0.0f;
#pragma unroll 1
        for (uint32_t e = lane; e < a.count; e += 64) sum += exp((double)(float)x[e] - most);
        inv = 1.0 / lane_sum<64>(sum);
    }
    auto score = [&](float l) { return a.sigmoid ? 1.0 / (1.0 + exp(-(double)l)) : exp((double)l - most) * inv; };
    wave_sync();
#pragma unroll 1
    for (uint32_t e = lane; e < a.count; e += 64) {
        const float l = (float)x[e], b = bias(e);
        keys[e] = l == -INFINITY || b == -INFINITY ? 0 : ordered(keyed ? score(l) + (double)b : (double)l + 0.0);
    }
    wave_sync();
    if (a.groups > 1) {
        // as (s + s') + (b + b'): groups of the same scores and biases are equal, whichever bias goes with which score
        const uint32_t size = a.count / a.groups;
        if (lane < a.groups) {
            const uint32_t begin = lane * size;
            uint32_t first = begin, second = begin;
            uint64_t best = 0, next = 0;
#pragma unroll 1
            for (uint32_t e = begin; e < begin + size; ++e) {
                const uint64_t k = keys[e];
                if (k > best) {
                    next = best;
                    second = first;
                    best = k;
                    first = e;
                } else if (k > next) {
                    next = k;
                    second = e;
                }
            }
            const double s = score((float)x[first]), s2 = next ? score((float)x[second]) : 0.0;
            const double b = (double)bias(first), b2 = next ? (double)bias(second) : 0.0;
            value[lane] = best ? ordered((s + s2) + (b + b2) + 0.0) : 0;
        }
        wave_sync();
        uint32_t ahead = 0;
        const uint64_t own = lane < a.groups ? value[lane] : 0;
#pragma unroll 1
        for (uint32_t h = 0; h < a.groups; ++h) ahead += value[h] > own || (value[h] == own && h < lane);
        const uint64_t kept = __ballot(own && ahead < a.top_groups);
#pragma unroll 1
        for (uint32_t e = lane; e < a.count; e += 64) {
            if (!(kept >> e / size & 1))
                keys[e] = 0;
            else if (!a.bias && keys[e])
                keys[e] = ordered((double)(float)x[e] + 0.0);
        }
        wave_sync();
    }
    uint32_t found = 0;
    for (; found < a.top_k; ++found) {
        uint64_t own = 0;
        uint32_t at = 0;
#pragma unroll 1
        for (uint32_t e = lane; e < a.count; e += 64) {
            const uint64_t k = keys[e];
            if (k > own) {
                own = k;
                at = e;
            }
        }
        const uint64_t best = lane_max<64>(own);
        if (!best) break;
        const uint32_t expert = ~lane_max<64>(own == best ? ~at : 0u);  // the lowest of equal ones
        if (own == best && at == expert) {
            keys[at] = 0;
            to[found] = ~expert;  // the lower half, as of a candidate
        }
        wave_sync();
    }
    return found;
}

// The best of a row's experts, V in each of L lanes one after the other, from their keys (0: closed). Candidates are those
// of at least the wanted-th largest of the half lanes' largest keys, in any order; each finds its place by those ahead of it.
// `to` gets key << 32 | ~expert. Returns how many there are of the `wanted`; more than kCandidates: there were too many.
// (65,536 rows of 256 in 8 groups, the best 8 of 4: the largest key taken nine times, a row to 64 lanes, 185 us.)
template <int L, int V>
__device__ inline uint32_t choose(const uint32_t (&key)[V], uint32_t wanted, uint32_t* lds, uint64_t* to) {
    const uint32_t lane = threadIdx.x % L;
    uint32_t* counter = lds + 2 * L;
    uint64_t* candidates = (uint64_t*)(lds + 2 * L + kMostGroups);
    uint32_t least = 1;
    wave_sync();
    if (lane == 0) *counter = 0;
    if constexpr (L >= 16) {  // fewer lanes: all open experts
        typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
        uint32_t one = key[0], two = key[V - 1];
#pragma unroll
        for (int v = 1; v < V / 2; ++v) {
            one = max(one, key[v]);
            two = max(two, key[V / 2 + v - 1]);
        }
        lds[2 * lane] = one;
        lds[2 * lane + 1] = two;
        wave_sync();
        uint32_t before_one = 0, before_two = 0;
#pragma unroll
        for (int l = 0; l < 2 * L; l += 4) {
            const u32x4 o = *(const u32x4*)(lds + l);
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                before_one += o[q] > one;
                before_two += o[q] > two;
            }
        }
        least = max(least, ~lane_max<L>(max(before_one < wanted ? ~one : 0u, before_two < wanted ? ~two : 0u)));
    }
    wave_sync();
    // `take`: the bits of a lane's keys that are candidates
    const auto gather = [&](uint32_t take) {
        uint32_t at = take ? atomicAdd(counter, __popc(take)) : 0;
#pragma unroll
        for (int v = 0; v < V; ++v)
            if (take >> v & 1) {
                if (at < kCandidates) candidates[at] = (uint64_t)key[v] << 32 | ~(lane * V + v);
                ++at;
            }
        wave_sync();
    };
    uint32_t take = 0;
#pragma unroll
    for (int v = 0; v < V; ++v) take |= key[v] >= least ? 1u << v : 0u;
    gather(take);
    if (L * V > kCandidates && *counter > kCandidates) {  // many of equal keys: those above them, and the first of them that are wanted
        uint32_t equal = 0;
#pragma unroll
        for (int v = 0; v < V; ++v) equal |= key[v] == least ? 1u << v : 0u;
        take &= ~equal;
        uint32_t above = __popc(take), upto = __popc(equal);
        for (int m = 1; m < L; m *= 2) {
            above += __shfl_xor(above, m);
            const uint32_t o = __shfl_up(upto, m, L);
            if (lane >= (uint32_t)m) upto += o;
        }
        const uint32_t room = above < wanted ? wanted - above : 0;
        for (uint32_t i = upto - __popc(equal); equal && i < room; ++i, equal &= equal - 1) take |= equal & -equal;
        wave_sync();
        if (lane == 0) *counter = 0;
        wave_sync();
        gather(take);
    }
    const uint32_t all = *counter, count = min(all, kCandidates);
    for (uint32_t i = lane; i < count; i += L) {
        const uint64_t c = candidates[i];
        uint32_t ahead = 0;
#pragma unroll 4
        for (uint32_t j = 0; j < count; ++j) ahead += candidates[j] > c;
        if (ahead < wanted) to[ahead] = c;
    }
    wave_sync();
    return all > kCandidates ? all : min(all, wanted);
}

// A group's value, the sum of its two largest keys (0: closed). Of keys near f32's lowest it is -infinity, but open.
__device__ inline uint32_t group_value(uint32_t best, uint32_t second) {
    return !best ? 0 : max(1u, ordered((second ? unordered(best) + unordered(second) : unordered(best)) + 0.0f));
}

// How far apart two f32 keys are, at least, that are in the exact order; `off`: what each is off by, but for its last rounding.
__device__ inline float apart(float off, float p, float q) { return 2.0f * off + 0x1p-23f * fmaxf(fabsf(p), fabsf(q)); }
// What a group's value is off by at most: two keys, their last roundings and the value's, and those of what it is compared with.
__device__ inline uint32_t group_off(float off, uint32_t best, uint32_t second) {
    return __float_as_uint(2.0f * off + 0x1.8p-23f * fabsf(unordered(best)) + (second ? 0x1.8p-23f * fabsf(unordered(second)) : 0.0f));
}

// Keys of the experts in groups other than the best top_groups to 0. False where values are too near each other for f32 to tell.
template <int L, int V>
__device__ inline bool keep_groups(const RouteArgs& a, float off, uint32_t (&key)[V], uint32_t* lds) {
    const uint32_t lane = threadIdx.x % L, first = lane * V, size = a.count / a.groups;
    uint32_t *value = lds + 2 * L, *offs = value + kMostGroups;  // the candidates' place
    const uint32_t lanes = size / V;  // of a group, where it takes whole ones
    wave_sync();
    if (lanes * V == size && (lanes & (lanes - 1)) == 0) {
        uint32_t best = key[0], second = 0;
#pragma unroll
        for (int v = 1; v < V; ++v) {
            second = max(second, min(best, key[v]));
            best = max(best, key[v]);
        }
        for (uint32_t m = 1; m < lanes; m *= 2) {
            const uint32_t b2 = __shfl_xor(best, m), s2 = __shfl_xor(second, m);
            second = max(max(second, s2), min(best, b2));
            best = max(best, b2);
        }
        if (lane % lanes == 0 && first < a.count) {
            value[first / size] = group_value(best, second);
            offs[first / size] = group_off(off, best, second);
        }
    } else {  // keys one lane after the other, groups in turn
        constexpr int Q = ((int)kMostGroups < L * V ? (int)kMostGroups + L - 1 : L * V) / L;  // groups a lane
        uint32_t* keys = offs;  // before they are known
        uint32_t best[Q] = {}, second[Q] = {};
        for (uint32_t base = 0; base < a.count; base += 2 * kCandidates) {
            const uint32_t end = min(base + 2 * kCandidates, a.count);
            wave_sync();
#pragma unroll
            for (int v = 0; v < V; ++v)
                if (first + v >= base && first + v < end) keys[first + v - base] = key[v];
            wave_sync();
#pragma unroll
            for (int q = 0; q < Q; ++q) {
                const uint32_t g = lane + q * L;
                if (g >= a.groups) continue;
#pragma unroll 2
                for (uint32_t e = max(g * size, base); e < min((g + 1) * size, end); ++e) {
                    const uint32_t k = keys[e - base];
                    second[q] = max(second[q], min(best[q], k));
                    best[q] = max(best[q], k);
                }
            }
        }
        wave_sync();
#pragma unroll
        for (int q = 0; q < Q; ++q)
            if (lane + q * L < a.groups) {
                value[lane + q * L] = group_value(best[q], second[q]);
                offs[lane + q * L] = group_off(off, best[q], second[q]);
            }
    }
    wave_sync();
    // a group stays if fewer than top_groups are ahead of it
    uint32_t least = ~0u, next = 0;  // what those that stay are at least, and the others at most
    uint64_t kept = 0;
    for (uint32_t g0 = 0; g0 < a.groups; g0 += L) {
        const uint32_t g = g0 + lane, own = g < a.groups ? value[g] : 0;
        uint32_t ahead = 0;
#pragma unroll 2
        for (uint32_t h = 0; h < a.groups; ++h) {
            const uint32_t other = value[h];
            ahead += other > own || (other == own && h < g);
        }
        const bool stays = own && ahead < a.top_groups;
        const float v = unordered(own), o = own ? __uint_as_float(offs[g]) : 0.0f;
        if (stays)
            least = min(least, ordered(v - o));
        else if (own)
            next = max(next, ordered(v + o));
        kept |= own_lanes<L>(__ballot(stays)) << g0;
    }
    next = lane_max<L>(next);
    least = ~lane_max<L>(~least);
    uint32_t g = first / size, left = size - first % size;
    if (size % V == 0) {
        const bool stays = kept >> (g & 63) & 1;
#pragma unroll
        for (int v = 0; v < V; ++v) key[v] = stays ? key[v] : 0;
    } else {
#pragma unroll
        for (int v = 0; v < V; ++v) {
            if (!(kept >> (g & 63) & 1)) key[v] = 0;
            if (--left == 0) {
                ++g;
                left = size;
            }
        }
    }
    return !next || unordered(least) > unordered(next);
}

// Rows to groups of L lanes. KEYED: with a bias or groups. A key s + b is off by at most (33 m + 1 + |key|) e, e = 2^-24 and m the
// row's largest score, where scores are a softmax's: a sum of exponentials (16 in a lane, then six levels), each 2 ulp off, of
// differences rounded once (x - max is off by |x - max| e, which exp(x - max) makes 0.37 e at most, and in the sum, whose error
// a row's keys have in common, its mean); the quotient; the key's own rounding. The hardware's exp2 and reciprocal leave sigma(x)
// off by s (1 - s) (|x| + 2) e + 3 s e, below 4 e. These bounds grow with the key by less than the key itself: keys further apart than two of
// them are in the exact order, and so is what lies behind. A bias that masks experts with a large finite value so leaves the
// others' keys as they are. A row with keys nearer than that (0.1 % of rows of 256 sigmoid scores) or with too many candidates is
// done again by its whole wave (all rows where groups tie, as those of a router that starts at zero: 375 us a call of the
// following size). 65,536 rows of 256 in 8 groups, the best 8 of 4, bf16: 49 us, of which the 38 MB that pass take 7: bound by the
// instructions for a key's score, group and place, 77 a key; while a CU is busy its vector units are, and CUs are busy for three
// quarters of that time, as blocks take 3.2 rounds. 4,096 rows of 8 f32: 4 us.
template <class T, int L, int V, bool KEYED>
__global__ __launch_bounds__(256) void k_route(RouteArgs a, uint64_t first_row) {
    extern __shared__ __align__(16) char shared[];
    constexpr uint32_t ROWS = 256 / L;
    const uint32_t lane = threadIdx.x % L, first = lane * V;
    const RouteLds size(L, a.count, a.top_k);
    char* of_wave = shared + threadIdx.x / 64 * size.wave;
    uint32_t* lds = (uint32_t*)(of_wave + (threadIdx.x & 63) / L * size.row);
    uint64_t* to = (uint64_t*)(lds + 2 * L + kMostGroups) + kCandidates;
    float b[V];
#pragma unroll
    for (int v = 0; v < V; ++v) b[v] = 0.0f;
    if (KEYED && a.bias && first < a.count) {
        if (a.bias_f32)
            load_unit<float, V>((const float*)a.bias + first, a.count - first, b);
        else
            load_unit<T, V>((const T*)a.bias + first, a.count - first, b);
    }
    // no loop over rows: what a loop would keep in registers from row to row halves the waves
    const uint64_t base = first_row + (uint64_t)blockIdx.x * ROWS;
    const uint64_t own = base + threadIdx.x / L, row = own < a.rows ? own : a.rows - 1;
    const T* x = (const T*)a.logits + row * a.stride;
    float s[V];
    if (first + V <= a.count) {
        const typename VecOf<T, V>::type w = *(const typename VecOf<T, V>::type*)(x + first);
#pragma unroll
        for (int v = 0; v < V; ++v) s[v] = (float)w[v];
    } else {
#pragma unroll
        for (int v = 0; v < V; ++v) s[v] = first + v < a.count ? (float)x[first + v] : -INFINITY;
    }
    // keys from what is -infinity for closed experts
    uint32_t key[V];
    float most = s[0], inv = 1.0f;
#pragma unroll
    for (int v = 0; v < V; ++v) {
        most = fmaxf(most, s[v]);
        if (!KEYED) key[v] = ordered(s[v] + 0.0f);
        if (KEYED) b[v] = s[v] == -INFINITY ? -INFINITY : b[v];
    }
    if (!a.sigmoid) {  // of all logits; a closed one's is 0
        most = lane_max<L>(most);
        most = most == -INFINITY ? 0.0f : most;
        float sum = 0.0f;
#pragma unroll
        for (int v = 0; v < V; ++v) {
            s[v] = expf(s[v] - most);
            sum += s[v];
        }
        inv = 1.0f / lane_sum<L>(sum);
    }
    bool certain = true;
    float off = 0.0f;
    if constexpr (KEYED) {
        off = 0x1p-24f * ((a.sigmoid ? 4.0f : 33.0f * inv) + 1.0f);
#pragma unroll
        for (int v = 0; v < V; ++v) {
            key[v] = ordered((a.sigmoid ? sigma(s[v]) : s[v] * inv) + b[v]);
            if (b[v] == -INFINITY) key[v] = 0;  // also where the score is NaN
        }
        if (a.groups > 1) certain = keep_groups<L, V>(a, off, key, lds);
        if (!a.bias) {  // of the groups that stay the logits order the experts, exactly (read again: few registers are free)
            float l[V];
            const uint32_t n = first < a.count ? a.count - first : 0;
            load_unit<T, V>(x + (n ? first : 0), n, l);
#pragma unroll
            for (int v = 0; v < V; ++v) key[v] = key[v] ? ordered(l[v] + 0.0f) : 0;
        }
    }
    uint32_t found = choose<L, V>(key, a.top_k, lds, to);
    if (found > kCandidates) certain = false;
    if (KEYED && a.bias) {
        // the same inputs: the lower expert, exactly
        const auto differ = [&](uint32_t d, uint32_t e) {
            return !((float)x[d] == (float)x[e] && load_param<T>(a.bias, a.bias_f32, d) == load_param<T>(a.bias, a.bias_f32, e));
        };
        bool near = false;
        for (uint32_t i = lane + 1; i < found && found <= kCandidates; i += L) {
            const uint32_t d = ~(uint32_t)to[i - 1], e = ~(uint32_t)to[i];
            const float p = unordered((uint32_t)(to[i - 1] >> 32)), q = unordered((uint32_t)(to[i] >> 32));
            if (!(p - q > apart(off, p, q))) near |= differ(d, e);
        }
        // and the last one chosen from every key that is left: one further down may be near it, too, behind its equals
        if (found == a.top_k) {
            const uint64_t last = to[found - 1];
            const uint32_t k = (uint32_t)(last >> 32), expert = ~(uint32_t)last;
            const float p = unordered(k);  // (twice the rounding of p: the difference is rounded, too)
            const uint32_t least = max(1u, min(k, ordered(p - apart(off, p, 2.0f * p))));
            uint32_t left = 0;  // and those chosen of the same key, whose inputs are the same, too, or are known not to be
#pragma unroll
            for (int v = 0; v < V; ++v) left |= key[v] - least <= k - least ? 1u << v : 0u;
            if (expert - first < V) left &= ~(1u << (expert - first));
            for (; left; left &= left - 1) near |= differ(first + __builtin_ctz(left), expert);
        }
        if (own_lanes<L>(__ballot(near))) certain = false;
    }
    found = min(found, a.top_k);
    // a row's choices, one to a lane of `step` (or several)
    auto finish = [&](uint32_t n, auto step_of, const uint64_t* list, uint64_t r, const T* logits, float m, float i) {
        constexpr int step = decltype(step_of)::value, TURNS = (int)kMostChoices > step ? (int)kMostChoices / step : 1;
        const uint32_t at = threadIdx.x % step;
        float w[TURNS], total = 0.0f;
#pragma unroll
        for (int q = 0; q < TURNS; ++q) {
            const uint32_t j = at + q * step;
            w[q] = 0.0f;
            if (j < n) {
                const float l = (float)logits[~(uint32_t)list[j]];
                w[q] = a.sigmoid ? sigmoid_of(l) : expf(l - m) * i;
            }
            total += w[q];
        }
        if (a.renormalise) total = lane_sum<step>(total) + kSumEps;
        if (r >= a.rows) return;
#pragma unroll
        for (int q = 0; q < TURNS; ++q) {
            const uint32_t j = at + q * step;
            if (j >= a.top_k) continue;
            a.experts[r * a.top_k + j] = j < n ? (int32_t)~(uint32_t)list[j] : -1;
            a.weights[r * a.top_k + j] = (a.renormalise ? w[q] / total : w[q]) * a.scale;
        }
    };
    finish(found, std::integral_constant<int, L>(), to, certain ? own : a.rows, x, most, inv);
    uint64_t again = __ballot(!certain && own < a.rows);
    while (again) {
        const uint32_t of = __builtin_ctzll(again) & ~(L - 1);
        again &= ~((L == 64 ? ~0ull : (1ull << (L & 63)) - 1) << of);
        const uint64_t r = base + (threadIdx.x & ~63u) / L + of / L;
        const T* logits = (const T*)a.logits + r * a.stride;
        const float m = __shfl(most, of), i = __shfl(inv, of);
        uint64_t* list = (uint64_t*)of_wave + a.count + kMostGroups;
        const uint32_t n = choose_exactly<T>(a, logits, KEYED, of_wave, list);
        finish(n, std::integral_constant<int, 64>(), list, r, logits, m, i);
    }
}

// The gradient of the logits. With Z = sum s_j + 1e-20 over the choices, ds_j = scale (g_j - sum g s / Z) / Z where
// the weights are renormalised, else scale g_j; dl = s (ds - sum_j ds_j s_j) through the softmax, where that sum is
// scale sum(g s) 1e-20 / Z^2 for renormalised weights (no difference of nearly equal sums); ds s (1 - s) through sigma.
// One pass, a row's logits in registers, and each choice's from the cache in all lanes, so that no lane waits for another's.
// Bound by what that repeats: each lane evaluates each choice's score, and vector units are active in 79 % of the cycles that
// CUs are busy. 65,536 rows of 8 f32 6.4 us, 5.2 MB; 20,011 of 123 f16, five choices, 12 us, 11 MB.
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
// A stable counting sort of 4 bytes an entry read and 8 written, bound by latency: a lane finds its place among its wave's by a
// ballot for each bit of the key, and no order depends on atomics. A block has a run of kChunk entries. 524,288 entries of 256:
// 5 us to count, 5 to scan, 11 to place; 8,192 of 8 in one block 10 us.
constexpr uint32_t kChunk = 2048, kSmallPlan = 8192, kFewBlocks = 16;

__device__ inline uint32_t plan_key(const PlanArgs& p, uint32_t i) { return min((uint32_t)p.chosen[i], p.experts); }

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

// A block's entries of each key: counts[key][block], or counts[block][key] where no scan follows
__global__ __launch_bounds__(256) void k_plan_count(PlanArgs p, uint32_t* counts, bool scan) {
    __shared__ uint32_t own[kMostExperts + 1];
    for (uint32_t e = threadIdx.x; e <= p.experts; e += 256) own[e] = 0;
    __syncthreads();
#pragma unroll
    for (uint32_t r = 0; r < kChunk / 256; ++r) {
        const uint32_t i = blockIdx.x * kChunk + r * 256 + threadIdx.x;
        if (i < p.entries) atomicAdd(own + plan_key(p, i), 1u);
    }
    __syncthreads();
    for (uint32_t e = threadIdx.x; e <= p.experts; e += 256)
        counts[scan ? (uint64_t)e * gridDim.x + blockIdx.x : (uint64_t)blockIdx.x * (p.experts + 1) + e] = own[e];
}

// A key's counts to their exclusive sums over the blocks, and its total to totals[key]
__global__ __launch_bounds__(256) void k_plan_scan(uint32_t* counts, uint32_t* totals, uint32_t blocks) {
    __shared__ uint32_t waves[4];
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

// Entries to their slots. Each wave has a part of the block's entries, 64 at a time, and knows from the lanes with the same
// key and from those before how many of the key precede; then come the waves before it, the blocks and the lower keys.
// `counts` null: one block has all entries. `totals` null: a block adds up the `blocks` blocks' counts itself.
template <int THREADS, int TURNS>
__global__ __launch_bounds__(THREADS) void k_plan_place(PlanArgs p, const uint32_t* counts, const uint32_t* totals, uint32_t blocks) {
    constexpr uint32_t WAVES = THREADS / 64;
    extern __shared__ uint32_t lds[];
    __shared__ uint32_t waves[WAVES];
    const uint32_t keys = p.experts + 1, wave = threadIdx.x / 64, lane = threadIdx.x & 63;
    uint32_t *base = lds, *next = lds + keys + wave * keys;  // next[wave][key]
    // a wave's entries lie one after the other: no more turns than the call's entries need
    const uint32_t turns = counts ? TURNS : (p.entries + THREADS - 1) / THREADS;
    const uint32_t begin = blockIdx.x * (THREADS * TURNS) + wave * turns * 64;
    uint32_t key[TURNS], before[TURNS];
#pragma unroll
    for (int r = 0; r < TURNS; ++r) {
        const uint32_t i = begin + r * 64 + lane;
        key[r] = (uint32_t)r < turns && i < p.entries ? plan_key(p, i) : ~0u;
    }
    for (uint32_t i = threadIdx.x; i < keys * WAVES; i += THREADS) lds[keys + i] = 0;
    __syncthreads();
    const int bits = 32 - __builtin_clz(p.experts);
#pragma unroll
    for (int r = 0; r < TURNS; ++r) {
        if ((uint32_t)r >= turns) break;
        const bool in = key[r] != ~0u;
        uint64_t same = __ballot(in);
        for (int b = 0; b < bits; ++b) {
            const uint64_t set = __ballot(key[r] >> b & 1);
            same &= key[r] >> b & 1 ? set : ~set;
        }
        if (in) {
            const uint32_t rank = __popcll(same & ((1ull << lane) - 1)), count = next[key[r]];
            before[r] = count + rank;
            wave_sync();
            if (rank == 0) next[key[r]] = count + __popcll(same);
        }
        wave_sync();
    }
    __syncthreads();
    for (uint32_t e = threadIdx.x; e < keys; e += THREADS) {
        uint32_t sum = 0;
        if (!counts) {
            for (uint32_t w = 0; w < WAVES; ++w) sum += lds[keys + w * keys + e];
        } else if (totals) {
            sum = totals[e];
        } else {
            uint32_t preceding = 0;
#pragma unroll 8
            for (uint32_t b = 0; b < blocks; ++b) {
                const uint32_t c = counts[b * keys + e];
                sum += c;
                preceding += b < blockIdx.x ? c : 0;
            }
            lds[keys * (WAVES + 1) + e] = preceding;  // read by this thread only
        }
        base[e] = sum;
    }
    __syncthreads();
    exclusive<THREADS>(base, keys, waves);
    for (uint32_t e = threadIdx.x; e < keys; e += THREADS) {
        uint32_t at = base[e];
        if (blockIdx.x == 0) p.offsets[e] = (int32_t)at;
        if (counts) at += totals ? counts[(uint64_t)e * gridDim.x + blockIdx.x] : lds[keys * (WAVES + 1) + e];
        for (uint32_t w = 0; w < WAVES; ++w) {
            const uint32_t c = lds[keys + w * keys + e];
            lds[keys + w * keys + e] = at;
            at += c;
        }
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < TURNS; ++r) {
        if (key[r] == ~0u) continue;
        const uint32_t i = begin + r * 64 + lane, slot = next[key[r]] + before[r];
        p.order[slot] = (int32_t)i;
        p.slots[i] = (int32_t)slot;
    }
}

// ------------------------------------------------------------------ rows from slots and back
// The entries past the experts' last slot have no expert: they add nothing, whatever their rows hold.
__device__ inline uint32_t live_slots(const CombineArgs& a) {
    const uint64_t all = a.rows * a.top_k;
    const uint32_t n = (uint32_t)a.offsets[a.experts];
    return n < all ? n : (uint32_t)all;
}

// out = residual + sum_j w_j y[slot_j], summed in the order of j; one pass, bound by memory and its latency. `lanes` lanes to a
// row, V elements each, as many rows to a block as find place (65,536 rows of two slots of 66 f32: 13.3 us, 15.8 where the
// lanes are a power of two).
template <class Y, class T>
__global__ __launch_bounds__(256) void k_combine(CombineArgs a, uint32_t lanes) {
    constexpr int V = 16 / sizeof(T);
    const uint32_t lane = threadIdx.x % lanes, rows = 256 / lanes, live = live_slots(a);
    if (threadIdx.x >= rows * lanes) return;
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
// L lanes to a row's entries in turn where the lanes are few, and else to an entry, a row's next to each other, so that dout
// is read from memory once. Bound by memory: 8,192 rows of two slots of 4,096 bf16 67 us, 5.0 TB/s (72 by rows).
template <class T, int L>
__global__ __launch_bounds__(256) void k_combine_adjoint(CombineArgs a) {
    constexpr int V = 16 / sizeof(T);
    constexpr uint32_t PER = 256 / L;
    __shared__ float part[4];
    const uint32_t lane = threadIdx.x % L, live = live_slots(a), turns = L < 64 ? a.top_k : 1;
    const uint64_t all = a.rows * a.top_k, units = L < 64 ? a.rows : all;
    for (uint64_t unit = (uint64_t)blockIdx.x * PER + threadIdx.x / L; unit < units; unit += (uint64_t)gridDim.x * PER)
    for (uint64_t entry = unit * turns; entry < (unit + 1) * turns; ++entry) {
        const uint64_t row = L < 64 ? unit : (uint32_t)entry / a.top_k;
        const T* dout = (const T*)a.dout + row * a.dout_stride;
        const uint32_t slot = (uint32_t)a.slots[entry];
        if (slot >= all) continue;
        const bool has = slot < live;
        const float w = !has ? 0.0f : a.weights ? a.weights[entry] : 1.0f;
        float dot = 0.0f;
#pragma unroll L < 64 ? 1 : 2
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
            dot = lane_sum<L < 64 ? L : 64>(dot);
            if (L > 64) {
                __syncthreads();
                if (threadIdx.x % 64 == 0) part[threadIdx.x / 64] = dot;
                __syncthreads();
                dot = (part[0] + part[1]) + (part[2] + part[3]);
            }
            if (lane == 0) a.dweights[entry] = dot;
        }
    }
}

// ------------------------------------------------------------------ launches
// A row's experts: V in each of L lanes.
#define NPA_EXPERTS(L, V) return f(std::integral_constant<int, L>(), std::integral_constant<int, V>())
// The choice takes candidates from the half lanes' largest keys: as many of these as choices, unless all experts are candidates.
template <class F>
hipError_t with_router(uint32_t count, uint32_t top_k, F f) {
    if (count <= 8) NPA_EXPERTS(8, 1);
    if (count <= 16) NPA_EXPERTS(8, 2);
    if (count <= 32) NPA_EXPERTS(8, 4);
    if (count <= 64) NPA_EXPERTS(16, 4);
    if (top_k < 16 && count <= 128) NPA_EXPERTS(16, 8);
    if (top_k < 16 && count <= 256) NPA_EXPERTS(16, 16);
    if (count <= 256) NPA_EXPERTS(64, 4);
    if (count <= 512) NPA_EXPERTS(64, 8);
    NPA_EXPERTS(64, 16);
}
template <class F>
hipError_t with_experts(uint32_t count, F f) {
    if (count <= 8) NPA_EXPERTS(8, 1);
    if (count <= 16) NPA_EXPERTS(8, 2);
    if (count <= 32) NPA_EXPERTS(8, 4);
    if (count <= 64) NPA_EXPERTS(16, 4);
    if (count <= 128) NPA_EXPERTS(32, 4);
    if (count <= 256) NPA_EXPERTS(64, 4);
    if (count <= 512) NPA_EXPERTS(64, 8);
    NPA_EXPERTS(64, 16);
}
#undef NPA_EXPERTS

template <class T>
hipError_t route_of(const RouteArgs& a, hipStream_t stream) {
    return with_router(a.count, a.top_k, [&](auto lanes, auto per) {
        constexpr int L = decltype(lanes)::value, V = decltype(per)::value;
        constexpr uint32_t rows = 256 / L;
        const uint32_t lds = 4 * RouteLds(L, a.count, a.top_k).wave;
        for (uint64_t first = 0; first < a.rows; first += kMostBlocks * rows) {
            const dim3 grid((uint32_t)std::min<uint64_t>((a.rows - first + rows - 1) / rows, kMostBlocks)), block(256);
            if (a.bias || a.groups > 1)
                hipLaunchKernelGGL((k_route<T, L, V, true>), grid, block, lds, stream, a, first);
            else
                hipLaunchKernelGGL((k_route<T, L, V, false>), grid, block, lds, stream, a, first);
            const hipError_t e = hipGetLastError();
            if (e != hipSuccess) return e;
        }
        return hipSuccess;
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
    const uint32_t lanes = std::min((a.width + V - 1) / V, 256u);
    const uint64_t blocks = (a.rows + 256 / lanes - 1) / (256 / lanes);
    hipLaunchKernelGGL((k_combine<Y, T>), dim3((uint32_t)std::min<uint64_t>(blocks, (uint64_t)cus * 32)), dim3(256), 0, stream, a, lanes);
    return hipGetLastError();
}

// A block to an entry where the entries are few: 250 rows of 8, 4,096 f32 19 us, 79 with a wave to a row's entries in turn.
template <class T>
hipError_t combine_adjoint_of(const CombineArgs& a, int cus, hipStream_t stream) {
    constexpr uint32_t V = 16 / sizeof(T);
    const uint64_t entries = a.rows * a.top_k;
    auto launch = [&](auto lanes) {
        constexpr int L = decltype(lanes)::value;
        const uint64_t units = L < 64 ? a.rows : entries, blocks = (units + 256 / L - 1) / (256 / L);
        hipLaunchKernelGGL((k_combine_adjoint<T, L>), dim3((uint32_t)std::min<uint64_t>(blocks, (uint64_t)cus * 32)), dim3(256), 0, stream, a);
        return hipGetLastError();
    };
    if (a.width <= 8 * V) return launch(std::integral_constant<int, 8>());
    if (a.width <= 16 * V) return launch(std::integral_constant<int, 16>());
    if (a.width > 64 * V && entries <= (uint64_t)cus * 8) return launch(std::integral_constant<int, 256>());
    return launch(std::integral_constant<int, 64>());
}

}  // namespace

hipError_t launch_route(const RouteArgs& a, hipStream_t stream) {
    if (!a.rows) return hipSuccess;
    if (a.type == NPA_TYPE_F32) return route_of<float>(a, stream);
    if (a.type == NPA_TYPE_BF16) return route_of<__bf16>(a, stream);
    return route_of<_Float16>(a, stream);
}

hipError_t launch_route_adjoint(const RouteArgs& a, int cus, hipStream_t stream) {
    if (!a.rows) return hipSuccess;
    if (a.type == NPA_TYPE_F32) return route_adjoint_of<float>(a, cus, stream);
    if (a.type == NPA_TYPE_BF16) return route_adjoint_of<__bf16>(a, cus, stream);
    return route_adjoint_of<_Float16>(a, cus, stream);
}

// Up to kSmallPlan entries are one block's, since a launch costs more than it saves (14,864 entries of 170: 21 us in one
// block, 11 in two launches; 8,192 of 8: 10). The block's waves count each key in LDS; with 512 experts or more there is room
// for half as many waves, and they take half as many entries (in one block and in two launches: 8 entries of 1,024 4.7 and 10.6 us,
// 4,096 10.6 and 14.5; 4,096 of 600 9.7 and 12.6). Up to kFewBlocks blocks find what precedes them from the others' counts, which
// a scan does where they are more (a call of 128,000 entries of 256, 63 blocks: 38 us without a scan, 35 with one).
hipError_t launch_plan(const PlanArgs& p, LayerWorkspace& ws, hipStream_t stream) {
    const uint32_t keys = p.experts + 1;
    const uint32_t* none = nullptr;
    if (p.entries <= kSmallPlan && keys <= 512) {
        constexpr int THREADS = 1024;
        const uint32_t lds = keys * (1 + THREADS / 64) * 4;
        if (p.entries <= kSmallPlan / 2)
            hipLaunchKernelGGL((k_plan_place<THREADS, 4>), dim3(1), dim3(THREADS), lds, stream, p, none, none, 1u);
        else
            hipLaunchKernelGGL((k_plan_place<THREADS, 8>), dim3(1), dim3(THREADS), lds, stream, p, none, none, 1u);
        return hipGetLastError();
    }
    if (p.entries <= kSmallPlan / 2) {
        constexpr int THREADS = 512;
        hipLaunchKernelGGL((k_plan_place<THREADS, 8>), dim3(1), dim3(THREADS), keys * (1 + THREADS / 64) * 4, stream, p, none, none, 1u);
        return hipGetLastError();
    }
    const uint32_t blocks = (p.entries + kChunk - 1) / kChunk;
    const bool scan = blocks > kFewBlocks;
    hipError_t e = ws.reserve(ws.counts, (uint64_t)keys * (blocks + 1) * 4, stream);
    if (e != hipSuccess) return e;
    uint32_t *counts = ws.counts.as<uint32_t>(), *totals = scan ? counts + (uint64_t)keys * blocks : nullptr;
    hipLaunchKernelGGL(k_plan_count, dim3(blocks), dim3(256), 0, stream, p, counts, scan);
    if ((e = hipGetLastError()) != hipSuccess) return e;
    if (scan) {
        hipLaunchKernelGGL(k_plan_scan, dim3(keys), dim3(256), 0, stream, counts, totals, blocks);
        if ((e = hipGetLastError()) != hipSuccess) return e;
    }
    hipLaunchKernelGGL((k_plan_place<256, kChunk / 256>), dim3(blocks), dim3(256), keys * 6 * 4, stream, p, (const uint32_t*)counts,
                       (const uint32_t*)totals, blocks);
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
