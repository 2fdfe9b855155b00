// npa_experts.hip - the linear layers of experts over the slots of a plan, and their adjoint.
//
// Slot s of expert e: y[s] = act(x[row of s] W_e^T + b_e), rows gathered through the plan or lying in the slots' order.
// Adjoint: dz = dy act'(z), dx[s] = dz W_e (a gathered row's slots summed), dW_e = dz^T x and db_e = sum dz over e's
// slots. Segments lie one after the other at offsets that only the device knows: launches have a block for every tile
// there can be, and a block finds its expert by the tiles of those before it.
#include "npa_tiles.hpp"

namespace npa {
namespace {

struct Segments {
    const int32_t* offsets = nullptr;
    uint32_t experts = 0, slots = 0;
    // Expert e's first slot; slots from `experts`' on have none.
    __device__ inline uint32_t begin(uint32_t e) const { return e > experts || !slots ? slots : min((uint32_t)offsets[e], slots); }
    __device__ inline uint32_t length(uint32_t e) const {
        const uint32_t a = begin(e), b = begin(e + 1);
        return b > a ? b - a : 0;
    }
};

// Inclusive sums over the lanes of a wave.
__device__ inline uint32_t lane_prefix(uint32_t v) {
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, true);  // the lane 1, 2, 4 and 8 before, in its row of 16
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, true);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, true);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, true);
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);  // row 0's last to row 1, row 2's to row 3
    v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);  // row 1's last to rows 2 and 3
    return v;
}

// The segments' tiles of `rows` rows, those of the slots without an expert last; every lane of a wave has some experts,
// one where there are no more than 63.
struct TileMap {
    uint32_t before, upto, total;  // tiles of the lanes before this one, and with this one's
    uint32_t per;                  // experts a lane
    uint32_t begin, length;        // of the lane's only one
    __device__ inline TileMap(const Segments& s, uint32_t rows) {
        const uint32_t lane = threadIdx.x & 63;
        per = (s.experts + 64) / 64;
        uint32_t own = 0;
        begin = length = 0;
        if (per == 1) {
            if (lane <= s.experts) {
                begin = s.begin(lane);
                length = s.length(lane);
            }
            own = (length + rows - 1) / rows;
        } else {
            for (uint32_t e = lane * per; e < min((lane + 1) * per, s.experts + 1); ++e) own += (s.length(e) + rows - 1) / rows;
        }
        upto = lane_prefix(own);
        before = upto - own;
        total = __builtin_amdgcn_readlane(upto, 63);
    }
    // Tile t < total: its expert, first slot and the expert's last slot + 1; the same in every lane, and scalars, as
    // addresses are built on them.
    __device__ inline void find(const Segments& s, uint32_t rows, uint32_t t, uint32_t& expert, uint32_t& first, uint32_t& end) const {
        const uint32_t at = __builtin_ctzll(__ballot(t < upto));
        uint32_t left = t - __builtin_amdgcn_readlane(before, at);
        if (per == 1) {
            expert = at;
            first = __builtin_amdgcn_readlane(begin, at) + left * rows;
            end = __builtin_amdgcn_readlane(begin, at) + __builtin_amdgcn_readlane(length, at);
            return;
        }
        for (expert = at * per; expert < s.experts; ++expert) {
            const uint32_t tiles = (s.length(expert) + rows - 1) / rows;
            if (left < tiles) break;
            left -= tiles;
        }
        expert = __builtin_amdgcn_readfirstlane(expert);
        end = __builtin_amdgcn_readfirstlane(s.begin(expert) + s.length(expert));
        first = __builtin_amdgcn_readfirstlane(s.begin(expert) + left * rows);
    }
};

struct ExpertProduct {
    ProductArgs g;  // of one expert: M all slots, the B operand, bias and results of expert 0
    Segments s;
    uint64_t b_step = 0, bias_step = 0;  // elements from expert to expert
};

// Rows first .. end - 1 and columns n0 .. n0 + cols - 1 of slots without an expert: zeros.
template <class T>
__device__ inline void zero_rows(const ProductArgs& g, uint32_t first, uint32_t end, uint32_t n0, uint32_t cols) {
    cols = min(cols, g.N - n0);
    for (uint32_t i = threadIdx.x; i < (end - first) * cols; i += blockDim.x) {
        const uint64_t row = first + i / cols, col = n0 + i % cols;
        if (g.e.out_f32)
            ((float*)g.e.out)[row * g.e.out_stride + col] = 0.0f;
        else
            ((T*)g.e.out)[row * g.e.out_stride + col] = (T)0.0f;
        if (g.e.z) ((T*)g.e.z)[row * g.e.z_stride + col] = (T)0.0f;
    }
}

// Block `id`'s tile of BM slots by BN columns, or the part of it at row, col of at most rows x cols: false where there is none
// left or its slots have no expert. `g` becomes the product of its expert, M its last slot + 1.
template <class T, int BM, int BN>
__device__ inline bool expert_tile(const ExpertProduct& p, const TileMap& map, uint32_t id, ProductArgs& g, uint32_t& first, uint32_t& n0,
                                   uint32_t row = 0, uint32_t col = 0, uint32_t rows = BM, uint32_t cols = BN) {
    g = p.g;
    g.tiles_m = map.total;
    if (id >= g.tiles_m * g.tiles_n) return false;
    uint32_t tm, tn, expert, end;
    tile_of(g, id, tm, tn);
    map.find(p.s, BM, tm, expert, first, end);
    n0 = tn * BN + col;
    first += row;
    if (first >= end || n0 >= g.N) return false;
    if (expert == p.s.experts) {
        zero_rows<T>(g, first, min(first + rows, end), n0, cols);
        return false;
    }
    g.M = end;
    g.b.p = (const T*)g.b.p + expert * p.b_step;
    if (g.e.bias) g.e.bias = (const char*)g.e.bias + expert * p.bias_step * (g.e.bias_f32 ? 4 : sizeof(T));
    return true;
}

// SPLIT: the product may be in parts, which lie next to each other in the order of blocks.
template <class X, class T, int BM, int BN, int WN, bool SPLIT = false>
__device__ inline void expert_block(ExpertProduct p, uint32_t id, char* lds) {
    ProductArgs g;
    uint32_t first, n0, split = 0, k0 = 0, k1 = p.g.K;
    if (SPLIT && p.g.splits > 1) {
        split = __builtin_amdgcn_readfirstlane(id % p.g.splits);
        id /= p.g.splits;
        k0 = split * (uint32_t)p.g.split_len;
        k1 = min(k1, k0 + (uint32_t)p.g.split_len);
        p.g.e.out = p.g.partials + (uint64_t)split * p.g.M * part_cols(p.g);  // of slots without an expert: zeros too
        p.g.e.out_stride = part_cols(p.g);
        p.g.e.out_f32 = true;
    }
    if (!expert_tile<T, BM, BN>(p, TileMap(p.s, BM), id, g, first, n0)) return;
    if (SPLIT && p.g.splits > 1) g.partials += (uint64_t)split * (p.g.M - g.M) * part_cols(g);  // store_tile adds split g.M's
    f32x16 acc[X::MI][X::NI];
    float none[8];
#pragma unroll
    for (int i = 0; i < X::MI; ++i)
#pragma unroll
        for (int j = 0; j < X::NI; ++j) acc[i][j] = f32x16{};
    X::sum(g.a, g.b, first, n0, g.M, g.N, k0, k1, g.K, false, lds, acc, none);
    store_tile<T, X::MI, X::NI>(g, split, first + threadIdx.x / 64 / WN * X::TM, n0 + threadIdx.x / 64 % WN * X::TN, (float*)lds, acc);
}

// Any type, alignment and size. 131,072 gathered slots of 8, 66 -> 128 f32, z kept: 59 us, 2.9 TB/s. A tile's lookup, loads,
// products and stores follow each other in all blocks at once: 42 us without the products, 44 without the stores. (Tiles of
// 64 x 64: 56 us where the calls before leave their operands in the caches, but 69 for 62 a call where they do not.)
template <class T, int BM, int BN, int WM, int WN, int DEPTH, bool GATHER>
__global__ __launch_bounds__(256, sizeof(T) == 4 && BM == 64 ? 3 : 2) void k_experts(ExpertProduct p) {
    using X = Tile<T, BM, BN, WM, WN, DEPTH, true, true, false, GATHER>;
    __shared__ __align__(16) char lds[X::LDS];
    expert_block<X, T, BM, BN, WN>(p, blockIdx.x, lds);
}

// Few slots an expert: its weights straight from memory to the matrix cores, 16 slots and 16 outputs a block. 1 row of 4 of
// 32, 2,048 -> 1,024 bf16: 8.3 us, the 17 MB of weights at 2 TB/s: latency.
template <class T, bool GATHER>
__global__ __launch_bounds__(kFewWaves * 64) void k_experts_few(ExpertProduct p) {
    __shared__ float red[kFewWaves][16][17];
    ProductArgs g;
    uint32_t first, n0;
    if (!expert_tile<T, 16, 16>(p, TileMap(p.s, 16), blockIdx.x, g, first, n0)) return;
    few_block<T, 1, GATHER>(g, first, min(first + 16, g.M), n0, red);
}

// 256 x 256 tiles, operands straight from memory to LDS, rows of x gathered as they are loaded. A last round of at most half as
// many tiles as CUs is done in quarters of them. 16,384 slots of 8, 2,048 -> 4,096 bf16, z kept: 295 us, 930 TFLOP/s (320 with
// the last round whole): bound by rounds of tiles, as the experts' last ones are not full, and by stores. (At 1.95 GHz; one call
// after the other the clock falls to 1.65, and they take up to 350.)
template <class T>
__global__ __launch_bounds__(512, 2) void k_experts_direct(ExpertProduct p, uint32_t cus) {
    using X = Direct<T, 256, 256, 64, 2, 4, 2, true, true>;
    using Q = Direct<T, 128, 128, 64, 2, 4, 4, true, true>;
    extern __shared__ __align__(16) char lds[];
    const TileMap map(p.s, 256);
    const uint32_t all = map.total * p.g.tiles_n, rest = all % cus, whole = rest * 2 <= cus ? all - rest : all;
    ProductArgs g;
    uint32_t first, n0;
    if (blockIdx.x < whole) {
        if (!expert_tile<T, 256, 256>(p, map, blockIdx.x, g, first, n0)) return;
        direct_tile<X, T, 256, 256, 4, true, true>(g, 0, first, n0, 0, g.K, g.a.order != nullptr, lds);
    } else {
        const uint32_t quarter = blockIdx.x - whole;
        if (!expert_tile<T, 256, 256>(p, map, whole + quarter / 4, g, first, n0, quarter % 2 * 128, quarter / 2 % 2 * 128, 128, 128)) return;
        direct_tile<Q, T, 128, 128, 4, true, true>(g, 0, first, n0, 0, g.K, g.a.order != nullptr, lds);
    }
}

// dW and the bias gradient: A dz [k][m], B x [k][n], both in slot order, k an expert's slots, in `splits` parts of its own
// length each.
struct ExpertGradient {
    ProductArgs g;  // of expert 0; partials and columns [splits][experts][..]
    Segments s;
};

// Block `id`'s tile, expert, part and slots.
struct GradientTile {
    uint32_t m0, n0, expert, split;
    uint64_t k0, k1;
    __device__ inline GradientTile(const ExpertGradient& p, uint32_t id, uint32_t bm, uint32_t bn, uint32_t bk) {
        const ProductArgs& g = p.g;
        // Experts in turn, as their sums differ in length: an XCD has an eighth of each one's tiles, in strips that share
        // operands. (A whole expert an XCD took 8,192 slots, 2,048 -> 4,096 from 300 to 370 us with the longest.)
        const uint32_t tiles = g.tiles_m * g.tiles_n, all = tiles * g.splits;
        expert = __builtin_amdgcn_readfirstlane(id / all);  // the same in every lane; scalars, as addresses are built on them
        const uint32_t in = id % all, own = all % 8 ? in : in % 8 * (all / 8) + in / 8, at = own % tiles;
        split = own / tiles;
        const uint32_t strip = at / (4 * g.tiles_n), height = min(g.tiles_m - strip * 4, 4u), r = at % (4 * g.tiles_n);
        m0 = __builtin_amdgcn_readfirstlane((strip * 4 + r % height) * bm);
        n0 = __builtin_amdgcn_readfirstlane(r / height * bn);
        const uint32_t first = p.s.begin(expert), length = p.s.length(expert);
        const uint32_t len = (length / bk + g.splits) / g.splits * bk;  // whole steps
        k0 = __builtin_amdgcn_readfirstlane(first + min(length, split * len));
        k1 = __builtin_amdgcn_readfirstlane(first + min(length, (split + 1) * len));
    }
    // The product of its expert.
    __device__ inline ProductArgs own(const ExpertGradient& p, uint32_t bytes) const {
        ProductArgs g = p.g;
        if (g.splits > 1)
            g.partials += ((uint64_t)split * p.s.experts + expert - split) * g.M * part_cols(g);  // store_tile adds split M's
        else
            g.e.out = (char*)g.e.out + (uint64_t)expert * g.M * g.e.out_stride * (g.e.out_f32 ? 4 : bytes);
        return g;
    }
};

template <class X, class T, int BM, int BN, int WN>
__device__ inline void gradient_block(const ExpertGradient& p, uint32_t id, char* lds) {
    const GradientTile tile(p, id, BM, BN, X::BK);
    const ProductArgs g = tile.own(p, sizeof(T));
    const uint32_t m0 = tile.m0, n0 = tile.n0;
    const bool sums = (g.columns || g.db) && n0 == 0;
    f32x16 acc[X::MI][X::NI];
    float columns[8] = {};
#pragma unroll
    for (int i = 0; i < X::MI; ++i)
#pragma unroll
        for (int j = 0; j < X::NI; ++j) acc[i][j] = f32x16{};
    X::sum(g.a, g.b, m0, n0, g.M, g.N, tile.k0, tile.k1, tile.k1, sums, lds, acc, columns);
    store_tile<T, X::MI, X::NI>(g, tile.split, m0 + threadIdx.x / 64 / WN * X::TM, n0 + threadIdx.x / 64 % WN * X::TN, (float*)lds, acc);
    if (sums) {
        const float s = tile_columns<X, BM>((float(*)[9])lds, columns);
        if (threadIdx.x < BM && m0 + threadIdx.x < g.M) {
            const uint64_t at = (uint64_t)tile.expert * g.M + m0 + threadIdx.x;
            if (g.db)
                store_param<T>(g.db, g.db_f32, g.db_accumulate, at, s);
            else
                g.columns[(uint64_t)tile.split * p.s.experts * g.M + at] = s;
        }
    }
}

// Both products of the adjoint in one launch, the one with the longer blocks first (`dx_last`: dW's): short ones fill what
// the long ones leave. GATHER: x is rows. Bound by latency: 131,072 slots of 8, 66 -> 128 f32 82 us, of which dz, x and dx take
// 25 from and to memory; 4,503 of 7, 777 -> 333 f16 28 us, a round of blocks of 6 to 20 steps.
template <class T, int BM, int BN, int WM, int WN, int DEPTH, bool SLOPE, bool GATHER>
__global__ __launch_bounds__(256, sizeof(T) == 4 && BM == 64 ? 3 : 2) void k_experts_adjoint(ExpertProduct dx, ExpertGradient dw, uint32_t first_blocks, bool dx_last) {
    using W = Tile<T, BM, BN, WM, WN, DEPTH, false, false, SLOPE, GATHER>;
    using X = Tile<T, BM, BN, WM, WN, DEPTH, true, false, SLOPE>;
    __shared__ __align__(16) char lds[W::LDS];
    const bool first = blockIdx.x < first_blocks;
    const uint32_t block = first ? blockIdx.x : blockIdx.x - first_blocks;
    if (first == dx_last)
        gradient_block<W, T, BM, BN, WN>(dw, block, lds);
    else
        expert_block<X, T, BM, BN, WN, true>(dx, block, lds);
}

// dx and dW in 256 x 256 tiles, in one launch: dx's, whose sums are longer where that pays, first, so that dW's fill the CUs
// that its last round leaves. 8,192 slots of 8, 2,048 -> 4,096 bf16: 290 us, 950 TFLOP/s.
template <class T>
__global__ __launch_bounds__(512, 2) void k_experts_direct_adjoint(ExpertProduct dx, ExpertGradient dw, uint32_t dx_blocks) {
    using X = Direct<T, 256, 256, 64, 2, 4, 2, true, false>;
    using W = Direct<T, 256, 256, 64, 2, 4, 2, false, false, true>;
    extern __shared__ __align__(16) char lds[];
    if (blockIdx.x < dx_blocks) {
        ProductArgs g;
        uint32_t first, n0;
        if (!expert_tile<T, 256, 256>(dx, TileMap(dx.s, 256), blockIdx.x, g, first, n0)) return;
        direct_tile<X, T, 256, 256, 4, true, false>(g, 0, first, n0, 0, g.K, false, lds);
    } else {
        const GradientTile tile(dw, blockIdx.x - dx_blocks, 256, 256, 64);
        const ProductArgs g = tile.own(dw, sizeof(T));
        direct_tile<W, T, 256, 256, 4, false, false>(g, 0, tile.m0, tile.n0, tile.k0, tile.k1, false, lds);
    }
}

// dz and its column sums by expert: block (x, y) has part y % parts of expert y / parts. Bound by memory: 131,072 slots of
// 128 f32 38 us, 5.3 TB/s.
template <class T, int ACT>
__global__ __launch_bounds__(256) void k_experts_slope(SlopeArgs g, Segments s, uint32_t parts) {
    __shared__ float shared[256][9];
    const uint32_t expert = blockIdx.y / parts, part = blockIdx.y % parts;
    const uint64_t first = s.begin(expert), length = s.length(expert);
    slope_block<T, ACT>(g, first + length * part / parts, first + length * (part + 1) / parts,
                        g.partials ? g.partials + ((uint64_t)part * s.experts + expert) * g.cols : nullptr, shared);
}

// Rows of x in the order of the slots, for tiles that load them straight to LDS with k across rows: a row's offset would be
// another in each step. 8,192 slots of 2,048 bf16 14 us, 4.8 TB/s.
template <class T>
__global__ __launch_bounds__(256) void k_experts_sort(Operand x, T* to, uint64_t to_stride, uint32_t width, uint32_t slots, uint32_t lanes) {
    constexpr uint32_t V = 16 / sizeof(T);
    const uint32_t lane = threadIdx.x % lanes, rows = 256 / lanes;
    for (uint64_t slot = (uint64_t)blockIdx.x * rows + threadIdx.x / lanes; slot < slots; slot += (uint64_t)gridDim.x * rows) {
        const T* from = (const T*)x.p + x.gathered(slot) * x.stride;
        for (uint32_t col = lane * V; col < width; col += lanes * V) {
            T* at = to + slot * to_stride + col;
            typedef typename VecOf<T, V>::type vec;
            if (width - col >= V)
                *(vec*)at = *(const vec*)(from + col);
            else
                for (uint32_t j = 0; j < width - col; ++j) at[j] = from[col + j];
        }
    }
}

// ------------------------------------------------------------------ launches
// Tiles of `rows` slots: at most so many, and about so many where the experts' shares are alike.
uint64_t most_tiles(const Segments& s, uint32_t rows) { return s.slots / rows + std::min<uint64_t>(s.experts + 1ull, s.slots); }
uint64_t usual_tiles(const Segments& s, uint32_t rows) {
    const uint64_t used = std::min(s.experts, s.slots);
    return std::max(used, s.slots / rows + used / 2);
}

// Tiles of 256 x 256 about, and whether the direct ones serve a product.
uint64_t direct_tiles(const ExpertProduct& p) { return usual_tiles(p.s, 256) * ((p.g.N + 255) / 256); }
uint64_t direct_tiles(const ExpertGradient& p) { return (uint64_t)p.s.experts * ((p.g.M + 255) / 256) * ((p.g.N + 255) / 256); }
template <class T, bool BF>
bool direct_serves(const ExpertProduct& p, bool gather) {
    const ProductArgs& g = p.g;
    if (sizeof(T) != 2 || g.N < 256 || g.K < 256 || g.K % 64) return false;
    if (!direct_operand<true>(g.a, 0) || !direct_operand<BF>(g.b, g.N) || p.b_step % 8) return false;
    return !gather || g.a.slow * g.a.stride * sizeof(T) < 1ull << 32;  // offsets of 32 bits
}
template <class T>
bool direct_serves(const ExpertGradient& p) {
    const ProductArgs& g = p.g;
    if (sizeof(T) != 2 || g.N < 256 || g.M < 256) return false;
    return direct_operand<false>(g.a, g.M) && (g.b.order || direct_operand<false>(g.b, g.N)) && g.N % 8 == 0;
}
// Whether they pay, alone: half a tile a CU or more, half a tile's slots an expert. (us, direct and else, gelu, bf16: 1,024
// slots of 8 experts, 2,048 -> 4,096: 47 and 50, 2,048 slots 55 and 84; 8,192 of 8, 512 -> 512, 72 tiles: 20 and 20.)
bool direct_pays(const ExpertProduct& p, int cus) {
    return p.s.slots >= 128ull * std::min(p.s.experts, p.s.slots) && direct_tiles(p) >= (uint64_t)cus / 2;
}
bool direct_pays(const ExpertGradient& p, int cus) { return p.s.slots >= 256ull * p.s.experts && direct_tiles(p) >= (uint64_t)cus / 2; }
// Both of an adjoint's, in one launch, in which the gradient's fill what dx's leave. (32 slots of 8, 2,048 -> 4,096: 96 and
// 125, 256 slots 102 and 134, 2,048 slots 143 and 192; 1,024 of 64, 512 -> 2,048: 106 and 118; 2,048 of 128, 512 -> 512: 84
// and 79; 4,096 of 64, 1,024 -> 1,024: 130 and 142; 8,192 of 8, 512 -> 512, 104 tiles in all: 66 and 57; 65,536 of 8,
// 256 -> 256, where the gradient has 8 tiles: 335 and 100, 128 with dx's only.)
bool direct_pays(const ExpertProduct& x, const ExpertGradient& w, int cus) {
    return x.s.slots >= 4ull * x.s.experts && direct_tiles(w) >= (uint64_t)cus / 2 && direct_tiles(x) >= (uint64_t)cus / 4;
}

template <class T>
hipError_t direct_forward(ExpertProduct p, int cus, hipStream_t stream) {
    using X = Direct<T, 256, 256, 64, 2, 4, 2, true, true>;
    const auto kernel = k_experts_direct<T>;
    static LdsLimitFlags flags;
    hipError_t e = raise_lds_limit((const void*)kernel, flags);
    if (e != hipSuccess) return e;
    p.g.tiles_n = (p.g.N + 255) / 256;
    hipLaunchKernelGGL(kernel, dim3((uint32_t)(most_tiles(p.s, 256) * p.g.tiles_n) + 2 * cus), dim3(512), X::LDS, stream, p, (uint32_t)cus);
    return hipGetLastError();
}

// Either of dx and dW, or both.
template <class T>
hipError_t direct_adjoint(ExpertProduct dx, ExpertGradient dw, bool want_dx, bool want_dw, hipStream_t stream) {
    using X = Direct<T, 256, 256, 64, 2, 4, 2, true, false>;
    const auto kernel = k_experts_direct_adjoint<T>;
    static LdsLimitFlags flags;
    hipError_t e = raise_lds_limit((const void*)kernel, flags);
    if (e != hipSuccess) return e;
    dx.g.tiles_n = (dx.g.N + 255) / 256;
    dw.g.tiles_m = (dw.g.M + 255) / 256;
    dw.g.tiles_n = (dw.g.N + 255) / 256;
    const uint32_t dx_blocks = want_dx ? (uint32_t)(most_tiles(dx.s, 256) * dx.g.tiles_n) : 0;
    const uint32_t dw_blocks = want_dw ? dw.g.tiles_m * dw.g.tiles_n * dw.s.experts : 0;
    hipLaunchKernelGGL(kernel, dim3(dx_blocks + dw_blocks), dim3(512), X::LDS, stream, dx, dw, dx_blocks);
    return hipGetLastError();
}

template <class T, bool GATHER>
hipError_t forward_of(ExpertProduct p, int cus, hipStream_t stream) {
    constexpr bool F32 = sizeof(T) == 4;
    constexpr uint64_t BK = F32 ? 32 : 64;
    ProductArgs& g = p.g;
    if constexpr (!F32) {
        if (direct_serves<T, true>(p, GATHER) && direct_pays(p, cus)) return direct_forward<T>(p, cus, stream);
    }
    const uint64_t steps = (g.K + BK - 1) / BK;
    int best = 0;
    Plan least;
    for (int k = 0; k < 3; ++k) {
        const Shape& s = kShapes[k];
        // up to 32 columns are the narrow tiles' (us, and in the others: 131,072 slots of 8, 128 -> 18 23 and 31, bf16 11.5 and 13.3, 128 -> 8
        // 21 and 28; 65,536 of 64, 512 -> 32 f16 17.6 and 20.3, of 128, 256 -> 16 23.8 and 23.6; 8,192 of 8, 128 -> 18 6.2 both, bf16 4.9 and 4.6)
        if ((k == 2) != (k && g.N <= 32) || (k && most_tiles(p.s, s.bm) * ((g.N + s.bn - 1) / s.bn) >= kTooManyTiles)) continue;
        const Plan q = plan(s, F32, false, usual_tiles(p.s, s.bm) * s.bm, g.N, steps, cus, 1);
        if (k == 0 || k == 2 || q.us < least.us) {
            least = q;
            best = k;
        }
    }
    // Weights straight to the matrix cores, by a model: a round of nine blocks a CU takes 4 us, a CU takes in 60 GB/s of operands,
    // memory gives 4.6 TB/s. (us, so and in tiles: 4 slots of 32 experts, 2,048 -> 1,024 bf16 12 and 24, 64 slots 32 and
    // 28, 256 slots 52 and 29; 256 slots of 8, 1,024 -> 1,024 f32 27 and 36; 131,072 of 8, 32 -> 128 bf16 99 and 25.)
    const uint64_t across = (g.N + 15) / 16, blocks = most_tiles(p.s, 16) * across;
    const double block_bytes = 16.0 * g.K * sizeof(T) * 2, usual = (double)usual_tiles(p.s, 16) * across;
    const double few_us = 4.0 * std::max(1.0, usual / (9.0 * cus)) +
                          std::max(std::ceil(usual / cus) * block_bytes / 60e3, usual * 16.0 * g.K * sizeof(T) / 4.6e6);
    if (blocks < 1u << 22 && few_us < least.us) {
        const uint32_t runs = (uint32_t)((g.K + 31) / 32);
        uint32_t waves = 1;
        while (waves < kFewWaves && waves * 4 < runs) waves *= 2;
        g.tiles_n = (uint32_t)across;
        hipLaunchKernelGGL((k_experts_few<T, GATHER>), dim3((uint32_t)blocks), dim3(waves * 64), 0, stream, p);
        return hipGetLastError();
    }
    const Shape& s = kShapes[best];
    g.tiles_n = (g.N + s.bn - 1) / s.bn;
    const dim3 grid((uint32_t)(most_tiles(p.s, s.bm) * g.tiles_n)), block(256);
    switch (best) {
        case 0: hipLaunchKernelGGL((k_experts<T, 128, 128, 2, 2, 2, GATHER>), grid, block, 0, stream, p); break;
        case 1: hipLaunchKernelGGL((k_experts<T, 64, 64, 2, 2, 3, GATHER>), grid, block, 0, stream, p); break;
        default: hipLaunchKernelGGL((k_experts<T, 128, 32, 4, 1, 2, GATHER>), grid, block, 0, stream, p);
    }
    return hipGetLastError();
}

Segments segments_of(const ExpertArgs& a) { return {a.offsets, a.experts, (uint32_t)a.entries}; }

template <class T>
hipError_t experts_of(const ExpertArgs& a, int cus, hipStream_t stream) {
    const LinearArgs& l = a.l;
    ExpertProduct p;
    p.s = segments_of(a);
    ProductArgs& g = p.g;
    g.M = (uint32_t)a.entries;
    g.N = l.out_dims;
    g.K = l.in_dims;
    g.a = {l.x, l.x_stride, l.rows};
    if (a.gather) {
        g.a.order = (const uint32_t*)a.order;
        g.a.per = a.top_k;
    }
    g.b = {l.w, l.w_stride, l.out_dims};
    Epilogue& e = g.e;
    e.out = l.out;
    e.out_stride = l.out_stride;
    e.bias = l.bias;
    e.bias_f32 = l.bias_f32;
    e.z = l.z;
    e.z_stride = l.z_stride;
    e.act = l.activation;
    e.out_f32 = sizeof(T) == 4;
    p.b_step = l.out_dims * l.w_stride;
    p.bias_step = l.out_dims;
    return a.gather ? forward_of<T, true>(p, cus, stream) : forward_of<T, false>(p, cus, stream);
}

inline uint64_t whole_units(uint64_t cols) { return (cols + 7) & ~7ull; }

// dz and the bias gradient's partial sums by a kernel of their own.
template <class T>
hipError_t slope_of(const ExpertArgs& a, LayerWorkspace& ws, int cus, BiasArgs& bias, hipStream_t stream) {
    const LinearArgs& l = a.l;
    SlopeArgs g;
    g.dy = l.dy;
    g.z = l.z;
    g.dy_stride = l.dy_stride;
    g.z_stride = l.z_stride;
    g.rows = a.entries;
    g.cols = l.out_dims;
    const uint32_t units = (g.cols + 7) / 8;
    for (g.lanes = 1; g.lanes < 32 && g.lanes < units;) g.lanes *= 2;
    const uint32_t across = (units + g.lanes - 1) / g.lanes;
    // about eight blocks a CU, each with two rows a thread or more where the experts' shares are alike
    const uint32_t parts = (uint32_t)std::max<uint64_t>(1, std::min({(uint64_t)(8 * cus) / across / a.experts, (uint64_t)(65535 / a.experts),
                                                                     a.entries * g.lanes / ((uint64_t)512 * a.experts)}));
    hipError_t e = hipSuccess;
    if (l.activation != NPA_ACT_IDENTITY && a.entries && (l.dx || l.dw)) {
        g.dz_stride = whole_units(l.out_dims);
        if ((e = ws.reserve(ws.dz, a.entries * g.dz_stride * sizeof(T), stream)) != hipSuccess) return e;
        g.dz = ws.dz.ptr;
    }
    if (l.db) {
        if ((e = ws.reserve(ws.columns, (uint64_t)parts * a.experts * g.cols * 4, stream)) != hipSuccess) return e;
        g.partials = ws.columns.as<float>();
        bias.partials = g.partials;
        bias.parts = parts;
    }
    const dim3 grid(across, parts * a.experts);
    const Segments s = segments_of(a);
    switch (l.activation) {
        case NPA_ACT_IDENTITY: hipLaunchKernelGGL((k_experts_slope<T, NPA_ACT_IDENTITY>), grid, dim3(256), 0, stream, g, s, parts); break;
        case NPA_ACT_RELU: hipLaunchKernelGGL((k_experts_slope<T, NPA_ACT_RELU>), grid, dim3(256), 0, stream, g, s, parts); break;
        case NPA_ACT_GELU: hipLaunchKernelGGL((k_experts_slope<T, NPA_ACT_GELU>), grid, dim3(256), 0, stream, g, s, parts); break;
        default: hipLaunchKernelGGL((k_experts_slope<T, NPA_ACT_SILU>), grid, dim3(256), 0, stream, g, s, parts);
    }
    return hipGetLastError();
}

template <class T, int BM, int BN, int WM, int WN, int DEPTH>
hipError_t launch_adjoint(const ExpertProduct& dx, const ExpertGradient& dw, uint32_t dx_blocks, uint32_t dw_blocks, bool slope,
                          hipStream_t stream) {
    const dim3 grid(dw_blocks + dx_blocks), block(256);
    const bool dx_last = !dx_blocks || (dw_blocks && dw.g.split_len >= dx.g.split_len), gather = dw.g.b.order != nullptr;
    const uint32_t first = dx_last ? dw_blocks : dx_blocks;
#define NPA_ADJOINT(SLOPE, GATHER) \
    hipLaunchKernelGGL((k_experts_adjoint<T, BM, BN, WM, WN, DEPTH, SLOPE, GATHER>), grid, block, 0, stream, dx, dw, first, dx_last)
    if (slope && gather)
        NPA_ADJOINT(true, true);
    else if (slope)
        NPA_ADJOINT(true, false);
    else if (gather)
        NPA_ADJOINT(false, true);
    else
        NPA_ADJOINT(false, false);
#undef NPA_ADJOINT
    return hipGetLastError();
}

template <class T>
hipError_t experts_adjoint_of(const ExpertArgs& a, LayerWorkspace& ws, int cus, hipStream_t stream) {
    constexpr bool F32 = sizeof(T) == 4;
    constexpr uint64_t BK = F32 ? 32 : 64;
    const LinearArgs& l = a.l;
    const bool active = l.activation != NPA_ACT_IDENTITY, want_dx = l.dx && a.entries, want_dw = l.dw;
    hipError_t err = hipSuccess;
    BiasArgs bias;
    bias.db = l.db;
    bias.cols = a.experts * l.out_dims;
    bias.f32 = l.grad_f32;
    bias.accumulate = l.accumulate;
    ExpertProduct px;
    px.s = segments_of(a);
    ProductArgs& dx = px.g;
    dx.M = (uint32_t)a.entries;
    dx.N = l.in_dims;
    dx.K = l.out_dims;
    dx.b = {l.w, l.w_stride, l.out_dims};
    px.b_step = l.out_dims * l.w_stride;
    dx.e.out = l.dx;
    dx.e.out_stride = l.dx_stride;
    dx.e.out_f32 = F32;
    ExpertGradient pw;
    pw.s = px.s;
    ProductArgs& dw = pw.g;
    dw.M = l.out_dims;
    dw.N = l.in_dims;
    dw.e.out = l.dw;
    dw.e.out_stride = l.in_dims;
    dw.e.out_f32 = l.grad_f32;
    dw.e.accumulate = l.accumulate;
    dw.b = {l.x, l.x_stride, l.rows};
    if (want_dx && a.gather) {  // a row's sum over its slots is of f32 gradients
        if ((err = ws.reserve(ws.spread, a.entries * whole_units(l.in_dims) * 4, stream)) != hipSuccess) return err;
        dx.e.out = ws.spread.ptr;
        dx.e.out_stride = whole_units(l.in_dims);
        dx.e.out_f32 = true;
    }
    if (want_dw && a.gather && a.entries) {
        dw.b.order = (const uint32_t*)a.order;
        dw.b.per = a.top_k;
    }
    // Large aligned products straight from memory: dz has to be there.
    dx.a = dw.a = active ? Operand{nullptr, whole_units(l.out_dims), a.entries} : Operand{l.dy, l.dy_stride, a.entries};
    const bool dx_served = want_dx && direct_serves<T, false>(px, false), dw_served = want_dw && direct_serves<T>(pw);
    const bool both = dx_served && dw_served && direct_pays(px, pw, cus);
    const bool direct_dx = both || (dx_served && !want_dw && direct_pays(px, cus));
    const bool direct_dw = both || (dw_served && !dx_served && direct_pays(pw, cus));
    // The slope in the products themselves where that is less than a pass of its own (as in the linear layer).
    const uint64_t again = (l.in_dims + 127) / 128;
    const bool staged = !direct_dx && !direct_dw && want_dw &&
                        (!active || a.entries * l.out_dims * again <= (1u << 19) || (l.activation == NPA_ACT_RELU && again == 1));
    if (!staged && (active || l.db)) {
        if ((err = slope_of<T>(a, ws, cus, bias, stream)) != hipSuccess) return err;
    }
    const bool slope = staged && active;
    if (slope) {
        dx.a = dw.a = {l.dy, l.dy_stride, a.entries};
        dx.a.z = dw.a.z = l.z;
        dx.a.z_stride = dw.a.z_stride = l.z_stride;
        dx.a.act = dw.a.act = l.activation;
    } else if (active) {
        dx.a.p = dw.a.p = ws.dz.ptr;
    }
    if (direct_dw && dw.b.order) {  // its loads take x in the slots' order
        const uint64_t stride = whole_units(l.in_dims);
        if ((err = ws.reserve(ws.sorted, a.entries * stride * sizeof(T), stream)) != hipSuccess) return err;
        uint32_t lanes = 1;
        while (lanes < 256 && lanes * (16 / sizeof(T)) < l.in_dims) lanes *= 2;
        const uint64_t blocks = (a.entries + 256 / lanes - 1) / (256 / lanes);
        hipLaunchKernelGGL(k_experts_sort<T>, dim3((uint32_t)std::min<uint64_t>(blocks, (uint64_t)cus * 32)), dim3(256), 0, stream, dw.b,
                           ws.sorted.as<T>(), stride, l.in_dims, (uint32_t)a.entries, lanes);
        if ((err = hipGetLastError()) != hipSuccess) return err;
        dw.b = {ws.sorted.ptr, stride, a.entries};
    }
    if constexpr (sizeof(T) == 2) {
        if ((direct_dx || direct_dw) && (err = direct_adjoint<T>(px, pw, direct_dx, direct_dw, stream)) != hipSuccess) return err;
    }
    ProductArgs whole;  // all experts' gradients, to join
    const bool tiled_dx = want_dx && !direct_dx, tiled_dw = want_dw && !direct_dw;
    if (tiled_dx || tiled_dw) {
        const uint64_t dw_steps = (a.entries / a.experts + BK) / BK, dx_steps = (dx.K + BK - 1) / BK;
        // A choice is seldom even, and the longest expert's sums end last: priced halfway between the mean and all rows, at
        // thrice the mean at most. (us, priced at the mean and so: 28,642 rows of 3 of 12, the longest 2.1 means, 781 -> 35
        // f16: 320 and 205; 22,910 of 8 of 152, the longest 5, 133 -> 37 f32: 268 and 160.)
        const double longest = std::min(3.0, 0.5 + 0.5 * std::max(1.0, (double)a.experts / a.top_k));
        int best = 0;
        double least = 0.0;
        Plan split, split_x;
        for (int k = 0; k < 3; ++k) {
            const Shape& s = kShapes[k];
            const uint64_t tiles = (tiled_dw ? tile_count(s, dw.M, dw.N) * a.experts : 0) +
                                   (tiled_dx ? most_tiles(px.s, s.bm) * ((dx.N + s.bn - 1) / s.bn) : 0);
            if ((k == 2 && dw.N > 32) || (k && tiles >= kTooManyTiles)) continue;
            Split w[kMostWays], x[kMostWays];
            double memory_w = 0.0, memory_x = 0.0;
            const int n = tiled_dw ? ways(s, (uint64_t)((dw.M + s.bm - 1) / s.bm) * s.bm * a.experts, dw.N, dw_steps, cus, kMostSplits, w, memory_w) : 1;
            const int nx = tiled_dx ? ways(s, usual_tiles(px.s, s.bm) * s.bm, dx.N, dx_steps, cus, kMostSplits, x, memory_x) : 1;
            const double memory = std::max(memory_w, memory_x) + 0.3 * std::min(memory_w, memory_x);
            for (int i = 0; i < n; ++i)
                for (int j = 0; j < nx; ++j) {
                    Split priced = tiled_dw ? w[i] : x[j];
                    if (tiled_dw) priced.plan.len = (uint64_t)(priced.plan.len * longest);
                    const double us = launch_us(s, F32, true, priced, tiled_dw && tiled_dx ? &x[j] : nullptr, cus, memory);
                    if (k + i + j > 0 && us >= least) continue;
                    least = us;
                    best = k;
                    if (tiled_dw) split = w[i].plan;
                    if (tiled_dx) split_x = x[j].plan;
                }
        }
        const Shape& s = kShapes[best];
        uint32_t dx_blocks = 0, dw_blocks = 0;
        if (tiled_dx) {
            set_plan(dx, split_x, s, BK);
            dx_blocks = (uint32_t)(most_tiles(px.s, s.bm) * dx.tiles_n) * dx.splits;
        }
        if (tiled_dw) {
            set_plan(dw, split, s, BK);
            dw_blocks = block_count(dw) * a.experts;
            whole = dw;
            whole.M = a.experts * dw.M;
        }
        const uint64_t dw_floats = tiled_dw ? part_floats(whole) : 0, dx_floats = tiled_dx ? part_floats(dx) : 0;
        if (dw_floats + dx_floats) {
            if ((err = ws.reserve(ws.partials, (dw_floats + dx_floats) * 4, stream)) != hipSuccess) return err;
            dw.partials = whole.partials = ws.partials.as<float>();
            dx.partials = ws.partials.as<float>() + dw_floats;
        }
        if (staged && l.db && dw.splits == 1) {
            dw.db = l.db;
            dw.db_f32 = l.grad_f32;
            dw.db_accumulate = l.accumulate;
            bias.db = nullptr;  // no parts to join
        } else if (staged && l.db) {
            if ((err = ws.reserve(ws.columns, (uint64_t)dw.splits * bias.cols * 4, stream)) != hipSuccess) return err;
            dw.columns = ws.columns.as<float>();
            bias.partials = dw.columns;
            bias.parts = dw.splits;
        }
        if (best == 0)
            err = launch_adjoint<T, 128, 128, 2, 2, 1>(px, pw, dx_blocks, dw_blocks, slope, stream);
        else if (best == 1)
            err = launch_adjoint<T, 64, 64, 2, 2, 3>(px, pw, dx_blocks, dw_blocks, slope, stream);
        else
            err = launch_adjoint<T, 128, 32, 4, 1, 2>(px, pw, dx_blocks, dw_blocks, slope, stream);
        if (err != hipSuccess) return err;
    }
    if ((err = join<T>(tiled_dw ? &whole : nullptr, tiled_dx ? &dx : nullptr, bias, stream)) != hipSuccess) return err;
    if (!want_dx || !a.gather) return hipSuccess;
    CombineArgs c;
    c.y = ws.spread.ptr;
    c.y_f32 = true;
    c.y_stride = whole_units(l.in_dims);
    c.offsets = a.offsets;
    c.slots = a.slots;
    c.out = l.dx;
    c.out_stride = l.dx_stride;
    c.rows = l.rows;
    c.experts = a.experts;
    c.top_k = a.top_k;
    c.width = l.in_dims;
    c.type = l.type;
    return launch_combine(c, cus, stream);
}

}  // namespace

// One object for each element type (all in one without NPA_PART).
#if !defined(NPA_PART) || NPA_PART == 0
hipError_t experts_f32(const ExpertArgs& a, int cus, hipStream_t stream) { return experts_of<float>(a, cus, stream); }
hipError_t experts_adjoint_f32(const ExpertArgs& a, LayerWorkspace& ws, int cus, hipStream_t stream) { return experts_adjoint_of<float>(a, ws, cus, stream); }

hipError_t launch_experts(const ExpertArgs& a, int cus, hipStream_t stream) {
    if (!a.entries) return hipSuccess;
    if (a.l.type == NPA_TYPE_F32) return experts_f32(a, cus, stream);
    return a.l.type == NPA_TYPE_BF16 ? experts_bf16(a, cus, stream) : experts_f16(a, cus, stream);
}

hipError_t launch_experts_adjoint(const ExpertArgs& a, LayerWorkspace& ws, int cus, hipStream_t stream) {
    if (a.l.type == NPA_TYPE_F32) return experts_adjoint_f32(a, ws, cus, stream);
    return a.l.type == NPA_TYPE_BF16 ? experts_adjoint_bf16(a, ws, cus, stream) : experts_adjoint_f16(a, ws, cus, stream);
}
#endif
#if !defined(NPA_PART) || NPA_PART == 1
hipError_t experts_bf16(const ExpertArgs& a, int cus, hipStream_t stream) { return experts_of<__bf16>(a, cus, stream); }
hipError_t experts_adjoint_bf16(const ExpertArgs& a, LayerWorkspace& ws, int cus, hipStream_t stream) { return experts_adjoint_of<__bf16>(a, ws, cus, stream); }
#endif
#if !defined(NPA_PART) || NPA_PART == 2
hipError_t experts_f16(const ExpertArgs& a, int cus, hipStream_t stream) { return experts_of<_Float16>(a, cus, stream); }
hipError_t experts_adjoint_f16(const ExpertArgs& a, LayerWorkspace& ws, int cus, hipStream_t stream) { return experts_adjoint_of<_Float16>(a, ws, cus, stream); }
#endif

}  // namespace npa
