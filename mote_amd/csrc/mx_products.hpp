// What the products of microscaled rows share: their arguments, and how an experts'
// product finds its rows.
#pragma once

#include <type_traits>

#include "mx.hpp"

namespace mote::mx {

// What a product's outputs become.
enum class Result {
    kF16,     // rows x outputs, binary16 (a linear)
    kF32,     // the same in 32 bits
    kGateUp,  // silu(gate) up of an expert's 2 outputs weight rows, binary16, row i of the plan
    kPairs,   // row i of the plan to the row of its pair, 32 bits (an expert's down projection)
};
struct ProductArgs {
    const uint8_t* x;        // values of the rows
    const uint8_t* x_scales;
    const uint8_t* w;        // values of the weights' rows, expert after expert
    const uint8_t* w_scales;
    void* output;
    const int32_t* offsets;  // [experts + 1] first row of the plan of each expert
    const int32_t* plan;     // the pair of each row of the plan
    uint32_t rows;           // of a linear's x; pairs of the experts'
    uint32_t outputs;        // columns of the output
    uint32_t kp;
    uint32_t experts, top;
};

// Tiles that keep the chip busy: one for three in four compute units.
constexpr uint64_t kEnoughTiles = 192;

// Products of many rows (mx_tiles.hip).
int launch_tiles(Result result, const ProductArgs& a, int bits, hipStream_t stream);

namespace {

template <Result R>
constexpr bool kOfExperts = R == Result::kGateUp || R == Result::kPairs;

// The rows of one tile: an expert's, `count` of them (0: no such tile) from row `first` of the
// plan, or a linear's.
struct Tile {
    uint32_t expert, first, count;
};

// The sum of v over the lanes before.
template <int Ctrl, int RowMask>
__device__ __forceinline__ uint32_t add_dpp(uint32_t v) {
    return v + static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), Ctrl, RowMask, 0xF, false));
}
__device__ __forceinline__ uint32_t lanes_before(uint32_t v) {
    uint32_t sum = add_dpp<0x111, 0xF>(v);  // row_shr:1, 2, 4, 8
    sum = add_dpp<0x112, 0xF>(sum);
    sum = add_dpp<0x114, 0xF>(sum);
    sum = add_dpp<0x118, 0xF>(sum);
    sum = add_dpp<0x142, 0xA>(sum);  // row_bcast:15 into rows 1 and 3
    sum = add_dpp<0x143, 0xC>(sum);  // row_bcast:31 into rows 2 and 3
    return sum - v;
}

// The tiles of PER rows of the experts: each has its rows / PER of them, rounded up.
// Every wave counts them by itself: lane l those of its run of experts, and a prefix sum over the
// lanes; a tile's run is found in that and walked.
template <uint32_t PER>
struct ExpertTiles {
    uint32_t upto;  // tiles of this lane's experts and the lanes' before

    // Kept inside the rows there are, whatever the offsets hold.
    __device__ __forceinline__ static uint32_t offset(const ProductArgs& a, uint32_t e) {
        return static_cast<uint32_t>(min(max(a.offsets[e], 0), static_cast<int32_t>(a.rows)));
    }
    __device__ __forceinline__ explicit ExpertTiles(const ProductArgs& a) {
        const uint32_t lane = threadIdx.x & 63, run = (a.experts + 63) / 64;
        const uint32_t e0 = min(lane * run, a.experts), e1 = min(e0 + run, a.experts);
        uint32_t mine = 0;
        if (e0 < e1) {
            uint32_t from = offset(a, e0);
            for (uint32_t e = e0; e < e1; ++e) {
                const uint32_t to = offset(a, e + 1);
                mine += to > from ? (to - from + PER - 1) / PER : 0;
                from = to;
            }
        }
        upto = lanes_before(mine) + mine;
    }
    __device__ __forceinline__ uint32_t total() const {
        return static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(upto), 63));
    }
    __device__ __forceinline__ Tile at(const ProductArgs& a, uint32_t unit) const {
        const uint32_t run = (a.experts + 63) / 64;
        const uint32_t owner = __builtin_popcountll(__builtin_amdgcn_ballot_w64(upto <= unit));
        if (owner == 64) return {0, 0, 0};
        uint32_t left = unit;
        if (owner > 0) left -= static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(upto), owner - 1));
        for (uint32_t e = owner * run; e < a.experts; ++e) {
            const uint32_t from = offset(a, e), to = offset(a, e + 1);
            const uint32_t n = to > from ? to - from : 0, tiles = (n + PER - 1) / PER;
            if (left < tiles) return {e, from + left * PER, min(n - left * PER, PER)};
            left -= tiles;
        }
        return {0, 0, 0};
    }
};
// A linear's, all of one matrix.
template <uint32_t PER>
struct RowTiles {
    uint32_t rows;
    __device__ __forceinline__ explicit RowTiles(const ProductArgs& a) : rows(a.rows) {}
    __device__ __forceinline__ uint32_t total() const { return (rows + PER - 1) / PER; }
    __device__ __forceinline__ Tile at(const ProductArgs&, uint32_t unit) const {
        return {0, unit * PER, min(rows - unit * PER, PER)};
    }
};
template <Result R, uint32_t PER>
using Tiles = std::conditional_t<kOfExperts<R>, ExpertTiles<PER>, RowTiles<PER>>;

// As many tiles as there may be.
inline uint64_t most_expert_tiles(uint64_t pairs, uint64_t experts, uint64_t per) {
    const uint64_t used = pairs < experts ? pairs : experts;
    const uint64_t tiles = pairs / per + used;
    return tiles < pairs ? tiles : pairs;
}

// silu(gate) up, the quotient by a reciprocal (good to 2^-23): gate / (1 + e^-gate) exactly
// rounded is a third of what a tile of outputs costs.
__device__ __forceinline__ float silu_product(float gate, float up) {
    return gate * __builtin_amdgcn_rcpf(1.0f + __expf(-gate)) * up;
}

// The row of x that row `first + i` of a tile multiplies.
template <Result R>
__device__ __forceinline__ uint32_t input_row(const ProductArgs& a, uint32_t row) {
    if constexpr (R == Result::kGateUp) {
        // An entry that names no pair reads row 0, in place of memory that is not x.
        const uint32_t pair = static_cast<uint32_t>(a.plan[row]);
        return pair < a.rows ? pair / a.top : 0;
    }
    return row;
}

}  // namespace
}  // namespace mote::mx
