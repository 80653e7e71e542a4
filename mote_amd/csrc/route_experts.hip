// The experts of each token, and the plan of their products.
//
// Scores of a token's logits x: softmax, exp(x_e - max) / sum, or sigmoid, 1 / (1 +
// exp(-x_e)); choice c_e = score + bias_e.  An expert whose logit or choice is not
// finite takes no part (a masked logit of -infinity: not in the sum either).  With
// groups of experts (each `size` of them, in order), a group's worth is the sum of its best
// one or two choices and only the experts of the best groups stay.  The `top`
// largest choices are taken, the lowest index first among equals.
//
// The choice is a comparison, and 64 bits do not tell all scores apart: sigmoids of 37 and
// more are 1, softmaxes of 746 under the largest 0.  Both scores grow with the logit, so without a
// bias the logits are compared, and equal choices by their logits (scores of different logits and biases never
// add up to the very same number).  Worths of two choices that are equal where it matters, between the last group that stays
// and the first that does not, are told apart by what 64 bits dropped (rest_of); the whole token is then
// done again, slowly: 4096 tokens of 256 logits that are all equal, in 8 groups, take 29 us.  What can still come in
// either order are choices of different biases, and worths, less than 2^-50 apart.
//
// A wave has a token, expert 64 v + lane in its lanes' slots v; a choice is compared as the unsigned number
// that orders like it, and the largest is found in the upper halves alone unless two
// lanes share it.  Bound by instructions: 4096 tokens of 256 experts in 8 groups, 8 of them, take 9.3 us one after
// another (their bytes 0.7), for the exponentials in 64 bits and a maximum over the lanes for each expert taken; one token
// of 128 experts 4.0 us, a launch's chain.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>

#include "mx_products.hpp"
#include "tile_ops.hpp"

namespace mote::mx {
namespace {

struct RouteArgs {
    const void* logits;
    const float* bias;  // or null
    int32_t* ids;
    float* weights;
    uint32_t tokens, experts, top, groups, size, top_groups, best;
    bool sigmoid, renormalize;
    float scale;
};

template <int Ctrl, int RowMask = 0xF>
__device__ __forceinline__ uint32_t max_dpp(uint32_t v) {
    const int b = static_cast<int>(v);
    return max(v, static_cast<uint32_t>(__builtin_amdgcn_update_dpp(b, b, Ctrl, RowMask, 0xF, false)));
}
__device__ __forceinline__ uint32_t wave_max(uint32_t v) {
    v = max_dpp<0xB1>(v);        // quad_perm [1,0,3,2]
    v = max_dpp<0x4E>(v);        // quad_perm [2,3,0,1]
    v = max_dpp<0x141>(v);       // row_half_mirror
    v = max_dpp<0x140>(v);       // row_mirror
    v = max_dpp<0x142, 0xA>(v);  // row_bcast:15 into rows 1 and 3
    v = max_dpp<0x143, 0xC>(v);  // row_bcast:31 into rows 2 and 3
    return static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(v), 63));
}
__device__ __forceinline__ uint64_t lane_value(uint64_t v, int lane) {
    const uint32_t lo = __builtin_amdgcn_readlane(static_cast<int>(v), lane);
    const uint32_t hi = __builtin_amdgcn_readlane(static_cast<int>(v >> 32), lane);
    return static_cast<uint64_t>(hi) << 32 | lo;
}
__device__ __forceinline__ double lane_value(double v, int lane) {
    return __builtin_bit_cast(double, lane_value(__builtin_bit_cast(uint64_t, v), lane));
}
template <int Ctrl, int RowMask = 0xF>
__device__ __forceinline__ double add_dpp64(double v) {
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = __builtin_amdgcn_update_dpp(0, static_cast<int>(b), Ctrl, RowMask, 0xF, false);
    const uint32_t hi = __builtin_amdgcn_update_dpp(0, static_cast<int>(b >> 32), Ctrl, RowMask, 0xF, false);
    return v + __builtin_bit_cast(double, static_cast<uint64_t>(hi) << 32 | lo);
}
__device__ __forceinline__ double wave_sum64(double v) {
    v = add_dpp64<0xB1>(v);        // as wave_max; a lane that a step leaves out adds 0
    v = add_dpp64<0x4E>(v);
    v = add_dpp64<0x141>(v);
    v = add_dpp64<0x140>(v);
    v = add_dpp64<0x142, 0xA>(v);
    v = add_dpp64<0x143, 0xC>(v);
    return lane_value(v, 63);
}
// Orders as the number does, above 0; 0 is for what takes no part.
__device__ __forceinline__ uint64_t order_of(double v) {
    const uint64_t b = __builtin_bit_cast(uint64_t, v + 0.0);  // -0 as 0
    return b >> 63 ? ~b : b | uint64_t{1} << 63;
}
__device__ __forceinline__ double value_of(uint64_t order) {
    return __builtin_bit_cast(double, order >> 63 ? order & ~(uint64_t{1} << 63) : ~order);
}
__device__ __forceinline__ uint32_t order_of(float v) {
    const uint32_t b = __builtin_bit_cast(uint32_t, v + 0.0f);
    return b >> 31 ? ~b : b | 0x80000000u;
}
// The largest of finite numbers and -infinity.
__device__ __forceinline__ float wave_max_float(float v) {
    const uint32_t most = wave_max(order_of(v));
    return __builtin_bit_cast(float, most >> 31 ? most & 0x7FFFFFFFu : ~most);
}
__device__ __forceinline__ bool finite(double v) { return __builtin_isfinite(v); }

// Of a logit that is finite, or -infinity for one that takes no part: all in the upper half.
__device__ __forceinline__ uint64_t logit_choice(float x) {
    return x != -__builtin_inff() ? static_cast<uint64_t>(order_of(x)) << 32 : 0;
}

// What tells groups of one worth apart, compared as they stand: the logit, where one choice is
// the worth.  Of two, the parts of their scores that 64 bits drop: a sigmoid is kept as its distance
// from 0 or 1, the nearer, their sum as its distance from the worth, and what that sum drops; softmaxes, which
// may all be 0, as the logarithm of their sum (but for the row's own sum) and the lower logit.
struct Rest {
    uint64_t first, second;
};
template <typename T>
__device__ Rest rest_of(const RouteArgs& a, const T* logits, const uint64_t* choices, uint64_t worth, uint32_t group) {
    uint64_t choice[2] = {};
    float x[2] = {-__builtin_inff(), -__builtin_inff()};
    double bias[2] = {};
    for (uint32_t e = group * a.size; e < (group + 1) * a.size; ++e) {
        const uint64_t c = choices[e];
        const float logit = static_cast<float>(logits[e]);
        const double b = a.bias != nullptr ? static_cast<double>(a.bias[e]) : 0.0;
        const bool best = c > choice[0] || (c == choice[0] && logit > x[0]);
        if (c != 0 && best) choice[1] = choice[0], x[1] = x[0], bias[1] = bias[0];
        if (c != 0 && (best || c > choice[1] || (c == choice[1] && logit > x[1])))
            choice[best ? 0 : 1] = c, x[best ? 0 : 1] = logit, bias[best ? 0 : 1] = b;
    }
    if (a.best == 1 || a.size == 1) return {order_of(static_cast<double>(x[0])), 0};
    // (With a bias the second may have the larger logit.)  e^most as 2^power e^left; what is left of logits so large
    // that it cannot be known is held to where it has to be, under ln 2, which is here in two parts.
    const double most = fmax(x[0], x[1]), least = fmin(x[0], x[1]);
    const double power = floor(most * 0x1.71547652b82fep0);  // log2 e
    const double left = fma(power, -0x1.abc9e3b39803fp-56, fma(power, -0x1.62e42fefa39efp-1, most));
    double t[2] = {a.sigmoid ? -fabs(static_cast<double>(x[0])) : least - most,
                   a.sigmoid ? -fabs(static_cast<double>(x[1])) : fmin(fmax(left, 0.0), 0x1.62e42fefa39efp-1)};
#pragma nounroll
    for (int i = 0; i < 2; ++i) {
        const double e = exp(t[0]);
        t[0] = t[1], t[1] = e;
    }
    if (!a.sigmoid) {
        const double size = (1.0 + t[0]) * t[1];
        return {order_of(size < 2.0 ? power + (size - 1.0) : power + size * 0.5), order_of(least)};
    }
    double whole = bias[0] + bias[1], distance[2] = {};
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        if (choice[i] == 0) continue;
        const double far = t[i] / (1.0 + t[i]);
        whole += x[i] > 0.0f ? 1.0 : 0.0;
        distance[i] = x[i] > 0.0f ? -far : far;
    }
    const double sum = distance[0] + distance[1], of_second = sum - distance[0];
    const double dropped = distance[0] - (sum - of_second) + (distance[1] - of_second);
    return {order_of(whole - value_of(worth) + sum), order_of(dropped)};
}

// Between a wave's writes to LDS and its other lanes' reads there.
__device__ __forceinline__ void wave_fence() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// SLOTS: experts of a lane.  GROUPED: LDS holds the choices and the groups' worths.
template <typename T, int SLOTS, bool GROUPED>
__global__ __launch_bounds__(256) void route_kernel(RouteArgs a) {
    constexpr uint32_t kRoom = GROUPED ? SLOTS * 64 : 1;
    __shared__ uint64_t choices[4][kRoom];
    __shared__ uint64_t worths[4][kRoom];
    const uint32_t wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const uint32_t token = __builtin_amdgcn_readfirstlane(blockIdx.x * 4 + wave);
    if (token >= a.tokens) return;
    const T* logits = static_cast<const T*>(a.logits) + static_cast<uint64_t>(token) * a.experts;
    float x[SLOTS];
    double score[SLOTS];
    uint64_t choice[SLOTS];
    // Without a bias the logits are compared, and so are groups whose worth is one choice.
    const bool by_score = a.bias != nullptr || (GROUPED && a.best == 2 && a.size > 1);
    const auto find_scores = [&] {
#pragma unroll
        for (int v = 0; v < SLOTS; ++v) {
            const uint32_t e = v * 64 + lane;
            x[v] = e < a.experts ? static_cast<float>(logits[e]) : -__builtin_inff();
            if (!__builtin_isfinite(x[v])) x[v] = -__builtin_inff();
        }
        if (a.sigmoid) {
#pragma unroll
            for (int v = 0; v < SLOTS; ++v) score[v] = 1.0 / (1.0 + exp(-static_cast<double>(x[v])));
        } else {
            float most = x[0];
#pragma unroll
            for (int v = 1; v < SLOTS; ++v) most = fmaxf(most, x[v]);
            most = wave_max_float(most);
            double sum = 0.0;
#pragma unroll
            for (int v = 0; v < SLOTS; ++v) {
                const bool there = x[v] != -__builtin_inff();
                score[v] = there ? exp(static_cast<double>(x[v]) - static_cast<double>(most)) : 0.0;
                sum += score[v];
            }
            const double part = 1.0 / wave_sum64(sum);  // of no expert: unused
#pragma unroll
            for (int v = 0; v < SLOTS; ++v) score[v] *= part;
        }
        if (by_score) {
#pragma unroll
            for (int v = 0; v < SLOTS; ++v) {
                const uint32_t e = v * 64 + lane;
                double c = score[v];
                if (a.bias != nullptr && e < a.experts) c += static_cast<double>(a.bias[e]);
                choice[v] = x[v] != -__builtin_inff() && finite(c) ? order_of(c) : 0;
            }
        } else {
#pragma unroll
            for (int v = 0; v < SLOTS; ++v) choice[v] = logit_choice(x[v]);
        }
    };
    find_scores();
    if constexpr (GROUPED) {
#pragma unroll
        for (int v = 0; v < SLOTS; ++v) choices[wave][v * 64 + lane] = choice[v];
        wave_fence();
        // `part` lanes share a group: its choices in turn, then their bests across the lanes.
        uint32_t part = 1;
        while (part * 2 * a.groups <= 64) part *= 2;
        for (uint32_t first_group = 0; first_group < a.groups; first_group += 64 / part) {
            const uint32_t g = first_group + lane / part;
            uint64_t first = 0, second = 0;
            if (g < a.groups) {
                for (uint32_t i = lane % part; i < a.size; i += part) {
                    const uint64_t c = choices[wave][g * a.size + i];
                    second = max(second, min(first, c));
                    first = max(first, c);
                }
            }
            for (uint32_t by = 1; by < part; by *= 2) {
                const uint64_t c = __shfl_xor(first, by, 64), d = __shfl_xor(second, by, 64);
                second = max(max(second, d), min(first, c));
                first = max(first, c);
            }
            if (a.best == 2 && second != 0) first = order_of(value_of(first) + value_of(second));
            if (g < a.groups && lane % part == 0) worths[wave][g] = first;
        }
        wave_fence();
        // Groups that fewer than top_groups others come before stay.
        const float part_of = 1.0f / static_cast<float>(a.size);  // e / size: e + 1/2 is 2^-11 away from the next
        uint64_t last_in = 0, first_out = 0;  // worths
        const auto note_border = [&](uint32_t before, uint64_t worth) {
            const uint64_t in = __builtin_amdgcn_ballot_w64(before == a.top_groups - 1);
            const uint64_t out = __builtin_amdgcn_ballot_w64(before == a.top_groups);
            if (in != 0) last_in = lane_value(worth, __builtin_ctzll(in));
            if (out != 0) first_out = lane_value(worth, __builtin_ctzll(out));
        };
        if (a.groups <= 64) {
            const uint64_t worth = lane < a.groups ? worths[wave][lane] : 0;
            uint32_t before = 0;
            for (uint32_t g = 0; g < a.groups; ++g) {
                const uint64_t other = lane_value(worth, g);
                before += other > worth || (other == worth && g < lane) ? 1 : 0;
            }
            note_border(before, worth);
            const uint64_t kept = __builtin_amdgcn_ballot_w64(before < a.top_groups);
#pragma unroll
            for (int v = 0; v < SLOTS; ++v) {
                const uint32_t g = static_cast<uint32_t>((static_cast<float>(v * 64 + lane) + 0.5f) * part_of);
                if (!(kept >> (g & 63) & 1)) choice[v] = 0;
            }
        } else {
#pragma unroll
            for (int v = 0; v < SLOTS; ++v) {
                const uint32_t mine = min((v * 64 + lane) / a.size, a.groups - 1);
                const uint64_t worth = worths[wave][mine];
                uint32_t before = 0;
                for (uint32_t g = 0; g < a.groups; ++g) {
                    const uint64_t other = worths[wave][g];
                    before += other > worth || (other == worth && g < mine) ? 1 : 0;
                }
                note_border(before, worth);
                if (before >= a.top_groups) choice[v] = 0;
            }
        }
        if (by_score && last_in == first_out && last_in != 0) {
            // What tells equal worths apart, over choices that have been read.  Then all once more: to
            // keep scores and choices meanwhile takes registers that halve the waves at work (16384 tokens of 256
            // experts 28 us, 25 as here, whether there are such worths or not).
            uint64_t* const rests = choices[wave];
            const uint32_t each = min(a.size, 2u), last = each - 1;
            for (uint32_t first_group = 0; first_group < a.groups; first_group += 64) {
                const uint32_t g = first_group + lane;
                Rest rest{};
                if (g < a.groups && worths[wave][g] != 0) rest = rest_of(a, logits, rests, worths[wave][g], g);
                wave_fence();
                if (g < a.groups) {
                    rests[g * each] = rest.first;
                    if (each == 2) rests[g * 2 + 1] = rest.second;
                }
                wave_fence();
            }
            memory_fence();
            find_scores();
#pragma unroll
            for (int v = 0; v < SLOTS; ++v) {
                const uint32_t mine = min((v * 64 + lane) / a.size, a.groups - 1);
                const uint64_t worth = worths[wave][mine], first = rests[mine * each], second = rests[mine * each + last];
                uint32_t before = 0;
                for (uint32_t g = 0; g < a.groups; ++g) {
                    const uint64_t w = worths[wave][g], f = rests[g * each], s = rests[g * each + last];
                    const bool level = w == worth && f == first;
                    before += w > worth || (w == worth && f > first) || (level && (s > second || (s == second && g < mine)))
                                  ? 1
                                  : 0;
                }
                if (before >= a.top_groups) choice[v] = 0;
            }
        }
    }
    if (GROUPED && by_score && a.bias == nullptr) {
#pragma unroll
        for (int v = 0; v < SLOTS; ++v) choice[v] = choice[v] != 0 ? logit_choice(x[v]) : 0;
    }
    // The largest, `top` times; lane j keeps the j-th.  The upper halves decide unless two are equal.
    int32_t id = -1;
    double weight = 0.0, total = 0.0;
    uint32_t high[SLOTS];
#pragma unroll
    for (int v = 0; v < SLOTS; ++v) high[v] = static_cast<uint32_t>(choice[v] >> 32);
    for (uint32_t j = 0; j < a.top; ++j) {
        uint32_t mine = high[0];
#pragma unroll
        for (int v = 1; v < SLOTS; ++v) mine = max(mine, high[v]);
        const uint32_t most = wave_max(mine);
        if (most == 0) break;  // nothing left: an order of 0 alone has an upper half of 0
        uint64_t holders[SLOTS];
        uint32_t count = 0, slot = 0;
#pragma unroll
        for (int v = SLOTS - 1; v >= 0; --v) {
            holders[v] = __builtin_amdgcn_ballot_w64(high[v] == most);
            count += __builtin_popcountll(holders[v]);
            slot = holders[v] ? v : slot;  // the lowest
        }
        if (count > 1) {
            uint32_t low = 0;
#pragma unroll
            for (int v = 0; v < SLOTS; ++v) low = max(low, high[v] == most ? static_cast<uint32_t>(choice[v]) : 0);
            low = wave_max(low);
#pragma unroll
            for (int v = SLOTS - 1; v >= 0; --v) {
                holders[v] = __builtin_amdgcn_ballot_w64(high[v] == most && static_cast<uint32_t>(choice[v]) == low);
                slot = holders[v] ? v : slot;
            }
            if (a.bias != nullptr) {  // equal sums: the larger logit (read again: few rows come here)
                uint32_t order[SLOTS], largest = 0;
#pragma unroll
                for (int v = 0; v < SLOTS; ++v) {
                    const bool holds = holders[v] >> lane & 1;
                    order[v] = holds ? order_of(static_cast<float>(logits[v * 64 + lane])) : 0;
                    largest = max(largest, order[v]);
                }
                largest = wave_max(largest);
#pragma unroll
                for (int v = SLOTS - 1; v >= 0; --v) {
                    holders[v] = __builtin_amdgcn_ballot_w64(order[v] == largest);
                    slot = holders[v] ? v : slot;
                }
            }
        }
        int winner = 0;
        double s = 0.0;
#pragma unroll
        for (int v = 0; v < SLOTS; ++v) {
            if (static_cast<uint32_t>(v) == slot) {  // the same in all lanes
                winner = __builtin_ctzll(holders[v]);
                s = lane_value(score[v], winner);
                high[v] = lane == static_cast<uint32_t>(winner) ? 0 : high[v];
            }
        }
        total += s;
        if (lane == j) {
            id = static_cast<int32_t>(slot * 64 + winner);
            weight = s;
        }
    }
    if (lane < a.top) {
        if (a.renormalize) weight = total > 0.0 ? weight / total : 0.0;
        const uint64_t out = static_cast<uint64_t>(token) * a.top + lane;
        a.ids[out] = id;
        a.weights[out] = static_cast<float>(weight * static_cast<double>(a.scale));
    }
}

struct PlanArgs {
    const int32_t* ids;
    int32_t* offsets;
    int32_t* rows;
    uint32_t pairs, experts;
};

// A workgroup for each expert: it counts the pairs of lower experts, which is where its own
// begin, and its own, then writes its own in their order.  No counter is shared, so the order is
// always the same.  A thread has four neighbouring pairs in each of up to kTurns turns, all
// in its registers (so up to 32768 pairs are read once, with whole lines to a wave); a wave's own are bits of
// ballots, and where they go is a prefix sum over turns and waves.  More pairs go by in rounds that are
// counted first.  Bound by the ids, which every workgroup reads from the L2 and compares: 32768 pairs of 256
// experts 7.9 to 8.4 us, a token's eight of 128 experts 2.9.
constexpr uint32_t kPlanThreads = 1024, kPlanWaves = kPlanThreads / 64, kMostTurns = 8;

// per: turns of a round, up to TURNS (one, where that is all: a single token's plan is bound by
// the reading of the code).
template <uint32_t TURNS>
__global__ __launch_bounds__(kPlanThreads) void plan_kernel(PlanArgs a, uint32_t per) {
    __shared__ uint32_t lower_of[kPlanWaves], own_of[TURNS * kPlanWaves];
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const uint32_t waves = blockDim.x >> 6, expert = blockIdx.x;
    const uint32_t round = blockDim.x * 4 * per, rounds = max((a.pairs + round - 1) / round, 1u);
    typedef int32_t i32x4_a4 __attribute__((ext_vector_type(4), aligned(4)));
    uint32_t of[TURNS][4];
    const auto first_of = [&](uint32_t r, uint32_t turn) { return r * round + (turn * blockDim.x + threadIdx.x) * 4; };
    const auto load = [&](uint32_t r) {
#pragma unroll
        for (uint32_t t = 0; t < TURNS; ++t) {
            const uint32_t first = first_of(r, t);
            if (t < per && first + 4 <= a.pairs) {
                const i32x4_a4 four = *reinterpret_cast<const i32x4_a4*>(a.ids + first);
#pragma unroll
                for (uint32_t j = 0; j < 4; ++j) of[t][j] = static_cast<uint32_t>(four[j]);
            } else {
#pragma unroll
                for (uint32_t j = 0; j < 4; ++j)
                    of[t][j] = t < per && first + j < a.pairs ? static_cast<uint32_t>(a.ids[first + j]) : ~0u;
            }
        }
    };
    const auto own_bits = [&](uint32_t t, uint32_t j) { return __builtin_amdgcn_ballot_w64(of[t][j] == expert); };
    const auto count_turns = [&] {  // each turn's own of the wave, to own_of
#pragma unroll
        for (uint32_t t = 0; t < TURNS; ++t) {
            uint32_t own = 0;
#pragma unroll
            for (uint32_t j = 0; j < 4; ++j) own += __builtin_popcountll(own_bits(t, j));
            if (lane == 0 && t < per) own_of[t * waves + wave] = own;
        }
    };
    uint32_t lower = 0;
    for (uint32_t r = 0; r < rounds; ++r) {
        load(r);
#pragma unroll
        for (uint32_t t = 0; t < TURNS; ++t)
#pragma unroll
            for (uint32_t j = 0; j < 4; ++j) lower += __builtin_popcountll(__builtin_amdgcn_ballot_w64(of[t][j] < expert));
    }
    if (rounds == 1) count_turns();
    if (lane == 0) lower_of[wave] = lower;
    __syncthreads();
    uint32_t at = 0;
    for (uint32_t w = 0; w < waves; ++w) at += lower_of[w];
    const uint32_t begin = at;
    for (uint32_t r = 0; r < rounds; ++r) {
        if (rounds > 1) {
            load(r);
            __syncthreads();  // the turns of the round before have been read
            count_turns();
            __syncthreads();
        }
        // Turn t of wave w is entry t waves + w: lane l adds up entries 2 l and 2 l + 1.
        const uint32_t entries = per * waves;
        const uint32_t a0 = 2 * lane < entries ? own_of[2 * lane] : 0;
        const uint32_t a1 = 2 * lane + 1 < entries ? own_of[2 * lane + 1] : 0;
        const uint32_t before = lanes_before(a0 + a1);
        const uint32_t all = static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(before + a0 + a1), 63));
#pragma unroll
        for (uint32_t t = 0; t < TURNS; ++t) {
            uint64_t bits[4], any = 0;
#pragma unroll
            for (uint32_t j = 0; j < 4; ++j) any |= bits[j] = own_bits(t, j);
            if (any == 0) continue;
            const uint32_t entry = t * waves + wave;
            uint32_t to = at + static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(before), entry / 2));
            if (entry & 1) to += static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(a0), entry / 2));
#pragma unroll
            for (uint32_t j = 0; j < 4; ++j)
                to += __builtin_popcountll(bits[j] & ((uint64_t{1} << lane) - 1));
#pragma unroll
            for (uint32_t j = 0; j < 4; ++j)
                if (of[t][j] == expert) a.rows[to++] = static_cast<int32_t>(first_of(r, t) + j);
        }
        at += all;
    }
    if (threadIdx.x == 0) a.offsets[expert] = static_cast<int32_t>(begin);
    if (expert + 1 == a.experts) {
        if (threadIdx.x == 0) a.offsets[a.experts] = static_cast<int32_t>(at);
        for (uint32_t p = at + threadIdx.x; p < a.pairs; p += blockDim.x) a.rows[p] = -1;
    }
}

template <typename T>
int route(const void* logits, const void* bias, void* ids, void* weights, uint64_t tokens, uint64_t experts,
          uint64_t top, int score, uint64_t groups, uint64_t top_groups, int group_best, int renormalize, float scale,
          void* stream) {
    if (!logits || !ids || !weights || !stream) return kInvalid;
    if (off_grid(logits, sizeof(T)) || off_grid(bias, 4) || off_grid(ids, 4) || off_grid(weights, 4)) return kInvalid;
    if (score < 0 || score > 1 || group_best < 1 || group_best > 2 || renormalize < 0 || renormalize > 1)
        return kInvalid;
    if (!std::isfinite(scale) || experts > kMostExperts || top > experts || top > kMostTop || tokens > kMostRows)
        return kInvalid;
    if (groups < 1 || top_groups < 1 || top_groups > groups) return kInvalid;
    if (tokens == 0 || experts == 0 || top == 0) return 0;
    if (experts % groups != 0 || top > top_groups * (experts / groups) || tokens * top > kMostRows) return kInvalid;
    const uint64_t workgroups = (tokens + 3) / 4;
    if (workgroups * 256 > kMostThreads) return kInvalid;
    const RouteArgs a{logits,
                      static_cast<const float*>(bias),
                      static_cast<int32_t*>(ids),
                      static_cast<float*>(weights),
                      static_cast<uint32_t>(tokens),
                      static_cast<uint32_t>(experts),
                      static_cast<uint32_t>(top),
                      static_cast<uint32_t>(groups),
                      static_cast<uint32_t>(experts / groups),
                      static_cast<uint32_t>(top_groups),
                      static_cast<uint32_t>(group_best),
                      score == 1,
                      renormalize == 1,
                      scale};
    const auto go = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, dim3(static_cast<uint32_t>(workgroups)), dim3(256), 0,
                           static_cast<hipStream_t>(stream), a);
    };
    const auto slots = [&](auto grouped) {
        constexpr bool kGrouped = decltype(grouped)::value;
        if (experts <= 64)
            go(route_kernel<T, 1, kGrouped>);
        else if (experts <= 128)
            go(route_kernel<T, 2, kGrouped>);
        else if (experts <= 256)
            go(route_kernel<T, 4, kGrouped>);
        else if (experts <= 512)
            go(route_kernel<T, 8, kGrouped>);
        else
            go(route_kernel<T, 16, kGrouped>);
    };
    if (top_groups < groups)
        slots(std::true_type{});
    else
        slots(std::false_type{});
    return static_cast<int>(hipGetLastError());
}

}  // namespace
}  // namespace mote::mx

MOTE_EXPORT int mote_hip_route_experts_f16(const void* logits, const void* bias, void* ids, void* weights,
                                           uint64_t tokens, uint64_t experts, uint64_t top, int score, uint64_t groups,
                                           uint64_t top_groups, int group_best, int renormalize, float scale,
                                           void* stream) noexcept {
    return mote::mx::route<_Float16>(logits, bias, ids, weights, tokens, experts, top, score, groups, top_groups,
                                     group_best, renormalize, scale, stream);
}
MOTE_EXPORT int mote_hip_route_experts_f32(const void* logits, const void* bias, void* ids, void* weights,
                                           uint64_t tokens, uint64_t experts, uint64_t top, int score, uint64_t groups,
                                           uint64_t top_groups, int group_best, int renormalize, float scale,
                                           void* stream) noexcept {
    return mote::mx::route<float>(logits, bias, ids, weights, tokens, experts, top, score, groups, top_groups,
                                  group_best, renormalize, scale, stream);
}

MOTE_EXPORT int mote_hip_plan_experts(const void* ids, void* offsets, void* rows, uint64_t tokens, uint64_t top,
                                      uint64_t experts, void* stream) noexcept {
    using namespace mote::mx;
    if (!ids || !offsets || !rows || !stream) return kInvalid;
    if (off_grid(ids, 4) || off_grid(offsets, 4) || off_grid(rows, 4)) return kInvalid;
    if (tokens > kMostRows || top > kMostTop || tokens * top > kMostRows || experts > kMostExperts) return kInvalid;
    if (experts == 0) return 0;
    const PlanArgs a{static_cast<const int32_t*>(ids), static_cast<int32_t*>(offsets), static_cast<int32_t*>(rows),
                     static_cast<uint32_t>(tokens * top), static_cast<uint32_t>(experts)};
    // Four pairs a thread, more turns where a thousand threads do not take them all.
    const uint32_t waves = a.pairs >= kPlanThreads * 4 ? kPlanWaves : std::max((a.pairs + 255) / 256, 1u);
    const uint32_t turns = (a.pairs + waves * 256 - 1) / (waves * 256);
    const uint32_t per = std::min(std::max(turns, 1u), kMostTurns);
    const auto go = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, dim3(a.experts), dim3(waves * 64), 0, static_cast<hipStream_t>(stream), a, per);
    };
    per == 1 ? go(plan_kernel<1>) : go(plan_kernel<kMostTurns>);
    return static_cast<int>(hipGetLastError());
}
