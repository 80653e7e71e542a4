// The experts of each token, and the plan of their products.
//
// Scores of a token's logits x: softmax, exp(x_e - max) / sum, or sigmoid, 1 / (1 +
// exp(-x_e)); choice c_e = score + bias_e.  An expert whose logit or choice is not
// finite takes no part (a masked logit of -infinity: not in the sum either).  With
// groups of experts (each `size` of them, in order), a group's worth is the sum of its best
// one or two choices and only the experts of the best groups stay.  The `top`
// largest choices are taken, the lowest index first among equals.
//
// The choice is a comparison, so scores, choices and worths are held in 64 bits: it is
// then that of the formula, not of roundings, but for logits that differ by less than 2^-50.  A wave
// has a token, expert 64 v + lane in its lanes' slots v; a choice is compared as the unsigned number
// that orders like it, and the largest is found in the upper halves alone unless two
// lanes share it.
#include <hip/hip_runtime.h>

#include <cstdint>
#include <cmath>

#include "mx_products.hpp"

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
__device__ __forceinline__ double lane_value(double v, int lane) {
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = __builtin_amdgcn_readlane(static_cast<int>(b), lane);
    const uint32_t hi = __builtin_amdgcn_readlane(static_cast<int>(b >> 32), lane);
    return __builtin_bit_cast(double, static_cast<uint64_t>(hi) << 32 | lo);
}
__device__ __forceinline__ double wave_sum64(double v) {
#pragma unroll
    for (int by = 1; by < 64; by *= 2) v += __shfl_xor(v, by, 64);
    return v;
}

// Orders as the number does, above 0; 0 is for what takes no part.
__device__ __forceinline__ uint64_t order_of(double v) {
    const uint64_t b = __builtin_bit_cast(uint64_t, v + 0.0);  // -0 as 0
    return b >> 63 ? ~b : b | uint64_t{1} << 63;
}
__device__ __forceinline__ double value_of(uint64_t order) {
    return __builtin_bit_cast(double, order >> 63 ? order & ~(uint64_t{1} << 63) : ~order);
}
__device__ __forceinline__ bool finite(double v) { return __builtin_isfinite(v); }

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
#pragma unroll
    for (int v = 0; v < SLOTS; ++v) {
        const uint32_t e = v * 64 + lane;
        x[v] = e < a.experts ? static_cast<float>(logits[e]) : -__builtin_inff();
        if (!__builtin_isfinite(x[v])) x[v] = -__builtin_inff();
    }
    double score[SLOTS];
    if (a.sigmoid) {
#pragma unroll
        for (int v = 0; v < SLOTS; ++v) score[v] = 1.0 / (1.0 + exp(-static_cast<double>(x[v])));
    } else {
        float most = x[0];
#pragma unroll
        for (int v = 1; v < SLOTS; ++v) most = fmaxf(most, x[v]);
#pragma unroll
        for (int by = 1; by < 64; by *= 2) most = fmaxf(most, __shfl_xor(most, by, 64));
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
    uint64_t choice[SLOTS];
#pragma unroll
    for (int v = 0; v < SLOTS; ++v) {
        const uint32_t e = v * 64 + lane;
        double c = score[v];
        if (a.bias != nullptr && e < a.experts) c += static_cast<double>(a.bias[e]);
        choice[v] = x[v] != -__builtin_inff() && finite(c) ? order_of(c) : 0;
    }
    if constexpr (GROUPED) {
#pragma unroll
        for (int v = 0; v < SLOTS; ++v) choices[wave][v * 64 + lane] = choice[v];
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
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
            double worth = first ? value_of(first) : 0.0;
            if (a.best == 2 && second) worth += value_of(second);
            if (g < a.groups && lane % part == 0) worths[wave][g] = first ? order_of(worth) : 0;
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        // Groups that fewer than top_groups others come before.
#pragma unroll
        for (int v = 0; v < SLOTS; ++v) {
            const uint32_t e = v * 64 + lane;
            if (e >= a.experts) continue;
            const uint32_t mine = e / a.size;
            const uint64_t worth = worths[wave][mine];
            uint32_t before = 0;
            for (uint32_t g = 0; g < a.groups; ++g) {
                const uint64_t other = worths[wave][g];
                before += other > worth || (other == worth && g < mine) ? 1 : 0;
            }
            if (before >= a.top_groups) choice[v] = 0;
        }
    }
    // The largest, `top` times; lane j keeps the j-th.
    int32_t id = -1;
    double weight = 0.0, total = 0.0;
    for (uint32_t j = 0; j < a.top; ++j) {
        uint64_t best = choice[0];
        uint32_t at = 0;
#pragma unroll
        for (int v = 1; v < SLOTS; ++v) {
            at = choice[v] > best ? v : at;
            best = max(best, choice[v]);
        }
        const uint32_t high = wave_max(static_cast<uint32_t>(best >> 32));
        if (high == 0) break;  // an order of 0 alone has an upper half of 0
        uint64_t holders = __builtin_amdgcn_ballot_w64(static_cast<uint32_t>(best >> 32) == high);
        if (holders & (holders - 1)) {
            const bool tied = static_cast<uint32_t>(best >> 32) == high;
            const uint32_t low = wave_max(tied ? static_cast<uint32_t>(best) : 0);
            const bool equal = tied && static_cast<uint32_t>(best) == low;
            holders = __builtin_amdgcn_ballot_w64(equal);
            const uint32_t least = ~wave_max(equal ? ~at : 0);  // the lowest slot, then the lowest lane
            holders = __builtin_amdgcn_ballot_w64(equal && at == least);
        }
        const int winner = __builtin_ctzll(holders);
        const uint32_t slot = static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(at), winner));
        double s = score[0];
#pragma unroll
        for (int v = 0; v < SLOTS; ++v) {
            const bool this_slot = static_cast<uint32_t>(v) == slot;
            s = this_slot ? score[v] : s;
            if (this_slot && lane == static_cast<uint32_t>(winner)) choice[v] = 0;
        }
        s = lane_value(s, winner);
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
// always the same.  A thread has a run of neighbouring pairs, up to kRun of them in its registers
// (so up to 32768 pairs are read once); more go by in rounds that are counted first.
constexpr uint32_t kPlanThreads = 1024;
constexpr uint32_t kRun = 32;

struct Run {
    uint32_t expert[kRun];
};
__device__ __forceinline__ void load_run(const PlanArgs& a, uint32_t first, uint32_t per, Run& run) {
    typedef int32_t i32x4_a4 __attribute__((ext_vector_type(4), aligned(4)));
#pragma unroll
    for (uint32_t i = 0; i < kRun; i += 4) {
        if (i < per && first + i + 4 <= a.pairs) {
            const i32x4_a4 four = *reinterpret_cast<const i32x4_a4*>(a.ids + first + i);
#pragma unroll
            for (uint32_t j = 0; j < 4; ++j) run.expert[i + j] = static_cast<uint32_t>(four[j]);
        } else {
#pragma unroll
            for (uint32_t j = 0; j < 4; ++j)
                run.expert[i + j] = i < per && first + i + j < a.pairs ? static_cast<uint32_t>(a.ids[first + i + j]) : ~0u;
        }
    }
}

// per: pairs of a thread's run in a round, a multiple of 4 up to kRun.
__global__ __launch_bounds__(kPlanThreads) void plan_kernel(PlanArgs a, uint32_t per) {
    __shared__ uint32_t lower_of[kPlanThreads / 64], own_of[kPlanThreads / 64];
    const uint32_t wave = threadIdx.x >> 6, lane = threadIdx.x & 63, waves = blockDim.x >> 6;
    const uint32_t expert = blockIdx.x;
    const uint32_t round = blockDim.x * per, rounds = max((a.pairs + round - 1) / round, 1u);
    const uint32_t mine = threadIdx.x * per;
    Run run;
    uint32_t lower = 0, all = 0;  // of this thread, all rounds
    for (uint32_t r = 0; r < rounds; ++r) {
        load_run(a, r * round + mine, per, run);
#pragma unroll
        for (uint32_t i = 0; i < kRun; ++i) {
            lower += run.expert[i] < expert ? 1 : 0;
            all += run.expert[i] == expert ? 1 : 0;
        }
    }
    // Those of the workgroup, and in one round those of the threads before.
    const uint32_t lower_before = lanes_before(lower), own_before = lanes_before(all);
    if (lane == 63) {
        lower_of[wave] = lower_before + lower;
        own_of[wave] = own_before + all;
    }
    __syncthreads();
    uint32_t begin = 0, total = 0, before = own_before;
    for (uint32_t w = 0; w < waves; ++w) {
        begin += lower_of[w];
        total += own_of[w];
        if (w < wave) before += own_of[w];
    }
    uint32_t at = begin;
    for (uint32_t r = 0; r < rounds && total > 0; ++r) {
        uint32_t own = all, own_total = total;
        if (rounds > 1) {
            load_run(a, r * round + mine, per, run);
            own = 0;
#pragma unroll
            for (uint32_t i = 0; i < kRun; ++i) own += run.expert[i] == expert ? 1 : 0;
            before = lanes_before(own);
            __syncthreads();  // the sums of the round before have been read
            if (lane == 63) own_of[wave] = before + own;
            __syncthreads();
            own_total = 0;
            for (uint32_t w = 0; w < waves; ++w) {
                own_total += own_of[w];
                if (w < wave) before += own_of[w];
            }
        }
        uint32_t to = at + before;
#pragma unroll
        for (uint32_t i = 0; i < kRun; ++i)
            if (run.expert[i] == expert) a.rows[to++] = static_cast<int32_t>(r * round + mine + i);
        at += own_total;
    }
    if (threadIdx.x == 0) a.offsets[expert] = static_cast<int32_t>(begin);
    if (expert + 1 == a.experts) {
        const uint32_t end = begin + total;
        if (threadIdx.x == 0) a.offsets[a.experts] = static_cast<int32_t>(end);
        for (uint32_t p = end + threadIdx.x; p < a.pairs; p += blockDim.x) a.rows[p] = -1;
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
    // Four pairs a thread, more where a thousand threads do not take them all.
    const uint32_t waves = a.pairs >= kPlanThreads * 4 ? kPlanThreads / 64 : max((a.pairs + 255) / 256, 1u);
    const uint32_t each = (a.pairs + waves * 64 - 1) / (waves * 64);
    const uint32_t per = min((max(each, 1u) + 3) & ~3u, kRun);
    hipLaunchKernelGGL(plan_kernel, dim3(a.experts), dim3(waves * 64), 0, static_cast<hipStream_t>(stream), a, per);
    return static_cast<int>(hipGetLastError());
}
