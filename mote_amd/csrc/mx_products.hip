// Products of microscaled rows: y = x W^T, and those of experts, each with its own
// weights and rows.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>
#include <utility>

#include "mx_products.hpp"

namespace mote::mx {
namespace {

// Few rows: HBM-bound on the weights.  A workgroup has one tile of up to 16 rows and the
// columns part, part + parts, ... of 16 outputs (of gate and of up each).  A wave has
// STEPS steps of K, the same for every column, and the waves' sums meet in LDS, in their order.
//
// A lane's operand is a 16-byte piece of a weights' row as it is stored, so nothing is
// unpacked; what costs time beside the memory is the number of load instructions (one row, 14336 x 4096, which
// the tiles take by now, 31 MB in the memory-side cache, 5.0 us at the rate of reads alone: weights alone 6.9 us, with
// their scales a word at a time and x at each step 11.5, as here 8.2).  So scales are loaded four steps at a
// time, x once for all of the workgroup's columns, and a step's weights for the next column as
// soon as they have been multiplied.
constexpr uint32_t kFewRows = 16;

template <typename F, int... I>
__device__ __forceinline__ void each_of(F f, std::integer_sequence<int, I...>) {
    (f(std::integral_constant<int, I>{}), ...);
}

template <int BITS, Result R, int STEPS, int MOST_WAVES>
__global__ __launch_bounds__(MOST_WAVES * 64) void few_rows_kernel(ProductArgs a, uint32_t parts) {
    constexpr int kSides = R == Result::kGateUp ? 2 : 1;
    typedef uint32_t u32x4_a4 __attribute__((ext_vector_type(4), aligned(4)));
    extern __shared__ f32x4 sums[];  // [2][waves][kSides][64]
    const uint32_t unit = blockIdx.x / parts, part = blockIdx.x % parts;
    const Tile tile = Tiles<R, kFewRows>(a).at(a, unit);
    if (tile.count == 0) return;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
    const uint32_t lane = threadIdx.x & 63, of16 = lane & 15, group = lane >> 4;
    const uint32_t columns = (a.outputs + 15) / 16;
    const uint32_t steps = a.kp / kStep, first = wave * STEPS;
    const uint32_t mine = first < steps ? min(steps - first, uint32_t{STEPS}) : 0;
    const auto step_at = [&](int i) { return min(first + i, steps - 1); };  // past the end the last again, unused
    const auto each_step = [](auto does) { each_of(does, std::make_integer_sequence<int, STEPS>{}); };

    u32x4 w[STEPS][kSides];
    uint32_t ws[STEPS][kSides];
    const uint8_t* w_row[kSides];
    const auto to_column = [&](uint32_t column) {  // and its scales
#pragma unroll
        for (int side = 0; side < kSides; ++side) {
            const uint64_t row = (static_cast<uint64_t>(tile.expert) * kSides + side) * a.outputs +
                                 min(column * 16 + of16, a.outputs - 1);
            w_row[side] = a.w + row * value_bytes(a.kp, 4);
            const uint32_t* scales = reinterpret_cast<const uint32_t*>(a.w_scales + row * scale_bytes(a.kp));
            if (mine == STEPS) {
#pragma unroll
                for (int i = 0; i < STEPS; i += 4) {
                    const u32x4 four = *reinterpret_cast<const u32x4_a4*>(scales + first + i);
#pragma unroll
                    for (int j = 0; j < 4; ++j) ws[i + j][side] = four[j];
                }
            } else {
#pragma unroll
                for (int i = 0; i < STEPS; ++i) ws[i][side] = scales[step_at(i)];
            }
        }
    };
    const auto load_w = [&](auto at) {
        constexpr int I = decltype(at)::value;
#pragma unroll
        for (int side = 0; side < kSides; ++side)
            w[I][side] = *reinterpret_cast<const u32x4*>(w_row[side] + step_at(I) * 64 + group * 16);
    };
    i32x8 x[STEPS];
    uint32_t xs[STEPS];
    if (mine > 0) {
        to_column(part);
        each_step(load_w);
        const uint64_t row = input_row<R>(a, tile.first + min(of16, tile.count - 1));
        const uint8_t* const values = a.x + row * value_bytes(a.kp, BITS);
        const uint32_t* const scales = reinterpret_cast<const uint32_t*>(a.x_scales + row * scale_bytes(a.kp));
        each_step([&](auto at) {
            constexpr int I = decltype(at)::value;
            x[I] = load_block<BITS>(values, a.kp, step_at(I) * 4 + group).operand();
            xs[I] = scales[step_at(I)] >> (8 * group);
        });
    }
    uint32_t buffer = 0, turn = 0;
    for (uint32_t column = part; column < columns; column += parts, buffer ^= 1) {
        f32x4 d[kSides] = {};
        if (mine > 0) {
            uint32_t now[STEPS][kSides];
#pragma unroll
            for (int i = 0; i < STEPS; ++i)
#pragma unroll
                for (int side = 0; side < kSides; ++side) now[i][side] = ws[i][side] >> (8 * group);
            const auto multiply = [&](auto at) {
                constexpr int I = decltype(at)::value;
                if (static_cast<uint32_t>(I) < mine) {
#pragma unroll
                    for (int side = 0; side < kSides; ++side)
                        d[side] = multiply16<BITS>(Block<4>{w[I][side]}.operand(), now[I][side], x[I], xs[I], d[side]);
                }
            };
            if (column + parts < columns) {
                to_column(column + parts);
                each_step([&](auto at) {
                    multiply(at);
                    load_w(at);
                });
            } else {
                each_step(multiply);
            }
        }
        f32x4* const of_buffer = sums + buffer * waves * (kSides * 64);
#pragma unroll
        for (int side = 0; side < kSides; ++side) of_buffer[(wave * kSides + side) * 64 + lane] = d[side];
        __syncthreads();  // (Two buffers: the one before has been read by all who are past this.)
        // The waves take turns, so that one adds while the others go on.
        const bool this_wave = turn == wave;
        turn = turn + 1 == waves ? 0 : turn + 1;
        if (!this_wave) continue;
        const uint32_t n = column * 16 + 4 * group;
        f32x4 total[kSides] = {};
        for (uint32_t v = 0; v < waves; ++v) {
#pragma unroll
            for (int side = 0; side < kSides; ++side) total[side] += of_buffer[(v * kSides + side) * 64 + lane];
        }
        if (of16 >= tile.count || n >= a.outputs) continue;
        uint64_t to = tile.first + of16;
        if constexpr (R == Result::kPairs) {
            to = static_cast<uint32_t>(a.plan[to]);
            if (to >= a.rows) continue;
        }
        to = to * a.outputs + n;
#pragma unroll
        for (uint32_t r = 0; r < 4; ++r) {
            if (n + r >= a.outputs) break;
            if constexpr (R == Result::kGateUp)
                static_cast<_Float16*>(a.output)[to + r] =
                    static_cast<_Float16>(silu_product(total[0][r], total[kSides - 1][r]));
            else if constexpr (R == Result::kF16)
                static_cast<_Float16*>(a.output)[to + r] = static_cast<_Float16>(total[0][r]);
            else
                static_cast<float*>(a.output)[to + r] = total[0][r];
        }
    }
}

// output[t] = the sum over j, in order, of weights[t][j] times the product of pair (t, j),
// left out where the pair has no expert.
struct CombineArgs {
    const float* products;  // [tokens top][hidden]
    const int32_t* ids;
    const float* weights;
    _Float16* output;
    uint32_t hidden, top, experts, parts;  // parts: workgroups of a token
};
__global__ __launch_bounds__(256) void combine_kernel(CombineArgs a) {
    const uint32_t token = blockIdx.x / a.parts;
    const uint32_t n = ((blockIdx.x % a.parts) * 256 + threadIdx.x) * 4;  // four outputs: hidden is whole blocks
    if (n >= a.hidden) return;
    f32x4 y = {};
    for (uint32_t j = 0; j < a.top; ++j) {
        const uint64_t pair = static_cast<uint64_t>(token) * a.top + j;
        if (static_cast<uint32_t>(a.ids[pair]) >= a.experts) continue;
        const f32x4 product = *reinterpret_cast<const f32x4*>(a.products + pair * a.hidden + n);
        const float weight = a.weights[pair];
#pragma unroll
        for (int r = 0; r < 4; ++r) y[r] = __builtin_fmaf(weight, product[r], y[r]);
    }
    typedef _Float16 f16x4_a2 __attribute__((ext_vector_type(4), aligned(2)));
    *reinterpret_cast<f16x4_a2*>(a.output + static_cast<uint64_t>(token) * a.hidden + n) =
        f16x4_a2{static_cast<_Float16>(y[0]), static_cast<_Float16>(y[1]), static_cast<_Float16>(y[2]),
                 static_cast<_Float16>(y[3])};
}

// Columns of a workgroup: more of them share the loads of x, but there have to be workgroups enough (gate/up of 32
// tokens' four experts of 2880 x 2880, some 5600 columns: one each 75 us, two 65, four 63, eight 62; one
// row, 4096 x 14336, 256 columns: 10.4 with one, 13.0 with two).
constexpr uint64_t kWorkgroups = 448, kMostColumns = 4;

template <int BITS, Result R, int STEPS, int MOST_WAVES>
int launch_few(const ProductArgs& a, hipStream_t stream) {
    constexpr uint32_t kSides = R == Result::kGateUp ? 2 : 1;
    const uint32_t columns = (a.outputs + 15) / 16, steps = a.kp / kStep;
    const uint64_t units = kOfExperts<R> ? most_expert_tiles(a.rows, a.experts, kFewRows)
                                         : (uint64_t{a.rows} + kFewRows - 1) / kFewRows;
    const uint64_t each = std::min(std::max(units * columns / kWorkgroups, uint64_t{1}), kMostColumns);
    const uint32_t parts = static_cast<uint32_t>((columns + each - 1) / each);
    const uint32_t waves = steps > STEPS ? (steps + STEPS - 1) / STEPS : 1;
    if (units * parts > kMostThreads / (waves * 64)) return kInvalid;
    hipLaunchKernelGGL((few_rows_kernel<BITS, R, STEPS, MOST_WAVES>), dim3(static_cast<uint32_t>(units * parts)),
                       dim3(waves * 64), 2 * waves * kSides * 1024, stream, a, parts);
    return static_cast<int>(hipGetLastError());
}

// Few rows, where the tiles (mx_tiles.hip) would leave much of the chip without one, or work with few of their rows:
// - a linear of up to 16 rows whose weights are few long rows (one row, 4096 x 14336 10.5 us, 13.2 in tiles;
//   4096 x 4096 5.8 and 5.1, 1024 x 8192 6.8 and 6.1; 14336 x 4096 9.4 in both, from the memory-side
//   cache 8.2 and 6.0);
// - gate/up of less than 8 rows of an expert in the mean (32 experts of 2880 x 2880, 6 bits: a row each 41 us and
//   44, 4 rows 63 and 66, 8 rows 74 and 71; 128 experts of 768 x 2048, 8 rows 54 and 45);
// - down of up to 8, where there are few tiles (8 experts of 4096 x 14336, 4 tokens of two: 256 tiles, 30 us
//   and 60; 64 experts of 4096 x 1408, 2 tokens of six: 384, 15.8 and 16.9; 128 of 2048 x 768, 4 of eight:
//   512, 15.3 and 13.0);
// - and K too short for the tiles' four steps, for any number of rows.  That is right but slow where there are
//   many: every 16 rows read the weights again, and results leave 2 or 4 bytes a lane (K 128, 256 and 384 here,
//   and 512 in tiles: 4096 x 4096 outputs 45, 65, 57 and 12 us; 8192 x 14336, 6 bits, 318, 451, 436 and 80; gate/up of
//   4096 tokens' four of 32 experts of 2880 181, 277, 254 and 91; down of 4096 tokens' eight of 128 experts to 2048
//   268, 333, 335 and 151; 16 x 4096 4.7, 4.8, 4.9 and 4.5).
template <Result R>
bool few_rows(const ProductArgs& a) {
    const uint64_t columns = a.outputs, steps = a.kp / kStep;
    if (steps < 4) return true;
    if constexpr (R == Result::kGateUp) return a.rows < 8 * uint64_t{a.experts} && steps <= 64;
    if constexpr (R == Result::kPairs)
        return a.rows <= 8 * uint64_t{a.experts} && steps <= 128 &&
               most_expert_tiles(a.rows, a.experts, 64) * ((columns + 127) / 128) < 512;
    return a.rows <= kFewRows && (columns + 31) / 32 < kEnoughTiles && steps > 64 && steps <= 128;
}

template <int BITS, Result R>
int launch_bits(const ProductArgs& a, hipStream_t stream) {
    if (!few_rows<R>(a)) return launch_tiles(R, a, BITS, stream);
    if constexpr (R != Result::kGateUp) {  // (twice the registers: no eight steps of K a wave)
        if (a.kp / kStep > 64) return launch_few<BITS, R, 8, 16>(a, stream);
    }
    return launch_few<BITS, R, 4, 16>(a, stream);
}

template <Result R>
int launch(const ProductArgs& a, int bits, hipStream_t stream) {
    return bits == 4 ? launch_bits<4, R>(a, stream) : launch_bits<6, R>(a, stream);
}

// Sizes and addresses that every product needs.
bool operands_ok(const void* x, const void* x_scales, const void* w, const void* w_scales, const void* stream,
                 uint64_t features, uint64_t outputs, int bits) {
    if (!x || !x_scales || !w || !w_scales || !stream || !known_bits(bits)) return false;
    if (off_grid(x, 16) || off_grid(w, 16) || off_grid(x_scales, 4) || off_grid(w_scales, 4)) return false;
    return features % kBlock == 0 && features <= kMostFeatures && outputs <= kMostFeatures;
}
bool experts_ok(uint64_t tokens, uint64_t top, uint64_t experts, uint64_t hidden, uint64_t inner) {
    return tokens <= kMostRows && top <= kMostTop && tokens * top <= kMostRows && experts <= kMostExperts &&
           hidden % kBlock == 0 && hidden <= kMostFeatures && inner % kBlock == 0 && inner <= kMostFeatures;
}

ProductArgs arguments(const void* x, const void* x_scales, const void* w, const void* w_scales, void* output,
                      uint64_t rows, uint64_t outputs, uint64_t features) {
    return {static_cast<const uint8_t*>(x),
            static_cast<const uint8_t*>(x_scales),
            static_cast<const uint8_t*>(w),
            static_cast<const uint8_t*>(w_scales),
            output,
            nullptr,
            nullptr,
            static_cast<uint32_t>(rows),
            static_cast<uint32_t>(outputs),
            padded(features),
            1,
            1};
}

template <Result R>
int linear(const void* x, const void* x_scales, const void* w, const void* w_scales, void* output, uint64_t rows,
           uint64_t outputs, uint64_t features, int bits, void* stream) {
    if (!output || !operands_ok(x, x_scales, w, w_scales, stream, features, outputs, bits)) return kInvalid;
    if (off_grid(output, R == Result::kF16 ? 2 : 4) || rows > kMostRows) return kInvalid;
    if (rows == 0 || outputs == 0) return 0;
    return launch<R>(arguments(x, x_scales, w, w_scales, output, rows, outputs, features), bits,
                     static_cast<hipStream_t>(stream));
}

// The products of the pairs, on the grid of the output's vector stores.
uint64_t down_bytes(uint64_t pairs, uint64_t hidden) { return pairs * hidden * 4; }

}  // namespace
}  // namespace mote::mx

MOTE_EXPORT int mote_hip_mx_linear_f16(const void* input_values, const void* input_scales, const void* weight_values,
                                       const void* weight_scales, void* output, uint64_t rows, uint64_t output_features,
                                       uint64_t input_features, int input_bits, void* stream) noexcept {
    return mote::mx::linear<mote::mx::Result::kF16>(input_values, input_scales, weight_values, weight_scales, output,
                                                    rows, output_features, input_features, input_bits, stream);
}
MOTE_EXPORT int mote_hip_mx_linear_f32(const void* input_values, const void* input_scales, const void* weight_values,
                                       const void* weight_scales, void* output, uint64_t rows, uint64_t output_features,
                                       uint64_t input_features, int input_bits, void* stream) noexcept {
    return mote::mx::linear<mote::mx::Result::kF32>(input_values, input_scales, weight_values, weight_scales, output,
                                                    rows, output_features, input_features, input_bits, stream);
}

MOTE_EXPORT int mote_hip_experts_gate_up_silu_mx_f16(const void* input_values, const void* input_scales,
                                                     const void* weight_values, const void* weight_scales,
                                                     const void* offsets, const void* plan_rows, void* output,
                                                     uint64_t tokens, uint64_t top, uint64_t experts, uint64_t hidden,
                                                     uint64_t inner, int input_bits, void* stream) noexcept {
    using namespace mote::mx;
    if (!output || !offsets || !plan_rows || off_grid(output, 2) || off_grid(offsets, 4) || off_grid(plan_rows, 4))
        return kInvalid;
    if (!operands_ok(input_values, input_scales, weight_values, weight_scales, stream, hidden, inner, input_bits) ||
        !experts_ok(tokens, top, experts, hidden, inner))
        return kInvalid;
    if (tokens == 0 || top == 0 || experts == 0 || inner == 0) return 0;
    ProductArgs a = arguments(input_values, input_scales, weight_values, weight_scales, output, tokens * top, inner, hidden);
    a.offsets = static_cast<const int32_t*>(offsets);
    a.plan = static_cast<const int32_t*>(plan_rows);
    a.experts = static_cast<uint32_t>(experts);
    a.top = static_cast<uint32_t>(top);
    return launch<Result::kGateUp>(a, input_bits, static_cast<hipStream_t>(stream));
}

MOTE_EXPORT int mote_hip_experts_down_workspace(uint64_t tokens, uint64_t top, uint64_t experts, uint64_t hidden,
                                                uint64_t inner, size_t* bytes) noexcept {
    using namespace mote::mx;
    if (!bytes || !experts_ok(tokens, top, experts, hidden, inner)) return kInvalid;
    *bytes = tokens == 0 || hidden == 0 ? 0 : down_bytes(tokens * top, hidden);
    return 0;
}

MOTE_EXPORT int mote_hip_experts_down_mx_f16(const void* input_values, const void* input_scales,
                                             const void* weight_values, const void* weight_scales, const void* ids,
                                             const void* offsets, const void* plan_rows, const void* pair_weights,
                                             void* output, uint64_t tokens, uint64_t top, uint64_t experts,
                                             uint64_t hidden, uint64_t inner, int input_bits, void* workspace,
                                             size_t workspace_bytes, void* stream) noexcept {
    using namespace mote::mx;
    if (!output || !ids || !offsets || !plan_rows || !pair_weights || off_grid(output, 2) || off_grid(ids, 4) ||
        off_grid(offsets, 4) || off_grid(plan_rows, 4) || off_grid(pair_weights, 4))
        return kInvalid;
    if (!operands_ok(input_values, input_scales, weight_values, weight_scales, stream, inner, hidden, input_bits) ||
        !experts_ok(tokens, top, experts, hidden, inner))
        return kInvalid;
    if (tokens == 0 || hidden == 0) return 0;
    const uint64_t need = down_bytes(tokens * top, hidden);
    if (need > 0 && (!workspace || off_grid(workspace, 16) || workspace_bytes < need)) return kInvalid;
    const uint32_t parts = static_cast<uint32_t>((hidden + 1023) / 1024);
    if (tokens * parts > kMostThreads / 256) return kInvalid;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    if (top > 0 && experts > 0) {
        ProductArgs a = arguments(input_values, input_scales, weight_values, weight_scales, workspace, tokens * top,
                                  hidden, inner);
        a.offsets = static_cast<const int32_t*>(offsets);
        a.plan = static_cast<const int32_t*>(plan_rows);
        a.experts = static_cast<uint32_t>(experts);
        a.top = static_cast<uint32_t>(top);
        const int status = launch<Result::kPairs>(a, input_bits, s);
        if (status != 0) return status;
    }
    const CombineArgs c{static_cast<const float*>(workspace),
                        static_cast<const int32_t*>(ids),
                        static_cast<const float*>(pair_weights),
                        static_cast<_Float16*>(output),
                        static_cast<uint32_t>(hidden),
                        static_cast<uint32_t>(top),
                        static_cast<uint32_t>(experts),
                        parts};
    hipLaunchKernelGGL(combine_kernel, dim3(static_cast<uint32_t>(tokens) * parts), dim3(256), 0, s, c);
    return static_cast<int>(hipGetLastError());
}
