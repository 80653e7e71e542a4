// Products of microscaled rows: y = x W^T, and those of experts, each with its own
// weights and rows.
#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdint>

#include "mx_products.hpp"

namespace mote::mx {
namespace {

// Few rows: HBM-bound on the weights.  A workgroup has 16 of the outputs (of gate and of
// up each) and up to 64 rows in 16-row fragments, of which only those that hold rows are
// multiplied; its waves divide the steps of K among them, two at a time, and add
// their sums through LDS, in the waves' order.  A lane's operand is a 16-byte piece of
// a weights' row as it is stored, so nothing is unpacked; the activations come from L2.
constexpr uint32_t kFewRows = 64;

template <int BITS, Result R, int WAVES>
__global__ __launch_bounds__(WAVES * 64) void few_rows_kernel(ProductArgs a, uint32_t column_tiles) {
    constexpr int kFragments = kFewRows / 16;
    constexpr int kSides = R == Result::kGateUp ? 2 : 1;
    __shared__ f32x4 sums[WAVES][kSides][kFragments][64];
    const uint32_t unit = blockIdx.x / column_tiles, column = blockIdx.x % column_tiles * 16;
    const Tile tile = find_tile<R, kFewRows>(a, unit);
    if (tile.count == 0) return;
    const uint32_t wave = threadIdx.x >> 6, lane = threadIdx.x & 63, of16 = lane & 15, group = lane >> 4;
    const uint32_t steps = a.kp / kStep;

    const uint8_t* w_row[kSides];
    const uint8_t* w_scale[kSides];
#pragma unroll
    for (int side = 0; side < kSides; ++side) {
        const uint64_t row = (static_cast<uint64_t>(tile.expert) * kSides + side) * a.outputs +
                             min(column + of16, a.outputs - 1);
        w_row[side] = a.w + row * value_bytes(a.kp, 4);
        w_scale[side] = a.w_scales + row * scale_bytes(a.kp);
    }
    const uint8_t* x_row[kFragments];
    const uint8_t* x_scale[kFragments];
    const uint32_t fragments = (tile.count + 15) / 16;
#pragma unroll
    for (int f = 0; f < kFragments; ++f) {
        const uint64_t row = input_row<R>(a, tile.first + min(f * 16 + of16, tile.count - 1));
        x_row[f] = a.x + row * value_bytes(a.kp, BITS);
        x_scale[f] = a.x_scales + row * scale_bytes(a.kp);
    }

    f32x4 d[kSides][kFragments] = {};
    for (uint32_t first = wave * 2; first < steps; first += WAVES * 2) {
#pragma unroll
        for (uint32_t j = 0; j < 2; ++j) {
            const uint32_t step = first + j;
            if (step >= steps) break;
            const uint32_t block = step * 4 + group;
            Block<4> w[kSides];
            uint32_t ws[kSides];
#pragma unroll
            for (int side = 0; side < kSides; ++side) {
                w[side] = load_block<4>(w_row[side], a.kp, block);
                ws[side] = reinterpret_cast<const uint32_t*>(w_scale[side])[step] >> (8 * group);
            }
#pragma unroll
            for (int f = 0; f < kFragments; ++f) {
                if (static_cast<uint32_t>(f) >= fragments) break;
                const Block<BITS> x = load_block<BITS>(x_row[f], a.kp, block);
                const uint32_t xs = reinterpret_cast<const uint32_t*>(x_scale[f])[step] >> (8 * group);
#pragma unroll
                for (int side = 0; side < kSides; ++side)
                    d[side][f] = multiply16<BITS>(w[side], ws[side], x, xs, d[side][f]);
            }
        }
    }
#pragma unroll
    for (int side = 0; side < kSides; ++side)
#pragma unroll
        for (int f = 0; f < kFragments; ++f)
            if (static_cast<uint32_t>(f) < fragments) sums[wave][side][f][lane] = d[side][f];
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < fragments * 64; i += WAVES * 64) {
        const uint32_t f = i / 64, l = i % 64;
        const uint32_t row = f * 16 + (l & 15), n = column + 4 * (l >> 4);
        if (row >= tile.count || n >= a.outputs) continue;
        f32x4 total[kSides];
#pragma unroll
        for (int side = 0; side < kSides; ++side) {
            total[side] = sums[0][side][f][l];
#pragma unroll
            for (int v = 1; v < WAVES; ++v) total[side] += sums[v][side][f][l];
        }
        uint64_t to = tile.first + row;
        if constexpr (R == Result::kPairs) {
            to = static_cast<uint32_t>(a.plan[to]);
            if (to >= a.rows) continue;
        }
        to = to * a.outputs + n;
#pragma unroll
        for (uint32_t r = 0; r < 4; ++r) {
            if (n + r >= a.outputs) break;
            if constexpr (R == Result::kGateUp)
                static_cast<_Float16*>(a.output)[to + r] = static_cast<_Float16>(silu(total[0][r]) * total[kSides - 1][r]);
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
    const uint32_t n = (blockIdx.x % a.parts) * 256 + threadIdx.x;
    if (n >= a.hidden) return;
    float y = 0.0f;
    for (uint32_t j = 0; j < a.top; ++j) {
        const uint64_t pair = static_cast<uint64_t>(token) * a.top + j;
        if (static_cast<uint32_t>(a.ids[pair]) >= a.experts) continue;
        y = __builtin_fmaf(a.weights[pair], a.products[pair * a.hidden + n], y);
    }
    a.output[static_cast<uint64_t>(token) * a.hidden + n] = static_cast<_Float16>(y);
}

template <Result R>
int launch(const ProductArgs& a, int bits, hipStream_t stream) {
    const uint32_t column_tiles = (a.outputs + 15) / 16;
    const uint64_t units = kOfExperts<R> ? most_expert_tiles(a.rows, a.experts, kFewRows)
                                         : (uint64_t{a.rows} + kFewRows - 1) / kFewRows;
    constexpr uint32_t kWaves = 8;
    if (units * column_tiles > kMostThreads / (kWaves * 64)) return kInvalid;
    const auto go = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, dim3(static_cast<uint32_t>(units * column_tiles)), dim3(kWaves * 64), 0, stream, a,
                           column_tiles);
    };
    bits == 4 ? go(few_rows_kernel<4, R, kWaves>) : go(few_rows_kernel<6, R, kWaves>);
    return static_cast<int>(hipGetLastError());
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
    const uint32_t parts = static_cast<uint32_t>((hidden + 255) / 256);
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
