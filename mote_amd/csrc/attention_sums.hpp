// The attentions' sums: those of a wave's rows, and the join of parts of the keys
// computed apart.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "attention.hpp"

namespace mote::attention {
namespace {

// The running sums of the row that a lane of a 32-row wave holds half of: of the 32
// D dimensions, 8 (r / 4) + 4 h + r % 4 of each 32 in o[.][r], h being the lane's half.
template <int D>
struct RowSums {
    f32x16 o[D];
    float m, l;  // l: of the lane's keys alone
    bool large;  // some row's m is: exponents are rounded before m is taken off

    static __device__ __forceinline__ f32x16 zero() {
        return f32x16{0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
    }
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int i = 0; i < D; ++i) o[i] = zero();
        m = -infinity();
        l = 0.0f;
        large = false;
    }
    // Makes room for exponents up to `top` (of the row, the same in both halves).
    __device__ __forceinline__ void grow_to(float top) {
        if (!wave_any(top - m > kReach)) return;
        const float to = reference(m, top);
        const float w = m == to ? 1.0f : exp2_fast(m - to);  // also where both are -inf
        m = to;
        l *= w;
#pragma unroll
        for (int i = 0; i < D; ++i) o[i] *= w;
        large = wave_any(fabsf(base()) > kLargeExponent);
    }
    __device__ __forceinline__ bool finite() const {
        float all = 0.0f;  // any that is not makes NaN
#pragma unroll
        for (int i = 0; i < D; ++i)
#pragma unroll
            for (int r = 0; r < 16; ++r) all = __builtin_fmaf(o[i][r], 0.0f, all);
        return all == 0.0f;
    }
    // What exponents are taken less of.
    __device__ __forceinline__ float base() const { return m == -infinity() ? 0.0f : m; }
    // The wave's results: through `stage`, 2 KB x D of LDS that is the wave's own, so
    // that whole rows leave in 16-byte chunks of neighbouring lanes (a lane's own
    // pieces are 8 bytes a row: 64 prompts of 128 tokens took 58 us so, 51 now).  row_at(i):
    // where row i goes, null for none.
    template <bool WHOLE, typename RowAt>
    __device__ __forceinline__ void write(uint8_t* stage, uint32_t head_dim, RowAt row_at) const {
        constexpr int CH = 4 * D, G = (CH & -CH) > 16 ? 16 : (CH & -CH);
        const int lane = threadIdx.x & 63, n = lane & 31, h = lane >> 5;
        const float all = sum_of(across_halves(l)), inv = all != 0.0f ? 1.0f / all : 0.0f;
        const auto chunk = [&](int row, int c) { return stage + (row * CH + (c ^ (row / (16 / G) % G))) * 16; };
#pragma unroll
        for (int i = 0; i < D; ++i)
#pragma unroll
            for (int r = 0; r < 16; r += 4) {
                const f16x2 lo = {static_cast<_Float16>(o[i][r] * inv), static_cast<_Float16>(o[i][r + 1] * inv)};
                const f16x2 hi = {static_cast<_Float16>(o[i][r + 2] * inv), static_cast<_Float16>(o[i][r + 3] * inv)};
                *reinterpret_cast<u32x2*>(chunk(n, 4 * i + r / 4) + 8 * h) =
                    u32x2{__builtin_bit_cast(uint32_t, lo), __builtin_bit_cast(uint32_t, hi)};
            }
        wave_lds_fence();
#pragma unroll
        for (int j = 0; j < CH / 2; ++j) {
            const int row = (64 * j + lane) / CH, c = (64 * j + lane) % CH;
            _Float16* const to = row_at(row);
            if (to != nullptr && (WHOLE || 8u * c < head_dim))
                *reinterpret_cast<u32x4_a2*>(to + 8 * c) = *reinterpret_cast<const u32x4*>(chunk(row, c));
        }
    }
    // The row's part, to row `at` of the statistics and sums.
    template <bool WHOLE>
    __device__ __forceinline__ void write_part(float2* stats, float* sums, uint64_t at, uint32_t head_dim) const {
        const int h = (threadIdx.x >> 5) & 1;
        const float all = sum_of(across_halves(l));
        if (h == 0) stats[at] = float2{m, all};
        if (all == 0.0f) return;  // saw nothing: not read
#pragma unroll
        for (int i = 0; i < D; ++i)
#pragma unroll
            for (int r = 0; r < 16; r += 4) {
                const uint32_t d = 32 * i + 2 * r + 4 * h;
                if (WHOLE || d < head_dim)
                    *reinterpret_cast<f32x4*>(sums + at * head_dim + d) = f32x4{o[i][r], o[i][r + 1], o[i][r + 2], o[i][r + 3]};
            }
    }
};

// Parts of the keys computed apart: part s of row r (token x heads + head) has
// (m, l) in stats[s][r] and sum_j 2^(c s_j - m) v_j in sums[s][r][head_dim].
// out = sum_s 2^(m_s - M) sums_s / sum_s 2^(m_s - M) l_s with M = max m_s; zeros
// where no part saw a key.  Rows that no workgroup computes are marked by
// l = kNotComputed in their first part and left as they are.  (The join looking for
// its row in the offsets took 0.8 to 1.3 us longer.)  W waves a row, each its share of
// the parts (64 at most, the statistics of one in a lane); a wave's lanes take four
// dimensions each and as many parts at a time as find room.
constexpr uint32_t kMostParts = 256;
constexpr float kNotComputed = -1.0f;

// Marks the rows of tokens [from, to) that belong to `count` heads from `head` on.
__device__ inline void mark_rows(float2* stats, uint32_t from, uint32_t to, uint32_t heads, uint32_t head,
                                 uint32_t count) {
    for (uint32_t t = from + threadIdx.x; t < to; t += blockDim.x)
        for (uint32_t i = 0; i < count; ++i)
            stats[static_cast<uint64_t>(t) * heads + head + i] = float2{-infinity(), kNotComputed};
}
// By one workgroup of a sequence and its heads: the sequence's rows past the first
// `most`, and beside the first and the last sequence those that none owns.
__device__ __forceinline__ void mark_not_computed(float2* stats, Span rows, uint32_t seq, uint32_t sequences,
                                                  uint32_t tokens, uint32_t most, uint32_t heads, uint32_t head,
                                                  uint32_t count) {
    const uint32_t at = static_cast<uint32_t>(rows.at), end = at + static_cast<uint32_t>(rows.n);
    if (end - at > most) mark_rows(stats, at + most, end, heads, head, count);
    if (seq == 0 && at != 0) mark_rows(stats, 0, at, heads, head, count);
    if (seq + 1 == sequences && end < tokens) mark_rows(stats, end, tokens, heads, head, count);
}

template <int W>
__global__ __launch_bounds__(256) void parts_join_kernel(const float2* __restrict__ stats,
                                                         const float* __restrict__ sums, _Float16* output,
                                                         uint32_t rows, uint32_t first_row, uint32_t parts,
                                                         uint32_t heads, uint32_t head_dim, uint32_t lanes,
                                                         uint64_t out_stride) {
    __shared__ __align__(16) float joined[W == 1 ? 1 : 4][W == 1 ? 4 : 256];
    __shared__ float2 joined_stats[4];
    __shared__ float weights[4][64];
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const uint32_t row = first_row + (W == 1 ? blockIdx.x * 4 + wave : blockIdx.x);
    if (row >= rows) return;
    const uint32_t share = (parts + W - 1) / W, first = W == 1 ? 0 : wave * share;
    const uint32_t mine = first < parts ? min(share, parts - first) : 0;
    const uint32_t d = (lane & (lanes - 1)) * 4;
    const uint32_t at_once = 64 / lanes, own = lane / lanes;  // lanes: a power of two, four times it at least head_dim
    const float* from = sums + (static_cast<uint64_t>(first) * rows + row) * head_dim + (d < head_dim ? d : 0);
    const uint64_t step = static_cast<uint64_t>(rows) * head_dim;
    f32x4 x[4];
    const auto load = [&](uint32_t s0) {  // past the last part: the first, weighing nothing
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t s = s0 + i * at_once + own;
            x[i] = *reinterpret_cast<const f32x4*>(from + (s < mine ? s : 0) * step);
        }
    };
    float2 ml = {-infinity(), 0.0f};
    if (lane < mine) ml = stats[static_cast<uint64_t>(first + lane) * rows + row];
    if (mine != 0) load(0);
    const float mark = __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, ml.y)));
    const float top = wave_max(ml.x);
    // A part that saw nothing has l = 0 and no sums; one with m = -inf and another l has NaN there.
    const float weight = ml.y == 0.0f ? 0.0f : ml.x == -infinity() ? ml.y : exp2_fast(ml.x - top);
    float l = wave_sum(weight * ml.y);
    weights[wave][lane] = weight;  // read by this wave alone
    wave_lds_fence();
    f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
    for (uint32_t s0 = 0; s0 < mine; s0 += 4 * at_once) {
        if (s0 != 0) load(s0);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t s = s0 + i * at_once + own;
            const float w = s < mine ? weights[wave][s] : 0.0f;
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[e] += w != 0.0f ? w * x[i][e] : 0.0f;
        }
    }
    for (uint32_t over = lanes; over < 64; over <<= 1)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[e] += __shfl_xor(acc[e], static_cast<int>(over), 64);
    if constexpr (W > 1) {
        if (lane < lanes) *reinterpret_cast<f32x4*>(&joined[wave][4 * lane]) = acc;
        if (lane == 0) joined_stats[wave] = float2{top, l};
        __syncthreads();
        if (wave != 0) return;
        float all = -infinity();
#pragma unroll
        for (int w = 0; w < 4; ++w) all = fmaxf(all, joined_stats[w].x);
        acc = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        l = 0.0f;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const float2 of = joined_stats[w];
            const float by = of.y == 0.0f ? 0.0f : of.x == -infinity() ? of.y : exp2_fast(of.x - all);
            l = __builtin_fmaf(by, of.y, l);
            acc += by * *reinterpret_cast<const f32x4*>(&joined[w][4 * (lane & (lanes - 1))]);
        }
    }
    if (lane >= lanes || d >= head_dim || mark == kNotComputed) return;
    acc *= l != 0.0f ? 1.0f / l : 0.0f;
    typedef _Float16 f16x4_a2 __attribute__((ext_vector_type(4), aligned(2)));
    _Float16* out = output + (row / heads) * out_stride + (row % heads) * static_cast<uint64_t>(head_dim) + d;
    *reinterpret_cast<f16x4_a2*>(out) =
        f16x4_a2{static_cast<_Float16>(acc.x), static_cast<_Float16>(acc.y), static_cast<_Float16>(acc.z),
                 static_cast<_Float16>(acc.w)};
}

// A workspace of `parts` parts: the statistics first, then the sums.
constexpr uint64_t stats_bytes(uint64_t rows, uint64_t parts) { return (rows * parts * 8 + 255) & ~uint64_t{255}; }
constexpr uint64_t parts_bytes(uint64_t rows, uint64_t parts, uint64_t head_dim) {
    return parts <= 1 ? 0 : stats_bytes(rows, parts) + rows * parts * head_dim * 4;
}

// How many parts the keys of `groups` workgroups are divided into, two at a time on
// each of 256 compute units, that walk up to `tiles` tiles of 64 keys: what a model
// of the time says is least.  A tile of 128 dimensions takes `alone` us where its
// workgroup has the unit to itself and `shared` us where two have; the parts' sums go
// out and come back at 4 MB a us, in a launch more of 4 us.
inline uint32_t choose_parts(uint64_t groups, uint64_t tiles, uint64_t rows, uint64_t head_dim, double alone,
                             double shared) {
    const double scale = head_dim < 64 ? 0.5 : static_cast<double>(head_dim) / 128.0;
    uint32_t best = 1;
    double least = 0.0;
    for (uint64_t parts = 1; parts <= kMostParts && (parts == 1 || 2 * parts <= tiles); ++parts) {
        const uint64_t all = groups * parts, rounds = (all + 511) / 512;
        const double walk = static_cast<double>((tiles + parts - 1) / parts) * scale *
                            (all <= 256 ? alone : shared * static_cast<double>(rounds));
        const double join = parts == 1 ? 0.0 : 4.0 + static_cast<double>(parts * rows * head_dim * 8) / 4e6;
        if (parts == 1 || walk + join < least) {
            best = static_cast<uint32_t>(parts);
            least = walk + join;
        }
        if (all > 2048) break;  // more only cost
    }
    return best;
}

inline int join_parts(const void* workspace, void* output, uint64_t rows, uint32_t parts, uint64_t heads,
                      uint64_t head_dim, uint64_t out_stride, hipStream_t stream) {
    uint32_t lanes = 2;
    while (lanes * 4 < head_dim) lanes *= 2;
    const bool many = parts > 8;
    const auto kernel = many ? parts_join_kernel<4> : parts_join_kernel<1>;
    const uint64_t per = many ? 1 : 4, most = most_groups(256) * per;
    for (uint64_t first = 0; first < rows; first += most) {
        const uint64_t now = rows - first < most ? rows - first : most;
        hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>((now + per - 1) / per)), dim3(256), 0, stream,
                           static_cast<const float2*>(workspace),
                           reinterpret_cast<const float*>(static_cast<const char*>(workspace) + stats_bytes(rows, parts)),
                           static_cast<_Float16*>(output), static_cast<uint32_t>(rows), static_cast<uint32_t>(first),
                           parts, static_cast<uint32_t>(heads), static_cast<uint32_t>(head_dim), lanes, out_stride);
        const int status = static_cast<int>(hipGetLastError());
        if (status != 0) return status;
    }
    return 0;
}

}  // namespace
}  // namespace mote::attention
