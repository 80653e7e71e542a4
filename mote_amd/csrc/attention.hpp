// What the attention kernels and the 8-bit cache share.
//
// Attention of query i (position i + keys - queries in its sequence) over the
// keys j it sees: o_i = sum_j p_ij v_j, p_ij = 2^(c q_i.k_j - m_i) / l_i, with
// c = scale log2(e), m_i a bound near the row's largest exponent and l_i the sum
// that makes the weights one.  One pass over the keys keeps (m, l, o) and
// rescales l and o by 2^(m - m') when m grows to m'; parts of the keys computed
// apart join the same way.  All of that is held in 32 bits.
#pragma once

#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdint>

#include "common.hpp"

namespace mote::attention {
namespace {

constexpr int kInvalid = -1;
constexpr uint32_t kBlockTokens = 32;             // tokens of a cache block
constexpr uint64_t kMostTokens = uint64_t{1} << 30;  // int32 offsets, with room for a window's
constexpr uint64_t kMostHeadDim = 256;
constexpr uint64_t kMostGrid = (uint64_t{1} << 32) / 256 - 1;  // workgroups of 256 threads in one launch

__host__ __device__ constexpr uint32_t padded_dim(uint32_t d) { return (d + 31u) & ~31u; }

// Eight binary16 values from an address of any element alignment.
typedef uint32_t u32x4_a2 __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t u32x2_a2 __attribute__((ext_vector_type(2), aligned(2)));

// Rows whose largest exponent grows by no more than this keep their reference
// m: weights then reach 2^(kGrowth + kShift) at most, within binary16 (2^16),
// and those that matter stay above its subnormals: kShift places the weight of
// the reference itself at 2^8, so weights down to 2^-22 of it keep all 11 bits.
constexpr float kGrowth = 6.0f;
constexpr float kShift = 8.0f;
constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ float infinity() { return __builtin_inff(); }

// v and the value of the lane 32 (16) away, in every lane.  (The results are
// copied before they are cast: a bit cast of a vector's element reads element 0.)
struct Both {
    float a, b;
};
__device__ __forceinline__ Both both_of(uint32_t a, uint32_t b) {
    return {__builtin_bit_cast(float, a), __builtin_bit_cast(float, b)};
}
__device__ __forceinline__ Both across_halves(float v) {
    const uint32_t x = __builtin_bit_cast(uint32_t, v);
    const auto r = __builtin_amdgcn_permlane32_swap(x, x, false, false);
    return both_of(r[0], r[1]);
}
__device__ __forceinline__ Both across_rows16(float v) {
    const uint32_t x = __builtin_bit_cast(uint32_t, v);
    const auto r = __builtin_amdgcn_permlane16_swap(x, x, false, false);
    return both_of(r[0], r[1]);
}
__device__ __forceinline__ float max_of(Both v) { return fmaxf(v.a, v.b); }
__device__ __forceinline__ float sum_of(Both v) { return v.a + v.b; }

// Packed sequences: tokens [at, at + n) of sequence s, from offsets held on the
// device, kept inside the `tokens` there are whatever the offsets hold.
struct Span {
    int at, n;
};
__device__ __forceinline__ Span span_of(const int32_t* offsets, uint32_t s, uint32_t tokens) {
    const int most = static_cast<int>(tokens);
    const int a = min(max(offsets[s], 0), most), b = min(max(offsets[s + 1], 0), most);
    return {a, max(b - a, 0)};
}

// Unit `unit` of the units of all sequences in order, count(s) of sequence s:
// its sequence and its number there.  Each wave looks it up by itself, 64
// sequences at a time.
struct Unit {
    uint32_t sequence, local, of;
    bool found;
};
template <typename Count>
__device__ __forceinline__ Unit locate(uint32_t unit, uint32_t sequences, Count count) {
    const uint32_t lane = threadIdx.x & 63;
    uint32_t base = 0;
    for (uint32_t s0 = 0; s0 < sequences; s0 += 64) {
        const uint32_t n = s0 + lane < sequences ? count(s0 + lane) : 0;
        uint32_t upto = n;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const uint32_t other = __shfl_up(upto, d, 64);
            if (lane >= static_cast<uint32_t>(d)) upto += other;
        }
        const uint64_t past = __builtin_amdgcn_ballot_w64(base + upto > unit);
        if (past != 0) {
            const int at = __builtin_ctzll(past);
            const uint32_t mine = __builtin_amdgcn_readlane(n, at);
            const uint32_t before = base + __builtin_amdgcn_readlane(upto, at) - mine;
            return {s0 + at, unit - before, mine, true};
        }
        base += __builtin_amdgcn_readlane(upto, 63);
    }
    return {0, 0, 0, false};
}

// Parts of the keys computed apart: part s of row r (token x heads + head) has
// (m, l) in stats[s][r] and sum_j 2^(c s_j - m) v_j in sums[s][r][head_dim].
// out = sum_s 2^(m_s - M) sums_s / sum_s 2^(m_s - M) l_s with M = max m_s; zeros
// where no part saw a key.  A wave per row, four dimensions a lane.
__global__ __launch_bounds__(256) void parts_join_kernel(const float2* __restrict__ stats,
                                                         const float* __restrict__ sums, _Float16* output,
                                                         uint32_t rows, uint32_t parts, uint32_t heads,
                                                         uint32_t head_dim, uint64_t out_stride) {
    const uint32_t row = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
    if (row >= rows) return;
    float top = -infinity();
    for (uint32_t s = 0; s < parts; ++s) top = fmaxf(top, stats[static_cast<uint64_t>(s) * rows + row].x);
    const uint32_t d = lane * 4;
    if (d >= head_dim) return;
    f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
    float l = 0.0f;
    for (uint32_t s = 0; s < parts; ++s) {
        const float2 ml = stats[static_cast<uint64_t>(s) * rows + row];
        if (ml.y == 0.0f) continue;  // saw nothing: its sums were not written
        const float w = ml.x == -infinity() ? ml.y : exp2_fast(ml.x - top);  // the first only where ml.y is NaN
        l = __builtin_fmaf(w, ml.y, l);
        acc += w * *reinterpret_cast<const f32x4*>(sums + (static_cast<uint64_t>(s) * rows + row) * head_dim + d);
    }
    const float inv = l != 0.0f ? 1.0f / l : 0.0f;
    acc *= inv;
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

inline int join_parts(const void* workspace, void* output, uint64_t rows, uint32_t parts, uint64_t heads,
                      uint64_t head_dim, uint64_t out_stride, hipStream_t stream) {
    hipLaunchKernelGGL(parts_join_kernel, dim3(static_cast<unsigned>((rows + 3) / 4)), dim3(256), 0, stream,
                       static_cast<const float2*>(workspace),
                       reinterpret_cast<const float*>(static_cast<const char*>(workspace) + stats_bytes(rows, parts)),
                       static_cast<_Float16*>(output), static_cast<uint32_t>(rows), parts,
                       static_cast<uint32_t>(heads), static_cast<uint32_t>(head_dim), out_stride);
    return static_cast<int>(hipGetLastError());
}

inline bool odd_address(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 1) != 0; }
inline bool off_grid(const void* p, uintptr_t grid) { return (reinterpret_cast<uintptr_t>(p) & (grid - 1)) != 0; }

}  // namespace
}  // namespace mote::attention
