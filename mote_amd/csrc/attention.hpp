// What the attention kernels and the 8-bit cache share.
//
// Attention of query i (position i + keys - queries in its sequence) over the
// keys j it sees: o_i = sum_j p_ij v_j, p_ij = 2^(c q_i.k_j - m_i) / l_i, with
// c = scale log2(e), m_i a reference near the row's largest exponent and l_i the sum
// that makes the weights one.  One pass over the keys keeps (m, l, o) and
// rescales l and o by 2^(m - m') when m grows to m'; parts of the keys computed
// apart join the same way.  All of that is held in 32 bits.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "common.hpp"

namespace mote::attention {
namespace {

constexpr int kInvalid = -1;
constexpr uint32_t kBlockTokens = 32;             // tokens of a cache block
constexpr uint64_t kMostTokens = uint64_t{1} << 30;  // int32 offsets, with room for a window's
constexpr uint64_t kMostHeadDim = 256;
// Workgroups of so many threads in one launch, whose threads are counted in 32 bits.
constexpr uint64_t most_groups(uint64_t threads) { return 0xFFFFFFFFu / threads; }

__host__ __device__ constexpr uint32_t padded_dim(uint32_t d) { return (d + 31u) & ~31u; }

// Eight binary16 values from an address of any element alignment.
typedef uint32_t u32x4_a2 __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t u32x2_a2 __attribute__((ext_vector_type(2), aligned(2)));

// A row's reference m lies kShift under the largest exponent it had when it was
// taken, so that the weight of that one is 2^8 and weights down to 2^-22 of it keep
// all 11 bits of binary16.  It is kept until an exponent lies more than kReach over
// it: weights stay within 2^14, and binary16 ends at 2^16.
constexpr float kShift = 8.0f;
constexpr float kReach = 14.0f;
// Where exponents are this large, their roundings to 32 bits show in 2^(x - m): a
// fused c s - m, next to an m taken from rounded products, would be off by as much.
// x is then rounded by itself, as what m was taken from.
constexpr float kLargeExponent = 0x1p22f;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLeastFactor = 0x1p-100f;  // of scores: a masked one stays -inf, others vanish
constexpr float kLeastScale = 0x1p-64f;  // of values: times 127 far below binary16, and its inverse in range

// Between a wave's own writes to LDS and what its other lanes read there.
__device__ __forceinline__ void wave_lds_fence() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

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

// A load whose address is the same in the whole wave, of memory that nothing writes
// while the kernel runs: said so that it stays a scalar load behind stores too.
template <typename T>
__device__ __forceinline__ T scalar_load(const T* p) {
    return *(const __attribute__((address_space(4))) T*)(p);
}

// The reference m where exponents reach up to `top` (-inf: none seen); no lower.
__device__ __forceinline__ float reference(float m, float top) {
    const float below = top - kShift;
    return fmaxf(m, top - below > kReach ? top : below);  // where floats are 16 apart, top - 8 may be 16 below
}
// c s, rounded before anything is added to it.
__device__ __forceinline__ float product(float s, float c) {
#pragma clang fp contract(off)
    return s * c;
}

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
__device__ __forceinline__ Span scalar_span_of(const int32_t* offsets, uint32_t s, uint32_t tokens) {
    const int32_t pair[2] = {scalar_load(offsets + s), scalar_load(offsets + s + 1)};
    return span_of(pair, 0, tokens);
}
__device__ __forceinline__ Span span_at(Span mine, int lane) {  // the span that `lane` holds
    return {__builtin_amdgcn_readlane(mine.at, lane), __builtin_amdgcn_readlane(mine.n, lane)};
}

// The largest of a wave's lanes, in all of them.
template <int Ctrl, int RowMask = 0xF>
__device__ __forceinline__ float max_dpp(float v) {
    const int b = __builtin_bit_cast(int, v);
    return fmaxf(v, __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(b, b, Ctrl, RowMask, 0xF, false)));
}
__device__ __forceinline__ float wave_max(float v) {
    v = max_dpp<0xB1>(v);        // quad_perm [1,0,3,2]
    v = max_dpp<0x4E>(v);        // quad_perm [2,3,0,1]
    v = max_dpp<0x141>(v);       // row_half_mirror
    v = max_dpp<0x140>(v);       // row_mirror
    v = max_dpp<0x142, 0xA>(v);  // row_bcast:15 into rows 1 and 3
    v = max_dpp<0x143, 0xC>(v);  // row_bcast:31 into rows 2 and 3
    return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), 63));
}

// Where work is divided by sequence: a sequence of n rows at offset a has its units
// from a / PER + EACH s on (its number being s), room for as many as n / PER + EACH.
// So a unit's sequence is found by its slot alone, from the offsets in order, 64 at
// a time: one load for up to 64 sequences, two for 4096.  Each wave looks it up by
// itself.  visit(s) is called, before it is known which is found, by a lane of each
// sequence that is near; `lane` is the one whose sequence it is.
struct Unit {
    uint32_t sequence, local;
    int lane;
    bool found;
};
template <uint32_t PER, uint32_t EACH, typename Visit>
__device__ __forceinline__ Unit locate(uint32_t unit, const int32_t* offsets, uint32_t sequences, uint32_t tokens,
                                       Visit visit) {
    const uint32_t lane = threadIdx.x & 63;
    uint32_t first = 0, count = sequences;
    for (;;) {
        const uint32_t stride = (count + 63) / 64;
        const uint32_t s = first + lane * stride;
        uint32_t slot = 0xFFFFFFFFu;
        if (lane * stride < count) {
            if (stride == 1) visit(s);
            slot = static_cast<uint32_t>(min(max(offsets[s], 0), static_cast<int>(tokens))) / PER + EACH * s;
        }
        const uint64_t before = __builtin_amdgcn_ballot_w64(slot <= unit);
        if (before == 0) return {0, 0, 0, false};
        const int at = 63 - __builtin_clzll(before);
        first += at * stride;
        count = min(stride, count - at * stride);
        if (stride == 1) return {first, unit - static_cast<uint32_t>(__builtin_amdgcn_readlane(slot, at)), at, true};
    }
}
// The units there are room for.
constexpr uint64_t units_of(uint64_t per, uint64_t each, uint64_t sequences, uint64_t tokens) {
    return tokens / per + each * sequences;
}

inline bool odd_address(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 1) != 0; }
inline bool off_grid(const void* p, uintptr_t grid) { return (reinterpret_cast<uintptr_t>(p) & (grid - 1)) != 0; }

}  // namespace
}  // namespace mote::attention
