// Microscaled formats, and what the kernels that multiply them share.
//
// A row of K elements is kept as Kp = K rounded up to 128 of them, in blocks of 32
// with a scale byte b that stands for 2^(b - 127) (255: not a number).  An element
// is E2M1 (4 bits: 0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives) or E2M3 (6 bits:
// 0 to 1.875 in eighths, to 3.75 in quarters, to 7.5 in halves); the lowest bits are the
// first elements'.  A block's 16 bytes of 4 bits, or the first 16 of its 24 bytes of 6,
// are at 16 (block) of the row, the last 8 at Kp / 2 + 8 (block): a lane of the matrix
// instruction holds one whole block, so both are loads of its operand as it stands.
// The padding is zeros, so no kernel has a case for the end of a row, and each four
// blocks' scales are one aligned word.
//
// The formats are the two that the matrix cores take at their full rate (registers
// only, random bits, 32 x 32 x 64: 4 x 4 bits 6.2 PFLOP/s, 4 x 6 6.1, 4 x 8 3.3), and
// whose block sums are exact: products are multiples of 1/16 below 2^6.  (Of 8-bit
// products they drop what lies 2^-14 under the largest of the block.)
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "common.hpp"

namespace mote::mx {
namespace {

constexpr int kInvalid = -1;
constexpr uint32_t kBlock = 32;     // elements of a scale
constexpr uint32_t kStep = 128;     // elements that rows are padded to; of a 16 x 16 matrix instruction
constexpr uint64_t kMostFeatures = uint64_t{1} << 24;  // byte offsets in a row, and its steps, in 32 bits
constexpr uint64_t kMostRows = uint64_t{1} << 30;
constexpr uint64_t kMostThreads = 0xFFFFFFFFu;  // of a launch
constexpr uint32_t kMostExperts = 1024;
constexpr uint32_t kMostTop = 64;  // experts of a token

// (Also of Kp itself; 32 bits on the device.)
__host__ __device__ constexpr uint32_t padded(uint64_t features) {
    return static_cast<uint32_t>((features + kStep - 1) / kStep * kStep);
}
__host__ __device__ constexpr uint32_t value_bytes(uint32_t kp, int bits) { return kp / 8 * bits; }
__host__ __device__ constexpr uint32_t scale_bytes(uint32_t kp) { return kp / kBlock; }

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x6 __attribute__((ext_vector_type(6)));

// The matrix instruction's code for an operand's format.
template <int BITS>
constexpr int kFormat = BITS == 4 ? 4 : 2;

// One lane's operand: a block.
template <int BITS>
struct Block;
template <>
struct Block<4> {
    u32x4 low;
    __device__ __forceinline__ i32x8 operand() const {
        return i32x8{static_cast<int>(low.x), static_cast<int>(low.y), static_cast<int>(low.z),
                     static_cast<int>(low.w), 0, 0, 0, 0};
    }
};
template <>
struct Block<6> {
    u32x4 low;
    u32x2 high;
    __device__ __forceinline__ i32x8 operand() const {
        return i32x8{static_cast<int>(low.x), static_cast<int>(low.y), static_cast<int>(low.z), static_cast<int>(low.w),
                     static_cast<int>(high.x), static_cast<int>(high.y), 0, 0};
    }
};

// Block `block` of the row at `row`.
template <int BITS>
__device__ __forceinline__ Block<BITS> load_block(const uint8_t* row, uint32_t kp, uint32_t block) {
    Block<BITS> b;
    b.low = *reinterpret_cast<const u32x4*>(row + 16 * block);
    if constexpr (BITS == 6) b.high = *reinterpret_cast<const u32x2*>(row + kp / 2 + 8 * block);
    return b;
}

// D[i][j] += sum over k of W[i][k] X[j][k] for 16 x 16 outputs and 128 elements: lane
// l holds block l / 16 of rows l % 16, and of D column j = l % 16, rows 4 (l / 16) + r.
// Scales are the lanes' low bytes.
template <int BITS>
__device__ __forceinline__ f32x4 multiply16(i32x8 w, uint32_t w_scale, i32x8 x, uint32_t x_scale, f32x4 d) {
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w, x, d, kFormat<4>, kFormat<BITS>, 0,
                                                            static_cast<int>(w_scale), 0, static_cast<int>(x_scale));
}

inline bool off_grid(const void* p, uintptr_t grid) { return (reinterpret_cast<uintptr_t>(p) & (grid - 1)) != 0; }
inline bool known_bits(int bits) { return bits == 4 || bits == 6; }

}  // namespace
}  // namespace mote::mx
