// Rows to microscaled 4 or 6 bits and back (mx.hpp has the formats).
//
// Scale of a block: 2^(floor(log2 m) - 2), m its largest magnitude, 2 the exponent of the
// largest element, and no smaller than 2^-127; an element is its value over that, rounded to
// the nearest (ties to even) and held to the format's largest, 6 or 7.5.  The
// scale is a power of two, so the quotient is exact and there is one rounding.  An infinity or NaN
// makes its block's scale 255 and its elements zeros: the block is NaN in all that reads it.
//
// A thread has a block: 64 or 128 bytes in, one conversion of the whole block (or one a
// pair), 16 and 8 bytes and a scale out, each contiguous over a wave.  Bound by the bytes: 4000 x 14336
// of f16 to 6 bits 25 to 26 us and back 25, 160 MB each, 6.2 to 6.4 TB/s (some of it from the
// memory-side cache); 64 x 4096 2.7 and 2.9 us, a launch's chain.
#include <hip/hip_runtime.h>

#include <cstdint>

#include "mx.hpp"

namespace mote::mx {
namespace {

typedef uint32_t u32x4_a2 __attribute__((ext_vector_type(4), aligned(2)));
typedef _Float16 f16x32 __attribute__((ext_vector_type(32)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x32 __attribute__((ext_vector_type(32)));

constexpr uint32_t kThreads = 256;

struct RowArgs {
    const void* input;
    void* output;
    const uint8_t* values_in;
    uint8_t* values;
    uint8_t* scales;
    uint64_t rows, stride;  // elements between the rows of f16 or f32
    uint32_t kp, blocks;    // Kp; blocks of K
};

// The row and block of this thread; false past the last row.
__device__ __forceinline__ bool block_of(const RowArgs& a, uint64_t& row, uint32_t& block) {
    const uint32_t per_row = a.kp / kBlock;
    const uint64_t first = static_cast<uint64_t>(blockIdx.x) * kThreads;  // of the workgroup: scalar
    const uint64_t first_row = first / per_row;
    const uint32_t at = static_cast<uint32_t>(first - first_row * per_row) + threadIdx.x;
    row = first_row + at / per_row;
    block = at % per_row;
    return row < a.rows;
}

// The scale byte for a largest magnitude with these bits (as a float).
__device__ __forceinline__ uint32_t scale_of(uint32_t most) {
    if (most >= 0x7F800000u) return 255;
    const uint32_t e = most >> 23;  // floor(log2 m) + 127; 0 below 2^-126
    return e > 2 ? e - 2 : 0;
}

// The conversions of a whole block write their result in several passes while they still read, and the
// compiler's own give result and operands the same registers where they can: elements then came out
// as others' bits.  So they are written here, where the result can be said to be written early.  (The
// compiler does not look into them for its wait states: two before and behind cover what a vector instruction needs
// of another.)
#ifdef __HIP_DEVICE_COMPILE__
#define MOTE_CONVERT_BLOCK(instruction, result, ...) \
    asm("s_nop 1\n\t" instruction "\n\ts_nop 1" : "=&v"(result) : __VA_ARGS__)
#else
#define MOTE_CONVERT_BLOCK(instruction, result, ...) (result = {})
#endif
__device__ __forceinline__ u32x6 to_six_bits(f16x32 v, float scale) {
    u32x6 w;
    MOTE_CONVERT_BLOCK("v_cvt_scalef32_pk32_fp6_f16 %0, %1, %2", w, "v"(v), "v"(scale));
    return w;
}
// (The instruction takes its elements from the two in turn.)
__device__ __forceinline__ u32x6 to_six_bits(f32x16 even, f32x16 odd, float scale) {
    u32x6 w;
    MOTE_CONVERT_BLOCK("v_cvt_scalef32_2xpk16_fp6_f32 %0, %1, %2, %3", w, "v"(even), "v"(odd), "v"(scale));
    return w;
}
__device__ __forceinline__ f32x32 from_six_bits(u32x6 codes) {
    f32x32 v;
    MOTE_CONVERT_BLOCK("v_cvt_scalef32_pk32_f32_fp6 %0, %1, 1.0", v, "v"(codes));
    return v;
}
#undef MOTE_CONVERT_BLOCK

template <int BITS>
__device__ __forceinline__ Block<BITS> convert(const _Float16 (&x)[32], float scale) {
    Block<BITS> b;
    if constexpr (BITS == 4) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            uint32_t word = 0;
            const _Float16* v = x + 8 * i;
            word = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(word, f16x2{v[0], v[1]}, scale, 0);
            word = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(word, f16x2{v[2], v[3]}, scale, 1);
            word = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(word, f16x2{v[4], v[5]}, scale, 2);
            word = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(word, f16x2{v[6], v[7]}, scale, 3);
            b.low[i] = word;
        }
    } else {
        f16x32 v;
#pragma unroll
        for (int i = 0; i < 32; ++i) v[i] = x[i];
        const u32x6 w = to_six_bits(v, scale);
        b.low = u32x4{w[0], w[1], w[2], w[3]};
        b.high = u32x2{w[4], w[5]};
    }
    return b;
}
template <int BITS>
__device__ __forceinline__ Block<BITS> convert(const float (&x)[32], float scale) {
    Block<BITS> b;
    if constexpr (BITS == 4) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            uint32_t word = 0;
            const float* v = x + 8 * i;
            word = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(word, v[0], v[1], scale, 0);
            word = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(word, v[2], v[3], scale, 1);
            word = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(word, v[4], v[5], scale, 2);
            word = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(word, v[6], v[7], scale, 3);
            b.low[i] = word;
        }
    } else {
        f32x16 even, odd;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            even[i] = x[2 * i];
            odd[i] = x[2 * i + 1];
        }
        const u32x6 w = to_six_bits(even, odd, scale);
        b.low = u32x4{w[0], w[1], w[2], w[3]};
        b.high = u32x2{w[4], w[5]};
    }
    return b;
}

template <typename T, int BITS>
__global__ __launch_bounds__(kThreads) void quantize_kernel(RowArgs a) {
    uint64_t row;
    uint32_t block;
    if (!block_of(a, row, block)) return;
    Block<BITS> b{};
    uint32_t byte = 0;
    if (block < a.blocks) {
        const T* in = static_cast<const T*>(a.input) + row * a.stride + block * kBlock;
        T x[32];
        constexpr int kPer = 16 / sizeof(T);
#pragma unroll
        for (int i = 0; i < 32 / kPer; ++i) {
            const u32x4 part = *reinterpret_cast<const u32x4_a2*>(in + i * kPer);
            __builtin_memcpy(x + i * kPer, &part, 16);
        }
        uint32_t most = 0;
        if constexpr (sizeof(T) == 2) {
#pragma unroll
            for (int i = 0; i < 32; ++i) most = max(most, __builtin_bit_cast(uint16_t, x[i]) & 0x7FFFu);
            most = most >= 0x7C00u ? 0x7F800000u
                                   : __builtin_bit_cast(uint32_t, static_cast<float>(__builtin_bit_cast(
                                                                      _Float16, static_cast<uint16_t>(most))));
        } else {
#pragma unroll
            for (int i = 0; i < 32; ++i) most = max(most, __builtin_bit_cast(uint32_t, x[i]) & 0x7FFFFFFFu);
        }
        byte = scale_of(most);
        if (byte < 255) {
            // Small scales, 2^-127 among them, are no normal numbers for the conversion, or
            // near it: both sides of its quotient times 2^64, which is exact.
            uint32_t by = byte;
            if constexpr (sizeof(T) == 4) {
                if (byte < 32) {
#pragma unroll
                    for (int i = 0; i < 32; ++i) x[i] *= 0x1p64f;
                    by = byte + 64;
                }
            } else {
                if (byte == 0) by = 127;  // zeros
            }
            b = convert<BITS>(x, __builtin_bit_cast(float, by << 23));
        }
    }
    uint8_t* out = a.values + row * value_bytes(a.kp, BITS);
    *reinterpret_cast<u32x4*>(out + 16 * block) = b.low;
    if constexpr (BITS == 6) *reinterpret_cast<u32x2*>(out + a.kp / 2 + 8 * block) = b.high;
    a.scales[row * scale_bytes(a.kp) + block] = static_cast<uint8_t>(byte);
}

// 2^(b - 127), NaN for 255.
__device__ __forceinline__ float scale_value(uint32_t byte) {
    const uint32_t bits = byte == 0 ? 0x00400000u : byte << 23;
    return byte == 255 ? __builtin_nanf("") : __builtin_bit_cast(float, bits);
}

// The blocks leave through LDS, so that a wave's stores are each 1024 bytes in a row.
template <typename T, int BITS>
__global__ __launch_bounds__(kThreads) void dequantize_kernel(RowArgs a) {
    constexpr int kPer = 16 / sizeof(T), kPieces = 32 / kPer;  // 16-byte pieces of a block
    constexpr int kRoom = kPieces * 16 + 16;                   // 16 bytes more: 8 lanes touch all banks
    __shared__ __attribute__((aligned(16))) uint8_t lds[kThreads / 64][64 * kRoom];
    uint64_t row;
    uint32_t block;
    const bool there = block_of(a, row, block) && block < a.blocks;
    const uint32_t lane = threadIdx.x & 63;
    uint8_t* const turn = lds[threadIdx.x >> 6];
    uint64_t to = 0;  // where the block goes; 0: nowhere
    if (there) {
        const Block<BITS> b = load_block<BITS>(a.values_in + row * value_bytes(a.kp, BITS), a.kp, block);
        const float scale = scale_value(a.scales[row * scale_bytes(a.kp) + block]);
        float v[32];
        if constexpr (BITS == 4) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const auto pair = [&](int at, f32x2 p) { v[8 * i + 2 * at] = p.x, v[8 * i + 2 * at + 1] = p.y; };
                pair(0, __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(b.low[i], 1.0f, 0));
                pair(1, __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(b.low[i], 1.0f, 1));
                pair(2, __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(b.low[i], 1.0f, 2));
                pair(3, __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(b.low[i], 1.0f, 3));
            }
        } else {
            const u32x6 codes = {b.low.x, b.low.y, b.low.z, b.low.w, b.high.x, b.high.y};
            const f32x32 w = from_six_bits(codes);
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] = w[i];
        }
#pragma unroll
        for (int i = 0; i < kPieces; ++i) {
            T part[kPer];
#pragma unroll
            for (int j = 0; j < kPer; ++j) part[j] = to_out<T>(v[i * kPer + j] * scale);
            u32x4 word;
            __builtin_memcpy(&word, part, 16);
            *reinterpret_cast<u32x4*>(turn + lane * kRoom + 16 * i) = word;
        }
        to = reinterpret_cast<uint64_t>(static_cast<T*>(a.output) + row * a.stride + block * kBlock);
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
        const uint32_t piece = i * 64 + lane, of = piece / kPieces;
        const uint64_t begin = __shfl(to, of, 64);
        if (begin == 0) continue;
        *reinterpret_cast<u32x4_a2*>(begin + piece % kPieces * 16) =
            *reinterpret_cast<const u32x4*>(turn + of * kRoom + piece % kPieces * 16);
    }
}

template <typename T>
int launch(bool back, const void* input, const void* values, const void* scales, void* output, uint64_t rows,
           uint64_t features, uint64_t stride, int bits, void* stream) {
    const void* plain = back ? output : input;
    if (!plain || !values || !scales || !stream || !known_bits(bits)) return kInvalid;
    if (features % kBlock != 0 || features > kMostFeatures || rows > kMostRows * 2 || stride < features ||
        stride > (uint64_t{1} << 40))
        return kInvalid;
    if (off_grid(plain, sizeof(T)) || off_grid(values, 16)) return kInvalid;
    if (rows == 0 || features == 0) return 0;
    const uint32_t kp = padded(features);
    const uint64_t threads = rows * (kp / kBlock);
    if (threads > kMostThreads - kThreads) return kInvalid;
    const RowArgs a{input,
                    output,
                    static_cast<const uint8_t*>(values),
                    static_cast<uint8_t*>(const_cast<void*>(values)),
                    static_cast<uint8_t*>(const_cast<void*>(scales)),
                    rows,
                    stride,
                    kp,
                    static_cast<uint32_t>(features / kBlock)};
    const dim3 grid(static_cast<uint32_t>((threads + kThreads - 1) / kThreads));
    const auto go = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, grid, dim3(kThreads), 0, static_cast<hipStream_t>(stream), a);
    };
    if (back)
        bits == 4 ? go(dequantize_kernel<T, 4>) : go(dequantize_kernel<T, 6>);
    else
        bits == 4 ? go(quantize_kernel<T, 4>) : go(quantize_kernel<T, 6>);
    return static_cast<int>(hipGetLastError());
}

}  // namespace
}  // namespace mote::mx

MOTE_EXPORT int mote_hip_mx_quantize_f16(const void* input, void* values, void* scales, uint64_t rows,
                                         uint64_t features, uint64_t input_stride, int bits, void* stream) noexcept {
    return mote::mx::launch<_Float16>(false, input, values, scales, nullptr, rows, features, input_stride, bits, stream);
}
MOTE_EXPORT int mote_hip_mx_quantize_f32(const void* input, void* values, void* scales, uint64_t rows,
                                         uint64_t features, uint64_t input_stride, int bits, void* stream) noexcept {
    return mote::mx::launch<float>(false, input, values, scales, nullptr, rows, features, input_stride, bits, stream);
}
MOTE_EXPORT int mote_hip_mx_dequantize_f16(const void* values, const void* scales, void* output, uint64_t rows,
                                           uint64_t features, uint64_t output_stride, int bits, void* stream) noexcept {
    return mote::mx::launch<_Float16>(true, nullptr, values, scales, output, rows, features, output_stride, bits,
                                      stream);
}
MOTE_EXPORT int mote_hip_mx_dequantize_f32(const void* values, const void* scales, void* output, uint64_t rows,
                                           uint64_t features, uint64_t output_stride, int bits, void* stream) noexcept {
    return mote::mx::launch<float>(true, nullptr, values, scales, output, rows, features, output_stride, bits, stream);
}
