// Keys and values into and out of the 8-bit cache.
//
// A block of 32 tokens has, for each head, a plane of keys and a plane of values
// of 32 P bytes (P: the head size rounded up to 32) and a 32-bit scale for each
// plane; a byte u stands for (u - 128) s.  With c = d / 32, the byte of element
// (token t of the block, dimension d) is at
//   keys:    [c][(d % 32) / 8][t % 16][t / 16][d % 8]               of [P/32][4][16][2][8]
//   values:  [c][(t % 16) / 4][d % 16][(d % 32) / 16][4 (t/16) + t % 4]
// which are the orders the 16 x 16 x 32 matrix instruction wants its operands
// in: the attention reads both planes with lane-linear 16-byte loads.
//
// Scale of a plane: s = max |x| / 127 over its tokens, byte = rint(x / s) + 128
// (x times the rounded reciprocal of s).  A plane that holds earlier tokens
// keeps its scale unless a new token needs a larger one; its bytes are then
// rounded again, rint((u - 128) s_old / s_new).  A value that is not finite
// makes the plane's scale NaN until the block is begun again, so it shows in
// every read and is never taken for a number.
#include <hip/hip_runtime.h>

#include <cstdint>

#include "attention.hpp"

namespace mote::attention {
namespace {

struct CacheArgs {
    const int32_t* offsets;    // [sequences + 1] packed rows of each sequence
    const int32_t* positions;  // [sequences] tokens before its first row
    const int32_t* table;      // [sequences][table_blocks]
    uint8_t* cache;            // [cache_blocks][heads][2][32 P]
    float* scales;             // [cache_blocks][heads][2]
    _Float16* k;
    _Float16* v;
    uint64_t k_stride, v_stride;  // elements between packed rows
    uint32_t sequences, tokens, heads, head_dim, table_blocks, cache_blocks;
};

// The part of a sequence's rows that lies in one block.
struct Piece {
    uint64_t plane;   // of scales and, times 32 P, of the cache
    uint64_t row;     // packed row of its first token
    uint32_t from, n; // its first slot and its tokens
    bool found;
};

__device__ __forceinline__ Piece piece_of(const CacheArgs& a, uint32_t unit, uint32_t head, uint32_t which) {
    Span rows;  // first of the lane's sequence, then of the workgroup's
    uint32_t first;
    const Unit u = locate(unit, a.sequences, [&](uint32_t s) {
        rows = span_of(a.offsets, s, a.tokens);
        first = max(a.positions[s], 0);
        return rows.n > 0 ? (first + rows.n - 1) / kBlockTokens - first / kBlockTokens + 1 : 0u;
    });
    Piece r{0, 0, 0, 0, false};
    if (!u.found) return r;
    rows = span_at(rows, u.lane);
    first = __builtin_amdgcn_readlane(first, u.lane);
    const uint32_t block = first / kBlockTokens + u.local;
    if (block >= a.table_blocks) return r;
    const int32_t id = a.table[static_cast<uint64_t>(u.sequence) * a.table_blocks + block];
    if (id < 0 || static_cast<uint32_t>(id) >= a.cache_blocks) return r;
    const uint32_t at = max(first, block * kBlockTokens);
    const uint32_t end = min(first + static_cast<uint32_t>(rows.n), (block + 1) * kBlockTokens);
    return {(static_cast<uint64_t>(id) * a.heads + head) * 2 + which, static_cast<uint64_t>(rows.at) + (at - first),
            at % kBlockTokens, end - at, true};
}

// Byte of element (t, d) of a plane.
template <bool VALUES>
__device__ __forceinline__ uint32_t byte_of(uint32_t t, uint32_t d) {
    const uint32_t c = d >> 5;
    if constexpr (VALUES)
        return (((c * 4 + ((t & 15) >> 2)) * 16 + (d & 15)) * 2 + ((d >> 4) & 1)) * 8 + (t >> 4) * 4 + (t & 3);
    else
        return (((c * 4 + ((d & 31) >> 3)) * 16 + (t & 15)) * 2 + (t >> 4)) * 8 + (d & 7);
}

constexpr uint32_t kMostPlane = 32 * 256;

__device__ __forceinline__ float scale_from_bits(uint32_t most) {
    // `most` is the largest magnitude's pattern: infinities and NaN order above every number.
    if (most >= 0x7C00u) return __builtin_nanf("");
    return static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(most))) / 127.0f;
}

__device__ __forceinline__ uint32_t to_byte(float x) {
    return static_cast<uint32_t>(static_cast<int>(fminf(fmaxf(__builtin_rintf(x), -127.0f), 127.0f)) + 128);
}

// One workgroup per (block piece, head, keys or values).
template <bool VALUES>
__device__ __forceinline__ void append_piece(const CacheArgs& a, uint32_t unit, uint32_t head) {
    __shared__ __align__(16) uint8_t image[kMostPlane];
    __shared__ uint32_t most_of[4];
    const Piece p = piece_of(a, unit, head, VALUES);
    if (!p.found) return;
    const uint32_t plane_bytes = kBlockTokens * padded_dim(a.head_dim);
    uint8_t* plane = a.cache + p.plane * plane_bytes;
    const _Float16* rows = (VALUES ? a.v + p.row * a.v_stride : a.k + p.row * a.k_stride) +
                           static_cast<uint64_t>(head) * a.head_dim;
    const uint64_t stride = VALUES ? a.v_stride : a.k_stride;
    const uint32_t t = threadIdx.x >> 3, sub = threadIdx.x & 7;  // eight threads a token
    const uint32_t chunks = a.head_dim / 8;
    constexpr int kChunks = 4;  // 16-byte chunks of a thread: 256 dimensions by eight threads
    u32x4 x[kChunks];
    uint32_t most = 0;
#pragma unroll
    for (int i = 0; i < kChunks; ++i) {
        const uint32_t c = sub + 8 * i;
        x[i] = u32x4{0, 0, 0, 0};
        if (t < p.n && c < chunks) x[i] = *reinterpret_cast<const u32x4_a2*>(rows + t * stride + c * 8);
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            most = max(most, x[i][w] & 0x7FFFu);
            most = max(most, (x[i][w] >> 16) & 0x7FFFu);
        }
    }
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) most = max(most, static_cast<uint32_t>(__shfl_xor(most, d, 64)));
    if ((threadIdx.x & 63) == 0) most_of[threadIdx.x >> 6] = most;
    float* const scale_at = a.scales + p.plane;
    const float old = p.from != 0 ? *scale_at : 0.0f;
    __syncthreads();
    most = max(max(most_of[0], most_of[1]), max(most_of[2], most_of[3]));
    const float need = scale_from_bits(most);
    const float scale = old != old || need != need ? __builtin_nanf("") : fmaxf(old, need);
    const float inverse = scale > 0.0f ? 1.0f / scale : 0.0f;  // 0 for an all-zero plane and for NaN: bytes 128
    const bool keep = p.from != 0 && scale == old;  // earlier bytes stay as they are
    // The plane's image: earlier tokens' bytes, rounded again where the scale has grown.
    if (p.from != 0) {
        const float ratio = old * inverse;
        for (uint32_t i = threadIdx.x; i < plane_bytes / 16; i += 256) {
            u32x4 b = reinterpret_cast<const u32x4*>(plane)[i];
            if (!keep) {
#pragma unroll
                for (int w = 0; w < 4; ++w) {
                    uint32_t r = 0;
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const float u = static_cast<float>((b[w] >> (8 * j)) & 255u) - 128.0f;
                        r |= to_byte(scale > 0.0f ? u * ratio : 0.0f) << (8 * j);
                    }
                    b[w] = r;
                }
            }
            reinterpret_cast<u32x4*>(image)[i] = b;
        }
        __syncthreads();
    } else if (p.n < kBlockTokens || a.head_dim % 32 != 0) {
        for (uint32_t i = threadIdx.x; i < plane_bytes / 16; i += 256)
            reinterpret_cast<u32x4*>(image)[i] = u32x4{0x80808080u, 0x80808080u, 0x80808080u, 0x80808080u};
        __syncthreads();
    }
    if (t < p.n) {
#pragma unroll
        for (int i = 0; i < kChunks; ++i) {
            const uint32_t c = sub + 8 * i;
            if (c >= chunks) break;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float e = (j & 1) ? half_hi_to_float(x[i][j / 2]) : half_lo_to_float(x[i][j / 2]);
                image[byte_of<VALUES>(p.from + t, c * 8 + j)] =
                    static_cast<uint8_t>(scale > 0.0f ? to_byte(e * inverse) : 128u);
            }
        }
    }
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < plane_bytes / 16; i += 256)
        reinterpret_cast<u32x4*>(plane)[i] = reinterpret_cast<const u32x4*>(image)[i];
    if (threadIdx.x == 0 && !keep) *scale_at = scale;
}

__global__ __launch_bounds__(256) void append_kernel(CacheArgs a) {
    if (blockIdx.z == 0)
        append_piece<false>(a, blockIdx.x, blockIdx.y);
    else
        append_piece<true>(a, blockIdx.x, blockIdx.y);
}

template <bool VALUES>
__device__ __forceinline__ void read_piece(const CacheArgs& a, uint32_t unit, uint32_t head) {
    const uint32_t t = threadIdx.x >> 3, sub = threadIdx.x & 7;
    const Piece p = piece_of(a, unit, head, VALUES);
    if (!p.found || t >= p.n) return;
    const uint32_t plane_bytes = kBlockTokens * padded_dim(a.head_dim);
    const uint8_t* plane = a.cache + p.plane * plane_bytes;
    const float scale = a.scales[p.plane];
    const uint64_t stride = VALUES ? a.v_stride : a.k_stride;
    _Float16* row = (VALUES ? a.v : a.k) + (p.row + t) * stride + static_cast<uint64_t>(head) * a.head_dim;
    for (uint32_t d = sub; d < a.head_dim; d += 8)
        row[d] = static_cast<_Float16>((static_cast<float>(plane[byte_of<VALUES>(p.from + t, d)]) - 128.0f) * scale);
}

__global__ __launch_bounds__(256) void read_kernel(CacheArgs a) {
    if (blockIdx.z == 0)
        read_piece<false>(a, blockIdx.x, blockIdx.y);
    else
        read_piece<true>(a, blockIdx.x, blockIdx.y);
}

// Checks shared by both directions; 1: go on.
int check_cache_call(const void* k, const void* v, const void* offsets, const void* positions, const void* table,
                     const void* cache, const void* scales, uint64_t sequences, uint64_t tokens, uint64_t heads,
                     uint64_t head_dim, uint64_t table_blocks, uint64_t cache_blocks, void* stream) {
    if (!k || !v || !offsets || !positions || !table || !cache || !scales || !stream) return kInvalid;
    if (head_dim % 8 != 0 || head_dim > kMostHeadDim) return kInvalid;
    if (tokens > kMostTokens || sequences > kMostTokens || heads > 65535) return kInvalid;
    if (table_blocks > kMostTokens / kBlockTokens || cache_blocks > 0x7FFFFFFFu) return kInvalid;
    if (odd_address(k) || odd_address(v) || off_grid(offsets, 4) || off_grid(positions, 4) || off_grid(table, 4) ||
        off_grid(scales, 4) || off_grid(cache, 16))
        return kInvalid;
    if (sequences == 0 || tokens == 0 || heads == 0 || head_dim == 0) return 0;
    return 1;
}

// Blocks that `tokens` new tokens of `sequences` sequences can touch: n tokens of
// one touch at most (n + 30) / 32 + 1.
uint64_t most_pieces(uint64_t sequences, uint64_t tokens) {
    const uint64_t with = sequences < tokens ? sequences : tokens;  // sequences with a token at all
    return (tokens + 30 * with) / kBlockTokens + with;
}

}  // namespace
}  // namespace mote::attention

MOTE_EXPORT int mote_hip_kv_cache_append_q8(const void* k, const void* v, const void* offsets, const void* positions,
                                           const void* block_table, void* cache, void* scales, uint64_t sequences,
                                           uint64_t tokens, uint64_t kv_heads, uint64_t head_dim, uint64_t k_stride,
                                           uint64_t v_stride, uint64_t table_blocks, uint64_t cache_blocks,
                                           void* stream) noexcept {
    using namespace mote::attention;
    const int go = check_cache_call(k, v, offsets, positions, block_table, cache, scales, sequences, tokens, kv_heads,
                                    head_dim, table_blocks, cache_blocks, stream);
    if (go != 1) return go;
    const uint64_t pieces = most_pieces(sequences, tokens);
    if (pieces > kMostGrid) return kInvalid;
    const CacheArgs a{static_cast<const int32_t*>(offsets), static_cast<const int32_t*>(positions),
                      static_cast<const int32_t*>(block_table), static_cast<uint8_t*>(cache),
                      static_cast<float*>(scales), static_cast<_Float16*>(const_cast<void*>(k)),
                      static_cast<_Float16*>(const_cast<void*>(v)), k_stride, v_stride,
                      static_cast<uint32_t>(sequences), static_cast<uint32_t>(tokens), static_cast<uint32_t>(kv_heads),
                      static_cast<uint32_t>(head_dim), static_cast<uint32_t>(table_blocks),
                      static_cast<uint32_t>(cache_blocks)};
    hipLaunchKernelGGL(append_kernel, dim3(static_cast<unsigned>(pieces), static_cast<unsigned>(kv_heads), 2),
                       dim3(256), 0, static_cast<hipStream_t>(stream), a);
    return static_cast<int>(hipGetLastError());
}

MOTE_EXPORT int mote_hip_kv_cache_read_q8_f16(const void* cache, const void* scales, const void* offsets,
                                             const void* positions, const void* block_table, void* k, void* v,
                                             uint64_t sequences, uint64_t tokens, uint64_t kv_heads,
                                             uint64_t head_dim, uint64_t k_stride, uint64_t v_stride,
                                             uint64_t table_blocks, uint64_t cache_blocks, void* stream) noexcept {
    using namespace mote::attention;
    const int go = check_cache_call(k, v, offsets, positions, block_table, cache, scales, sequences, tokens, kv_heads,
                                    head_dim, table_blocks, cache_blocks, stream);
    if (go != 1) return go;
    if (k_stride < kv_heads * head_dim || v_stride < kv_heads * head_dim) return kInvalid;
    const uint64_t pieces = most_pieces(sequences, tokens);
    if (pieces > kMostGrid) return kInvalid;
    const CacheArgs a{static_cast<const int32_t*>(offsets), static_cast<const int32_t*>(positions),
                      static_cast<const int32_t*>(block_table), static_cast<uint8_t*>(const_cast<void*>(cache)),
                      static_cast<float*>(const_cast<void*>(scales)), static_cast<_Float16*>(k),
                      static_cast<_Float16*>(v), k_stride, v_stride, static_cast<uint32_t>(sequences),
                      static_cast<uint32_t>(tokens), static_cast<uint32_t>(kv_heads), static_cast<uint32_t>(head_dim),
                      static_cast<uint32_t>(table_blocks), static_cast<uint32_t>(cache_blocks)};
    hipLaunchKernelGGL(read_kernel, dim3(static_cast<unsigned>(pieces), static_cast<unsigned>(kv_heads), 2), dim3(256),
                       0, static_cast<hipStream_t>(stream), a);
    return static_cast<int>(hipGetLastError());
}
