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
//
// Prompts (8 of up to 2000 tokens, 8 heads of 128, 42 MB each way): read 9.1 us, 4.6
// TB/s; append 12.3 us, 3.4 TB/s, its waves waiting 56 % of their time (four barriers
// between loads and stores) and the vector ALUs busy 59 % of the cycles.  Single tokens
// are bound by the chain of loads offsets, table, rows (64 sequences: 5.4 and 5.3 us).
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
    uint32_t sequences, tokens, heads, head_dim, table_blocks, cache_blocks, first;  // first: unit of the launch
};

// The part of a sequence's rows that lies in one block.
struct Piece {
    uint64_t planes;   // its head's plane of keys; of scales and, times 32 P, of the cache
    uint64_t row;      // packed row of its first token
    uint32_t from, n;  // its first slot and its tokens
    bool found;
};

__device__ __forceinline__ Piece piece_of(const CacheArgs& a, uint32_t unit, uint32_t head) {
    Span rows;  // first of the lane's sequence, then of the workgroup's
    uint32_t first;
    const Unit u = locate<kBlockTokens, 2>(unit, a.offsets, a.sequences, a.tokens, [&](uint32_t s) {
        rows = span_of(a.offsets, s, a.tokens);
        first = max(a.positions[s], 0);
    });
    Piece r{0, 0, 0, 0, false};
    if (!u.found) return r;
    rows = span_at(rows, u.lane);
    first = __builtin_amdgcn_readlane(first, u.lane);
    const uint32_t block = first / kBlockTokens + u.local;
    if (block * kBlockTokens >= first + static_cast<uint32_t>(rows.n)) return r;  // room that it does not need
    if (block >= a.table_blocks) return r;
    const int32_t id = a.table[static_cast<uint64_t>(u.sequence) * a.table_blocks + block];
    if (id < 0 || static_cast<uint32_t>(id) >= a.cache_blocks) return r;
    const uint32_t at = max(first, block * kBlockTokens);
    const uint32_t end = min(first + static_cast<uint32_t>(rows.n), (block + 1) * kBlockTokens);
    return {(static_cast<uint64_t>(id) * a.heads + head) * 2, static_cast<uint64_t>(rows.at) + (at - first),
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

constexpr uint32_t kMostPlane = kBlockTokens * kMostHeadDim;

__device__ __forceinline__ float scale_from_bits(uint32_t most) {
    // `most` is the largest magnitude's pattern: infinities and NaN order above every number.
    if (most >= 0x7C00u) return __builtin_nanf("");
    return static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(most))) / 127.0f;
}

// rint(x) held to [-127, 127], plus 128, in the low byte: the sum has no bits below one.
__device__ __forceinline__ uint32_t to_byte(float x) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_fmed3f(x, -127.0f, 127.0f) + (12582912.0f + 128.0f));
}
__device__ __forceinline__ uint32_t four_bytes(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    const uint32_t lo = __builtin_amdgcn_perm(b, a, 0x0C0C0400u), hi = __builtin_amdgcn_perm(d, c, 0x0C0C0400u);
    return lo | hi << 16;
}

// The largest of a wave's lanes, in lane 63.
__device__ __forceinline__ uint32_t wave_most(uint32_t v) {
    const auto with = [&](int other) { v = max(v, static_cast<uint32_t>(other)); };
    with(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), 0x111, 0xF, 0xF, false));  // row_shr:1, 2, 4, 8
    with(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), 0x112, 0xF, 0xF, false));
    with(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), 0x114, 0xF, 0xF, false));
    with(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), 0x118, 0xF, 0xF, false));
    with(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), 0x142, 0xA, 0xF, false));  // row_bcast:15
    with(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), 0x143, 0xC, 0xF, false));  // row_bcast:31
    return v;
}

// The plane's scale after the new tokens, whose largest magnitude's pattern is
// `most`; `old` is 0 for a block begun anew.
struct Scale {
    float scale, inverse;  // inverse: 0 for an all-zero plane and for NaN (bytes 128)
    float old;
};
__device__ __forceinline__ Scale new_scale(uint32_t most, float old) {
    const float need = scale_from_bits(most);
    const float scale = old != old || need != need ? __builtin_nanf("") : fmaxf(old, need);
    return {scale, scale > 0.0f ? 1.0f / scale : 0.0f, old};
}

// Of a token's bytes in LDS: rows read together lie in different banks.
constexpr uint32_t stage_row(int chunks) { return 64 * chunks + 8; }

// Writes the new tokens' bytes, `x` being the thread's chunks of its token.
template <bool VALUES, int CHUNKS>
__device__ __forceinline__ void write_plane(const CacheArgs& a, const Piece& p, u32x4 (&x)[CHUNKS], const Scale& s,
                                            uint8_t* image, uint8_t* stage) {
    constexpr uint32_t kStageRow = stage_row(CHUNKS);
    const uint32_t padded = padded_dim(a.head_dim), plane_bytes = kBlockTokens * padded;
    uint8_t* const plane = a.cache + (p.planes + VALUES) * plane_bytes;
    const uint32_t t = threadIdx.x >> 3, sub = threadIdx.x & 7, chunks = a.head_dim / 8;
    const bool keep = p.from != 0 && s.scale == s.old;  // the earlier bytes stay as they are: only the new are written
    const bool turn = VALUES && p.from == 0;
    if (!(s.scale > 0.0f)) {
#pragma unroll
        for (int i = 0; i < CHUNKS; ++i) x[i] = u32x4{0, 0, 0, 0};
    }
    // Otherwise the plane goes through its image in LDS: the earlier tokens' bytes
    // rounded again to the larger scale, or zeros where none is written.
    if (p.from != 0 && !keep) {
        const float ratio = s.scale > 0.0f ? s.old * s.inverse : 0.0f;
        for (uint32_t i = threadIdx.x; i < plane_bytes / 16; i += 256) {
            u32x4 b = reinterpret_cast<const u32x4*>(plane)[i];
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                uint32_t r[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) r[j] = to_byte((static_cast<float>((b[w] >> (8 * j)) & 255u) - 128.0f) * ratio);
                b[w] = four_bytes(r[0], r[1], r[2], r[3]);
            }
            reinterpret_cast<u32x4*>(image)[i] = b;
        }
        __syncthreads();
    } else if (!keep && !turn && (p.n < kBlockTokens || a.head_dim % 32 != 0)) {
        for (uint32_t i = threadIdx.x; i < plane_bytes / 16; i += 256)
            reinterpret_cast<u32x4*>(image)[i] = u32x4{0x80808080u, 0x80808080u, 0x80808080u, 0x80808080u};
        __syncthreads();
    }
    if (t < p.n) {
#pragma unroll
        for (int i = 0; i < CHUNKS; ++i) {
            const uint32_t c = sub + 8 * i;
            if (c >= chunks) break;
            uint32_t b[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const uint32_t pair = x[i][j / 2];
                b[j] = to_byte(((j & 1) ? half_hi_to_float(pair) : half_lo_to_float(pair)) * s.inverse);
            }
            const u32x2 eight = {four_bytes(b[0], b[1], b[2], b[3]), four_bytes(b[4], b[5], b[6], b[7])};
            if (turn) {
                *reinterpret_cast<u32x2*>(stage + t * kStageRow + c * 8) = eight;
            } else if constexpr (VALUES) {  // dimensions are 16 bytes apart
                uint8_t* const to = (keep ? plane : image) + byte_of<true>(p.from + t, c * 8);
#pragma unroll
                for (int j = 0; j < 8; ++j) to[16 * j] = static_cast<uint8_t>(b[j]);
            } else {
                *reinterpret_cast<u32x2*>((keep ? plane : image) + byte_of<false>(p.from + t, c * 8)) = eight;
            }
        }
    }
    if (turn) {
        // A block of values begun anew: four tokens of a dimension are neighbours in
        // the plane, so four by four bytes are turned at a time.
        __syncthreads();
        for (uint32_t i = threadIdx.x; i < plane_bytes / 16; i += 256) {
            const uint32_t d = i % (padded / 4) * 4, slot = i / (padded / 4) * 4;
            uint32_t r[4];
#pragma unroll
            for (uint32_t j = 0; j < 4; ++j) {
                r[j] = 0x80808080u;
                if (slot + j < p.n && d < a.head_dim)
                    r[j] = *reinterpret_cast<const uint32_t*>(stage + (slot + j) * kStageRow + d);
            }
            const auto pick = [](uint32_t hi, uint32_t lo, uint32_t sel) { return __builtin_amdgcn_perm(hi, lo, sel); };
            const uint32_t ab02 = pick(r[1], r[0], 0x06020400u), ab13 = pick(r[1], r[0], 0x07030501u);
            const uint32_t cd02 = pick(r[3], r[2], 0x06020400u), cd13 = pick(r[3], r[2], 0x07030501u);
            uint8_t* const to = image + byte_of<true>(slot, d);
            *reinterpret_cast<uint32_t*>(to) = pick(cd02, ab02, 0x05040100u);
            *reinterpret_cast<uint32_t*>(to + 16) = pick(cd13, ab13, 0x05040100u);
            *reinterpret_cast<uint32_t*>(to + 32) = pick(cd02, ab02, 0x07060302u);
            *reinterpret_cast<uint32_t*>(to + 48) = pick(cd13, ab13, 0x07060302u);
        }
    }
    if (keep) return;
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < plane_bytes / 16; i += 256)
        reinterpret_cast<u32x4*>(plane)[i] = reinterpret_cast<const u32x4*>(image)[i];
    if (threadIdx.x == 0) a.scales[p.planes + VALUES] = s.scale;
}

// One workgroup per (block piece, head): eight threads a token, which hold its
// values of both planes, CHUNKS 16-byte chunks each, while the planes' scales are
// found.  (8 prompts of 2000 tokens at most, 8 heads of 128: with room for 256
// dimensions in registers and LDS, which leaves four workgroups a compute unit, 13 %
// longer than with room for 128.)
template <int CHUNKS>
__global__ __launch_bounds__(256) void append_kernel(CacheArgs a) {
    __shared__ __align__(16) uint8_t image[2][kBlockTokens * 64 * CHUNKS];
    __shared__ __align__(16) uint8_t stage[kBlockTokens * stage_row(CHUNKS)];
    __shared__ uint32_t most_of[2][4];
    const uint32_t head = blockIdx.y;
    const Piece p = piece_of(a, a.first + blockIdx.x, head);
    if (!p.found) return;
    const float old_k = p.from != 0 ? a.scales[p.planes] : 0.0f, old_v = p.from != 0 ? a.scales[p.planes + 1] : 0.0f;
    const uint32_t t = threadIdx.x >> 3, sub = threadIdx.x & 7, chunks = a.head_dim / 8;
    const _Float16* const k = a.k + (p.row + t) * a.k_stride + static_cast<uint64_t>(head) * a.head_dim;
    const _Float16* const v = a.v + (p.row + t) * a.v_stride + static_cast<uint64_t>(head) * a.head_dim;
    u32x4 xk[CHUNKS], xv[CHUNKS];
    uint32_t most_k = 0, most_v = 0;
#pragma unroll
    for (int i = 0; i < CHUNKS; ++i) {
        const uint32_t c = sub + 8 * i;
        xk[i] = xv[i] = u32x4{0, 0, 0, 0};
        if (t < p.n && c < chunks) {
            xk[i] = *reinterpret_cast<const u32x4_a2*>(k + c * 8);
            xv[i] = *reinterpret_cast<const u32x4_a2*>(v + c * 8);
        }
    }
#pragma unroll
    for (int i = 0; i < CHUNKS; ++i)
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            most_k = max(most_k, max(xk[i][w] & 0x7FFFu, (xk[i][w] >> 16) & 0x7FFFu));
            most_v = max(most_v, max(xv[i][w] & 0x7FFFu, (xv[i][w] >> 16) & 0x7FFFu));
        }
    most_k = wave_most(most_k);
    most_v = wave_most(most_v);
    if ((threadIdx.x & 63) == 63) {
        most_of[0][threadIdx.x >> 6] = most_k;
        most_of[1][threadIdx.x >> 6] = most_v;
    }
    __syncthreads();
    const auto all = [&](const uint32_t (&of)[4]) { return max(max(of[0], of[1]), max(of[2], of[3])); };
    write_plane<false>(a, p, xk, new_scale(all(most_of[0]), old_k), image[0], stage);
    write_plane<true>(a, p, xv, new_scale(all(most_of[1]), old_v), image[1], stage);
}

// (u - 128) s in binary16 for the bytes of a dword.
__device__ __forceinline__ void values_of(uint32_t b, float scale, _Float16 (&out)[4]) {
#pragma unroll
    for (int j = 0; j < 4; ++j)
        out[j] = static_cast<_Float16>((static_cast<float>((b >> (8 * j)) & 255u) - 128.0f) * scale);
}

// One workgroup per (block piece, head): planes come in 16 bytes a thread, pass
// through LDS as rows of tokens and leave in 16-byte chunks of a row.
__global__ __launch_bounds__(256) void read_kernel(CacheArgs a) {
    constexpr uint32_t kMostRow = kMostHeadDim + 8;  // rows 16 bytes past a multiple of the banks
    __shared__ __align__(16) _Float16 rows[kBlockTokens * kMostRow];
    const uint32_t head = blockIdx.y;
    const Piece p = piece_of(a, a.first + blockIdx.x, head);
    if (!p.found) return;
    const uint32_t padded = padded_dim(a.head_dim), loads = kBlockTokens * padded / 16, row = padded + 8;
    const float scale_k = a.scales[p.planes], scale_v = a.scales[p.planes + 1];
    const u32x4* const plane = reinterpret_cast<const u32x4*>(a.cache + p.planes * (kBlockTokens * padded));
    constexpr int kLoads = kMostPlane / 16 / 256;
    u32x4 bk[kLoads], bv[kLoads];
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
        const uint32_t at = threadIdx.x + 256 * i;
        bk[i] = bv[i] = u32x4{0, 0, 0, 0};
        if (at < loads) {
            bk[i] = plane[at];
            bv[i] = plane[loads + at];
        }
    }
    const uint32_t chunks = a.head_dim / 8;
    const auto store = [&](_Float16* to, uint64_t stride) {
        __syncthreads();
        for (uint32_t i = threadIdx.x; i < p.n * chunks; i += 256) {
            const uint32_t t = i / chunks, c = i % chunks;
            *reinterpret_cast<u32x4_a2*>(to + (p.row + t) * stride + static_cast<uint64_t>(head) * a.head_dim + 8 * c) =
                *reinterpret_cast<const u32x4*>(rows + (p.from + t) * row + 8 * c);
        }
    };
    // Position of 16 bytes: (c, g, m); keys: tokens m and 16 + m, dimensions 32 c + 8 g ..
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
        const uint32_t at = threadIdx.x + 256 * i, m = at & 15, d = (at >> 4) * 8;
        if (at >= loads) break;
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            _Float16 x[8];
            values_of(bk[i][2 * half], scale_k, reinterpret_cast<_Float16(&)[4]>(x[0]));
            values_of(bk[i][2 * half + 1], scale_k, reinterpret_cast<_Float16(&)[4]>(x[4]));
            f16x8 y;
#pragma unroll
            for (int j = 0; j < 8; ++j) y[j] = x[j];
            *reinterpret_cast<f16x8*>(rows + (m + 16 * half) * row + d) = y;
        }
    }
    store(a.k, a.k_stride);
    __syncthreads();
    // values: dimensions 32 c + m and 16 more, tokens 4 g .. and 16 + 4 g ..
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
        const uint32_t at = threadIdx.x + 256 * i, m = at & 15, g = (at >> 4) & 3, c = at >> 6;
        if (at >= loads) break;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            _Float16 x[4];
            values_of(bv[i][w], scale_v, x);
#pragma unroll
            for (int j = 0; j < 4; ++j) rows[(16 * (w & 1) + 4 * g + j) * row + 32 * c + 16 * (w >> 1) + m] = x[j];
        }
    }
    store(a.v, a.v_stride);
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

// A workgroup for each piece there is room for and each head.
int launch_pieces(void (*kernel)(CacheArgs), CacheArgs a, void* stream) {
    const uint64_t pieces = units_of(kBlockTokens, 2, a.sequences, a.tokens), most = most_groups(256);
    for (uint64_t first = 0; first < pieces; first += most) {
        a.first = static_cast<uint32_t>(first);
        const uint64_t now = pieces - first < most ? pieces - first : most;
        hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(now), a.heads), dim3(256), 0,
                           static_cast<hipStream_t>(stream), a);
        const int status = static_cast<int>(hipGetLastError());
        if (status != 0) return status;
    }
    return 0;
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
    const CacheArgs a{static_cast<const int32_t*>(offsets), static_cast<const int32_t*>(positions),
                      static_cast<const int32_t*>(block_table), static_cast<uint8_t*>(cache),
                      static_cast<float*>(scales), static_cast<_Float16*>(const_cast<void*>(k)),
                      static_cast<_Float16*>(const_cast<void*>(v)), k_stride, v_stride,
                      static_cast<uint32_t>(sequences), static_cast<uint32_t>(tokens), static_cast<uint32_t>(kv_heads),
                      static_cast<uint32_t>(head_dim), static_cast<uint32_t>(table_blocks),
                      static_cast<uint32_t>(cache_blocks), 0};
    const auto kernel = head_dim <= 64 ? append_kernel<1> : head_dim <= 128 ? append_kernel<2> : append_kernel<4>;
    return launch_pieces(kernel, a, stream);
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
    const CacheArgs a{static_cast<const int32_t*>(offsets), static_cast<const int32_t*>(positions),
                      static_cast<const int32_t*>(block_table), static_cast<uint8_t*>(const_cast<void*>(cache)),
                      static_cast<float*>(const_cast<void*>(scales)), static_cast<_Float16*>(k),
                      static_cast<_Float16*>(v), k_stride, v_stride, static_cast<uint32_t>(sequences),
                      static_cast<uint32_t>(tokens), static_cast<uint32_t>(kv_heads), static_cast<uint32_t>(head_dim),
                      static_cast<uint32_t>(table_blocks), static_cast<uint32_t>(cache_blocks), 0};
    return launch_pieces(read_kernel, a, stream);
}
