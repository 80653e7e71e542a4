// Attention over the 8-bit cache: the last n tokens of each sequence (one when
// decoding, several for drafts or a chunk of a prompt) over all its cached
// tokens, or the last `window` of them.
//
// The query heads of a key head and the sequence's query tokens are the rows of
// one small matrix product, so each cached byte is read once for all of them:
// S^T = K Q^T and O^T = V^T P^T on the 16 x 16 x 32 matrix instruction, 16 rows a
// tile.  With keys as the instruction's rows, a lane ends with the scores of one
// query row for tokens 4 g .. 4 g + 3 of each half block (g = lane / 16), which is
// the operand that the second product wants of it: no score leaves its register.
// Bytes become the exact binary16 integers u - 128; the planes' scales join the
// scores and the exponents in 32 bits.
//
// One pass is bound by the cache's bytes.  A workgroup takes `chunk` blocks of
// one (sequence, rows, key head), its waves a block each in turn, and joins the
// waves' sums through LDS; the chunks' sums join in a second launch.  With 8 key
// heads of 128: 1 x 131 000 tokens 52.5 us (5.11 TB/s, the join included), 64 sequences
// of up to 8192 tokens 106.5 us (4.83 TB/s), 1 x 600 tokens 7.0 us; a copy reaches 5.05
// to 5.18 TB/s here.  The vector ALUs, which turn bytes into operands, are busy 43 % of
// the cycles.  Chunks are cut from max_context: with a window far shorter, or lengths
// far below it, few of the workgroups have blocks (a window of 4096 over 131 072 tokens
// 24 us, 4096 tokens without one 12).
#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdint>

#include "attention_sums.hpp"
#include "tile_ops.hpp"

namespace mote::attention {
namespace {

struct CacheAttentionArgs {
    const _Float16* q;
    const uint8_t* cache;
    const float* scales;
    const int32_t* offsets;  // null: one query of each sequence
    const int32_t* lengths;
    const int32_t* table;
    _Float16* output;
    float2* stats;  // null: one part, written to output
    float* sums;
    uint64_t q_stride, out_stride;
    uint32_t sequences, tokens, max_queries, row_tiles, heads, kv_heads, head_dim;
    uint32_t table_blocks, cache_blocks, window, chunk, parts, first;
    float exponent;  // scale log2(e)
};

__device__ __forceinline__ f32x4 mfma16(const f16x8& a, const f16x8& b, const f32x4& c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

// Eight bytes as the binary16 integers u - 128: a byte under 0x64 reads 1024 + u.
__device__ __forceinline__ f16x8 values_of(uint32_t lo, uint32_t hi) {
    const f16x2 bias = {static_cast<_Float16>(-1152.0f), static_cast<_Float16>(-1152.0f)};
    const uint32_t top = 0x64646464u;
    const f16x2 a = as_h2(__builtin_amdgcn_perm(top, lo, 0x04010400u)) + bias;
    const f16x2 b = as_h2(__builtin_amdgcn_perm(top, lo, 0x04030402u)) + bias;
    const f16x2 c = as_h2(__builtin_amdgcn_perm(top, hi, 0x04010400u)) + bias;
    const f16x2 d = as_h2(__builtin_amdgcn_perm(top, hi, 0x04030402u)) + bias;
    return f16x8{a.x, a.y, b.x, b.y, c.x, c.y, d.x, d.y};
}

// Waves of a workgroup: sixteen, one workgroup a compute unit, where a wave does
// with 128 registers.  (One sequence of 131 000 tokens, 8 key heads of 128: 52 us,
// with four waves and four times the workgroups 58; 32 of 6000: 71 and 79; 64 of up
// to 8192: 107 and 113.)
constexpr int waves_of(int c, int nt) { return c * nt <= 4 ? 16 : 4; }

// C: 32-dimension groups of the padded head; NT: 16-row tiles of a workgroup.
template <int C, int NT>
__global__ __launch_bounds__(64 * waves_of(C, NT), waves_of(C, NT) == 16 ? 4 : NT * C <= 8 ? 2 : 1) void
cache_attention_kernel(CacheAttentionArgs a) {
    constexpr int WAVES = waves_of(C, NT);
    constexpr int kRows = 16 * NT;
    constexpr int kJoin = 4 / NT;               // dimension groups joined at a time: 256 pieces of 8
    constexpr int kRowFloats = 32 * kJoin + 4;  // padded: rows start 4 banks apart
    __shared__ __align__(16) float sums_of[WAVES][kRows][kRowFloats];
    __shared__ float2 stats_of[WAVES][kRows];

    uint32_t id = a.first + blockIdx.x;
    const uint32_t part = id % a.parts;
    id /= a.parts;
    const uint32_t kv_head = id % a.kv_heads;
    id /= a.kv_heads;
    const uint32_t row_tile = id % a.row_tiles, seq = id / a.row_tiles;

    const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n = lane & 15, g = lane >> 4;
    const uint32_t group = a.heads / a.kv_heads;
    Span rows = {static_cast<int>(seq), 1};
    if (a.offsets != nullptr) rows = scalar_span_of(a.offsets, seq, a.tokens);
    const auto mark = [&] {  // done last: before the walk, 80 rows of 16 x 8000 tokens took 110 us for 107
        if (a.stats != nullptr && part == 0 && row_tile == 0)
            mark_not_computed(a.stats, rows, seq, a.sequences, a.tokens, a.max_queries, a.heads, kv_head * group, group);
    };
    const uint32_t row0 = row_tile * kRows, all_rows = min(static_cast<uint32_t>(rows.n), a.max_queries) * group;
    if (row0 >= all_rows) return mark();
    const uint32_t here = min(all_rows - row0, static_cast<uint32_t>(kRows));
    const int most_length = static_cast<int>(a.table_blocks * kBlockTokens);
    const int length = min(max(scalar_load(a.lengths + seq), 0), most_length);
    const int shift = length - rows.n;  // position of the first query; below 0: it sees nothing
    const int first_token = static_cast<int>(row0 / group), last_token = static_cast<int>((row0 + here - 1) / group);
    // Blocks that any of the rows sees: [b0, b1)
    const int last_seen = shift + last_token;
    const int first_seen = a.window ? max(0, shift + first_token - static_cast<int>(a.window) + 1) : 0;
    const int start = first_seen / static_cast<int>(kBlockTokens);
    const int b0 = start + static_cast<int>(part * a.chunk);
    const int end = (last_seen + 1 + 31) / static_cast<int>(kBlockTokens);
    const int b1 = part + 1 == a.parts ? end : min(b0 + static_cast<int>(a.chunk), end);  // the last part: all that is left

    // Queries: the lane's row of each tile, and its position.
    f16x8 qf[NT][C];
    int pos[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        const uint32_t r = min(row0 + 16 * t + n, all_rows - 1);  // rows past the last are not written
        const uint32_t token = r / group, head = kv_head * group + r % group;
        pos[t] = shift + static_cast<int>(token);
        const _Float16* q = a.q + static_cast<uint64_t>(rows.at + token) * a.q_stride +
                            static_cast<uint64_t>(head) * a.head_dim;
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const uint32_t d = 32 * c + 8 * g;
            u32x4 v = {0, 0, 0, 0};
            if (d < a.head_dim) v = *reinterpret_cast<const u32x4_a2*>(q + d);
            qf[t][c] = __builtin_bit_cast(f16x8, v);
        }
    }

    const f32x4 zero = {0.0f, 0.0f, 0.0f, 0.0f};
    f32x4 o[NT][2 * C];
    float m[NT], l[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        m[t] = -infinity();
        l[t] = 0.0f;
#pragma unroll
        for (int i = 0; i < 2 * C; ++i) o[t][i] = zero;
    }

    const int32_t* table = a.table + static_cast<uint64_t>(seq) * a.table_blocks;
    constexpr uint32_t kPlane = 1024 * C;
    const uint32_t seen = a.window ? a.window : 0x80000000u;  // a row sees tokens (pos - seen, pos]
    // A block's numbers are read two blocks ahead; its keys are on their way from
    // where the last block's have been used, its values likewise, in the same registers.
    struct Place {
        const uint8_t* planes;
        float key_scale, value_scale;
        bool there;
    };
    const auto number = [&](int b) { return b < b1 ? scalar_load(table + b) : -1; };
    const auto place_of = [&](int32_t block) {
        Place f;
        f.there = block >= 0 && static_cast<uint32_t>(block) < a.cache_blocks;
        const uint64_t at = static_cast<uint64_t>(f.there ? block : 0) * a.kv_heads + kv_head;
        f.planes = a.cache + at * (2 * kPlane) + lane * 16;
        f.key_scale = scalar_load(a.scales + at * 2);
        f.value_scale = scalar_load(a.scales + at * 2 + 1);
        return f;
    };
    u32x4 kb[C], vb[C];
    const auto load = [&](u32x4 (&to)[C], const uint8_t* from) {
#pragma unroll
        for (int c = 0; c < C; ++c) to[c] = *reinterpret_cast<const u32x4*>(from + 1024 * c);
    };
    int b = b0 + static_cast<int>(wave);
    if (a.cache_blocks == 0) b = b1;  // nothing to point at
    int32_t next = number(b + WAVES);
    Place f{}, ahead{};
    if (b < b1) {
        f = place_of(number(b));
        load(kb, f.planes);
        load(vb, f.planes + kPlane);
    }
    for (; b < b1; b += WAVES) {
        const bool more_to_come = b + WAVES < b1;
        if (more_to_come) ahead = place_of(next);
        next = number(b + 2 * WAVES);
        f32x4 s[NT][2];
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const f16x8 k0 = values_of(kb[c][0], kb[c][1]), k1 = values_of(kb[c][2], kb[c][3]);
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                s[t][0] = mfma16(k0, qf[t][c], c == 0 ? zero : s[t][0]);
                s[t][1] = mfma16(k1, qf[t][c], c == 0 ? zero : s[t][1]);
            }
        }
        if (more_to_come) load(kb, ahead.planes);
        const int j0 = b * static_cast<int>(kBlockTokens);
        const bool edge = !f.there || j0 + 31 > shift + first_token ||
                          (a.window && j0 <= last_seen - static_cast<int>(a.window));
        // The values' scale joins the exponent, 2^(x + log2 s), so that the products
        // of all blocks add up in one sum; the weights' sum is divided by it again.
        // A scale of zero counts as one too small to show.
        const float factor = f.key_scale * a.exponent;
        const float scale = f.value_scale < kLeastScale ? kLeastScale : f.value_scale;
        const float more = __builtin_amdgcn_logf(scale);
        const float less = scale == scale ? __builtin_amdgcn_rcpf(scale) : 1.0f;
        f16x8 p[NT];
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            float x[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = __builtin_fmaf(s[t][i >> 2][i & 3], factor, more);
            if (edge) {
                const int from_last = (f.there ? pos[t] : -static_cast<int>(kMostTokens)) - j0 - 4 * g;
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if (static_cast<uint32_t>(from_last - (16 * (i >> 2) + (i & 3))) >= seen) x[i] = -infinity();
            }
            float top = fmaxf(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])), fmaxf(fmaxf(x[4], x[5]), fmaxf(x[6], x[7])));
            top = max_of(across_halves(max_of(across_rows16(top))));
            if (wave_any(top - m[t] > kReach)) {
                const float to = reference(m[t], top);
                const float w = m[t] == to ? 1.0f : exp2_fast(m[t] - to);  // also where both are -inf
                m[t] = to;
                l[t] *= w;
#pragma unroll
                for (int i = 0; i < 2 * C; ++i) o[t][i] *= w;
            }
            const float base = m[t] == -infinity() ? 0.0f : m[t];
            float sum = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float e = exp2_fast(x[i] - base);
                sum += e;
                p[t][i] = static_cast<_Float16>(e);
            }
            l[t] = __builtin_fmaf(sum, less, l[t]);
        }
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const f16x8 v0 = values_of(vb[c][0], vb[c][1]), v1 = values_of(vb[c][2], vb[c][3]);
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                o[t][2 * c] = mfma16(v0, p[t], o[t][2 * c]);
                o[t][2 * c + 1] = mfma16(v1, p[t], o[t][2 * c + 1]);
            }
        }
        if (more_to_come) load(vb, ahead.planes + kPlane);
        f = ahead;
    }

    // The waves' sums join, a few dimension groups at a time.
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        const float all = sum_of(across_halves(sum_of(across_rows16(l[t]))));
        if (g == 0) stats_of[wave][16 * t + n] = float2{m[t], all};
    }
    const uint64_t part_row = static_cast<uint64_t>(part) * a.tokens * a.heads;
    constexpr int kPieces = 4 * kJoin;  // of eight dimensions, a row
    const uint32_t row = threadIdx.x / kPieces, piece = threadIdx.x % kPieces;
    const uint32_t r = row0 + row, token = r / group, head = kv_head * group + r % group;
#pragma unroll
    for (int c0 = 0; c0 < C; c0 += kJoin) {
        if (c0 != 0) __syncthreads();
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int i = 0; i < 2 * kJoin; ++i)
                if (c0 * 2 + i < 2 * C)
                    *reinterpret_cast<f32x4*>(&sums_of[wave][16 * t + n][16 * i + 4 * g]) = o[t][c0 * 2 + i];
        __syncthreads();
        const uint32_t d = 32 * c0 + 8 * piece;
        if (row >= here || d >= a.head_dim) continue;
        float top = -infinity();
#pragma unroll
        for (int w = 0; w < WAVES; ++w) top = fmaxf(top, stats_of[w][row].x);
        f32x4 lo = {0.0f, 0.0f, 0.0f, 0.0f}, hi = lo;
        float sum = 0.0f;
#pragma unroll
        for (int w = 0; w < WAVES; ++w) {
            const float2 ml = stats_of[w][row];
            const float weight = ml.x == -infinity() ? ml.y : exp2_fast(ml.x - top);  // saw nothing: 0, or NaN
            sum = __builtin_fmaf(weight, ml.y, sum);
            lo += weight * *reinterpret_cast<const f32x4*>(&sums_of[w][row][8 * piece]);
            hi += weight * *reinterpret_cast<const f32x4*>(&sums_of[w][row][8 * piece + 4]);
        }
        if (a.stats == nullptr) {
            const float inv = sum != 0.0f ? 1.0f / sum : 0.0f;
            lo *= inv;
            hi *= inv;
            const f16x8 y = {static_cast<_Float16>(lo.x), static_cast<_Float16>(lo.y), static_cast<_Float16>(lo.z),
                             static_cast<_Float16>(lo.w), static_cast<_Float16>(hi.x), static_cast<_Float16>(hi.y),
                             static_cast<_Float16>(hi.z), static_cast<_Float16>(hi.w)};
            _Float16* out = a.output + static_cast<uint64_t>(rows.at + token) * a.out_stride +
                            static_cast<uint64_t>(head) * a.head_dim + d;
            *reinterpret_cast<u32x4_a2*>(out) = __builtin_bit_cast(u32x4, y);
        } else {
            const uint64_t at = part_row + static_cast<uint64_t>(rows.at + token) * a.heads + head;
            if (d == 0) a.stats[at] = float2{top, sum};
            if (sum == 0.0f) continue;  // saw nothing: not read
            float* out = a.sums + at * a.head_dim + d;
            *reinterpret_cast<f32x4*>(out) = lo;
            *reinterpret_cast<f32x4*>(out + 4) = hi;
        }
    }
    mark();
}

// Many rows: 128 of a (sequence, key head), 32 a wave, over tiles of two blocks
// that the four waves share through LDS as binary16, each byte converted once for
// all rows.  As in the prompts' kernel S^T = K Q^T and O^T = V^T P^T run on the
// 32 x 32 x 16 instruction; the planes' order makes both operands of a lane 16
// consecutive bytes of LDS, key row 16 c + 8 b + 4 h + r of a tile being token
// 16 b + 8 c + 4 h + r of the block.  512 queries of 32 heads over 8192 tokens of 8
// key heads of 128: 91 to 95 us, 700 to 730 TFLOP/s (in 16-row tiles 243), 10 of them the
// join of four parts; matrix cores busy 38 % and vector ALUs 51 % of the cycles.  (The next
// tile's scores under this one's weights, with two tiles' in registers: 99.)
// CT: 32-dimension groups there is room for.
constexpr uint32_t kTileRows = 128;

template <int CT>
__global__ __launch_bounds__(256, CT <= 4 ? 2 : 1) void cache_tiles_kernel(CacheAttentionArgs a) {
    constexpr int KS = 2 * CT;
    constexpr int kPlaneHalfs = 1024 * CT;             // a block's plane as binary16
    constexpr int kTileBytes = 2 * 2 * kPlaneHalfs;    // two blocks of keys, or of values
    constexpr int kLoads = (2 * 64 * CT + 255) / 256;  // 16-byte chunks of a thread in two planes
    __shared__ __align__(1024) uint8_t lds[4 * kTileBytes];  // two of [keys | values]

    uint32_t id = a.first + blockIdx.x;
    const uint32_t kv_head = id % a.kv_heads;
    id /= a.kv_heads;
    const uint32_t part = id % a.parts;
    id /= a.parts;
    const uint32_t row_tile = id % a.row_tiles, seq = id / a.row_tiles;

    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n = lane & 31, h = lane >> 5;
    const uint32_t group = a.heads / a.kv_heads, groups = padded_dim(a.head_dim) / 32;
    Span rows = {static_cast<int>(seq), 1};
    if (a.offsets != nullptr) rows = scalar_span_of(a.offsets, seq, a.tokens);
    if (a.stats != nullptr && part == 0 && row_tile == 0)
        mark_not_computed(a.stats, rows, seq, a.sequences, a.tokens, a.max_queries, a.heads, kv_head * group, group);
    const uint32_t row0 = row_tile * kTileRows, all_rows = min(static_cast<uint32_t>(rows.n), a.max_queries) * group;
    if (row0 >= all_rows) return;
    const int length = min(max(scalar_load(a.lengths + seq), 0), static_cast<int>(a.table_blocks * kBlockTokens));
    const int shift = length - rows.n;  // position of the first query
    const int window = static_cast<int>(a.window);
    const auto position = [&](uint32_t r) { return shift + static_cast<int>(min(r, all_rows - 1) / group); };
    const int last_of_tile = position(row0 + kTileRows - 1);
    const uint32_t wave_row = row0 + 32 * wave, r = wave_row + n;
    const int wave_first = position(wave_row), wave_last = position(wave_row + 31), pos = position(r);

    // Tiles of 64 tokens that any row sees, and this part's.
    const int end = max(last_of_tile + 1, 0);
    const int begin = window ? min(max(position(row0) - window + 1, 0), end) & ~63 : 0;
    const int tiles = (end - begin + 63) / 64;
    const int per_part = (tiles + static_cast<int>(a.parts) - 1) / static_cast<int>(a.parts);
    const int tile0 = static_cast<int>(part) * per_part;
    const int tile1 = a.cache_blocks == 0 ? tile0 : min(tiles, tile0 + per_part);

    const int32_t* const table = a.table + static_cast<uint64_t>(seq) * a.table_blocks;
    const int last_block = (end + 31) / 32 - 1;
    struct Scales {
        float key[2], value[2];
        bool there[2];
    };
    u32x4 raw_k[kLoads], raw_v[kLoads];
    const auto load_tile = [&](int tile) {
        Scales f;
        uint64_t at[2];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const int b = begin / 32 + 2 * tile + t;
            const int32_t block = scalar_load(table + min(b, last_block));
            f.there[t] = b <= last_block && block >= 0 && static_cast<uint32_t>(block) < a.cache_blocks;
            at[t] = static_cast<uint64_t>(f.there[t] ? block : 0) * a.kv_heads + kv_head;
            f.key[t] = scalar_load(a.scales + at[t] * 2);
            f.value[t] = scalar_load(a.scales + at[t] * 2 + 1);
        }
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            const int wave_at = 4 * i + wave, t = wave_at / CT;  // 64 chunks a wave: dimension group wave_at % CT of block t
            const uint32_t c = static_cast<uint32_t>(wave_at % CT);
            raw_k[i] = raw_v[i] = u32x4{0x80808080u, 0x80808080u, 0x80808080u, 0x80808080u};
            if (t < 2 && c < groups) {
                const uint8_t* const from = a.cache + (t ? at[1] : at[0]) * (2048 * groups) + 1024 * c + lane * 16;
                raw_k[i] = *reinterpret_cast<const u32x4*>(from);
                raw_v[i] = *reinterpret_cast<const u32x4*>(from + 1024 * groups);
            }
        }
        return f;
    };
    const auto store_tile = [&](uint8_t* to) {
        const int g = lane >> 4, at = lane & 15;
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            const int wave_at = 4 * i + wave, t = wave_at / CT, c = wave_at % CT;
            if (t >= 2) break;
            // keys: tokens `at` and 16 + at, dimensions 32 c + 8 g ..
            uint8_t* const key = to + ((t * KS + 2 * c + (g >> 1)) * 64 + 32 * (g & 1) + 16 * (at >> 3) + (at & 7)) * 16;
            *reinterpret_cast<f16x8*>(key) = values_of(raw_k[i][0], raw_k[i][1]);
            *reinterpret_cast<f16x8*>(key + 128) = values_of(raw_k[i][2], raw_k[i][3]);
            // values: dimensions 32 c + at and 16 more, tokens 4 g .. and 16 + 4 g ..
            uint8_t* const value = to + kTileBytes + ((t * KS + 2 * c + (g >> 1)) * 64 + 32 * (g & 1) + at) * 16;
            *reinterpret_cast<f16x8*>(value) = values_of(raw_v[i][0], raw_v[i][1]);
            *reinterpret_cast<f16x8*>(value + 256) = values_of(raw_v[i][2], raw_v[i][3]);
        }
    };

    Scales scales{};
    if (tile0 < tile1) scales = load_tile(tile0);
    f16x8 qf[KS];
    const uint32_t valid = min(r, all_rows - 1), token = valid / group, head = kv_head * group + valid % group;
    {
        const _Float16* const q = a.q + static_cast<uint64_t>(rows.at + token) * a.q_stride +
                                  static_cast<uint64_t>(head) * a.head_dim;
#pragma unroll
        for (int i = 0; i < KS; ++i) {
            const uint32_t d = 16 * i + 8 * h;
            u32x4 x = {0, 0, 0, 0};
            if (d < a.head_dim) x = *reinterpret_cast<const u32x4_a2*>(q + d);
            qf[i] = __builtin_bit_cast(f16x8, x);
        }
    }
    if (tile0 < tile1) store_tile(lds);
    RowSums<CT> sums;
    sums.clear();
    const uint32_t seen = window ? a.window : 0x80000000u;  // the row sees tokens (pos - seen, pos]

    for (int tile = tile0; tile < tile1; ++tile) {
        uint8_t* const here = lds + ((tile - tile0) & 1) * 2 * kTileBytes;
        uint8_t* const there = lds + (1 - ((tile - tile0) & 1)) * 2 * kTileBytes;
        __syncthreads();
        const Scales now = scales;
        if (tile + 1 < tile1) scales = load_tile(tile + 1);
        const int j0 = begin + tile * 64;
        if (j0 <= wave_last && !(window && j0 + 63 <= wave_first - window)) {
            f32x16 s[2];
#pragma unroll
            for (int i = 0; i < KS; ++i)
#pragma unroll
                for (int t = 0; t < 2; ++t)
                    s[t] = mfma32(*reinterpret_cast<const f16x8*>(here + ((t * KS + i) * 64 + lane) * 16), qf[i],
                                  i == 0 ? RowSums<CT>::zero() : s[t]);
            // Exponents are s factor + more: see the few rows' kernel for the values' scale.
            float factor[2], more[2], less[2];
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                const float by = now.key[t] * a.exponent, scale = now.value[t] < kLeastScale ? kLeastScale : now.value[t];
                factor[t] = by < kLeastFactor ? kLeastFactor : by;
                more[t] = __builtin_amdgcn_logf(scale);
                less[t] = scale == scale ? __builtin_amdgcn_rcpf(scale) : 1.0f;
                if (!now.there[t] || j0 + 32 * t + 31 > wave_first || (window && j0 + 32 * t <= wave_last - window)) {
                    const int from_last = (now.there[t] ? pos : -static_cast<int>(kMostTokens)) - j0 - 32 * t - 4 * h;
                    bool any = false;
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const int j = 16 * ((i >> 2) & 1) + 8 * (i >> 3) + (i & 3);
                        const bool sees = static_cast<uint32_t>(from_last - j) < seen;
                        any |= sees;
                        s[t][i] = sees ? s[t][i] : -infinity();
                    }
                    if (!any) factor[t] = 1.0f, more[t] = 0.0f;  // whatever the block's scales are
                }
            }
            float top[2];
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                top[t] = s[t][0];
#pragma unroll
                for (int i = 1; i < 16; ++i) top[t] = fmaxf(top[t], s[t][i]);
                top[t] = __builtin_fmaf(top[t], factor[t], more[t]);
            }
            sums.grow_to(max_of(across_halves(fmaxf(top[0], top[1]))));
            const float base = sums.base();
            if (sums.large) {
#pragma unroll
                for (int t = 0; t < 2; ++t) {
#pragma unroll
                    for (int i = 0; i < 16; ++i) s[t][i] = __builtin_fmaf(s[t][i], factor[t], more[t]);
                    factor[t] = 1.0f, more[t] = 0.0f;
                }
            }
            f16x8 p[4];
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                const float add = more[t] - base;
                float sum = 0.0f;
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const float e = exp2_fast(__builtin_fmaf(s[t][i], factor[t], add));
                    sum += e;
                    p[2 * t + (i >> 3)][i & 7] = static_cast<_Float16>(e);
                }
                sums.l = __builtin_fmaf(sum, less[t], sums.l);
            }
#pragma unroll
            for (int c = 0; c < 4; ++c)
#pragma unroll
                for (int i = 0; i < CT; ++i)
                    sums.o[i] = mfma32(*reinterpret_cast<const f16x8*>(here + kTileBytes +
                                                                       (((c >> 1) * KS + 2 * i + (c & 1)) * 64 + lane) * 16),
                                       p[c], sums.o[i]);
        }
        if (tile + 1 < tile1) store_tile(there);
    }
    if (a.stats == nullptr) {
        __syncthreads();  // no tile is read any more
        sums.template write<false>(lds + wave * (2048 * CT), a.head_dim, [&](int i) -> _Float16* {
            const uint32_t row = wave_row + i;
            if (row >= all_rows) return nullptr;
            return a.output + static_cast<uint64_t>(rows.at + row / group) * a.out_stride +
                   static_cast<uint64_t>(kv_head * group + row % group) * a.head_dim;
        });
    } else if (r < all_rows) {
        const uint64_t all = static_cast<uint64_t>(a.tokens) * a.heads;
        sums.template write_part<false>(a.stats, a.sums,
                                        part * all + static_cast<uint64_t>(rows.at + token) * a.heads + head, a.head_dim);
    }
}

struct CachePlan {
    uint32_t row_tiles, tile_rows, chunk, parts, waves;
};

CachePlan plan_cache_attention(uint64_t sequences, uint64_t max_queries, uint64_t max_context, uint64_t heads,
                               uint64_t kv_heads, uint64_t head_dim) {
    const uint64_t rows = max_queries * (heads / kv_heads);
    CachePlan p{};
    // Two small tiles that read the blocks twice, from cache, beat one of twice the
    // rows, whose registers leave room for few waves: heads of 128, 16 sequences of
    // 8000 tokens, 20 rows 52 us on 16-row tiles and 57 on one of 32; 48 rows 84 on
    // 16, 75 on 32, 98 on one of 64 and 105 on one of 128; 80 rows 116, 107 and (128)
    // 111; 120 rows 157, 123 and 116.  Heads of 256, 3000 tokens, 64 rows: 74 on 16, 84 on 128.
    p.tile_rows = rows <= 32 || (head_dim > 128 && rows <= 64) ? 16 : rows <= 96 && head_dim <= 128 ? 32 : kTileRows;
    p.row_tiles = static_cast<uint32_t>((rows + p.tile_rows - 1) / p.tile_rows);
    const uint64_t groups = sequences * p.row_tiles * kv_heads;
    if (p.tile_rows == kTileRows) {
        p.waves = 4;
        p.parts = choose_parts(groups, (max_context + 63) / 64 + 1, sequences * max_queries * heads, head_dim, 1.8, 2.2);
        return p;
    }
    // Sixteen waves to a compute unit, none with less than one block (of sixteen) or
    // two (of four).  Contexts of up to three blocks for each of sixteen waves stay in
    // one launch: 600 tokens 6.9 us against 9.8 in parts, 1500 tokens 10.0 both ways.
    p.waves = static_cast<uint32_t>(waves_of(static_cast<int>(padded_dim(static_cast<uint32_t>(head_dim)) / 32),
                                             static_cast<int>(p.tile_rows / 16)));
    const uint64_t blocks = (max_context + kBlockTokens - 1) / kBlockTokens + 1;
    const uint64_t wanted = p.waves == 16 ? 256 : 1024, least = p.waves == 16 ? 16 : 8;
    uint64_t parts = groups >= wanted || (p.waves == 16 && blocks <= 48) ? 1 : (wanted + groups - 1) / groups;
    if (parts > kMostParts) parts = kMostParts;
    uint64_t chunk = (blocks + parts - 1) / parts;
    if (chunk < least) chunk = least;
    p.chunk = static_cast<uint32_t>(chunk);
    p.parts = static_cast<uint32_t>((blocks + chunk - 1) / chunk);
    return p;
}

auto kernel_of(uint32_t tile_rows, uint32_t c) -> void (*)(CacheAttentionArgs) {
    if (tile_rows == 16) switch (c) {
        case 1: return cache_attention_kernel<1, 1>;
        case 2: return cache_attention_kernel<2, 1>;
        case 3: return cache_attention_kernel<3, 1>;
        case 4: return cache_attention_kernel<4, 1>;
        case 5: return cache_attention_kernel<5, 1>;
        case 6: return cache_attention_kernel<6, 1>;
        case 7: return cache_attention_kernel<7, 1>;
        default: return cache_attention_kernel<8, 1>;
    }
    if (tile_rows == 32) switch (c) {
        case 1: return cache_attention_kernel<1, 2>;
        case 2: return cache_attention_kernel<2, 2>;
        case 3: return cache_attention_kernel<3, 2>;
        default: return cache_attention_kernel<4, 2>;
    }
    switch (c) {
        case 1:
        case 2: return cache_tiles_kernel<2>;
        case 3: return cache_tiles_kernel<3>;
        case 4: return cache_tiles_kernel<4>;
        case 5:
        case 6: return cache_tiles_kernel<6>;
        default: return cache_tiles_kernel<8>;
    }
}

bool bad_shape(uint64_t sequences, uint64_t query_tokens, uint64_t max_queries, uint64_t max_context, uint64_t heads,
               uint64_t kv_heads, uint64_t head_dim) {
    if (head_dim % 8 != 0 || head_dim > kMostHeadDim || heads > 65535 || kv_heads > heads) return true;
    if (heads != 0 && (kv_heads == 0 || heads % kv_heads != 0)) return true;
    return query_tokens > kMostTokens || sequences > kMostTokens || max_queries > kMostTokens ||
           max_context > kMostTokens || query_tokens * heads > 0xFFFFFFFFull || max_queries * heads > 0x7FFFFFFFull;
}

}  // namespace
}  // namespace mote::attention

MOTE_EXPORT int mote_hip_cache_attention_workspace(uint64_t sequences, uint64_t query_tokens, uint64_t max_queries,
                                                  uint64_t max_context, uint64_t q_heads, uint64_t kv_heads,
                                                  uint64_t head_dim, size_t* bytes) noexcept {
    using namespace mote::attention;
    if (!bytes) return kInvalid;
    *bytes = 0;
    if (bad_shape(sequences, query_tokens, max_queries, max_context, q_heads, kv_heads, head_dim)) return kInvalid;
    if (sequences == 0 || query_tokens == 0 || max_queries == 0 || q_heads == 0 || head_dim == 0) return 0;
    const CachePlan p = plan_cache_attention(sequences, max_queries, max_context, q_heads, kv_heads, head_dim);
    *bytes = static_cast<size_t>(parts_bytes(query_tokens * q_heads, p.parts, head_dim));
    return 0;
}

MOTE_EXPORT int mote_hip_cache_attention_q8_f16(const void* q, const void* cache, const void* scales,
                                               const void* query_offsets, const void* lengths,
                                               const void* block_table, void* output, uint64_t sequences,
                                               uint64_t query_tokens, uint64_t max_queries, uint64_t max_context,
                                               uint64_t q_heads, uint64_t kv_heads, uint64_t head_dim,
                                               uint64_t q_stride, uint64_t output_stride, uint64_t table_blocks,
                                               uint64_t cache_blocks, float scale, uint64_t window, void* workspace,
                                               size_t workspace_bytes, void* stream) noexcept {
    using namespace mote::attention;
    if (!q || !cache || !scales || !lengths || !block_table || !output || !stream) return kInvalid;
    if (bad_shape(sequences, query_tokens, max_queries, max_context, q_heads, kv_heads, head_dim)) return kInvalid;
    const float exponent = scale * kLog2e;
    if (!(scale > 0.0f) || !std::isfinite(exponent)) return kInvalid;
    if (table_blocks > kMostTokens / kBlockTokens || cache_blocks > 0x7FFFFFFFu) return kInvalid;
    if (!query_offsets && (query_tokens != sequences || max_queries > 1)) return kInvalid;
    if (output_stride < q_heads * head_dim) return kInvalid;
    if (odd_address(q) || odd_address(output) || off_grid(cache, 16) || off_grid(scales, 4) ||
        off_grid(query_offsets, 4) || off_grid(lengths, 4) || off_grid(block_table, 4))
        return kInvalid;
    if (sequences == 0 || query_tokens == 0 || max_queries == 0 || q_heads == 0 || head_dim == 0) return 0;
    const CachePlan p = plan_cache_attention(sequences, max_queries, max_context, q_heads, kv_heads, head_dim);
    const uint64_t rows = query_tokens * q_heads;
    const uint64_t need = parts_bytes(rows, p.parts, head_dim);
    if (need > 0 && (!workspace || off_grid(workspace, 16) || workspace_bytes < need)) return kInvalid;
    if (sequences * p.row_tiles > 0xFFFFFFFFu / kv_heads / p.parts) return kInvalid;  // workgroups: 32 bits
    CacheAttentionArgs a{};
    a.q = static_cast<const _Float16*>(q);
    a.cache = static_cast<const uint8_t*>(cache);
    a.scales = static_cast<const float*>(scales);
    a.offsets = static_cast<const int32_t*>(query_offsets);
    a.lengths = static_cast<const int32_t*>(lengths);
    a.table = static_cast<const int32_t*>(block_table);
    a.output = static_cast<_Float16*>(output);
    if (p.parts > 1) {
        a.stats = static_cast<float2*>(workspace);
        a.sums = reinterpret_cast<float*>(static_cast<char*>(workspace) + stats_bytes(rows, p.parts));
    }
    a.q_stride = q_stride;
    a.out_stride = output_stride;
    a.sequences = static_cast<uint32_t>(sequences);
    a.tokens = static_cast<uint32_t>(query_tokens);
    a.max_queries = static_cast<uint32_t>(max_queries);
    a.row_tiles = p.row_tiles;
    a.heads = static_cast<uint32_t>(q_heads);
    a.kv_heads = static_cast<uint32_t>(kv_heads);
    a.head_dim = static_cast<uint32_t>(head_dim);
    a.table_blocks = static_cast<uint32_t>(table_blocks);
    a.cache_blocks = static_cast<uint32_t>(cache_blocks);
    a.window = window >= table_blocks * kBlockTokens ? 0 : static_cast<uint32_t>(window);  // no shorter than any context
    a.chunk = p.chunk;
    a.parts = p.parts;
    a.exponent = exponent;
    const auto kernel = kernel_of(p.tile_rows, padded_dim(a.head_dim) / 32);
    const auto s = static_cast<hipStream_t>(stream);
    const uint64_t groups = sequences * p.row_tiles * kv_heads * p.parts, most = most_groups(64 * p.waves);
    for (uint64_t first = 0; first < groups; first += most) {
        a.first = static_cast<uint32_t>(first);
        const uint64_t now = groups - first < most ? groups - first : most;
        hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(now)), dim3(64 * p.waves), 0, s, a);
        const int status = static_cast<int>(hipGetLastError());
        if (status != 0) return status;
    }
    if (p.parts <= 1) return 0;
    return join_parts(workspace, output, rows, p.parts, q_heads, head_dim, output_stride, s);
}
