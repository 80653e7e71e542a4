// Attention of packed prompts: sequences of different lengths one behind the
// other, grouped heads, causal or not, with or without a sliding window, over
// binary16 keys and values.
//
// A workgroup takes 128 query rows of one head, 32 a wave, and walks the keys
// they see in tiles of 64 or 32 that the four waves share through LDS.  S^T = K Q^T
// and O^T = V^T P^T on the 32 x 32 x 16 matrix instruction: with keys as the
// instruction's rows a lane ends with the scores of one query row, the running
// maximum and sum need one exchange between the wave's halves, and the scores
// are the operand of the second product where they lie.  Its other operand,
// V^T, comes out of the row-major tile through LDS transpose reads.
//
// 64 x 32 scores of 128 dimensions are 32 matrix instructions (1024 cycles) and
// about 150 vector instructions, a fifth of them exponentials (1050 cycles); the
// workgroups of a compute unit run the one under the other.  1 x 8192 tokens, 32 heads
// of 128, causal: 557 to 590 us by the card, 930 to 990 TFLOP/s (a large library
// product: 1310 to 1325).  Power bounds it: the matrix cores are busy 60 % of the cycles,
// of which the card gives 1.5 GHz over the launch (1.9 in light ones).  Short prompts wait
// for their starts: 6300 cycles before a workgroup's first product, 24 prompts of up to
// 1000 tokens 123 to 128 us, 530 to 550 TFLOP/s.
#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdint>
#include <type_traits>

#include "attention_sums.hpp"
#include "tile_ops.hpp"

namespace mote::attention {
namespace {

constexpr uint32_t kTileRows = 128;

struct PromptArgs {
    const _Float16* q;
    const _Float16* k;
    const _Float16* v;
    _Float16* output;
    const int32_t* query_offsets;
    const int32_t* key_offsets;
    float2* stats;  // null: one part, written to output
    float* sums;
    uint64_t q_stride, k_stride, v_stride, out_stride;
    uint32_t sequences, tokens, keys, heads, kv_heads, head_dim, window, causal, parts, first;
    float exponent;  // scale log2(e)
};

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4* lds_s16x4;

// Four rows by sixteen columns of a row-major binary16 tile, transposed: lane i
// of each sixteen gives the address of piece i % 4 of row i / 4 and gets column i.
__device__ __forceinline__ u32x2 read_transposed(const uint8_t* at) {
    return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)(at)));
}

// Position of 16-byte chunk c of row r in a tile of CH chunks a row: chunks of a
// row are exchanged within aligned groups of G, a power of two, so that what is read
// together lies in different banks, of which 16 chunks fill all: conflicts are 0.8 %
// of the LDS cycles for 8192 tokens (a third with c ^ r for keys and c ^ 2 r for
// values), 7 % for 24 packed prompts, 5 % for windows of 512 with heads of 64.
// 16 / G neighbouring rows differ by their place alone.
template <int CH>
struct Swizzle {
    static constexpr int G = (CH & -CH) > 16 ? 16 : (CH & -CH);
    // Keys: chunks c and c + 1 of any 8 neighbouring rows, and c of any 16.
    static __device__ __forceinline__ int key(int r, int c) {
        const int q = r / (16 / G);
        return r * CH + (c ^ ((q * 2) % G | (q / (G / 2)) % 2));
    }
    // Values: four chunks of any 4 neighbouring rows.
    static __device__ __forceinline__ int value(int r, int c) { return r * CH + (c ^ (4 * (r / (16 / G)) % G)); }
};

// The pair with halves that are not finite replaced by zero.
__device__ __forceinline__ uint32_t finite_of(uint32_t pair) {
    uint32_t r = pair;
    if ((pair & 0x7C00u) == 0x7C00u) r &= 0xFFFF0000u;
    if ((pair & 0x7C000000u) == 0x7C000000u) r &= 0x0000FFFFu;
    return r;
}

// DP: the padded head size.  DIRECT: rows and addresses on the 16-byte grid and
// head_dim = DP, so tiles go from memory to LDS without passing registers.  (Heads
// of 64: four workgroups a compute unit, for which three registers go to scratch, 95
// us for windows of 512 against 98 with the three that fit without the bound.)
//
// KEYS: of a tile.  Tiles of 32 keys leave room for three workgroups of 128
// dimensions a compute unit, which cover each other's starts where there are many:
// 64 prompts of 64 tokens 25 us against 30, of 256 92 against 103, 24 of up to 1000
// 122 against 129, 8192 tokens level; with few workgroups tiles of 64 have the
// fewer turns: 1024 tokens 26 against 32, 333 queries over 7333 keys 62 against 65.
template <int DP, bool DIRECT, int KEYS>
__global__ __launch_bounds__(256, DIRECT && DP == 64 ? 4 : KEYS == 32 ? 3 : DP <= 128 ? 2 : 1) void
prompt_attention_kernel(PromptArgs a) {
    constexpr int CH = DP / 8, KS = DP / 16, DT = DP / 32;
    constexpr int kLoads = KEYS * CH / 256;       // 16-byte chunks of a thread in each tile
    constexpr int kTileBytes = KEYS * CH * 16;
    __shared__ __align__(1024) uint8_t lds[4 * kTileBytes];  // two of [keys | values]
    __shared__ int not_finite;  // a wave's sums are not
    __shared__ int taken_out;   // the last tile, from 1, with values that are not finite taken out

    // Key heads first, so that with eight of them each XCD's L2 keeps one; then the
    // query heads that share them; then the tiles.
    const uint32_t kv_head = blockIdx.x;
    const uint32_t head = kv_head * gridDim.y + blockIdx.y;
    Span queries, keys;  // first of the lane's sequence, then of the workgroup's
    const uint32_t z = a.first + blockIdx.z;
    const uint32_t part = a.parts == 1 ? 0 : z % a.parts;
    const Unit u = locate<kTileRows, 1>(a.parts == 1 ? z : z / a.parts, a.query_offsets, a.sequences, a.tokens,
                                        [&](uint32_t s) {
                                            queries = span_of(a.query_offsets, s, a.tokens);
                                            keys = span_of(a.key_offsets, s, a.keys);
                                        });
    if (!u.found) return;
    queries = span_at(queries, u.lane);
    keys = span_at(keys, u.lane);
    if (a.stats != nullptr && part == 0 && u.local == 0)
        mark_not_computed(a.stats, queries, u.sequence, a.sequences, a.tokens, a.tokens, a.heads, head, 1);
    const uint32_t row_tiles = (static_cast<uint32_t>(queries.n) + kTileRows - 1) / kTileRows;
    if (u.local >= row_tiles) return;  // room that the sequence does not need
    const int row0 = static_cast<int>((row_tiles - 1 - u.local) * kTileRows);  // the longest walks first
    const int shift = keys.n - queries.n;  // position of the first query
    const int last_row = min(row0 + static_cast<int>(kTileRows), queries.n) - 1;
    const int window = static_cast<int>(a.window);

    // The keys that any row of the tile sees, and this part's tiles of them.
    const int end = a.causal ? min(max(last_row + shift + 1, 0), keys.n) : keys.n;
    const int begin = window ? min(max(row0 + shift - window + 1, 0), end) & ~(KEYS - 1) : 0;
    const int tiles = (end - begin + KEYS - 1) / KEYS;
    const int per_part = (tiles + static_cast<int>(a.parts) - 1) / static_cast<int>(a.parts);
    const int tile0 = static_cast<int>(part) * per_part, tile1 = min(tiles, tile0 + per_part);

    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n = lane & 31, h = lane >> 5;
    const int wave_row = row0 + 32 * wave;
    const int row = wave_row + n;
    const int pos = row + shift;
    // The row sees keys (last_seen - seen, last_seen].
    const int last_seen = a.causal ? pos : keys.n - 1;
    const uint32_t seen = window ? a.window : 0x80000000u;
    const int wave_last = min(wave_row + 31, queries.n - 1) + shift;  // position of the wave's last row

    const _Float16* const k = a.k + static_cast<uint64_t>(keys.at) * a.k_stride + static_cast<uint64_t>(kv_head) * a.head_dim;
    const _Float16* const v = a.v + static_cast<uint64_t>(keys.at) * a.v_stride + static_cast<uint64_t>(kv_head) * a.head_dim;

    // Chunk i of a thread lies at position 256 i + thread of a tile.
    u32x4 next_k[DIRECT ? 1 : kLoads], next_v[DIRECT ? 1 : kLoads];
    uint32_t source_k[kLoads], source_v[kLoads];  // DIRECT: their bytes from the tile's first row
    const auto set_source = [&](int i, int last) {
        const int at = static_cast<int>(threadIdx.x) + 256 * i, r = at / CH, c = at % CH;
        const uint32_t from = static_cast<uint32_t>(min(r, last));
        source_k[i] = (from * static_cast<uint32_t>(a.k_stride) + 8 * (Swizzle<CH>::key(r, c) - r * CH)) * 2;
        source_v[i] = (from * static_cast<uint32_t>(a.v_stride) + 8 * (Swizzle<CH>::value(r, c) - r * CH)) * 2;
    };
    if constexpr (DIRECT) {
#pragma unroll
        for (int i = 0; i < kLoads; ++i) set_source(i, KEYS - 1);
    }
    const auto load_tile = [&](int tile, uint8_t* to) {
        const int j0 = begin + tile * KEYS;
        if constexpr (DIRECT) {
            const Buffer kb = buffer_at(k + static_cast<uint64_t>(j0) * a.k_stride);
            const Buffer vb = buffer_at(v + static_cast<uint64_t>(j0) * a.v_stride);
            const int last = keys.n - 1 - j0;
            if (last < KEYS - 1) {  // rows past the last repeat it; no row sees them
#pragma unroll
                for (int i = 0; i < kLoads; ++i) set_source(i, last);
            }
#pragma unroll
            for (int i = 0; i < kLoads; ++i) {
                uint8_t* const dst = to + (256 * i + 64 * wave) * 16;
                load_lds16(kb, source_k[i], 0, dst);
                load_lds16(vb, source_v[i], 0, dst + kTileBytes);
            }
        } else {
#pragma unroll
            for (int i = 0; i < kLoads; ++i) {
                const int at = static_cast<int>(threadIdx.x) + 256 * i, r = at / CH, c = at % CH;
                next_k[i] = next_v[i] = u32x4{0, 0, 0, 0};
                if (j0 + r < keys.n && 8u * c < a.head_dim) {
                    next_k[i] = *reinterpret_cast<const u32x4_a2*>(k + static_cast<uint64_t>(j0 + r) * a.k_stride + 8 * c);
                    next_v[i] = *reinterpret_cast<const u32x4_a2*>(v + static_cast<uint64_t>(j0 + r) * a.v_stride + 8 * c);
                }
            }
        }
    };
    const auto store_tile = [&](uint8_t* to) {  // what load_tile left in registers
        if constexpr (!DIRECT) {
#pragma unroll
            for (int i = 0; i < kLoads; ++i) {
                const int at = static_cast<int>(threadIdx.x) + 256 * i, r = at / CH, c = at % CH;
                *reinterpret_cast<u32x4*>(to + Swizzle<CH>::key(r, c) * 16) = next_k[i];
                *reinterpret_cast<u32x4*>(to + kTileBytes + Swizzle<CH>::value(r, c) * 16) = next_v[i];
            }
        }
    };

    if (threadIdx.x == 0) not_finite = taken_out = 0;
    if (tile0 < tile1) {
        load_tile(tile0, lds);
        store_tile(lds);
    }

    f16x8 qf[KS];
    {
        const _Float16* q = a.q + static_cast<uint64_t>(queries.at + min(row, queries.n - 1)) * a.q_stride +
                            static_cast<uint64_t>(head) * a.head_dim;
#pragma unroll
        for (int i = 0; i < KS; ++i) {
            const uint32_t d = 16 * i + 8 * h;
            u32x4 x = {0, 0, 0, 0};
            if (DIRECT || d < a.head_dim) x = *reinterpret_cast<const u32x4_a2*>(q + d);
            qf[i] = __builtin_bit_cast(f16x8, x);
        }
    }

    RowSums<DT> sums;
    sums.clear();

    // Lane addresses in a tile: of its key's chunks, of its piece of the values.
    uint32_t key_at[KS], value_at[DT];
#pragma unroll
    for (int i = 0; i < KS; ++i) key_at[i] = Swizzle<CH>::key(n, 2 * i + h) * 16;
#pragma unroll
    for (int i = 0; i < DT; ++i) {
        const int r = 4 * h + ((lane & 15) >> 2), piece = lane & 3;
        const int chunk = 4 * i + 2 * ((lane >> 4) & 1) + (piece >> 1);
        value_at[i] = kTileBytes + Swizzle<CH>::value(r, chunk) * 16 + 8 * (piece & 1);
    }

    // A value that is not finite, in a key that some row of the tile does not see,
    // reaches that row through a weight of zero as NaN.  None is looked for on the
    // way: where sums end up not finite the walk is done again, carefully.  (Looking
    // at each partly seen tile first cost 24 packed prompts 9 of 143 us.)
    const auto walk = [&](auto kind) {
        constexpr bool careful = decltype(kind)::value;
        if (tile0 < tile1) {
            if constexpr (DIRECT && careful) {  // the last tile may have cut them
#pragma unroll
                for (int i = 0; i < kLoads; ++i) set_source(i, KEYS - 1);
            }
            if constexpr (careful) {
                load_tile(tile0, lds);
                store_tile(lds);
            }
        }
        for (int tile = tile0; tile < tile1; ++tile) {
            uint8_t* const here = lds + ((tile - tile0) & 1) * 2 * kTileBytes;
            uint8_t* const there = lds + (1 - ((tile - tile0) & 1)) * 2 * kTileBytes;
            if constexpr (DIRECT) {
                // The tile has come; what this wave read of the last one has arrived,
                // since the others load over it once they are past the barrier.  (Said
                // in assembly: after the builtin the compiler made the first LDS read
                // wait for the loads of the next tile, 8192 tokens 5 % longer.)
                asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
                wait_counts<vm_wait(0)>();
                group_barrier();
                order_fence();
            } else {
                __syncthreads();
            }
            const int j0 = begin + tile * KEYS;
            // Carefully: such values are taken out of tiles that some row of the workgroup
            // does not see all of, and added below to the rows that do.
            if (careful && (j0 + KEYS > keys.n || (a.causal && j0 + KEYS - 1 > row0 + shift) ||
                            (window && j0 <= last_row + shift - window))) {
                bool bad = false;
#pragma unroll
                for (int i = 0; i < kLoads; ++i) {
                    u32x4* const at = reinterpret_cast<u32x4*>(here + kTileBytes) + threadIdx.x + 256 * i;
                    const u32x4 x = *at;
                    u32x4 fine;
#pragma unroll
                    for (int w = 0; w < 4; ++w) fine[w] = finite_of(x[w]);
                    if (fine[0] != x[0] || fine[1] != x[1] || fine[2] != x[2] || fine[3] != x[3]) {
                        *at = fine;
                        bad = true;
                    }
                }
                if (bad) taken_out = tile + 1;
                __syncthreads();
            }
            if (tile + 1 < tile1) load_tile(tile + 1, there);
            if (!(a.causal && (j0 > wave_last || (window && j0 + KEYS - 1 <= wave_row + shift - window)))) {
                // Products that follow each other go to different sums (1 to 5 % over
                // one sum after the other).
                f32x16 s[KEYS / 32];
#pragma unroll
                for (int i = 0; i < KS; ++i)
#pragma unroll
                    for (int t = 0; t < KEYS / 32; ++t)
                        s[t] = mfma32(*reinterpret_cast<const f16x8*>(here + key_at[i] + 32 * CH * 16 * t), qf[i],
                                      i == 0 ? RowSums<DT>::zero() : s[t]);
                if (j0 + KEYS > keys.n || (a.causal && j0 + KEYS - 1 > wave_row + shift) ||
                    (window && j0 <= wave_last - window)) {
                    const int from_last = last_seen - j0 - 4 * h;
#pragma unroll
                    for (int i = 0; i < KEYS / 2; ++i) {
                        const int j = 32 * (i >> 4) + 8 * ((i & 15) >> 2) + (i & 3);
                        if (static_cast<uint32_t>(from_last - j) >= seen) s[i >> 4][i & 15] = -infinity();
                    }
                }
                float top = s[0][0];
#pragma unroll
                for (int i = 1; i < KEYS / 2; ++i) top = fmaxf(top, s[i >> 4][i & 15]);
                sums.grow_to(product(max_of(across_halves(top)), a.exponent));
                const float base = sums.base();
                float exponent = a.exponent;
                if (sums.large) {
                    exponent = 1.0f;
#pragma unroll
                    for (int i = 0; i < KEYS / 2; ++i) s[i >> 4][i & 15] = product(s[i >> 4][i & 15], a.exponent);
                }
                f16x8 p[KEYS / 16];
#pragma unroll
                for (int i = 0; i < KEYS / 2; ++i) {
                    const float e = exp2_fast(__builtin_fmaf(s[i >> 4][i & 15], exponent, -base));
                    sums.l += e;
                    p[i >> 3][i & 7] = static_cast<_Float16>(e);
                }
                // V^T: dimensions 32 i + n, keys 16 c + {4 h .. 4 h + 3, 8 + 4 h ..}.
#pragma unroll
                for (int c = 0; c < KEYS / 16; ++c)
#pragma unroll
                    for (int i = 0; i < DT; ++i) {
                        const uint8_t* at = here + value_at[i] + 16 * CH * 16 * c;
                        const u32x2 lo = read_transposed(at), hi = read_transposed(at + 8 * CH * 16);
                        sums.o[i] = mfma32(__builtin_bit_cast(f16x8, u32x4{lo.x, lo.y, hi.x, hi.y}), p[c], sums.o[i]);
                    }
                if (careful && taken_out == tile + 1) {
#pragma unroll 1
                    for (int j = j0; j < min(j0 + KEYS, keys.n); ++j) {
                        const bool sees = static_cast<uint32_t>(last_seen - j) < seen;
                        const _Float16* at = v + static_cast<uint64_t>(j) * a.v_stride + 4 * h;
#pragma unroll
                        for (int i = 0; i < DT; ++i) {
#pragma unroll
                            for (int r = 0; r < 16; r += 4) {
                                const uint32_t d = 32 * i + 2 * r;
                                if (!DIRECT && d >= a.head_dim) continue;
                                const u32x2 four = *reinterpret_cast<const u32x2_a2*>(at + d);
                                const float x[4] = {half_lo_to_float(four.x), half_hi_to_float(four.x),
                                                    half_lo_to_float(four.y), half_hi_to_float(four.y)};
#pragma unroll
                                for (int e = 0; e < 4; ++e)
                                    sums.o[i][r + e] += sees && !(fabsf(x[e]) < infinity()) ? x[e] : 0.0f;
                            }
                            order_fence();  // rare, and not to be paid for in registers
                        }
                    }
                }
            }
            if (tile + 1 < tile1) store_tile(there);
        }
    };
    walk(std::false_type());
    if (wave_any(!sums.finite())) not_finite = 1;
    __syncthreads();
    if (not_finite) {
        sums.clear();
        walk(std::true_type());
        __syncthreads();
    }

    // No tile is read any more.
    if (a.stats == nullptr) {
        sums.template write<DIRECT>(lds + wave * (64 * DP), a.head_dim, [&](int i) -> _Float16* {
            if (wave_row + i >= queries.n) return nullptr;
            return a.output + static_cast<uint64_t>(queries.at + wave_row + i) * a.out_stride +
                   static_cast<uint64_t>(head) * a.head_dim;
        });
    } else if (row < queries.n) {
        const uint64_t rows = static_cast<uint64_t>(a.tokens) * a.heads;
        sums.template write_part<DIRECT>(a.stats, a.sums,
                                         part * rows + static_cast<uint64_t>(queries.at + row) * a.heads + head,
                                         a.head_dim);
    }
}

struct PromptPlan {
    uint64_t tiles;
    uint32_t parts;
};

PromptPlan plan_prompt(uint64_t sequences, uint64_t tokens, uint64_t max_keys, uint64_t heads, uint64_t head_dim) {
    PromptPlan p{};
    p.tiles = units_of(kTileRows, 1, sequences, tokens);
    p.parts = choose_parts(p.tiles * heads, (max_keys + 63) / 64, tokens * heads, head_dim, 1.4, 2.0);
    return p;
}

bool bad_shape(uint64_t sequences, uint64_t tokens, uint64_t keys, uint64_t max_keys, uint64_t heads,
               uint64_t kv_heads, uint64_t head_dim) {
    if (head_dim % 8 != 0 || head_dim > kMostHeadDim || heads > 65535 || kv_heads > heads) return true;
    if (heads != 0 && (kv_heads == 0 || heads % kv_heads != 0)) return true;
    return tokens > kMostTokens || keys > kMostTokens || max_keys > kMostTokens || sequences > kMostTokens ||
           tokens * heads > 0xFFFFFFFFull;
}

}  // namespace
}  // namespace mote::attention

MOTE_EXPORT int mote_hip_prompt_attention_workspace(uint64_t sequences, uint64_t query_tokens, uint64_t key_tokens,
                                                   uint64_t max_keys, uint64_t q_heads, uint64_t kv_heads,
                                                   uint64_t head_dim, size_t* bytes) noexcept {
    using namespace mote::attention;
    if (!bytes) return kInvalid;
    *bytes = 0;
    if (bad_shape(sequences, query_tokens, key_tokens, max_keys, q_heads, kv_heads, head_dim)) return kInvalid;
    if (sequences == 0 || query_tokens == 0 || q_heads == 0 || head_dim == 0) return 0;
    const PromptPlan p = plan_prompt(sequences, query_tokens, max_keys, q_heads, head_dim);
    *bytes = static_cast<size_t>(parts_bytes(query_tokens * q_heads, p.parts, head_dim));
    return 0;
}

MOTE_EXPORT int mote_hip_prompt_attention_f16(const void* q, const void* k, const void* v, void* output,
                                             const void* query_offsets, const void* key_offsets, uint64_t sequences,
                                             uint64_t query_tokens, uint64_t key_tokens, uint64_t max_keys,
                                             uint64_t q_heads, uint64_t kv_heads, uint64_t head_dim,
                                             uint64_t q_stride, uint64_t k_stride, uint64_t v_stride,
                                             uint64_t output_stride, float scale, int causal, uint64_t window,
                                             void* workspace, size_t workspace_bytes, void* stream) noexcept {
    using namespace mote::attention;
    if (!q || !k || !v || !output || !query_offsets || !stream) return kInvalid;
    if (bad_shape(sequences, query_tokens, key_tokens, max_keys, q_heads, kv_heads, head_dim)) return kInvalid;
    const float exponent = scale * kLog2e;
    if (!(scale > 0.0f) || !std::isfinite(exponent)) return kInvalid;
    if ((causal != 0 && causal != 1) || (!causal && window != 0)) return kInvalid;
    if (!key_offsets && key_tokens != query_tokens) return kInvalid;
    if (output_stride < q_heads * head_dim) return kInvalid;
    if (odd_address(q) || odd_address(k) || odd_address(v) || odd_address(output) || off_grid(query_offsets, 4) ||
        off_grid(key_offsets, 4))
        return kInvalid;
    if (sequences == 0 || query_tokens == 0 || q_heads == 0 || head_dim == 0) return 0;
    const PromptPlan p = plan_prompt(sequences, query_tokens, max_keys, q_heads, head_dim);
    const uint64_t rows = query_tokens * q_heads, need = parts_bytes(rows, p.parts, head_dim);
    if (need > 0 && (!workspace || off_grid(workspace, 16) || workspace_bytes < need)) return kInvalid;
    PromptArgs a{};
    a.q = static_cast<const _Float16*>(q);
    a.k = static_cast<const _Float16*>(k);
    a.v = static_cast<const _Float16*>(v);
    a.output = static_cast<_Float16*>(output);
    a.query_offsets = static_cast<const int32_t*>(query_offsets);
    a.key_offsets = static_cast<const int32_t*>(key_offsets ? key_offsets : query_offsets);
    if (p.parts > 1) {
        a.stats = static_cast<float2*>(workspace);
        a.sums = reinterpret_cast<float*>(static_cast<char*>(workspace) + stats_bytes(rows, p.parts));
    }
    a.q_stride = q_stride;
    a.k_stride = k_stride;
    a.v_stride = v_stride;
    a.out_stride = output_stride;
    a.sequences = static_cast<uint32_t>(sequences);
    a.tokens = static_cast<uint32_t>(query_tokens);
    a.keys = static_cast<uint32_t>(key_tokens);
    a.heads = static_cast<uint32_t>(q_heads);
    a.kv_heads = static_cast<uint32_t>(kv_heads);
    a.head_dim = static_cast<uint32_t>(head_dim);
    a.window = window >= key_tokens ? 0 : static_cast<uint32_t>(window);  // no shorter than any sequence
    a.causal = static_cast<uint32_t>(causal);
    a.parts = p.parts;
    a.exponent = exponent;
    const bool direct = !off_grid(k, 16) && !off_grid(v, 16) && k_stride % 8 == 0 && v_stride % 8 == 0 &&
                        k_stride < (uint64_t{1} << 24) && v_stride < (uint64_t{1} << 24);
    const bool many = p.tiles * q_heads >= 1024;
    const auto kernel = direct && head_dim == 64            ? prompt_attention_kernel<64, true, 64>
                        : direct && head_dim == 96          ? prompt_attention_kernel<96, true, 64>
                        : direct && head_dim == 128 && many ? prompt_attention_kernel<128, true, 32>
                        : direct && head_dim == 128         ? prompt_attention_kernel<128, true, 64>
                        : direct && head_dim == 192         ? prompt_attention_kernel<192, true, 64>
                        : direct && head_dim == 256         ? prompt_attention_kernel<256, true, 64>
                        : head_dim <= 64                    ? prompt_attention_kernel<64, false, 64>
                        : head_dim <= 96                    ? prompt_attention_kernel<96, false, 64>
                        : head_dim <= 128                   ? prompt_attention_kernel<128, false, 64>
                        : head_dim <= 192                   ? prompt_attention_kernel<192, false, 64>
                                                            : prompt_attention_kernel<256, false, 64>;
    const auto s = static_cast<hipStream_t>(stream);
    constexpr uint64_t kMostZ = 65535;
    for (uint64_t first = 0; first < p.tiles * p.parts; first += kMostZ) {
        const uint64_t left = p.tiles * p.parts - first;
        a.first = static_cast<uint32_t>(first);
        hipLaunchKernelGGL(kernel, dim3(a.kv_heads, a.heads / a.kv_heads, static_cast<unsigned>(left < kMostZ ? left : kMostZ)),
                           dim3(256), 0, s, a);
        const int status = static_cast<int>(hipGetLastError());
        if (status != 0) return status;
    }
    if (p.parts <= 1) return 0;
    return join_parts(workspace, output, rows, p.parts, q_heads, head_dim, output_stride, s);
}
