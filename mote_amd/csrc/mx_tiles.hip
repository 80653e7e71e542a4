// Products of many microscaled rows, bound by the matrix cores.
//
// A workgroup has a tile of BN weight rows (gate/up: BN / 2 of each) by BM rows of x. Both
// operands' bytes, 128 elements of K a stage, go from memory straight into a ring of
// stages in LDS: 64 bytes of a row of 4 bits, for x of 6 bits 32 more, and each row's four
// scales.  A wave multiplies 32 x 32 x 64 (half the time of 16 x 16 x 128 a
// product), reading operands as the instruction takes them.  A row's 16-byte pieces lie
// at piece ^ (row / 4 % 4), so 16 lanes that read the same piece of 16 rows touch every
// bank once; but lanes l and l + 32 read neighbouring pieces, and those two of 8 rows fall on 8 of the 16 places,
// two on each: 35 to 40 % of the LDS cycles are conflicts.  One barrier a stage: behind it, all waves' loads of
// the stage have landed and the stage before is free to be loaded again.
//
// What bounds large ones (4096 x 14336 x 4096 in 4 bits, 142 to 151 us from card to card, 3.2 to 3.4 PFLOP/s of the 6.2
// that the instruction reaches on registers alone; each part taken out in turn): the matrix instructions alone some 98 us, in four
// rounds of 3.5 rounds' tiles; the results, which all compute units write at one time, 24; the loads 22, LDS
// reads 13.  Stages of 256 elements, whose loads have pieces of 128 bytes (53 bytes a cycle and compute
// unit in place of 36), were level (152 and 154 us) and slower for experts (130 and 122).
#include <hip/hip_runtime.h>

#include <cstdint>

#include "mx_products.hpp"
#include "tile_ops.hpp"

namespace mote::mx {
namespace {

// D[i][j] += sum over k of W[i][k] X[j][k], 32 x 32 outputs and 64 elements: lane l holds
// block l / 32 of rows l % 32, and of D column j = l % 32, rows i = 8 (r / 4) + 4 (l / 32)
// + r % 4.  SCALE: the byte of the lanes' scale words.
template <int BITS, int SCALE>
__device__ __forceinline__ f32x16 multiply32(i32x8 w, uint32_t w_scale, i32x8 x, uint32_t x_scale,
                                             f32x16 d) {
    return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(w, x, d, kFormat<4>, kFormat<BITS>,
                                                           SCALE, static_cast<int>(w_scale), SCALE,
                                                           static_cast<int>(x_scale));
}

// Between a wave's writes to LDS and its other lanes' reads there.
__device__ __forceinline__ void wave_fence() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4_a2 __attribute__((ext_vector_type(4), aligned(2)));

// The tile of workgroup `at`.  Workgroups go to the 8 XCDs in turn: each gets a run of
// tiles, of BAND row tiles by all columns, columns outside, so that those it
// computes at one time share rows of both operands in its L2.  (Experts have bands of one, as the next
// tile of rows is often another's: 5000 tokens' four of 32 experts of 2880 x 2880, down, 265 us, 284 in
// bands of four.  Linears: 4096 x 28672 x 1024 141 us in bands of one, 136 of four, 131 of eight; 8192 x 4096 x 4096
// 89, 87 and 94.)
struct Place {
    uint32_t unit, column;
};
template <uint32_t BAND>
__device__ __forceinline__ Place place_of(uint32_t at, uint32_t units, uint32_t columns) {
    const uint32_t total = units * columns;
    const uint32_t xcd = at % 8, each = total / 8, more = total % 8;
    const uint32_t t = xcd * each + min(xcd, more) + at / 8;
    const uint32_t band = t / (BAND * columns), in_band = t - band * BAND * columns;
    const uint32_t height = min(BAND, units - band * BAND);
    return {band * BAND + in_band % height, in_band / height};
}

// WN x WM waves divide a tile, or WK waves divide K and add their sums at the end, in their order.
template <int BITS, Result R, int BN, int BM, int WN, int WM, int WK, int STAGES>
__global__ __launch_bounds__(64 * WN * WM * WK) void tiles_kernel(ProductArgs a, uint32_t columns) {
    constexpr int kThreads = 64 * WN * WM * WK;
    constexpr int NF = BN / WN / 32, MF = BM / WM / 32;  // 32 x 32 products of a wave
    constexpr bool kGate = R == Result::kGateUp;
    constexpr int kColumns = kGate ? BN / 2 : BN;  // outputs of a tile
    static_assert(!kGate || NF % 2 == 0, "a wave has a gate and its up");
    // Waves that divide K have a whole tile each, with rings and loads of their own: nothing of theirs
    // meets before the end, so there is no barrier to wait at.
    constexpr bool kAlone = WK > 1;
    static_assert(!kAlone || WN * WM == 1, "waves divide the tile or K");
    constexpr int kLoaders = kAlone ? 64 : kThreads;  // threads that load a stage, a step of K
    // The parts of a stage, and the loads that a thread issues for each.  Where a part has fewer
    // pieces than there are threads, some are loaded twice, to the same place: every wave then
    // waits for the same number.
    constexpr int kW = BN * 64, kX = BM * 64, kHigh = BITS == 6 ? BM * 32 : 0, kStage = kW + kX + kHigh;
    // Scales come four steps at a time, 16 bytes of a row (a word of each row at every step was half
    // of all requests to the L2), to a ring of their own.
    constexpr int kScaleRows = (BN + BM + 63) / 64 * 64;  // whole loads of a wave
    constexpr int kScales = kScaleRows * 16;
    constexpr auto loads_of = [](int pieces) { return (pieces + kLoaders - 1) / kLoaders; };
    constexpr int kWLoads = loads_of(kW / 16), kXLoads = loads_of(kX / 16), kHighLoads = loads_of(kHigh / 16);
    constexpr int kScaleLoads = loads_of(kScaleRows), kLoads = kWLoads + kXLoads + kHighLoads;
    constexpr int kRing = STAGES * kStage, kOwn = kRing + 2 * kScales, kPairsAt = WK * kOwn;
    constexpr int kLds = kPairsAt + (R == Result::kPairs ? BM * 4 : 0);
    static_assert(kLds <= 160 * 1024 && (STAGES - 2) * kLoads + kScaleLoads < 64, "LDS and waits");
    static_assert(kW / 16 % 64 == 0 && kX / 16 % 64 == 0 && kHigh / 16 % 64 == 0, "whole loads of a wave");
    __shared__ __attribute__((aligned(1024))) uint8_t lds[kLds];

    // (The grid has room for the most tiles that the experts may have: those there are
    // go to all XCDs alike.)
    const Tiles<R, BM> tiles(a);
    const uint32_t units = tiles.total();
    if (blockIdx.x >= units * columns) return;
    const Place place = place_of<kOfExperts<R> ? 1 : 4>(blockIdx.x, units, columns);
    const Tile tile = tiles.at(a, place.unit);
    if (tile.count == 0) return;  // (offsets of no plan)
    const uint32_t column = place.column * kColumns;
    const int lane = static_cast<int>(threadIdx.x) & 63;
    const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) >> 6);
    const int wn = wave % WN, wm = wave / WN % WM, wk = wave / (WN * WM);
    const uint32_t steps = a.kp / kStep, each = (steps + WK - 1) / WK;
    const uint32_t first_step = min(wk * each, steps), stages = min(each, steps - first_step);
    uint8_t* const own = lds + wk * kOwn;

    // Row `row` of the tile's weights, rows past the last being the last again.
    const auto w_row = [&](uint32_t row) -> uint64_t {
        if constexpr (kGate) {
            const uint32_t side = row / (BN / 2), n = min(column + row % (BN / 2), a.outputs - 1);
            return (static_cast<uint64_t>(tile.expert) * 2 + side) * a.outputs + n;
        }
        return static_cast<uint64_t>(tile.expert) * a.outputs + min(column + row, a.outputs - 1);
    };
    const auto x_row = [&](uint32_t row) -> uint64_t {
        return input_row<R>(a, tile.first + min(row, tile.count - 1));
    };
    if constexpr (R == Result::kPairs) {  // where the rows of the results go, at hand when they do
        for (uint32_t row = threadIdx.x; row < BM; row += kThreads)
            reinterpret_cast<uint32_t*>(lds + kPairsAt)[row] =
                row < tile.count ? static_cast<uint32_t>(a.plan[tile.first + row]) : ~0u;
    }
    // What this thread loads: the row's first step, and the step of the stage.  (A load's place
    // in the part is the wave's; `piece` is the lane's own.)
    const int loader = kAlone ? 0 : wave;
    const auto piece_of = [&](int i, int pieces) { return (i * kLoaders + loader * 64) % pieces + lane; };
    const uint8_t* w_from[kWLoads];
    const uint8_t* x_from[kXLoads];
    const uint8_t* high_from[kHighLoads > 0 ? kHighLoads : 1];
    const uint8_t* scale_from[kScaleLoads];
#pragma unroll
    for (int i = 0; i < kWLoads; ++i) {
        const uint32_t at = piece_of(i, kW / 16), row = at / 4, block = (at % 4) ^ (row / 4 % 4);
        w_from[i] = a.w + w_row(row) * value_bytes(a.kp, 4) + block * 16;
    }
#pragma unroll
    for (int i = 0; i < kXLoads; ++i) {
        const uint32_t at = piece_of(i, kX / 16), row = at / 4, block = (at % 4) ^ (row / 4 % 4);
        x_from[i] = a.x + x_row(row) * value_bytes(a.kp, BITS) + block * 16;
    }
    if constexpr (BITS == 6) {
#pragma unroll
        for (int i = 0; i < kHighLoads; ++i) {  // two blocks' 8 bytes, at pair ^ (row / 8 % 2)
            const uint32_t at = piece_of(i, kHigh / 16), row = at / 2, pair = (at % 2) ^ (row / 8 % 2);
            high_from[i] = a.x + x_row(row) * value_bytes(a.kp, BITS) + a.kp / 2 + pair * 16;
        }
    }
#pragma unroll
    for (int i = 0; i < kScaleLoads; ++i) {
        const uint32_t row = min(piece_of(i, kScaleRows), BN + BM - 1);
        scale_from[i] = row < BN ? a.w_scales + w_row(row) * scale_bytes(a.kp)
                                 : a.x_scales + x_row(row - BN) * scale_bytes(a.kp);
    }
    // The scales of the group of four steps; of the last four of all where that passes the end.
    const auto first_of = [&](uint32_t group) { return min(first_step + 4 * group, steps - 4); };
    const auto load_scales = [&](uint32_t group) {
        uint8_t* const to = own + kRing + group % 2 * kScales;
#pragma unroll
        for (int i = 0; i < kScaleLoads; ++i)
            load_lds16(scale_from[i] + first_of(group) * 4, to + (piece_of(i, kScaleRows) - lane) * 16);
    };
    // Load `i` of stage `stage`, to a slot.
    const auto load_one = [&](uint32_t stage, uint32_t slot, int i) {
        uint8_t* const to = own + slot * kStage;
        const uint32_t step = first_step + stage;
        if (i < kWLoads)
            load_lds16(w_from[i] + step * 64, to + (piece_of(i, kW / 16) - lane) * 16);
        else if (i < kWLoads + kXLoads)
            load_lds16(x_from[i - kWLoads] + step * 64, to + kW + (piece_of(i - kWLoads, kX / 16) - lane) * 16);
        else if constexpr (BITS == 6)
            load_lds16(high_from[i - kWLoads - kXLoads] + step * 32,
                       to + kW + kX + (piece_of(i - kWLoads - kXLoads, kHigh / 16) - lane) * 16);
    };
    const auto load_stage = [&](uint32_t stage, uint32_t slot) {
#pragma unroll
        for (int i = 0; i < kLoads; ++i) load_one(stage, slot, i);
    };

    // This lane's rows of the wave's products, in the tile.
    const uint32_t of32 = lane & 31, half = lane >> 5;
    const auto w_in_tile = [&](int f) -> uint32_t {
        if constexpr (kGate)
            return f / (NF / 2) * (BN / 2) + (wn * (NF / 2) + f % (NF / 2)) * 32;
        else
            return (wn * NF + f) * 32;
    };
    const auto x_in_tile = [&](int f) -> uint32_t { return (wm * MF + f) * 32; };
    f32x16 d[NF][MF] = {};
    // Operands of half a step (blocks 2 S and 2 S + 1) and a step's scales, from LDS.
    u32x4 w[2][NF], x_low[2][MF];
    u32x2 x_high[2][MF];  // (of 6 bits)
    uint32_t w_words[NF], x_words[MF], ws[NF], xs[MF];
    const auto read_scales = [&](uint32_t stage) {
        const uint32_t group = stage / 4;
        const uint32_t* const scales = reinterpret_cast<const uint32_t*>(own + kRing + group % 2 * kScales) +
                                       (first_step + stage - first_of(group));
#pragma unroll
        for (int f = 0; f < NF; ++f) w_words[f] = scales[(w_in_tile(f) + of32) * 4];
#pragma unroll
        for (int f = 0; f < MF; ++f) x_words[f] = scales[(BN + x_in_tile(f) + of32) * 4];
    };
    const auto take_scales = [&] {  // this lane's bytes, blocks `half` and 2 + half, to bits 0 and 16
#pragma unroll
        for (int f = 0; f < NF; ++f) ws[f] = w_words[f] >> (8 * half);
#pragma unroll
        for (int f = 0; f < MF; ++f) xs[f] = x_words[f] >> (8 * half);
    };
    const auto read_half = [&](uint32_t slot, auto which) {
        constexpr int S = decltype(which)::value;
        const uint8_t* const at = own + slot * kStage;
        const uint32_t block = 2 * S + half;
#pragma unroll
        for (int f = 0; f < MF; ++f) {
            const uint32_t row = x_in_tile(f) + of32;
            x_low[S][f] = *reinterpret_cast<const u32x4*>(at + kW + row * 64 + (block ^ (row / 4 % 4)) * 16);
            if constexpr (BITS == 6)
                x_high[S][f] =
                    *reinterpret_cast<const u32x2*>(at + kW + kX + row * 32 + (S ^ (row / 8 % 2)) * 16 + half * 8);
        }
#pragma unroll
        for (int f = 0; f < NF; ++f) {
            const uint32_t row = w_in_tile(f) + of32;
            w[S][f] = *reinterpret_cast<const u32x4*>(at + row * 64 + (block ^ (row / 4 % 4)) * 16);
        }
    };
    // Products `first` up to `last` of a half.
    const auto multiply_half = [&](auto which, int first, int last) {
        constexpr int S = decltype(which)::value;
#pragma unroll
        for (int g = 0; g < MF; ++g) {
            Block<BITS> x;
            x.low = x_low[S][g];
            if constexpr (BITS == 6) x.high = x_high[S][g];
#pragma unroll
            for (int f = 0; f < NF; ++f)
                if (g * NF + f >= first && g * NF + f < last)
                    d[f][g] = multiply32<BITS, 2 * S>(Block<4>{w[S][f]}.operand(), ws[f], x.operand(), xs[g], d[f][g]);
        }
    };
    constexpr std::integral_constant<int, 0> k0;
    constexpr std::integral_constant<int, 1> k1;

    const auto next = [](uint32_t slot) { return slot + 1 == STAGES ? 0 : slot + 1; };
    uint32_t loading = 0, reading = 0;
    // Until all but `later` of the loads have landed, for all waves that share them.
    const auto arrive = [&](auto later) {
        wait_counts<vm_wait(decltype(later)::value) & kLgkmWait>();
        order_fence();
        if constexpr (!kAlone) group_barrier();
        order_fence();
    };
    // While one half of a step is multiplied the next one is read: behind the first of its
    // products, so that the wait for what that one needs is not for these too.
    const auto run_stage = [&](uint32_t stage, auto loads, auto later) {
        constexpr int kLater = decltype(later)::value;  // loads under way when the next stage has landed; -1: none
        take_scales();
        multiply_half(k0, 0, 1);
        order_fence();
        read_half(reading, k1);
        order_fence();
        // The loads of a later stage between the products: one after the other they would hold up
        // the wave, and the others at the barrier, for longer than the products take.
        constexpr int kProducts = NF * MF, kGaps = kProducts > 1 ? kProducts - 1 : 1;
#pragma unroll
        for (int i = 0; i < kGaps; ++i) {
            multiply_half(k0, i + 1, i + 2);
            order_fence();
            if constexpr (decltype(loads)::value) {
#pragma unroll
                for (int l = i * kLoads / kGaps; l < (i + 1) * kLoads / kGaps; ++l)
                    load_one(stage + STAGES - 1, loading, l);
                order_fence();
            }
        }
        if constexpr (decltype(loads)::value) loading = next(loading);
        reading = next(reading);
        if constexpr (kLater >= 0) arrive(later);
        multiply_half(k1, 0, 1);
        order_fence();
        if constexpr (kLater >= 0) {
            read_scales(stage + 1);
            read_half(reading, k0);
            order_fence();
        }
        multiply_half(k1, 1, kProducts);
        order_fence();
    };
    if (!kAlone || stages > 0) {
        load_scales(0);
#pragma unroll
        for (uint32_t s = 0; s < STAGES - 1; ++s)
            if (!kAlone || s < stages) load_stage(s, loading), loading = next(loading);
        constexpr std::integral_constant<int, (STAGES - 2) * kLoads> kSteady;
        if (!kAlone || stages >= STAGES - 1)
            arrive(kSteady);
        else
            arrive(k0);
        read_scales(0);
        read_half(0, k0);
        uint32_t stage = 0;
        for (; stage + STAGES + 2 < stages; stage += 4) {  // in fours: straight code with the scales' loads
            load_scales(stage / 4 + 1);
            run_stage(stage, std::true_type{}, std::integral_constant<int, (STAGES - 2) * kLoads + kScaleLoads>{});
            run_stage(stage + 1, std::true_type{}, kSteady);
            run_stage(stage + 2, std::true_type{}, kSteady);
            run_stage(stage + 3, std::true_type{}, kSteady);
        }
        for (; stage + STAGES - 1 < stages; ++stage) {
            if (stage % 4 == 0) load_scales(stage / 4 + 1);
            run_stage(stage, std::true_type{}, kSteady);
        }
        if constexpr (kAlone) {
            for (; stage + 1 < stages; ++stage) {
                if (stage % 4 == 0) load_scales(stage / 4 + 1);
                run_stage(stage, std::false_type{}, k0);
            }
        } else {  // two stages more, K having four at least, in straight code (in a loop: 256 registers for 206)
            static_assert(STAGES == 3, "the last two stages");
            run_stage(stage++, std::false_type{}, k0);
        }
        run_stage(stage, std::false_type{}, std::integral_constant<int, -1>{});
    }
    __syncthreads();  // the last stage has been read
    if constexpr (WK > 1) {
        constexpr int kGroup = WN * WM * NF * MF;  // products of a group of waves
        static_assert((WK - 1) * kGroup * 4096 <= kPairsAt, "LDS");
        f32x4* const sums = reinterpret_cast<f32x4*>(lds) + lane;
        const int of_wave = wn + WN * wm;
        const auto place_in = [&](int group, int f, int g, int q) {
            return (((group - 1) * WN * WM + of_wave) * NF * MF + f * MF + g) * 256 + q * 64;
        };
#pragma unroll
        for (int f = 0; f < NF; ++f)
#pragma unroll
            for (int g = 0; g < MF; ++g)
#pragma unroll
                for (int q = 0; q < 4; ++q)
                    if (wk > 0)
                        sums[place_in(wk, f, g, q)] =
                            f32x4{d[f][g][4 * q], d[f][g][4 * q + 1], d[f][g][4 * q + 2], d[f][g][4 * q + 3]};
        __syncthreads();
        if (wk > 0) return;
#pragma unroll
        for (int f = 0; f < NF; ++f)
#pragma unroll
            for (int g = 0; g < MF; ++g)
#pragma unroll
                for (int q = 0; q < 4; ++q)
#pragma unroll
                    for (int group = 1; group < WK; ++group) {
                        const f32x4 more = sums[place_in(group, f, g, q)];
#pragma unroll
                        for (int r = 0; r < 4; ++r) d[f][g][4 * q + r] += more[r];
                    }
    }

    // Results leave as whole rows: a wave turns 32 rows of up to 256 bytes at a time in LDS of
    // its own (rows 16 bytes apart more, so that 8 lanes writing 16 or 8 bytes touch all banks).
    // Those of the largest tiles, tens of megabytes of all compute units at one time, go past the caches
    // (500 rows each, down of 128 experts of 2048 x 768 331 -> 312 us; 900 rows, 64 of 2048 x 1408 408 -> 374;
    // 4096 x 14336 x 4096 151 -> 148).
    constexpr bool kPast = BN * BM == 256 * 256;
    constexpr bool kHalf = R == Result::kGateUp || R == Result::kF16;
    constexpr int kSize = kHalf ? 2 : 4;
    constexpr int kOut = kGate ? NF / 2 : NF;                         // 32-column products of the wave
    constexpr int kPass = kOut < 8 / kSize ? kOut : 8 / kSize;        // of them, those turned together
    constexpr int kRowBytes = kPass * 32 * kSize, kRowRoom = kRowBytes + 16;
    static_assert((WK - 1) * WN * WM * NF * MF * 4096 + WN * WM * 32 * kRowRoom <= kPairsAt && kOut % kPass == 0, "LDS");
    constexpr int kRowLanes = kRowBytes / 16, kPer = 16 / kSize;
    uint8_t* const turn = lds + (WK > 1 ? (WK - 1) * WN * WM * NF * MF * 4096 : 0) + wave * (32 * kRowRoom);
#pragma unroll
    for (int g = 0; g < MF; ++g) {
        if (x_in_tile(g) >= tile.count) break;
#pragma unroll
        for (int pass = 0; pass < kOut; pass += kPass) {
#pragma unroll
            for (int f = 0; f < kPass; ++f) {
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    f32x4 y;
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        y[r] = d[pass + f][g][4 * q + r];
                        if constexpr (kGate) y[r] = silu_product(y[r], d[pass + f + NF / 2][g][4 * q + r]);
                    }
                    uint8_t* const at = turn + of32 * kRowRoom + (f * 32 + 8 * q + 4 * half) * kSize;
                    if constexpr (kHalf)
                        *reinterpret_cast<f16x4*>(at) = f16x4{static_cast<_Float16>(y[0]), static_cast<_Float16>(y[1]),
                                                              static_cast<_Float16>(y[2]), static_cast<_Float16>(y[3])};
                    else
                        *reinterpret_cast<f32x4*>(at) = y;
                }
            }
            wave_fence();
            const uint32_t n = column + (wn * kOut + pass) * 32 + lane % kRowLanes * kPer;
#pragma unroll
            for (int r = 0; r < 32; r += 64 / kRowLanes) {
                const uint32_t in_product = r + lane / kRowLanes, row = x_in_tile(g) + in_product;
                if (row >= tile.count || n >= a.outputs) continue;
                const u32x4 word =
                    *reinterpret_cast<const u32x4*>(turn + in_product * kRowRoom + lane % kRowLanes * 16);
                uint64_t to = tile.first + row;
                if constexpr (R == Result::kPairs) {
                    to = reinterpret_cast<const uint32_t*>(lds + kPairsAt)[row];
                    if (to >= a.rows) continue;
                }
                uint8_t* const out = static_cast<uint8_t*>(a.output) + (to * a.outputs + n) * kSize;
                if (n + kPer <= a.outputs) {
                    if constexpr (kPast)
                        __builtin_nontemporal_store(static_cast<u32x4_a2>(word), reinterpret_cast<u32x4_a2*>(out));
                    else
                        *reinterpret_cast<u32x4_a2*>(out) = word;
                } else {  // the last of a row that is no whole number of pieces
                    for (uint32_t i = 0; n + i < a.outputs; ++i) {
                        if constexpr (kHalf)
                            reinterpret_cast<uint16_t*>(out)[i] = static_cast<uint16_t>(word[i / 2] >> (i % 2 * 16));
                        else
                            reinterpret_cast<uint32_t*>(out)[i] = word[i];
                    }
                }
            }
            wave_fence();
        }
    }
}

template <Result R>
uint64_t row_tiles(const ProductArgs& a, uint32_t rows) {
    return kOfExperts<R> ? most_expert_tiles(a.rows, a.experts, rows) : (uint64_t{a.rows} + rows - 1) / rows;
}
template <Result R>
uint32_t column_tiles(const ProductArgs& a, uint32_t weight_rows) {
    const uint32_t columns = R == Result::kGateUp ? weight_rows / 2 : weight_rows;
    return (a.outputs + columns - 1) / columns;
}

template <int BITS, Result R, int BN, int BM, int WN, int WM, int WK, int STAGES>
int launch(const ProductArgs& a, hipStream_t stream) {
    constexpr uint32_t kThreads = 64 * WN * WM * WK;
    const uint32_t columns = column_tiles<R>(a, BN);
    const uint64_t units = row_tiles<R>(a, BM);
    if (units * columns > kMostThreads / kThreads) return kInvalid;
    hipLaunchKernelGGL((tiles_kernel<BITS, R, BN, BM, WN, WM, WK, STAGES>),
                       dim3(static_cast<uint32_t>(units * columns)), dim3(kThreads), 0, stream, a, columns);
    return static_cast<int>(hipGetLastError());
}

// A linear takes the largest tile, no taller than its rows need, of which there is one for three in
// four compute units: a workgroup's time hardly depends on how many others run (4096 outputs
// of 4096, 6 bits: 64 rows in 32, 64 and 256 tiles of 128 x 64, 64 x 64 and 32 x 32: 14.3, 10.4 and 6.8 us;
// 256 rows in 64, 128 and 256 of 128 x 128, 128 x 64 and 64 x 64: 17.8, 14.5 and 12.0; 4096 rows in 256, 1024
// and 2048 of 256 x 256, 128 x 128 and 128 x 64: 50, 78 and 96).  In the small ones waves divide K.
template <int BITS, Result R>
int choose(const ProductArgs& a, hipStream_t stream) {
    const auto enough = [&](uint32_t weight_rows, uint32_t rows) {
        return row_tiles<R>(a, rows) * column_tiles<R>(a, weight_rows) >= kEnoughTiles;
    };
    if constexpr (kOfExperts<R>) {
        // An expert's rows seldom fill its last tile, so tiles follow the mean of the rows (gate/up, 6 bits, us;
        // 32 experts of 2880 x 2880, and 128 of 768 x 2048):
        //   rows         8        16        32        64       128       256       500
        //   256 x 32    71  45    85  53  102  61  136  82
        //   128 x 64    74  48    80  54   91  59  121  74  165 106  272 170  488 288
        //   128 x 128             81  60   92  66  104  73  134  92  201 143  355 236
        //   256 x 256            101  74  104  77  114  94  140 104  183 137  274 197
        // (4 bits, 8 rows: 75 and 45 in 256 x 32, 68 and 45 in 128 x 64; down, 64 rows: 75 and 62 in 128 x 64, 75 and
        // 65 in 128 x 128.)
        const uint64_t mean = a.rows / a.experts;
        if (mean >= 256 && enough(256, 256)) return launch<BITS, R, 256, 256, 2, 2, 1, 3>(a, stream);
        if (mean >= 64) return launch<BITS, R, 128, 128, 2, 2, 1, 3>(a, stream);
        if constexpr (R == Result::kGateUp && BITS == 6) {
            if (mean < 16) return launch<BITS, R, 256, 32, 4, 1, 1, 3>(a, stream);
        }
        return launch<BITS, R, 128, 64, 2, 2, 1, 3>(a, stream);
    } else {
        if (a.rows > 32) {
            if (enough(256, 256)) return launch<BITS, R, 256, 256, 2, 2, 1, 3>(a, stream);
            if (enough(128, 128)) return launch<BITS, R, 128, 128, 2, 2, 1, 3>(a, stream);
            if (enough(128, 64)) return launch<BITS, R, 128, 64, 2, 2, 1, 3>(a, stream);
            if (enough(64, 64)) return launch<BITS, R, 64, 64, 1, 1, 4, 3>(a, stream);
        }
        if (enough(64, 32)) return launch<BITS, R, 64, 32, 1, 1, 2, 4>(a, stream);
        return launch<BITS, R, 32, 32, 1, 1, 4, 4>(a, stream);
    }
}

}  // namespace

int launch_tiles(Result result, const ProductArgs& a, int bits, hipStream_t stream) {
    const auto of = [&](auto r) {
        constexpr Result R = decltype(r)::value;
        return bits == 4 ? choose<4, R>(a, stream) : choose<6, R>(a, stream);
    };
    switch (result) {
        case Result::kF16: return of(std::integral_constant<Result, Result::kF16>{});
        case Result::kF32: return of(std::integral_constant<Result, Result::kF32>{});
        case Result::kGateUp: return of(std::integral_constant<Result, Result::kGateUp>{});
        default: return of(std::integral_constant<Result, Result::kPairs>{});
    }
}

}  // namespace mote::mx
