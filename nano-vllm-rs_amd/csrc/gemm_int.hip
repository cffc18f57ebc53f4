// Products in 8-bit integers (nv_gemm_i8), and of the gate's and the up
// projection's weights with SiLU·up behind them (nv_gemm_i8_silu). No counterpart
// in the reference, whose projections are bf16 products (kernels/kernels.cu:98-106,
// src/model.rs:659-678, :753-780).
//
// Semantics. Token i as 8-bit integers xq with the scale xs (nvr_int8.h), channel j
// of the weight as wq with ws:
//   y[i, j] = bf16(sum_l xq[i, l] wq[j, l] * xs[i] * ws[j]),
// the sum exact in 32 bits (k <= 131071: 2^14 k < 2^31, a weight of -128 too), its
// value in fp32, two products in fp32 and one rounding to bf16. Gated, with g and u
// those fp32 values of channels j and inter + j: bf16(g / (1 + e^-g) * u).
// Integer sums have no order, so every form gives the same bits for a token,
// whatever the batch.
//
// Three forms. Up to 16 tokens over short rows are made into integers by every
// block, and up to 32 over some wide weights are brought to LDS; gemm_rows_i8 then
// streams the weights through registers, each byte once, bound by HBM and, in the
// smallest calls, by one chain: tokens, their largest value, products, outputs. All
// others go by tiles (gemm_int_tiles.hip). On MI355X: 1 token over 1024 x 2048 3.4
// us, 8 with sum and norm over 4096 x 1024 4.2 us; 32 over 151936 x 1024 39.6 us with
// the tokens' launch, 4.2 TB/s.
#include "../../include/nano_hip.h"
#include "nvr_int8.h"
#include "nvr_internal.h"

namespace {

using nvr::kWave;
using nvr::Scale;
using nvr::Tokens;
typedef int i32x4_t __attribute__((ext_vector_type(4)));

constexpr int kWaves = 8, kThreads = kWaves * kWave;
constexpr int kRowPad = 16;  // behind a token's row in LDS: 16 tokens' pieces of one column lie in different banks
constexpr int kFewTokens = 32;
constexpr int kMostLds = 160 * 1024;

// Where the tokens' integers come from: made by each block (of x, the norm, or the norm of the sum), or by a launch of
// quantize_rows and brought to LDS.
enum class Source { kPlain, kNorm, kAddNorm, kCopied };

struct RowsArgs {
    nvr::ProductArgs p;
    nvr::TokenArgs t;
    int log_parts;              // 2^log_parts waves share the k of a tile: 1, 2, 4 or 8
    int per, more;              // a block has `per` tiles, the first `more` blocks one more
    int share, units;           // lines of 128 bytes of k a wave has of a tile; loads of STEPS steps
};

// LDS of a block: partial sums (parts > 1), scales, tokens.
template <int MT>
constexpr int kSumBytes = 2 * kWaves * MT * kWave * 16;
template <int MT>
int64_t rows_lds(int m, int x_pitch) {
    return kSumBytes<MT> + MT * 16 * 4 + int64_t(m) * (x_pitch + kRowPad);
}

// Few tokens: the weights stream through registers, once, STEPS pieces of 64 bytes of k in flight together as a unit, and
// two units; 16 rows of the weight are a product's first operand, so that nothing of it passes LDS. ONE: every wave has one
// unit at most in all.
template <Source SRC, bool WHOLE, int CH, int RW, int MT, bool GATED, int STEPS, bool ONE>
__global__ __launch_bounds__(kThreads) void gemm_rows_i8(RowsArgs a) {
    constexpr bool kMade = SRC != Source::kCopied;
    constexpr int kChannels = GATED ? 8 : 16;  // of a tile: 16 rows of the weight, or 8 of gate, then 8 of up
    extern __shared__ __align__(16) unsigned char smem[];
    const nvr::ProductArgs& p = a.p;
    const int lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int i = lane % 16, g = lane / 16;
    const int parts = 1 << a.log_parts, groups = kWaves >> a.log_parts, group = wave >> a.log_parts, part = wave & (parts - 1);
    const int first = int(blockIdx.x) * a.per + min(int(blockIdx.x), a.more);
    // Of a block's tiles, and of a group's of waves.
    const int mine = a.per + (int(blockIdx.x) < a.more ? 1 : 0);  // >= 1
    const int rounds = (mine + groups - 1) >> (3 - a.log_parts);  // the same in every wave
    static_assert(kWaves == 8, "rounds");
    const int even = mine >> (3 - a.log_parts), odd = mine & (groups - 1);
    const int tile0 = first + group * even + min(group, odd), tile_count = even + (group < odd ? 1 : 0);
    // A wave's steps of each of its tiles.
    const int lines = p.x_pitch / 128, units = a.units;
    const int s0 = min(part * a.share, lines) * 2, s1 = min((part + 1) * a.share, lines) * 2;

    i32x4_t* red = reinterpret_cast<i32x4_t*>(smem);                   // [2][kWaves][MT][64]
    float* xs = reinterpret_cast<float*>(smem + kSumBytes<MT>);        // [MT * 16]
    unsigned char* xq = reinterpret_cast<unsigned char*>(xs + MT * 16);  // [m][pitch]
    const int pitch = p.x_pitch + kRowPad;

    // The weights of a unit: lane l has row l % 16, 16 bytes at 16 (l / 16) of each step. Behind the wave's steps, which are
    // not multiplied, its last one again (lines of another wave's would cost: 4 tokens over 4096 x 1024 6.0 us for 4.3), and
    // behind a row's end, where x is zero, any bytes of the row.
    const int last_step = max(s1, 1) - 1;
    struct Unit {
        uint4 w[STEPS];
        float ws[4];  // of the lane's outputs
    };
    Unit unit[2];
    int ahead_round = 0, ahead = 0;  // the next unit to load
    auto load = [&](Unit& u) {
        const int tile = tile0 + max(min(ahead_round, tile_count - 1), 0);  // its own last one, if any, where it has no more
        const int64_t row = GATED ? int64_t(i < 8 ? 0 : p.n) + min(tile * 8 + i % 8, p.n - 1) : min(tile * 16 + i, p.n - 1);
        const uint8_t* w = p.wq + row * p.w_pitch;
        const int s = s0 + ahead * STEPS;
#pragma unroll
        for (int e = 0; e < STEPS; ++e)
            u.w[e] = *reinterpret_cast<const uint4*>(w + min(min(s + e, last_step) * 64 + 16 * g, p.w_pitch - 16));
#pragma unroll
        for (int r = 0; r < 4; ++r)
            u.ws[r] = GATED ? p.ws[int64_t(g < 2 ? 0 : p.n) + min(tile * 8 + 4 * (g % 2) + r, p.n - 1)]
                            : p.ws[min(tile * 16 + 4 * g + r, p.n - 1)];
        if (++ahead == units) {
            ahead = 0;
            ++ahead_round;
        }
    };
    if constexpr (kMade) {
        // A wave's loads return in order: its tokens' come before the weights'.
        constexpr Tokens T = SRC == Source::kPlain ? Tokens::kPlain : SRC == Source::kNorm ? Tokens::kNorm : Tokens::kAddNorm;
        const nvr::NormChunks<CH> norm = nvr::load_norm<T, WHOLE, CH, 1>(a.t, lane, 0);
        nvr::RowChunks<T, CH> chunks[RW];
#pragma unroll
        for (int i = 0; i < RW; ++i)
            chunks[i] = nvr::load_row<T, WHOLE, CH, 1>(a.t, min(wave + i * kWaves, p.m - 1), lane, 0);
        // The compiler would mix them otherwise (1 token over 1024 x 2048 4.5 us for 3.4).
        __builtin_amdgcn_sched_barrier(0);
        load(unit[0]);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < RW; ++i) {
            const int row = wave + i * kWaves;
            if (row >= p.m) break;
            const nvr::RowStep step = nvr::quantize_row<T, WHOLE, CH, 1>(
                a.t, row, chunks[i], norm, p.x_pitch, blockIdx.x == 0 && a.t.residual_out != nullptr, lane, 0,
                nvr::NoJoin{}, [&](int j, uint2 eight) { *reinterpret_cast<uint2*>(xq + row * pitch + j) = eight; });
            if (lane == 0) xs[row] = step.scale;
        }
    } else {
        for (int row = wave; row < p.m; row += kWaves)
#pragma unroll 4
            for (int c = lane * 16; c < p.x_pitch; c += kWave * 16)
                *reinterpret_cast<uint4*>(xq + row * pitch + c) =
                    *reinterpret_cast<const uint4*>(p.xq + int64_t(row) * p.x_pitch + c);
        if (int(threadIdx.x) < p.m) xs[threadIdx.x] = p.xs[threadIdx.x];
        load(unit[0]);  // behind the tokens, for the same reason
    }
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");  // leaves the weights in flight
    if constexpr (!ONE) load(unit[1]);

    // Tokens behind the last repeat it and are not stored.
    const unsigned char* xrow[MT];
#pragma unroll
    for (int t = 0; t < MT; ++t)
        xrow[t] = xq + min(t * 16 + i, p.m - 1) * pitch + 16 * g;
    i32x4_t acc[MT];
    float ws[4];
    // A wave that has its tiles to itself, and several, keeps its outputs until they fill lines of 128 bytes.
    const bool lines_kept = !ONE && parts == 1 && p.n % 8 == 0;
    unsigned char* kept = smem + wave * (MT * 16 * 128);  // [MT * 16][128], where the sums would be
    static_assert(kWaves * MT * 16 * 128 == kSumBytes<MT>, "its place");
    int round = 0, at = 0;  // the unit to multiply
    // Lane l has token l % 16 of 16, rows 4 (l / 16) .. + 3 of the tile.
    auto finish = [&](int t, const i32x4_t& sum) {
        const int token = t * 16 + i;
        const Scale x = nvr::split_scale(xs[min(token, p.m - 1)]);
        float y[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            y[r] = nvr::scaled(sum[r], x, nvr::split_scale(ws[r]));
            if constexpr (GATED) y[r] = nvr::gated(y[r], nvr::xor_lane(y[r], 32));  // the other half has the up rows
        }
        if (round >= tile_count) return;
        const int channel = (tile0 + round) * kChannels + 4 * (GATED ? g % 2 : g);
        const bool stored = token < p.m && !(GATED && g >= 2);
        if (lines_kept) {
            if (stored)
                *reinterpret_cast<uint2*>(kept + token * 128 + channel % 64 * 2) =
                    make_uint2(nvr::pack_bf16x2(y[0], y[1]), nvr::pack_bf16x2(y[2], y[3]));
            return;
        }
        if (stored) nvr::store_outputs(p.y + int64_t(token) * p.n + channel, y, channel, p.n);
    };
    // A wave's tiles that fill a line of 64 channels, or its last: 8 tokens' lines a store.
    auto flush = [&] {
        const int end = (tile0 + round + 1) * kChannels;
        if (round >= tile_count || (end % 64 != 0 && round + 1 < tile_count)) return;
        // finish wrote values of another type, which the compiler may take to be elsewhere; the wave's LDS accesses themselves
        // are in order, and so are the next lines' writes behind these reads.
        asm volatile("" ::: "memory");
        const int channel = (end - 1) / 64 * 64 + lane % 8 * 8;
        if (channel < tile0 * kChannels || channel >= min(end, p.n)) return;
#pragma unroll
        for (int r = 0; r < MT * 16; r += 8)
            if (r + lane / 8 < p.m)
                nvr::store8(p.y + int64_t(r + lane / 8) * p.n + channel,
                            *reinterpret_cast<const uint4*>(kept + (r + lane / 8) * 128 + lane % 8 * 16));
        asm volatile("" ::: "memory");
    };
    auto multiply = [&](const Unit& u) {
        if (at == 0) {
#pragma unroll
            for (int t = 0; t < MT; ++t) acc[t] = i32x4_t{0, 0, 0, 0};
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) ws[r] = u.ws[r];
        const int s = s0 + at * STEPS;
        auto tokens = [&](int t, int e) { return *reinterpret_cast<const i32x4_t*>(xrow[t] + (s + e) * 64); };
        auto product = [](i32x4_t& sum, const uint4& w, i32x4_t x) {
            sum = __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i32x4_t, w), x, sum, 0, 0, 0);
        };
        if (s + STEPS <= s1) {
            i32x4_t x[STEPS][MT];
#pragma unroll
            for (int e = 0; e < STEPS; ++e)
#pragma unroll
                for (int t = 0; t < MT; ++t) x[e][t] = tokens(t, e);
#pragma unroll
            for (int e = 0; e < STEPS; ++e)
#pragma unroll
                for (int t = 0; t < MT; ++t)
                    product(acc[t], u.w[e], x[e][t]);
        } else {
#pragma unroll
            for (int e = 0; e < STEPS; ++e) {
                if (s + e >= s1) break;
#pragma unroll
                for (int t = 0; t < MT; ++t)
                    product(acc[t], u.w[e], tokens(t, e));
            }
        }
        ++at;
    };
    // After the loads that follow: a wait for those of one unit then leaves the stores of the one before in flight.
    auto settle = [&] {
        if (at < units) return;
        if (parts == 1) {
#pragma unroll
            for (int t = 0; t < MT; ++t) finish(t, acc[t]);
            if (lines_kept) flush();
        } else {
            i32x4_t* sums = red + (round & 1) * (kWaves * MT * kWave) + lane;
#pragma unroll
            for (int t = 0; t < MT; ++t) sums[(wave * MT + t) * kWave] = acc[t];
            asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
#pragma unroll
            for (int t = 0; t < MT; ++t) {
                if (((round * MT + t) & (parts - 1)) != part) continue;  // the waves take turns
                i32x4_t sum[kWaves];
#pragma unroll
                for (int q = 0; q < kWaves; ++q)
                    if (q < parts) sum[q] = sums[(((wave & -parts) + q) * MT + t) * kWave];
#pragma unroll
                for (int q = 1; q < kWaves; ++q)
                    if (q < parts) sum[0] += sum[q];
                finish(t, sum[0]);
            }
        }
        at = 0;
        ++round;
    };
    if constexpr (ONE) {
        multiply(unit[0]);
        settle();
        return;
    }
    for (int left = rounds * units;; left -= 2) {
        multiply(unit[0]);
        if (left <= 2) {
            settle();
            if (left == 2) {
                multiply(unit[1]);
                settle();
            }
            break;
        }
        load(unit[0]);
        settle();
        multiply(unit[1]);
        if (left == 3) {
            settle();
            multiply(unit[0]);
            settle();
            break;
        }
        load(unit[1]);
        settle();
    }
}

template <Source SRC, bool WHOLE, int CH, int RW, int MT, bool GATED, int STEPS, bool ONE>
void launch_rows_as(nv_context* c, const RowsArgs& a, int blocks) {
    hipLaunchKernelGGL((gemm_rows_i8<SRC, WHOLE, CH, RW, MT, GATED, STEPS, ONE>), dim3(unsigned(blocks)), dim3(kThreads),
                       size_t(rows_lds<MT>(a.p.m, a.p.x_pitch)), c->stream, a);
}

void plan_rows(RowsArgs& a, int tiles, int parts, int blocks) {
    const int lines = a.p.x_pitch / 128;
    a.log_parts = __builtin_ctz(unsigned(parts));
    a.per = tiles / blocks;
    a.more = tiles % blocks;
    a.share = (lines + parts - 1) / parts;
}

template <Source SRC, bool WHOLE, bool GATED>
void launch_rows(nv_context* c, RowsArgs a) {
    constexpr bool kMade = SRC != Source::kCopied;
    const int tiles = (a.p.n + (GATED ? 8 : 16) - 1) / (GATED ? 8 : 16);
    const int cus = c->cu_count > 0 ? c->cu_count : 256;
    const int lines = a.p.x_pitch / 128;
    // As many waves for a tile as leave each one tile, if its share of k is then one unit; else up to four turns of them. On
    // MI355X, weights cold, in us by 1, 2, 4 and 8 waves a tile: 1 token over 4096 x 1024 6.1, 4.4, 3.5, 3.1; over 16384 x 1024
    // 6.7, 5.6, 6.2, 7.7; 16 over 4096 x 1024 7.2, 4.9, 4.6, 4.4; gated 1 over 4096 x 1024 6.9, 5.3, 4.6, 5.8, over 11008 x 4096
    // 21.8, 24.3, 19.5, 21.8; 4 with sum and norm over 8192 x 4096 21.3, 14.3, 11.4, 11.7, over 65536 x 4096 57.1, 50.6, 49.6,
    // 51.3; 8 with norm over 151936 x 1024 32.6, 33.1, 34.4, 48.8. Takes more waves than are best for 1 over 65536 at k 256, 1024
    // (2, where 1 and 2 are 5.8, 14.9 and 7.9, 16.0) and 16384 x 4096 (8: 19.6, 14.2, 14.6, 16.2).
    auto fits = [&](int parts) { return int64_t(tiles) * parts <= int64_t(cus) * kWaves && (lines + parts - 1) / parts <= 4; };
    int parts = fits(8) ? 8 : fits(4) ? 4 : fits(2) ? 2 : fits(1) ? 1 : 8;
    if (!fits(parts))
        while (parts > 1 && (parts > lines || int64_t(tiles) * parts > int64_t(cus) * kWaves * 4)) parts /= 2;
    const int blocks = std::min(cus, (tiles * parts + kWaves - 1) / kWaves);
    plan_rows(a, tiles, parts, blocks);
    const bool alone = (a.per + (a.more != 0)) * parts <= kWaves;  // a wave has one tile at most
    auto run = [&](auto chunks, auto rows, auto tiles16) {
        constexpr int CH = decltype(chunks)::value, RW = decltype(rows)::value, MT = decltype(tiles16)::value;
        auto with = [&](auto steps, auto one) {
            constexpr int STEPS = decltype(steps)::value;
            a.units = (a.share * 2 + STEPS - 1) / STEPS;
            launch_rows_as<SRC, WHOLE, CH, RW, MT, GATED, STEPS, decltype(one)::value>(c, a, blocks);
        };
        // The fewest loads that hold a wave's share: each is made, also behind it. On MI355X, in us, as here, by the next larger
        // unit, and by two of 8 steps in turn: 1 token over 4096 at k 1024 (2 steps) 3.1, 3.3, 5.6, with sum and norm 3.5, 3.8,
        // 5.9; at k 2048 (4) 4.2, 5.2, 6.4; at k 4096 (8) 6.1, -, 7.9. Of several tiles in turn, over 65536 at k 128, 256 (4)
        // 5.0, 7.9, by 8 6.4, 11.2. Tokens brought to LDS meet wide weights: several tiles a wave, without one unit's forms.
        const auto one = std::true_type{};
        if constexpr (WHOLE && kMade) {
            if (alone && a.share == 1) return with(std::integral_constant<int, 2>{}, one);
        }
        if constexpr (WHOLE) {
            if (!alone && a.share <= 2) return with(std::integral_constant<int, 4>{}, std::false_type{});
        }
        if constexpr (kMade) {
            if (alone && a.share <= 2) return with(std::integral_constant<int, 4>{}, one);
            if (alone && a.share <= 4) return with(std::integral_constant<int, 8>{}, one);
        }
        with(std::integral_constant<int, 8>{}, std::false_type{});
    };
    using std::integral_constant;
    const integral_constant<int, 1> one;
    const integral_constant<int, 2> two;
    if constexpr (SRC == Source::kCopied) {
        a.p.m <= 16 ? run(one, one, one) : run(one, one, two);
    } else {
        const integral_constant<int, 4> four;
        const int chunks = (a.p.x_pitch + nvr::kWaveChunk - 1) / nvr::kWaveChunk;
        if (a.p.m > kWaves) {
            if constexpr (SRC == Source::kPlain && WHOLE)
                if (chunks > 2) return run(four, two, one);
            run(two, two, one);
        } else if (chunks <= 2) {
            run(two, one, one);
        } else if (!WHOLE || chunks <= 4) {
            run(four, one, one);
        } else if constexpr (WHOLE) {
            run(integral_constant<int, 8>{}, one, one);
        }
    }
}

// Whether each block makes the tokens' integers by itself, a row or two a wave: one launch less, for work that all blocks
// repeat. On MI355X in a graph, weights cold, n 4096, made and by a launch of their own, in us:
//   k 1024: 1 token 3.1, 5.6; 8 with sum and norm 4.2, 6.2; 16 4.4, 5.7, with sum and norm 5.6, 6.1;
//   k 2048: 8 5.0, 6.7, with sum and norm 6.3, 7.3; 9 and 16 5.1, 6.2 and 6.8, 7.0; 16 with sum and norm 8.8, 7.8;
//   k 4096: 8 8.2, 8.6; with sum and norm 4 8.1, 9.0, but 6 10.5, 9.1: two waves of a SIMD then have a row each, and a row's
//   chunks, sums and norm weights fill the registers beside the weights.
// What every block repeats does not grow with n, and neither does what it saves. 16 at k 2048 over n 1024, 8192, 16384, 32768,
// 65536: 5.4, 7.7, 11.8, 17.5, 28.4 and 6.0, 8.0, 11.2, 19.0, 30.8; 16 with sum and norm at k 1024 5.3, 6.2, 7.9, 12.0, 17.7 and
// 5.9, 7.3, 8.6, 13.2, 19.9; 8 at k 4096 5.9, 12.2, 17.4, 28.2, 51.3 and 7.3, 12.0, 18.8, 29.2, 53.1.
// Chunks of a k that is no multiple of 8 take shifts, so half as many: 8 at k 2041 5.2, 6.8, at 4090 9.7, 8.8; 1 with sum and
// norm at 2041 6.8, 7.6, at 4090 15.0, 9.6; 8 at 1001 5.2, 6.7, at 1111 7.5, 7.0; 16 at 1001 5.0, 5.9, at 1111 7.1, 6.4.
bool tokens_in_block(const nvr::TokenArgs& t) {
    const int most = t.rows <= 4 ? 8 : t.rows <= kWaves ? 4 : 2;  // chunks of a row with a norm
    const int chunks = t.norm_weight != nullptr ? most : t.rows <= kWaves ? 8 : 4;
    return t.rows <= 2 * kWaves && t.k <= (t.k % nvr::kChunk == 0 ? chunks : chunks / 2) * nvr::kWaveChunk;
}

// Whether few tokens, made by a launch of their own, take gemm_rows_i8 rather than gemm_split's tiles of 32 rows of the weight.
// On MI355X, weights cold, tokens' launch included, this and that in us:
//   more than 16 tokens over a wide weight of short rows, of which a tile is mostly its start and its end: 32 over 151936 at
//   k 520, 1024, 1030 27.2, 39.1, 43.2 and 32.7, 43.6, 48.5; over 65536 15.9, 21.7, 26.2 and 17.9, 23.8, 25.2; over 40000
//   (five turns of the CUs) 12.8, 16.3, 20.1 and 13.0, 16.4, 18.5. Of longer rows the tiles are mostly the faster ones: at k
//   2048 over 40000, 100000, 151936 25.9, 52.0, 70.6 and 23.4, 49.1, 70.6; 24 over 100000 x 4096 97, 84, but 32 over 151936 x
//   3000 98, 106. 16 tokens: over 40000 x 1024 14.7, 13.6, over 151936 at k 1024, 4096 36.2, 132 and 36.2, 112;
//   where the runs of tiles that the XCDs take lie a power of two apart, 8 MB or more, so that all eight read the same memory
//   channels in step, and there is more than a tile a CU: 16 tokens over 16384 at k 4096, 8192 19.2, 30.8 and 21.5, 36.8; over
//   32768 29.8, 52.4 and 33.6, 72.3; over 65536 56.3, 106 and 58.3, 133; gated over 16384 x 4096 31.0, 35.5; at 16384 x 16384
//   53.4, 53.4. Beside them: 16384 at k 3000, 4104, 6144 17.6, 23.2, 27.5 and 15.3, 19.5, 22.8; 20480 at k 4096, 8192 22.2,
//   39.9 and 22.1, 36.7; 8192 x 8192 (a tile a CU) 20.2, 17.9; 12288 x 8192 25.0, 25.5. Gated 24 over 11008 x 4096 24.7, 25.2.
// Up to 8 tokens over one to two turns of long rows would gain: 8 over 11008, 12288, 13824 at k 12288 31.5, 32.7, 40.0 and
// 37.0, 36.4, 38.5.
bool weight_streams(const nv_context* c, const nvr::ProductArgs& p, bool gated) {
    const int64_t rows = gated ? 2 * int64_t(p.n) : p.n, cus = c->cu_count > 0 ? c->cu_count : 256, tiles = (rows + 31) / 32;
    const int64_t run = tiles / nvr::kXcds * (gated ? 16 : 32) * p.w_pitch;  // bytes from an XCD's tiles to the next one's
    const bool in_step = tiles > cus && run >= 8 << 20 && (run & (run - 1)) == 0;
    const bool wide = p.m > 16 && tiles >= 8 * cus && p.x_pitch <= 1152;
    return p.m <= kFewTokens && (in_step || wide) &&
           (p.m <= 16 ? rows_lds<1>(p.m, p.x_pitch) : rows_lds<2>(p.m, p.x_pitch)) <= kMostLds;
}

constexpr int kStepBytes = 128;  // tokens' rows in the workspace end in zeros at a multiple of this
int64_t token_pitch(int64_t k) { return (k + kStepBytes - 1) / kStepBytes * kStepBytes; }

size_t workspace_bytes(int64_t m, int64_t k) { return size_t(m * token_pitch(k) + (m * 4 + 15) / 16 * 16); }

int check_sizes(const char* op, int m, int n, int k, bool gated) {
    if (m <= 0 || n <= 0 || k <= 0 || k > nvr::kMostSummed)
        return nvr::fail(-2, "%s: m %d, n %d, k %d; k goes from 1 to %d", op, m, n, k, nvr::kMostSummed);
    if (n > (gated ? INT32_MAX / 2 : INT32_MAX) - 256)
        return nvr::fail(-2, "%s: n %d is too large", op, n);
    return 0;
}

template <bool GATED>
int product(nv_context* c, const char* op, const void* x, const void* residual, void* residual_out,
            const void* norm_weight, const void* w, const void* w_scales, void* y, void* workspace, int m, int n, int k,
            float eps) {
    NVR_ACTIVATE(c);
    if (int error = check_sizes(op, m, n, k, GATED)) return error;
    if (x == nullptr || w == nullptr || w_scales == nullptr || y == nullptr || workspace == nullptr)
        return nvr::fail(-2, "%s: x, w, w_scales, the output and the workspace are required", op);
    if (residual != nullptr && norm_weight == nullptr)
        return nvr::fail(-2, "%s: a residual needs a norm_weight", op);
    if (residual == nullptr && residual_out != nullptr)
        return nvr::fail(-2, "%s: residual_out needs a residual to add", op);
    if (!nvr::aligned(w, 16) || !nvr::aligned(workspace, 16) || !nvr::aligned(w_scales, 4) || !nvr::aligned(x, 2) ||
        !nvr::aligned(residual, 2) || !nvr::aligned(residual_out, 2) || !nvr::aligned(norm_weight, 2) || !nvr::aligned(y, 2))
        return nvr::fail(-2, "%s: w and the workspace start at multiples of 16 bytes, scales of 4, others of 2", op);
    // Blocks read while others write.
    const int64_t in_bytes = int64_t(m) * k * 2, channels = GATED ? 2 * int64_t(n) : n;
    if (nvr::overlap({{residual_out, in_bytes}, {y, int64_t(m) * n * 2}, {workspace, int64_t(workspace_bytes(m, k))}},
                     {{x, in_bytes}, {residual, in_bytes}, {norm_weight, int64_t(k) * 2}, {w, channels * nvr::i8_pitch(k)},
                      {w_scales, channels * 4}}))
        return nvr::fail(-2, "%s: an output or the workspace overlaps another argument", op);
    const nvr::TokenArgs t{static_cast<const uint16_t*>(x),
                           static_cast<const uint16_t*>(residual),
                           static_cast<uint16_t*>(residual_out),
                           static_cast<const uint16_t*>(norm_weight),
                           m,
                           k,
                           eps};
    const int pitch = int(token_pitch(k));
    uint8_t* xq = static_cast<uint8_t*>(workspace);
    float* xs = reinterpret_cast<float*>(xq + int64_t(m) * pitch);
    const nvr::ProductArgs p{xq, xs, static_cast<const uint8_t*>(w), static_cast<const float*>(w_scales),
                             static_cast<uint16_t*>(y), m, n, pitch, int(nvr::i8_pitch(k))};
    const RowsArgs few{p, t, 0, 0, 0, 0, 0};
    if (tokens_in_block(t)) {
        auto run = [&](auto whole) {
            constexpr bool WHOLE = decltype(whole)::value;
            if (norm_weight == nullptr) launch_rows<Source::kPlain, WHOLE, GATED>(c, few);
            else if (residual == nullptr) launch_rows<Source::kNorm, WHOLE, GATED>(c, few);
            else launch_rows<Source::kAddNorm, WHOLE, GATED>(c, few);
        };
        k % nvr::kChunk == 0 ? run(std::true_type{}) : run(std::false_type{});
        return nvr::launch_status();
    }
    const bool streams = weight_streams(c, p, GATED);
    if (!streams)
        if (int error = nvr::launch_product_tiles(c, p, GATED, true)) return error;
    nvr::launch_quantize(c, t, xq, xs, pitch);
    if (!streams) return nvr::launch_product_tiles(c, p, GATED, false);
    launch_rows<Source::kCopied, true, GATED>(c, few);
    return nvr::launch_status();
}

}  // namespace

extern "C" {

int nv_gemm_i8_workspace(int m, int n, int k, size_t* bytes) {
    if (int error = check_sizes("gemm_i8_workspace", m, n, k, false)) return error;
    *bytes = workspace_bytes(m, k);
    return 0;
}

int nv_gemm_i8(nv_context* c, const void* x, const void* residual, void* residual_out, const void* norm_weight,
               const void* w, const void* w_scales, void* y, void* workspace, int m, int n, int k, float eps) {
    return product<false>(c, "gemm_i8", x, residual, residual_out, norm_weight, w, w_scales, y, workspace, m, n, k, eps);
}

int nv_gemm_i8_silu_workspace(int m, int intermediate, int k, size_t* bytes) {
    if (int error = check_sizes("gemm_i8_silu_workspace", m, intermediate, k, true)) return error;
    *bytes = workspace_bytes(m, k);
    return 0;
}

int nv_gemm_i8_silu(nv_context* c, const void* x, const void* residual, void* residual_out, const void* norm_weight,
                    const void* w, const void* w_scales, void* act, void* workspace, int m, int intermediate, int k,
                    float eps) {
    return product<true>(c, "gemm_i8_silu", x, residual, residual_out, norm_weight, w, w_scales, act, workspace, m,
                         intermediate, k, eps);
}

}  // extern "C"
