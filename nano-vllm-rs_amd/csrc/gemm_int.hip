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
#include "../../include/nano_hip.h"
#include "nvr_int8.h"
#include "nvr_internal.h"

namespace {

using nvr::kWave;
using nvr::Scale;
using nvr::Tokens;
typedef int i32x4_t __attribute__((ext_vector_type(4)));
typedef int i32x16_t __attribute__((ext_vector_type(16)));

constexpr int kWaves = 8, kThreads = kWaves * kWave;
constexpr int kUnit = 8;     // steps of 64 bytes of k whose weights are in flight together
constexpr int kRowPad = 16;  // behind a token's row in LDS: 16 tokens' pieces of one column lie in different banks
constexpr int kFewTokens = 32;
constexpr int kKeptChunks = 8;       // a made token's row stays in registers: k <= 4096
constexpr int kMadeTokens = 32768;   // values that each block makes
constexpr int kMostLds = 160 * 1024;

// Where the tokens' integers come from: made by each block (of x, the norm, or the norm of the sum), or by a launch of
// quantize_rows, and then brought to LDS, or read where they are used.
enum class Source { kPlain, kNorm, kAddNorm, kCopied, kMemory };

struct RowsArgs {
    nvr::ProductArgs p;
    nvr::TokenArgs t;
    int parts;  // waves that share the k of a tile: 1, 2, 4 or 8
};

// LDS of a block: partial sums (parts > 1), scales, tokens.
template <int MT>
constexpr int kSumBytes = 2 * kWaves * MT * kWave * 16;
template <Source SRC, int MT>
int64_t rows_lds(int m, int x_pitch) {
    return kSumBytes<MT> + MT * 16 * 4 + (SRC == Source::kMemory ? 0 : int64_t(m) * (x_pitch + kRowPad));
}

// Few tokens: the weights stream through registers, once.
template <Source SRC, int MT, bool GATED>
__global__ __launch_bounds__(kThreads) void gemm_rows_i8(RowsArgs a) {
    constexpr bool kMade = SRC != Source::kCopied && SRC != Source::kMemory;
    constexpr int kChannels = GATED ? 8 : 16;  // of a tile: 16 rows of the weight, or 8 of gate, then 8 of up
    extern __shared__ __align__(16) unsigned char smem[];
    const nvr::ProductArgs& p = a.p;
    const int lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int i = lane % 16, g = lane / 16;
    const int parts = a.parts, groups = kWaves / parts, group = wave / parts, part = wave % parts;
    // A block's tiles lie side by side, so the pieces of y's rows fill lines in one XCD's L2.
    const int tiles = (p.n + kChannels - 1) / kChannels;
    const int first = int(int64_t(blockIdx.x) * tiles / gridDim.x);
    const int mine = int(int64_t(blockIdx.x + 1) * tiles / gridDim.x) - first;  // >= 1
    const int rounds = (mine + groups - 1) / groups;                            // the same in every wave
    // A wave's steps of each of its tiles: whole lines of 128 bytes.
    const int lines = p.x_pitch / 128, share = (lines + parts - 1) / parts;
    const int s0 = min(part * share, lines) * 2, s1 = min((part + 1) * share, lines) * 2;
    const int units = (share * 2 + kUnit - 1) / kUnit;

    i32x4_t* red = reinterpret_cast<i32x4_t*>(smem);                   // [2][kWaves][MT][64]
    float* xs = reinterpret_cast<float*>(smem + kSumBytes<MT>);        // [MT * 16]
    unsigned char* xq = reinterpret_cast<unsigned char*>(xs + MT * 16);  // [m][pitch]
    const int pitch = SRC == Source::kMemory ? p.x_pitch : p.x_pitch + kRowPad;

    // The weights of a unit: lane l has row l % 16, 16 bytes at 16 (l / 16) of each step. Behind a row's end, where x is
    // zero, and behind the wave's steps, which are not multiplied, any bytes of the row will do.
    struct Unit {
        uint4 w[kUnit];
        float ws[4];  // of the lane's outputs; with a tile's first unit
    };
    Unit unit[2];
    int ahead_round = 0, ahead = 0;  // the next unit to load
    auto load = [&](Unit& u) {
        const int tile = first + min(ahead_round * groups + group, mine - 1);
        const int64_t row = GATED ? int64_t(i < 8 ? 0 : p.n) + min(tile * 8 + i % 8, p.n - 1) : min(tile * 16 + i, p.n - 1);
        const uint8_t* w = p.wq + row * p.w_pitch;
        const int s = s0 + ahead * kUnit;
#pragma unroll
        for (int e = 0; e < kUnit; ++e) u.w[e] = nvr::load_stream(w + min((s + e) * 64 + 16 * g, p.w_pitch - 16));
        if (ahead == 0) {
#pragma unroll
            for (int r = 0; r < 4; ++r)
                u.ws[r] = GATED ? p.ws[int64_t(g < 2 ? 0 : p.n) + min(tile * 8 + 4 * (g % 2) + r, p.n - 1)]
                                : p.ws[min(tile * 16 + 4 * g + r, p.n - 1)];
        }
        if (++ahead == units) {
            ahead = 0;
            ++ahead_round;
        }
    };
    load(unit[0]);

    if constexpr (kMade) {
        constexpr Tokens T = SRC == Source::kPlain ? Tokens::kPlain : SRC == Source::kNorm ? Tokens::kNorm : Tokens::kAddNorm;
        for (int row = wave; row < p.m; row += kWaves) {
            const nvr::RowStep step = nvr::quantize_row<T, true, true, kKeptChunks, 1>(
                a.t, row, p.x_pitch, blockIdx.x == 0 && a.t.residual_out != nullptr, lane, 0, nvr::NoJoin{},
                [&](int j, uint2 eight) { *reinterpret_cast<uint2*>(xq + row * pitch + j) = eight; });
            if (lane == 0) xs[row] = step.scale;
        }
    } else {
        if constexpr (SRC == Source::kCopied) {
            const int pieces = p.x_pitch / 16;
            for (int at = threadIdx.x; at < p.m * pieces; at += kThreads)
                *reinterpret_cast<uint4*>(xq + at / pieces * pitch + at % pieces * 16) =
                    *reinterpret_cast<const uint4*>(p.xq + int64_t(at) * 16);
        }
        if (int(threadIdx.x) < p.m) xs[threadIdx.x] = p.xs[threadIdx.x];
    }
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");  // leaves the weights in flight

    // Tokens behind the last repeat it and are not stored.
    const unsigned char* xrow[MT];
#pragma unroll
    for (int t = 0; t < MT; ++t)
        xrow[t] = (SRC == Source::kMemory ? p.xq : xq) + int64_t(min(t * 16 + i, p.m - 1)) * pitch + 16 * g;
    i32x4_t acc[MT];
    float ws[4];
    int round = 0, at = 0;  // the unit to multiply
    // Lane l has token l % 16 of 16, rows 4 (l / 16) .. + 3 of the tile.
    auto finish = [&](int t, const i32x4_t& sum) {
        const int token = t * 16 + i, tile = round * groups + group;
        const Scale x = nvr::split_scale(xs[min(token, p.m - 1)]);
        float y[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            y[r] = nvr::scaled(sum[r], x, nvr::split_scale(ws[r]));
            if constexpr (GATED) y[r] = nvr::silu_mul(y[r], nvr::xor_lane(y[r], 32));  // the other half has the up rows
        }
        if (tile >= mine || token >= p.m || (GATED && g >= 2)) return;
        const int channel = (first + tile) * kChannels + 4 * (GATED ? g % 2 : g);
        uint16_t* out = p.y + int64_t(token) * p.n + channel;
        if (p.n % 4 == 0 && nvr::aligned(p.y, 8)) {
            if (channel < p.n)
                *reinterpret_cast<uint2*>(out) = make_uint2(nvr::pack_bf16x2(y[0], y[1]), nvr::pack_bf16x2(y[2], y[3]));
        } else {
#pragma unroll
            for (int r = 0; r < 4; ++r)
                if (channel + r < p.n) out[r] = nvr::f32_to_bf16(y[r]);
        }
    };
    auto multiply = [&](const Unit& u) {
        if (at == 0) {
#pragma unroll
            for (int t = 0; t < MT; ++t) acc[t] = i32x4_t{0, 0, 0, 0};
#pragma unroll
            for (int r = 0; r < 4; ++r) ws[r] = u.ws[r];
        }
        const int s = s0 + at * kUnit;
#pragma unroll
        for (int e = 0; e < kUnit; ++e) {
            if (s + e >= s1) break;
#pragma unroll
            for (int t = 0; t < MT; ++t)
                acc[t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i32x4_t, u.w[e]),
                                                               *reinterpret_cast<const i32x4_t*>(xrow[t] + (s + e) * 64),
                                                               acc[t], 0, 0, 0);
        }
        if (++at < units) return;
        if (parts == 1) {
#pragma unroll
            for (int t = 0; t < MT; ++t) finish(t, acc[t]);
        } else {
            i32x4_t* sums = red + (round & 1) * (kWaves * MT * kWave) + lane;
#pragma unroll
            for (int t = 0; t < MT; ++t) sums[(wave * MT + t) * kWave] = acc[t];
            asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
#pragma unroll
            for (int t = 0; t < MT; ++t) {
                if ((round * MT + t) % parts != part) continue;  // the waves take turns
                i32x4_t sum = sums[(group * parts * MT + t) * kWave];
                for (int q = 1; q < parts; ++q) sum += sums[((group * parts + q) * MT + t) * kWave];
                finish(t, sum);
            }
        }
        at = 0;
        ++round;
    };
    const int total = rounds * units;
    for (int u = 0; u < total; u += 2) {
        if (u + 1 < total) load(unit[1]);
        multiply(unit[0]);
        if (u + 1 >= total) break;
        if (u + 2 < total) load(unit[0]);
        multiply(unit[1]);
    }
}

template <Source SRC, int MT, bool GATED>
void launch_rows_as(nv_context* c, const RowsArgs& a, int blocks) {
    hipLaunchKernelGGL((gemm_rows_i8<SRC, MT, GATED>), dim3(unsigned(blocks)), dim3(kThreads),
                       size_t(rows_lds<SRC, MT>(a.p.m, a.p.x_pitch)), c->stream, a);
}

template <Source SRC, bool GATED>
void launch_rows(nv_context* c, RowsArgs a) {
    const int tiles = (a.p.n + (GATED ? 8 : 16) - 1) / (GATED ? 8 : 16);
    const int cus = c->cu_count > 0 ? c->cu_count : 256;
    const int units = (a.p.x_pitch / 64 + kUnit - 1) / kUnit;
    a.parts = 8;
    while (a.parts > 1 && (units * 2 <= a.parts || int64_t(tiles) * a.parts > int64_t(cus) * kWaves * 4)) a.parts /= 2;
    const int blocks = std::min(cus, (tiles * a.parts + kWaves - 1) / kWaves);
    a.p.m <= 16 ? launch_rows_as<SRC, 1, GATED>(c, a, blocks) : launch_rows_as<SRC, 2, GATED>(c, a, blocks);
}

// Whether each block makes the tokens' integers by itself: they fit its LDS and registers, and are few enough.
bool tokens_in_block(const nvr::TokenArgs& t) {
    return t.k <= kKeptChunks * nvr::kWaveChunk && nvr::tokens_aligned(t) && int64_t(t.rows) * t.k <= kMadeTokens;
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
    const RowsArgs few{p, t, 0};
    if (m <= kFewTokens && tokens_in_block(t)) {
        if (norm_weight == nullptr) launch_rows<Source::kPlain, GATED>(c, few);
        else if (residual == nullptr) launch_rows<Source::kNorm, GATED>(c, few);
        else launch_rows<Source::kAddNorm, GATED>(c, few);
        return nvr::launch_status();
    }
    nvr::launch_quantize(c, t, xq, xs, pitch);
    if (m > kFewTokens) nvr::launch_product_tiles(c, p, GATED);
    else if ((m <= 16 ? rows_lds<Source::kCopied, 1>(m, pitch) : rows_lds<Source::kCopied, 2>(m, pitch)) <= kMostLds)
        launch_rows<Source::kCopied, GATED>(c, few);
    else launch_rows<Source::kMemory, GATED>(c, few);
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
