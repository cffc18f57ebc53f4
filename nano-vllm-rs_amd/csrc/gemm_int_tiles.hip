// Tiles of nv_gemm_i8 and nv_gemm_i8_silu (gemm_int.hip has the semantics).
#include "../../include/nano_hip.h"
#include "nvr_int8.h"
#include "nvr_internal.h"

namespace {

using nvr::kWave;
using nvr::Scale;
typedef int i32x4_t __attribute__((ext_vector_type(4)));
typedef int i32x16_t __attribute__((ext_vector_type(16)));

constexpr int kStep = 128;  // bytes of k a stage holds of each row
constexpr int kXcds = 8;

template <int BM_, int BN_, int WM_, int WN_>
struct Shape {
    static constexpr int BM = BM_, BN = BN_, WM = WM_, WN = WN_, WAVES = WM * WN, THREADS = WAVES * kWave;
    static constexpr int TM = BM / WM, TN = BN / WN, MI = TM / 32, NI = TN / 32;
    static constexpr int XR = BM / WAVES, WR = BN / WAVES;  // rows of each operand that a wave copies
    static constexpr int kStageBytes = (BM + BN) * kStep;
    static_assert(XR % 8 == 0 && WR % 8 == 0 && TM % 32 == 0 && TN % 32 == 0, "whole copies and products");
};

// The tile of a block: neighbours in a group of 4 tiles of tokens share an XCD, so that the 32 blocks that run there
// read few rows of either operand.
__device__ __forceinline__ int2 tile_of(unsigned block, unsigned blocks, int mt, int nt) {
    // Blocks go to XCDs in turn; each XCD takes a run of tiles.
    const unsigned xcd = block % kXcds, at = block / kXcds, whole = blocks / kXcds, more = blocks % kXcds;
    const unsigned tile = xcd * whole + min(xcd, more) + at;
    constexpr unsigned kGroup = 4;
    const unsigned per = kGroup * unsigned(nt), group = tile / per, in = tile % per;
    const unsigned rows = min(kGroup, unsigned(mt) - group * kGroup);
    return make_int2(int(group * kGroup + in % rows), int(in / rows));
}

template <class S, bool GATED>
__global__ __launch_bounds__(S::THREADS) void gemm_tiles(nvr::ProductArgs p, int mt, int nt) {
    extern __shared__ __align__(16) unsigned char smem[];
    const int lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int2 tile = tile_of(blockIdx.x, gridDim.x, mt, nt);
    const int64_t m0 = int64_t(tile.x) * S::BM;
    const int n0 = tile.y * (GATED ? S::BN / 2 : S::BN);  // < n
    const int steps = p.x_pitch / kStep;

    // Copies: a wave's instruction brings 8 rows of 128 bytes, 16 a lane, to LDS in order of lanes. The 16-byte piece c of
    // row r goes to place c ^ (r % 8) of its 8, so 8 rows' pieces of one column lie in 8 places.
    const int piece = (lane % 8) ^ (lane / 8);
    uint32_t xoff[S::XR / 8], woff[S::WR / 8];
#pragma unroll
    for (int u = 0; u < S::XR / 8; ++u) {
        const int64_t row = min(m0 + wave * S::XR + u * 8 + lane / 8, int64_t(p.m) - 1);
        xoff[u] = uint32_t(row - m0) * uint32_t(p.x_pitch) + piece * 16;
    }
    // Gated, every 32 rows of gate are followed by the 32 of up for the same channels.
    const bool up = GATED && (wave * S::WR / 32) % 2 != 0;
    static_assert(!GATED || 32 % S::WR == 0, "a wave copies rows of one kind");
#pragma unroll
    for (int u = 0; u < S::WR / 8; ++u) {
        const int r = wave * S::WR + u * 8 + lane / 8;
        const int row = min(n0 + (GATED ? r / 64 * 32 + r % 32 : r), p.n - 1);
        woff[u] = uint32_t(row - n0) * uint32_t(p.w_pitch) + piece * 16;
    }
    const uint8_t* xbase = p.xq + m0 * p.x_pitch;
    const uint8_t* wbase = p.wq + (int64_t(n0) + (up ? int64_t(p.n) : 0)) * p.w_pitch;
    const uint32_t lds = __builtin_amdgcn_readfirstlane(nvr::lds_address(smem));
    // Inline asm, so that the compiler, which would make every later LDS read wait for them, never sees the copies:
    // the waits below order them. M0 holds the LDS address and is restored.
    auto copy = [&](const uint8_t* base, uint32_t off, uint32_t dst) {
        uint32_t saved;
        asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %3\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2\n\ts_mov_b32 m0, %0"
                     : "=&s"(saved)
                     : "v"(off), "s"(base), "s"(dst)
                     : "memory");
    };
    auto stage = [&](int step) {
        const uint32_t dst = lds + (step & 1) * S::kStageBytes;
        if (step == steps - 1) {  // past its row a weight's bytes meet zeros of x: any byte of the row will do
            const int past = p.w_pitch - 16 - step * kStep;
            if (piece * 16 > past) {
#pragma unroll
                for (int u = 0; u < S::WR / 8; ++u) woff[u] += uint32_t(past - piece * 16);
            }
        }
#pragma unroll
        for (int u = 0; u < S::XR / 8; ++u)
            copy(xbase + step * kStep, xoff[u], dst + (wave * S::XR + u * 8) * kStep);
#pragma unroll
        for (int u = 0; u < S::WR / 8; ++u)
            copy(wbase + step * kStep, woff[u], dst + (S::BM + wave * S::WR + u * 8) * kStep);
    };

    // Operands: lane l has row l % 32, bytes 16 (l / 32) .. of each 32.
    const int wm = wave % S::WM, wn = wave / S::WM;
    const int read = lane % 32 * kStep + (((lane / 32) ^ (lane % 8)) << 4);
    auto operand = [&](const unsigned char* rows, int i, int ks) {
        return *reinterpret_cast<const i32x4_t*>(rows + i * 32 * kStep + (read ^ (ks << 5)));
    };
    i32x16_t acc[S::NI][S::MI];
#pragma unroll
    for (int i = 0; i < S::NI; ++i)
#pragma unroll
        for (int j = 0; j < S::MI; ++j) acc[i][j] = i32x16_t{};
    i32x4_t xf[2][S::MI], wf[2][S::NI];
    auto fetch = [&](int slot, int buffer, int ks) {
        const unsigned char* at = smem + buffer * S::kStageBytes;
#pragma unroll
        for (int i = 0; i < S::NI; ++i) wf[slot][i] = operand(at + (S::BM + wn * S::TN) * kStep, i, ks);
#pragma unroll
        for (int j = 0; j < S::MI; ++j) xf[slot][j] = operand(at + wm * S::TM * kStep, j, ks);
    };
    stage(0);
    asm volatile("s_waitcnt vmcnt(0)\n\ts_barrier" ::: "memory");
    if (steps > 1) stage(1);
    fetch(0, 0, 0);
    for (int step = 0; step < steps; ++step) {
#pragma unroll
        for (int ks = 0; ks < 4; ++ks) {
            if (ks < 3) {
                fetch((ks + 1) & 1, step & 1, ks + 1);
            } else if (step + 1 < steps) {
                // This stage is read and the next one here, in every wave: its place takes the one after.
                asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
                if (step + 2 < steps) stage(step + 2);
                fetch(0, (step + 1) & 1, 0);
            }
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int i = 0; i < S::NI; ++i)
#pragma unroll
                for (int j = 0; j < S::MI; ++j)
                    acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(wf[ks & 1][i], xf[ks & 1][j], acc[i][j], 0, 0, 0);
            __builtin_amdgcn_sched_barrier(0);
        }
    }

    // Lane l has token l % 32 of each 32, and channels 8 q + 4 (l / 32) + r, in its element 4 q + r.
#pragma unroll
    for (int j = 0; j < S::MI; ++j) {
        const int64_t token = m0 + wm * S::TM + j * 32 + lane % 32;
        if (token >= p.m) continue;
        const Scale xs = nvr::split_scale(p.xs[token]);
        uint16_t* row = p.y + token * p.n;
#pragma unroll
        for (int i = 0; i < S::NI; i += GATED ? 2 : 1) {
            const int first = n0 + (GATED ? (wn * S::TN + i * 32) / 2 : wn * S::TN + i * 32) + 4 * (lane / 32);
#pragma unroll
            for (int q = 0; q < 4; ++q) {
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int channel = first + 8 * q + r;
                    if (channel >= p.n) continue;
                    float y = nvr::scaled(acc[i][j][4 * q + r], xs, nvr::split_scale(p.ws[channel]));
                    if constexpr (GATED)
                        y = nvr::silu_mul(y, nvr::scaled(acc[i + 1][j][4 * q + r], xs,
                                                         nvr::split_scale(p.ws[int64_t(p.n) + channel])));
                    row[channel] = nvr::f32_to_bf16(y);
                }
            }
        }
    }
}

template <class S, bool GATED>
void launch(nv_context* c, const nvr::ProductArgs& p) {
    constexpr int kChannels = GATED ? S::BN / 2 : S::BN;
    const int mt = int((int64_t(p.m) + S::BM - 1) / S::BM), nt = (p.n + kChannels - 1) / kChannels;
    hipLaunchKernelGGL((gemm_tiles<S, GATED>), dim3(unsigned(mt) * unsigned(nt)), dim3(S::THREADS), 2 * S::kStageBytes,
                       c->stream, p, mt, nt);
}

}  // namespace

namespace nvr {

void launch_product_tiles(nv_context* c, const ProductArgs& p, bool gated) {
    using Large = Shape<256, 256, 2, 4>;
    gated ? launch<Large, true>(c, p) : launch<Large, false>(c, p);
}

}  // namespace nvr
