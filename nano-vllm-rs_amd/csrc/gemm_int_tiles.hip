// Tiles of nv_gemm_i8 and nv_gemm_i8_silu (gemm_int.hip has the semantics).
#include "../../include/nano_hip.h"
#include "nvr_int8.h"
#include "nvr_internal.h"

namespace {

using nvr::kWave;
using nvr::Scale;
typedef int i32x4_t __attribute__((ext_vector_type(4)));
typedef int i32x16_t __attribute__((ext_vector_type(16)));

constexpr int kXcds = 8;

// A block's tile of BM tokens and BN channels (gated: BN / 2 of gate and of up), by WM x WN waves; STAGES stages in LDS of
// KB bytes of k of each row.
template <int BM_, int BN_, int WM_, int WN_, int KB_, int STAGES_>
struct Shape {
    static constexpr int BM = BM_, BN = BN_, WM = WM_, WN = WN_, KB = KB_, STAGES = STAGES_;
    static constexpr int WAVES = WM * WN, THREADS = WAVES * kWave;
    static constexpr int TM = BM / WM, TN = BN / WN, MI = TM / 32, NI = TN / 32;  // a wave's products of 32 x 32
    static constexpr int SUB = KB / 32;                                          // products' depths in a stage
    static constexpr int PIECES = KB / 16, ROWS = kWave / PIECES;                // of a copy: pieces of a row, rows
    static constexpr int XR = BM / WAVES, WR = BN / WAVES;                       // rows that a wave copies
    static constexpr int COPIES = (XR + WR) / ROWS;                              // instructions of a wave a stage
    static constexpr int kStageBytes = (BM + BN) * KB;
    static_assert(XR % ROWS == 0 && WR % ROWS == 0 && TM % 32 == 0 && TN % 32 == 0, "whole copies and products");
    static_assert(STAGES * kStageBytes <= 160 * 1024 && (KB == 64 || KB == 128), "LDS");
};

// Waits until all but the last `late` stages' copies of this wave have landed.
template <class S>
__device__ __forceinline__ void wait_stages(int late) {
    static_assert(S::STAGES <= 6 && (S::STAGES - 2) * S::COPIES < 64, "vmcnt");
    switch (late) {
        case 0: asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); break;
        case 1: asm volatile("s_waitcnt vmcnt(%0)" ::"n"(S::COPIES) : "memory"); break;
        case 2: asm volatile("s_waitcnt vmcnt(%0)" ::"n"(2 * S::COPIES) : "memory"); break;
        case 3: asm volatile("s_waitcnt vmcnt(%0)" ::"n"(3 * S::COPIES) : "memory"); break;
        default: asm volatile("s_waitcnt vmcnt(%0)" ::"n"(4 * S::COPIES) : "memory"); break;
    }
}

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
    const int steps = (p.w_pitch + S::KB - 1) / S::KB;  // x holds zeros to the end of the last

    // Copies: a wave's instruction brings ROWS rows of KB bytes, 16 a lane, to LDS in order of lanes. The 16-byte piece c
    // of row r goes to place c ^ (r / 2 % 8) (of 4 places: c ^ (r / 4 % 4)), so that 16 rows' pieces of one column lie in
    // different ones of the 64 banks.
    auto place = [](int r, int c) { return S::PIECES == 8 ? c ^ (r / 2 % 8) : c ^ (r / 4 % 4); };
    const int at = lane / S::PIECES;  // a copy's row of this lane
    auto piece = [&](int u) { return place(u * S::ROWS + at, lane % S::PIECES); };
    uint32_t xoff[S::XR / S::ROWS], woff[S::WR / S::ROWS];
#pragma unroll
    for (int u = 0; u < S::XR / S::ROWS; ++u) {
        const int64_t row = min(m0 + wave * S::XR + u * S::ROWS + at, int64_t(p.m) - 1);
        xoff[u] = uint32_t(row - m0) * uint32_t(p.x_pitch) + piece(u) * 16;
    }
    // Gated, every 32 rows of gate are followed by the 32 of up for the same channels.
    const bool up = GATED && (wave * S::WR / 32) % 2 != 0;
    static_assert(!GATED || 32 % S::WR == 0, "a wave copies rows of one kind");
#pragma unroll
    for (int u = 0; u < S::WR / S::ROWS; ++u) {
        const int r = wave * S::WR + u * S::ROWS + at;
        const int row = min(n0 + (GATED ? r / 64 * 32 + r % 32 : r), p.n - 1);
        woff[u] = uint32_t(row - n0) * uint32_t(p.w_pitch) + piece(u) * 16;
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
    auto stage = [&](int step, int buffer) {
        const uint32_t dst = lds + buffer * S::kStageBytes;
        const int past = p.w_pitch - 16 - step * S::KB;
        if (past < S::KB - 16) {  // the last: past its row a weight's bytes meet zeros of x, any bytes of the row will do
#pragma unroll
            for (int u = 0; u < S::WR / S::ROWS; ++u) woff[u] -= max(piece(u) * 16 - past, 0);
        }
#pragma unroll
        for (int u = 0; u < S::XR / S::ROWS; ++u)
            copy(xbase + step * S::KB, xoff[u], dst + (wave * S::XR + u * S::ROWS) * S::KB);
#pragma unroll
        for (int u = 0; u < S::WR / S::ROWS; ++u) copy(wbase + step * S::KB, woff[u], dst + (S::BM + wave * S::WR + u * S::ROWS) * S::KB);
    };

    // Operands: lane l has row l % 32, bytes 16 (l / 32) .. of each 32.
    const int wm = wave % S::WM, wn = wave / S::WM;
    const int read = lane % 32 * S::KB + place(lane % 32, lane / 32) * 16;
    auto operand = [&](const unsigned char* rows, int i, int ks) {
        return *reinterpret_cast<const i32x4_t*>(rows + i * 32 * S::KB + (read ^ (ks << 5)));
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
        for (int i = 0; i < S::NI; ++i) wf[slot][i] = operand(at + (S::BM + wn * S::TN) * S::KB, i, ks);
#pragma unroll
        for (int j = 0; j < S::MI; ++j) xf[slot][j] = operand(at + wm * S::TM * S::KB, j, ks);
    };
    for (int s = 0; s < S::STAGES && s < steps; ++s) stage(s, s);
    wait_stages<S>(min(steps, S::STAGES) - 1);
    asm volatile("s_barrier" ::: "memory");
    fetch(0, 0, 0);
    int buffer = 0;
    for (int step = 0; step < steps; ++step) {
        const int next = buffer + 1 == S::STAGES ? 0 : buffer + 1;
#pragma unroll
        for (int ks = 0; ks < S::SUB; ++ks) {
            if (ks + 1 < S::SUB) {
                fetch((ks + 1) & 1, buffer, ks + 1);
            } else if (step + 1 < steps) {
                // This stage is read and the next one here, in every wave: its place takes another.
                wait_stages<S>(min(steps - 2 - step, S::STAGES - 2));
                asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
                if (step + S::STAGES < steps) stage(step + S::STAGES, buffer);
                fetch(0, next, 0);
            }
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int i = 0; i < S::NI; ++i)
#pragma unroll
                for (int j = 0; j < S::MI; ++j)
                    acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(wf[ks & 1][i], xf[ks & 1][j], acc[i][j], 0, 0, 0);
            __builtin_amdgcn_sched_barrier(0);
        }
        buffer = next;
    }

    // Lane l has token l % 32 of each 32, and channels 8 q + 4 (l / 32) + r, in its element 4 q + r. A wave brings its
    // outputs through LDS, so that it stores rows of OUT channels.
    constexpr int OUT = GATED ? S::TN / 2 : S::TN, UNITS = OUT / 8;
    static_assert(S::WAVES * S::TM * OUT * 2 <= S::STAGES * S::kStageBytes, "a wave's outputs");
    static_assert(UNITS == 4 || UNITS == 8, "banks");
    auto unit = [](int r, int c) { return UNITS == 8 ? c ^ (r / 2 % 8) : c ^ (r / 4 % 4); };
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    unsigned char* mine = smem + wave * (S::TM * OUT * 2);
    const int64_t t0 = m0 + wm * S::TM;
    const int c0 = n0 + wn * OUT;
    float xs[S::MI];
    bool plain = true;
#pragma unroll
    for (int j = 0; j < S::MI; ++j) {
        xs[j] = p.xs[min(t0 + j * 32 + lane % 32, int64_t(p.m) - 1)];
        plain = plain && nvr::middling(xs[j]);
    }
    auto outputs = [&](auto scale) {
#pragma unroll
        for (int i = 0; i < S::NI; i += GATED ? 2 : 1) {
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int at = (GATED ? i / 2 : i) * 32 + 8 * q + 4 * (lane / 32);
                float ws[4], us[4];
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int channel = min(c0 + at + r, p.n - 1);
                    ws[r] = p.ws[channel];
                    if constexpr (GATED) us[r] = p.ws[int64_t(p.n) + channel];
                }
#pragma unroll
                for (int j = 0; j < S::MI; ++j) {
                    float y[4];
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        y[r] = scale(acc[i][j][4 * q + r], xs[j], ws[r]);
                        if constexpr (GATED) y[r] = nvr::silu_mul(y[r], scale(acc[i + 1][j][4 * q + r], xs[j], us[r]));
                    }
                    const int row = j * 32 + lane % 32;
                    *reinterpret_cast<uint2*>(mine + row * (OUT * 2) + unit(row, at / 8) * 16 + lane / 32 * 8) =
                        make_uint2(nvr::pack_bf16x2(y[0], y[1]), nvr::pack_bf16x2(y[2], y[3]));
                }
            }
        }
    };
#pragma unroll 1
    for (int c = lane; c < OUT; c += kWave) {
        plain = plain && nvr::middling(p.ws[min(c0 + c, p.n - 1)]);
        if constexpr (GATED) plain = plain && nvr::middling(p.ws[int64_t(p.n) + min(c0 + c, p.n - 1)]);
    }
    if (__all(plain)) outputs([](int sum, float x, float w) { return float(sum) * x * w; });
    else outputs([](int sum, float x, float w) { return nvr::scaled(sum, nvr::split_scale(x), nvr::split_scale(w)); });
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // its own region only
    auto store = [&](auto kind) {
        using T = decltype(kind);
        constexpr int PER = sizeof(T) / 2, LANES = OUT / PER, ROWS = kWave / LANES;
        const int c = lane % LANES * PER;
        if (c0 + c >= p.n) return;  // a T lies inside n or outside
#pragma unroll 4
        for (int r = lane / LANES; r < S::TM; r += ROWS) {
            if (t0 + r >= p.m) break;
            const T v = *reinterpret_cast<const T*>(mine + r * (OUT * 2) + unit(r, c / 8) * 16 + c % 8 * 2);
            *reinterpret_cast<T*>(p.y + (t0 + r) * p.n + c0 + c) = v;
        }
    };
    if (p.n % 8 == 0 && nvr::aligned(p.y, 16)) store(uint4{});
    else if (p.n % 2 == 0 && nvr::aligned(p.y, 4)) store(uint32_t{});
    else store(uint16_t{});
}

template <class S, bool GATED>
void launch(nv_context* c, const nvr::ProductArgs& p) {
    constexpr int kChannels = GATED ? S::BN / 2 : S::BN;
    const int mt = int((int64_t(p.m) + S::BM - 1) / S::BM), nt = (p.n + kChannels - 1) / kChannels;
    hipLaunchKernelGGL((gemm_tiles<S, GATED>), dim3(unsigned(mt) * unsigned(nt)), dim3(S::THREADS), S::STAGES * S::kStageBytes,
                       c->stream, p, mt, nt);
}

}  // namespace

namespace nvr {

void launch_product_tiles(nv_context* c, const ProductArgs& p, bool gated) {
    using Large = Shape<256, 256, 2, 4, 128, 2>;
    using Small = Shape<128, 128, 2, 2, 128, 2>;
    const int channels = gated ? 2 * p.n : p.n;
    const int64_t large = ((int64_t(p.m) + 255) / 256) * ((int64_t(channels) + 255) / 256);
    if (large >= c->cu_count) gated ? launch<Large, true>(c, p) : launch<Large, false>(c, p);
    else gated ? launch<Small, true>(c, p) : launch<Small, false>(c, p);
}

}  // namespace nvr
