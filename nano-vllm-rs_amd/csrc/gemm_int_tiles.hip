// Tiles of nv_gemm_i8 and nv_gemm_i8_silu (gemm_int.hip has the semantics). No counterpart in the reference
// (kernels/kernels.cu:98-106 calls a library's bf16 product).
//
// gemm_tiles is bound by the matrix units' power: products of random integers alone, from registers, run at 4.0 POPS in
// 16 x 16 x 64 and 3.35 in 32 x 32 x 32 (the same work a cycle, more energy), with their operands' LDS reads at 3.4 and 3.0,
// at clocks near 1.8 GHz; of constant data at 4.9. Therefore 16 x 16 x 64 (8192 tokens over 12288 x 4096 349 us for 380), and
// tiles of 256 x 256, whose operands are read from LDS 64 rows for 128, the largest that registers hold beside two depths of
// operands. 8192 over 12288 x 4096 takes 350 us, 2.36 POPS; the library's product without scales, in raw 32-bit integers,
// 389 us, and at 8192 x 8192 x 8192 2.07 POPS.
//   The two stages of 128 bytes of k take 128 KB of LDS. Three or four stages of 64 bytes, whose barriers come twice as often,
//   380 us for 349. A depth's operands are read one depth ahead, a read between two products, so that the units never wait.
//   Outputs go through LDS, so that a store writes whole rows of 128 bytes: 8 bytes a lane into 16 rows at once 631 us for
//   393. Products with their operands' reads alone would take 241 us. Of the 108 over them 53 do not grow with k (k 2048,
//   4096, 8192 199, 349, 635 us): the first stage's way to LDS and the outputs, in each of 6 turns. The others, in the loop,
//   are its barriers, copies and waits, not told apart.
#include "../../include/nano_hip.h"
#include "nvr_int8.h"
#include "nvr_internal.h"

namespace {

using nvr::kWave;
using nvr::Scale;
typedef int i32x4_t __attribute__((ext_vector_type(4)));

// A block's tile of BM tokens and BN channels (gated: BN / 2 of gate and of up), by WM x WN waves; STAGES stages in LDS of
// KB bytes of k of each row.
template <int BM_, int BN_, int WM_, int WN_, int STAGES_>
struct Shape {
    static constexpr int BM = BM_, BN = BN_, WM = WM_, WN = WN_, KB = 128, STAGES = STAGES_;
    static constexpr int WAVES = WM * WN, THREADS = WAVES * kWave;
    static constexpr int TM = BM / WM, TN = BN / WN, MI = TM / 16, NI = TN / 16;  // a wave's products of 16 x 16
    static constexpr int SUB = KB / 64;                                          // products' depths of a stage
    static constexpr int PIECES = KB / 16, ROWS = kWave / PIECES;                // of a copy: pieces of a row, rows
    static constexpr int XR = BM / WAVES, WR = BN / WAVES;                       // rows that a wave copies
    static constexpr int COPIES = (XR + WR) / ROWS;                              // instructions of a wave a stage
    static constexpr int kStageBytes = (BM + BN) * KB;
    static constexpr int kLds = STAGES * kStageBytes + (BM + BN) * 4;            // and the scales
    static_assert(XR % ROWS == 0 && WR % ROWS == 0 && TM % 16 == 0 && TN % 32 == 0, "whole copies and products");
    static_assert(kLds <= 160 * 1024, "LDS");
};

// Waits until all but the last `late` stages' copies of this wave have landed.
template <class S>
__device__ __forceinline__ void wait_stages(int late) {
    constexpr int C = S::COPIES;
    static_assert(S::STAGES <= 3 && (S::STAGES - 1) * C < 64, "vmcnt");
    if (late == 0) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    else if (S::STAGES == 2 || late == 1) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(C) : "memory");
    else asm volatile("s_waitcnt vmcnt(%0)" ::"n"(2 * C) : "memory");
}

// The tile of a block: neighbours in a group of 4 tiles of tokens share an XCD, so that the 32 blocks that run there
// read few rows of either operand.
__device__ __forceinline__ int2 tile_of(unsigned block, unsigned blocks, int mt, int nt) {
    // Blocks go to XCDs in turn; each XCD takes a run of tiles.
    const unsigned xcd = block % nvr::kXcds, at = block / nvr::kXcds, whole = blocks / nvr::kXcds, more = blocks % nvr::kXcds;
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
    // of row r goes to place c ^ (r / 2 % 8), so that 16 rows' pieces of one column lie in different ones of the 64 banks.
    static_assert(S::PIECES == 8, "place");
    auto place = [](int r, int c) { return c ^ (r / 2 % 8); };
    const int at = lane / S::PIECES;  // a copy's row of this lane
    auto piece = [&](int rows, int u) { return place(wave * rows + u * S::ROWS + at, lane % S::PIECES); };
    uint32_t xoff[S::XR / S::ROWS], woff[S::WR / S::ROWS];
#pragma unroll
    for (int u = 0; u < S::XR / S::ROWS; ++u) {
        const int64_t row = min(m0 + wave * S::XR + u * S::ROWS + at, int64_t(p.m) - 1);
        xoff[u] = uint32_t(row - m0) * uint32_t(p.x_pitch) + piece(S::XR, u) * 16;
    }
    // Gated, every 32 rows of gate are followed by the 32 of up for the same channels.
    const bool up = GATED && (wave * S::WR / 32) % 2 != 0;
    static_assert(!GATED || 32 % S::WR == 0, "a wave copies rows of one kind");
#pragma unroll
    for (int u = 0; u < S::WR / S::ROWS; ++u) {
        const int r = wave * S::WR + u * S::ROWS + at;
        const int row = min(n0 + (GATED ? r / 64 * 32 + r % 32 : r), p.n - 1);
        woff[u] = uint32_t(row - n0) * uint32_t(p.w_pitch) + piece(S::WR, u) * 16;
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
            for (int u = 0; u < S::WR / S::ROWS; ++u) woff[u] -= max(piece(S::WR, u) * 16 - past, 0);
        }
#pragma unroll
        for (int u = 0; u < S::XR / S::ROWS; ++u)
            copy(xbase + step * S::KB, xoff[u], dst + (wave * S::XR + u * S::ROWS) * S::KB);
#pragma unroll
        for (int u = 0; u < S::WR / S::ROWS; ++u)
            copy(wbase + step * S::KB, woff[u], dst + (S::BM + wave * S::WR + u * S::ROWS) * S::KB);
    };

    // Operands: lane l has row l % 16, bytes 16 (l / 16) .. of each 64.
    const int wm = wave % S::WM, wn = wave / S::WM;
    const int lane_at = lane % 16 * S::KB + place(lane % 16, lane / 16) * 16;
    auto operand = [&](const unsigned char* rows, int i, int ks) {
        return *reinterpret_cast<const i32x4_t*>(rows + i * 16 * S::KB + (lane_at ^ (ks << 6)));
    };
    i32x4_t acc[S::NI][S::MI];
#pragma unroll
    for (int i = 0; i < S::NI; ++i)
#pragma unroll
        for (int j = 0; j < S::MI; ++j) acc[i][j] = i32x4_t{0, 0, 0, 0};
    // Operands of two depths: those of the next are read while the products of one are formed, a read before a product.
    constexpr int READS = S::NI + S::MI, PRODUCTS = S::NI * S::MI;
    i32x4_t xf[2][S::MI], wf[2][S::NI];
    auto fetch = [&](int slot, const unsigned char* stage_at, int ks, int r) {  // the r-th operand
        if (r == 0) wf[slot][0] = operand(stage_at + (S::BM + wn * S::TN) * S::KB, 0, ks);
        else if (r <= S::MI) xf[slot][r - 1] = operand(stage_at + wm * S::TM * S::KB, r - 1, ks);
        else wf[slot][r - S::MI] = operand(stage_at + (S::BM + wn * S::TN) * S::KB, r - S::MI, ks);
    };
    auto product = [&](int slot, int q) {
        const int i = q / S::MI, j = q % S::MI;
        acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wf[slot][i], xf[slot][j], acc[i][j], 0, 0, 0);
    };
    // The scales come first, so that no epilogue waits for them: [BM] of tokens, [BN] of channels (gated: half of gate, half
    // of up).
    float* scales = reinterpret_cast<float*>(smem + S::STAGES * S::kStageBytes);
    for (int i = threadIdx.x; i < S::BM + S::BN; i += S::THREADS) {
        const int c = i - S::BM, half = GATED ? S::BN / 2 : S::BN;
        scales[i] = c < 0 ? p.xs[min(m0 + i, int64_t(p.m) - 1)]
                          : p.ws[(c < half ? 0 : int64_t(p.n)) + min(n0 + (c < half ? c : c - half), p.n - 1)];
    }
    for (int s = 0; s < S::STAGES && s < steps; ++s) stage(s, s);
    wait_stages<S>(min(steps, S::STAGES) - 1);
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
#pragma unroll
    for (int r = 0; r < READS; ++r) fetch(0, smem, 0, r);
    int buffer = 0;
    for (int step = 0; step < steps; ++step) {
        const int next = buffer + 1 == S::STAGES ? 0 : buffer + 1;
#pragma unroll
        for (int ks = 0; ks < S::SUB; ++ks) {
            const bool last = ks + 1 == S::SUB;
            const int slot = ks & 1;
            static_assert(S::SUB == 2, "slots");
            const int first = last ? PRODUCTS / 2 : 0;
            if (last) {
#pragma unroll
                for (int q = 0; q < first; ++q) product(slot, q);
                __builtin_amdgcn_sched_barrier(0);
                if (step + 1 < steps) {
                    // This stage is read and the next one here, in every wave: its place takes another.
                    wait_stages<S>(min(steps - 2 - step, S::STAGES - 2));
                    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
                    if (step + S::STAGES < steps) stage(step + S::STAGES, buffer);
                }
            }
            // Behind the last stage: what lies in LDS is read and not used.
            const unsigned char* at = smem + (last ? next : buffer) * S::kStageBytes;
#pragma unroll
            for (int q = 0; q < std::max(READS, PRODUCTS - first); ++q) {
                if (q < READS) fetch(slot ^ 1, at, last ? 0 : ks + 1, q);
                if (first + q < PRODUCTS) product(slot, first + q);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        buffer = next;
    }

    // Lane l has token l % 16 of each 16, and channels 4 (l / 16) .. + 3 of each 16. A wave brings its outputs through LDS,
    // so that it stores rows of OUT channels.
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
        xs[j] = scales[wm * S::TM + j * 16 + lane % 16];
        plain = plain && nvr::middling(xs[j]);
    }
    const float* wscales = scales + S::BM + wn * OUT;
    if (lane < OUT) {
        plain = plain && nvr::middling(wscales[lane]);
        if constexpr (GATED) plain = plain && nvr::middling(wscales[S::BN / 2 + lane]);
    }
    auto outputs = [&](auto scale) {
#pragma unroll
        for (int o = 0; o < OUT / 16; ++o) {
            const int i = GATED ? o / 2 * 4 + o % 2 : o;  // gated: 32 rows of gate, 32 of up
            const int at = o * 16 + 4 * (lane / 16);
            float ws[4], us[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                ws[r] = wscales[at + r];
                us[r] = GATED ? wscales[S::BN / 2 + at + r] : 0.0f;
            }
#pragma unroll
            for (int j = 0; j < S::MI; ++j) {
                float y[4];
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    y[r] = scale(acc[i][j][r], xs[j], ws[r]);
                    if constexpr (GATED) y[r] = nvr::gated(y[r], scale(acc[i + 2][j][r], xs[j], us[r]));
                }
                const int row = j * 16 + lane % 16;
                *reinterpret_cast<uint2*>(mine + row * (OUT * 2) + unit(row, at / 8) * 16 + at % 8 * 2) =
                    make_uint2(nvr::pack_bf16x2(y[0], y[1]), nvr::pack_bf16x2(y[2], y[3]));
            }
        }
    };
    if (__all(plain)) outputs([](int sum, float x, float w) { return float(sum) * x * w; });
    else outputs([](int sum, float x, float w) { return nvr::scaled(sum, nvr::split_scale(x), nvr::split_scale(w)); });
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // its own region only
    constexpr int ROWS = kWave / UNITS;
    const int c = lane % UNITS * 8;
#pragma unroll 4
    for (int r = lane / UNITS; r < S::TM; r += ROWS) {
        if (t0 + r >= p.m) break;
        const unsigned char* at = mine + r * (OUT * 2) + unit(r, c / 8) * 16;
        uint16_t* out = p.y + (t0 + r) * p.n + c0 + c;
        if (c0 + c + 8 <= p.n) {
            nvr::store8(out, *reinterpret_cast<const uint4*>(at));
        } else {
            for (int e = 0; e < 8 && c0 + c + e < p.n; ++e) out[e] = *reinterpret_cast<const uint16_t*>(at + 2 * e);
        }
    }
}

// Fewer tokens: tiles of TOK tokens by SIDE rows of the weight (gated: half of gate, half of up), a wave for every fourth
// unit of 128 bytes of k. A wave copies and reads its units by itself, SLOTS of them in LDS, so the loop has no barrier; each
// byte of LDS is read once, where four waves side by side would read it twice, and one group's products cover the next one's
// reads. Bound by the copies: what a CU brings to LDS from L2 (110 to 130 bytes a ns; 27 from beyond), or by their
// latency: 16 tokens over 4096 x 12288, 50 MB of cold weights, 16.6 us with the tokens' launch, 3.0 TB/s. 100 over 6144 x 4096
// 11.4 us without it, 5.1 of them at any k (the launch, first copies, the waves' sums, outputs); the others are 84 bytes a ns
// a CU, with cold weights 61.
constexpr int kUnitBytes = 128, kSplit = 4, kSplitThreads = kSplit * kWave;

template <int TOK, int SIDE, int SLOTS, bool GATED>
__global__ __launch_bounds__(kSplitThreads) void gemm_split(nvr::ProductArgs p, int mt, int nt) {
    extern __shared__ __align__(16) unsigned char smem[];
    const int lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int2 tile = tile_of(blockIdx.x, gridDim.x, mt, nt);
    const int64_t m0 = int64_t(tile.x) * TOK;
    const int n0 = tile.y * (GATED ? SIDE / 2 : SIDE);  // < n
    constexpr bool kHalves = GATED && SIDE == 16;  // a product's 16 rows are 8 of gate, then 8 of up
    constexpr int NI = SIDE / 16, MJ = TOK / 16, SLOT = (TOK + SIDE) * kUnitBytes;
    const int units = (p.w_pitch + kUnitBytes - 1) / kUnitBytes;  // x holds zeros to the end of the last
    const int mine = (units - wave + kSplit - 1) / kSplit;        // wave, wave + 4, ...

    // A copy brings 8 rows of 128 bytes; the piece c of row r goes to place c ^ (r / 2 % 8), as in gemm_tiles.
    auto place = [](int r, int c) { return c ^ (r / 2 % 8); };
    constexpr int XC = TOK / 8, WC = SIDE / 8;
    uint32_t xoff[XC], woff[WC];
#pragma unroll
    for (int u = 0; u < XC; ++u) {
        const int r = u * 8 + lane / 8;
        xoff[u] = uint32_t(min(m0 + r, int64_t(p.m) - 1) - m0) * uint32_t(p.x_pitch) + place(r, lane % 8) * 16;
    }
#pragma unroll
    for (int u = 0; u < WC; ++u) {
        const int r = u * 8 + lane / 8;
        const int row = min(n0 + (GATED ? r % (SIDE / 2) : r), p.n - 1);
        woff[u] = uint32_t(row - n0) * uint32_t(p.w_pitch) + place(r, lane % 8) * 16;
    }
    const uint8_t* xbase = p.xq + m0 * p.x_pitch;
    const uint8_t* wbase = p.wq + int64_t(n0) * p.w_pitch;
    const uint8_t* ubase = GATED ? wbase + int64_t(p.n) * p.w_pitch : wbase;  // of the tile's upper half
    const uint32_t lds = __builtin_amdgcn_readfirstlane(nvr::lds_address(smem)) + wave * (SLOTS * SLOT);
    // Two copies to places of 1 KB side by side; inline asm for the reasons given in gemm_tiles.
    auto copy2 = [&](const uint8_t* base, uint32_t off0, uint32_t off1, uint32_t dst) {
        uint32_t saved;
        asm volatile(
            "s_mov_b32 %0, m0\n\ts_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %3, %1\n\t"
            "s_add_u32 m0, m0, 0x400\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %4, %1\n\ts_mov_b32 m0, %0"
            : "=&s"(saved)
            : "s"(base), "s"(dst), "v"(off0), "v"(off1)
            : "memory", "scc");
    };
    auto copy1 = [&](const uint8_t* base, uint32_t off, uint32_t dst) {
        uint32_t saved;
        asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %3, %1\n\ts_mov_b32 m0, %0"
                     : "=&s"(saved)
                     : "s"(base), "s"(dst), "v"(off)
                     : "memory");
    };
    auto copy = [&](int i) {  // this wave's i-th unit
        const int k = (wave + i * kSplit) * kUnitBytes;
        const uint32_t dst = lds + i % SLOTS * SLOT;
        const int past = p.w_pitch - 16 - k;
        if (past < kUnitBytes - 16) {  // past its row a weight's bytes meet zeros of x: any bytes of the row will do
#pragma unroll
            for (int u = 0; u < WC; ++u) woff[u] -= max(place(u * 8 + lane / 8, lane % 8) * 16 - past, 0);
        }
#pragma unroll
        for (int u = 0; u < XC; u += 2) copy2(xbase + k, xoff[u], xoff[u + 1], dst + u * 1024);
        if constexpr (kHalves) {
            copy1(wbase + k, woff[0], dst + XC * 1024);
            copy1(ubase + k, woff[1], dst + (XC + 1) * 1024);
        } else {
#pragma unroll
            for (int u = 0; u < WC; u += 2)
                copy2((u < WC / 2 ? wbase : ubase) + k, woff[u], woff[u + 1], dst + (XC + u) * 1024);
        }
    };
    const int lane_at = lane % 16 * kUnitBytes + place(lane % 16, lane / 16) * 16;
    const unsigned char* ring = smem + wave * (SLOTS * SLOT);
    struct Operands {
        i32x4_t x[MJ], w[NI];
    };
    auto fetch = [&](Operands& o, int i, int ks) {
        const unsigned char* at = ring + i % SLOTS * SLOT + (lane_at ^ (ks << 6));
#pragma unroll
        for (int j = 0; j < MJ; ++j) o.x[j] = *reinterpret_cast<const i32x4_t*>(at + j * 2048);
#pragma unroll
        for (int i16 = 0; i16 < NI; ++i16) o.w[i16] = *reinterpret_cast<const i32x4_t*>(at + (MJ + i16) * 2048);
    };
    i32x4_t acc[NI][MJ];
#pragma unroll
    for (int i = 0; i < NI; ++i)
#pragma unroll
        for (int j = 0; j < MJ; ++j) acc[i][j] = i32x4_t{0, 0, 0, 0};
    auto products = [&](const Operands& o) {
#pragma unroll
        for (int i = 0; i < NI; ++i)
#pragma unroll
            for (int j = 0; j < MJ; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(o.w[i], o.x[j], acc[i][j], 0, 0, 0);
        __builtin_amdgcn_sched_barrier(0);
    };
    auto landed = [&](int late) {  // this wave's copies, but those of the last `late` units
        constexpr int C = XC + WC;
        static_assert((SLOTS == 2 || SLOTS == 4) && (SLOTS - 1) * C < 64, "vmcnt");
        if (late == 0) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        else if (SLOTS == 2 || late == 1) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(C) : "memory");
        else if (late == 2) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(2 * C) : "memory");
        else asm volatile("s_waitcnt vmcnt(%0)" ::"n"(SLOTS == 2 ? 0 : 3 * C) : "memory");
    };
    Operands a, b;
    if (mine > 0) {
        for (int i = 0; i < SLOTS && i < mine; ++i) copy(i);
        landed(min(mine, SLOTS) - 1);
        fetch(a, 0, 0);
        for (int i = 0; i < mine; ++i) {
            fetch(b, i, 1);
            __builtin_amdgcn_sched_barrier(0);
            products(a);
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the unit is read
            if (i + SLOTS < mine) copy(i + SLOTS);
            if (i + 1 < mine) {
                landed(min(mine - i - 2, SLOTS - 1));
                fetch(a, i + 1, 0);
            }
            __builtin_amdgcn_sched_barrier(0);
            products(b);
        }
    }
    // The waves' sums, of 16 tokens by 16 rows (gated: and the 16 of up), each in one wave.
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    i32x4_t* sums = reinterpret_cast<i32x4_t*>(smem) + lane;  // [wave][16 tokens][16 rows][64]
    static_assert(MJ * NI * kWave * 16 <= SLOTS * SLOT, "its place");
#pragma unroll
    for (int j = 0; j < MJ; ++j)
#pragma unroll
        for (int i = 0; i < NI; ++i) sums[((wave * MJ + j) * NI + i) * kWave] = acc[i][j];
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    constexpr int OI = GATED && !kHalves ? NI / 2 : NI;  // a token's 16 channels (8)
#pragma unroll
    for (int at = 0; at < MJ * OI; at += kSplit) {
        const int q = at + wave, j = q / OI, i = q % OI;
        if (q >= MJ * OI) break;
        auto whole = [&](int row16) {
            i32x4_t part[kSplit];
#pragma unroll
            for (int v = 0; v < kSplit; ++v) part[v] = sums[((v * MJ + j) * NI + row16) * kWave];
            return part[0] + part[1] + (part[2] + part[3]);
        };
        static_assert(kSplit == 4, "whole");
        const i32x4_t sum = whole(i), up = GATED && !kHalves ? whole(i + NI / 2) : sum;
        const int64_t token = m0 + j * 16 + lane % 16;
        const int channel = n0 + i * 16 + 4 * (kHalves ? lane / 16 % 2 : lane / 16);
        const float* ws = p.ws + (kHalves && lane >= 32 ? int64_t(p.n) : 0);
        const Scale xs = nvr::split_scale(p.xs[min(token, int64_t(p.m) - 1)]);
        float y[4], u[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) {  // all scales are asked for before the first gate's branch
            const int c = min(channel + r, p.n - 1);
            y[r] = nvr::scaled(sum[r], xs, nvr::split_scale(ws[c]));
            if constexpr (kHalves) u[r] = nvr::xor_lane(y[r], 32);  // the other half has the up rows
            else if constexpr (GATED) u[r] = nvr::scaled(up[r], xs, nvr::split_scale(p.ws[int64_t(p.n) + c]));
        }
        if constexpr (GATED) {
#pragma unroll
            for (int r = 0; r < 4; ++r) y[r] = nvr::gated(y[r], u[r]);
        }
        if (token >= p.m || (kHalves && lane >= 32)) continue;
        nvr::store_outputs(p.y + token * p.n + channel, y, channel, p.n);
    }
}

// A grid dimension holds fewer than 2^32 work-items.
int refuse_grid(int64_t mt, int64_t nt, int threads) {
    if (mt * nt < (int64_t(1) << 32) / threads) return 0;
    return nvr::fail(-2, "gemm_i8: %lld tiles of tokens by %lld of channels are more than one launch", (long long)mt,
                     (long long)nt);
}

template <class S, bool GATED>
int launch(nv_context* c, const nvr::ProductArgs& p, bool check) {
    constexpr int kChannels = GATED ? S::BN / 2 : S::BN;
    const int mt = int((int64_t(p.m) + S::BM - 1) / S::BM), nt = (p.n + kChannels - 1) / kChannels;
    if (check) return refuse_grid(mt, nt, S::THREADS);
    hipLaunchKernelGGL((gemm_tiles<S, GATED>), dim3(unsigned(mt) * unsigned(nt)), dim3(S::THREADS), S::kLds, c->stream, p, mt,
                       nt);
    return nvr::launch_status();
}

template <int TOK, int SIDE, int SLOTS, bool GATED>
int launch_split(nv_context* c, const nvr::ProductArgs& p, bool check) {
    constexpr int kChannels = GATED ? SIDE / 2 : SIDE;
    const int mt = int((int64_t(p.m) + TOK - 1) / TOK), nt = (p.n + kChannels - 1) / kChannels;
    if (check) return refuse_grid(mt, nt, kSplitThreads);
    hipLaunchKernelGGL((gemm_split<TOK, SIDE, SLOTS, GATED>), dim3(unsigned(mt) * unsigned(nt)), dim3(kSplitThreads),
                       kSplit * SLOTS * (TOK + SIDE) * kUnitBytes, c->stream, p, mt, nt);
    return nvr::launch_status();
}

}  // namespace

namespace nvr {

// The tile by tokens and by turns: how often the CUs are filled. On MI355X, weights cold, in us, first of whole calls:
//   tiles of 16 rows of the weight while there is at most one a CU, against 32 rows, which leave half of the CUs without:
//   16 tokens over 4096 at k 2056, 4104, 12288 7.6, 9.6, 17.0 and 8.4, 11.2, 20.7; over 6144 (more than one) 9.0, 12.7, 25.4
//   and 8.8, 12.0, 23.6; 32 tokens over 4096 at k 4104 11.1, 12.5; 64 12.8, 14.9; 256 over 1000 at k 1030 6.7, 7.7. Few
//   such tokens are latency: four units of k in LDS instead of two, 16 over 1024 at k 12288 13.3, 14.7; 64 tokens
//   by two over 1024 at k 4104 10.4, by three 10.7. Eight waves for a tile's k: 32 over 4096 at k 8192 14.8,
//   four 14.7; over 200 9.9, 10.6. Gated, 8 rows of gate and of up against 16: 32 over 1376 at k 4104 10.5, 12.1; over 2048 at
//   k 1111 7.0, 7.3.
// Of the product alone:
//   a tile's k over four waves while there is a tile a CU: 256 tokens over 1024 x 2048 by tiles of 64 x 32, 64 x 64 and
//   128 x 128 5.2, 7.3, 11.2; 100 over 6144 x 4096 13.1 (in two turns), 10.9, 15.2; 512 over 4096 x 1024 (two turns of 64 x
//   64) -, 10.7, 7.9;
//   up to 64 tokens past a tile of 64 x 64 a CU, by 64 x 128 (just past it 129 blocks), 64 x 64 in two turns and 128 x 128,
//   whole calls: 64 over 16640 x 1024 11.3, 15.9, 13.8, at k 4096 27.2, 33.3, 36.3; over 22016 x 4096 29.2, 35.1, 38.2; 33 over
//   16640 x 4096 25.2, 30.1, 35.9; over 32768 x 4096 36.8, 37.7, 41.9; 64 over 40000 x 4096 48.3, 50.6, 47.5; over 65536 x 4096
//   65.9, 75.9, 71.0; gated 64 over 11008 x 4096 28.6, 35.0, 38.4; the product of 64 over 151936 x 1024 41.2, -, 46.1;
//   256 x 256 against 128 x 128, two of which share a CU: 8192 over 12288 x 4096 (6 turns, 24) 356, 422; 4096 over 4096 x
//   1024 (1, 4) 23.2, 24.6; 768 over 12288 x 4096 (1, 3) 48.9, 52.1; 1500 over 4096 x 12288 (1, 2) 125, 85; 2048 over 4096 x
//   1024 (1, 2) 20.8, 14.2. Where k is short, a tile is mostly its outputs, which two blocks overlap: 5327 over 18704 x 176
//   (7, 25) 77.6, 67.6; 8192 over 8192 x 512 (4, 16) 59.9, 65.8; gated 2244 over 8001 x 1024 (3, 9) 63.2, 57.0.
int launch_product_tiles(nv_context* c, const ProductArgs& p, bool gated, bool check) {
    using Large = Shape<256, 256, 2, 4, 2>;
    using Medium = Shape<128, 128, 4, 2, 2>;
    using Wide = Shape<64, 128, 4, 2, 3>;
    constexpr int kShort = 384;
    const int64_t cus = c->cu_count > 0 ? c->cu_count : 256, rows = gated ? 2 * int64_t(p.n) : p.n;
    auto tiles = [&](int tokens, int side) { return (int64_t(p.m) + tokens - 1) / tokens * ((rows + side - 1) / side); };
    auto turns = [&](int64_t t) { return (t + cus - 1) / cus; };
    auto run = [&](auto g) {
        constexpr bool G = decltype(g)::value;
        if (p.m <= 16 && tiles(16, 16) <= cus) return launch_split<16, 16, 4, G>(c, p, check);
        if (p.m <= 32 && tiles(32, 16) <= cus) return launch_split<32, 16, 4, G>(c, p, check);
        if (tiles(64, 16) <= cus) return launch_split<64, 16, 2, G>(c, p, check);
        if (p.m <= 16) return launch_split<16, 32, 2, G>(c, p, check);
        if (p.m <= 32) return launch_split<32, 32, 2, G>(c, p, check);
        if (tiles(64, 32) <= cus) return launch_split<64, 32, 2, G>(c, p, check);
        if (tiles(64, 64) <= cus) return launch_split<64, 64, 2, G>(c, p, check);
        if (p.m <= 64) return launch<Wide, G>(c, p, check);
        const int64_t large = 3 * turns(tiles(256, 256)) + (p.w_pitch <= 1024 ? 1 : 0);
        if (p.w_pitch <= kShort || large > turns(tiles(128, 128))) return launch<Medium, G>(c, p, check);
        return launch<Large, G>(c, p, check);
    };
    return gated ? run(std::true_type{}) : run(std::false_type{});
}

}  // namespace nvr
