// Rows of bf16 as 8-bit integers with a scale a row (nv_quantize_rows), and the
// tokens of nv_gemm_i8 and nv_gemm_i8_silu where a launch of its own makes them.
// No counterpart in the reference, whose weights and products are bf16
// (kernels/kernels.cu:98-106). The arithmetic is in nvr_int8.h.
//
// Bound by memory: 3 bytes an element move (7 with a residual). A row is read
// once and stays in registers: up to 4096 values by one wave, so no barrier is
// waited for, up to 16384 by the four waves of a block; longer rows are read again
// for each step. With few rows four waves a row are taken below 4096 too, for
// more loads in flight.
#include "../../include/nano_hip.h"
#include "nvr_int8.h"
#include "nvr_internal.h"

namespace {

using nvr::kWave;
using nvr::Tokens;

constexpr int kThreads = 256, kRowChunks = 8;

// The four waves of a row exchange through LDS.
struct BlockJoin {
    float* sum;
    uint32_t* top;
    int lane, wave;
    __device__ void sums(float* s) const {
        if (lane == 0) sum[wave] = s[0];
        __syncthreads();
#pragma unroll
        for (int i = 0; i < nvr::kClasses; ++i) s[i] = sum[i];
    }
    __device__ void most(uint32_t& t) const {
        if (lane == 0) top[wave] = t;
        __syncthreads();
        t = max(max(top[0], top[1]), max(top[2], top[3]));
    }
};

template <Tokens T, bool VEC, bool KEEP, int WAVES>
__global__ __launch_bounds__(kThreads) void quantize_rows(nvr::TokenArgs t, uint8_t* __restrict__ q,
                                                          float* __restrict__ scales, int pitch) {
    __shared__ float sum[nvr::kClasses];
    __shared__ uint32_t top[nvr::kClasses];
    const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
    constexpr int kRows = kThreads / kWave / WAVES;  // rows of a block at a time
    for (int64_t row = int64_t(blockIdx.x) * kRows + (WAVES == 1 ? wave : 0); row < t.rows;
         row += int64_t(gridDim.x) * kRows) {
        uint8_t* out = q + row * pitch;
        auto put = [&](int j, uint2 eight) { *reinterpret_cast<uint2*>(out + j) = eight; };
        const bool keep_sum = t.residual_out != nullptr;
        nvr::RowStep step;
        if constexpr (WAVES == 1) {
            step = nvr::quantize_row<T, VEC, KEEP, kRowChunks, 1>(t, row, pitch, keep_sum, lane, 0, nvr::NoJoin{}, put);
        } else {
            step = nvr::quantize_row<T, VEC, KEEP, kRowChunks, WAVES>(t, row, pitch, keep_sum, lane, wave,
                                                                     BlockJoin{sum, top, lane, wave}, put);
        }
        if (lane == 0 && (WAVES == 1 || wave == 0)) scales[row] = step.scale;
        if constexpr (WAVES != 1) __syncthreads();  // sum and top are read
    }
}

template <Tokens T, bool VEC>
void launch(nv_context* c, const nvr::TokenArgs& t, uint8_t* q, float* scales, int pitch) {
    constexpr int kWaveRow = kRowChunks * nvr::kWaveChunk, kBlockRow = 4 * kWaveRow;
    constexpr int64_t kMostBlocks = 1 << 20;  // further rows are taken in turn
    const int64_t quarter = (int64_t(t.rows) + 3) / 4;
    const dim3 block(kThreads);
    if (pitch <= kWaveRow && quarter >= c->cu_count)
        hipLaunchKernelGGL((quantize_rows<T, VEC, true, 1>), dim3(unsigned(std::min(quarter, kMostBlocks))), block, 0,
                           c->stream, t, q, scales, pitch);
    else if (pitch <= kBlockRow)
        hipLaunchKernelGGL((quantize_rows<T, VEC, true, 4>), dim3(unsigned(std::min<int64_t>(t.rows, kMostBlocks))), block,
                           0, c->stream, t, q, scales, pitch);
    else
        hipLaunchKernelGGL((quantize_rows<T, VEC, false, 4>), dim3(unsigned(std::min<int64_t>(t.rows, kMostBlocks))), block,
                           0, c->stream, t, q, scales, pitch);
}

}  // namespace

namespace nvr {

bool tokens_aligned(const TokenArgs& t) {
    return t.k % kChunk == 0 && aligned(t.x, 16) && aligned(t.residual, 16) && aligned(t.residual_out, 16) &&
           aligned(t.norm_weight, 16);
}

void launch_quantize(nv_context* c, const TokenArgs& t, uint8_t* q, float* scales, int pitch) {
    const bool vec = tokens_aligned(t);
    auto run = [&](auto tokens) {
        constexpr Tokens T = decltype(tokens)::value;
        vec ? launch<T, true>(c, t, q, scales, pitch) : launch<T, false>(c, t, q, scales, pitch);
    };
    if (t.norm_weight == nullptr) run(std::integral_constant<Tokens, Tokens::kPlain>{});
    else if (t.residual == nullptr) run(std::integral_constant<Tokens, Tokens::kNorm>{});
    else run(std::integral_constant<Tokens, Tokens::kAddNorm>{});
}

}  // namespace nvr

extern "C" int nv_quantize_rows(nv_context* c, const void* x, void* q, void* scales, int rows, int k) {
    NVR_ACTIVATE(c);
    if (rows <= 0 || k <= 0 || k > nvr::kMostSummed)
        return nvr::fail(-2, "quantize_rows: rows %d, k %d; k goes from 1 to %d", rows, k, nvr::kMostSummed);
    if (x == nullptr || q == nullptr || scales == nullptr)
        return nvr::fail(-2, "quantize_rows: x, q and scales are required");
    if (!nvr::aligned(x, 2) || !nvr::aligned(q, 16) || !nvr::aligned(scales, 4))
        return nvr::fail(-2, "quantize_rows: q starts at a multiple of 16 bytes, x of 2, scales of 4");
    const nvr::TokenArgs t{static_cast<const uint16_t*>(x), nullptr, nullptr, nullptr, rows, k, 0.0f};
    nvr::launch_quantize(c, t, static_cast<uint8_t*>(q), static_cast<float*>(scales), int(nvr::i8_pitch(k)));
    return nvr::launch_status();
}
