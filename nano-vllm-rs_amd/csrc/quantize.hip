// Rows of bf16 as 8-bit integers with a scale a row (nv_quantize_rows), and the
// tokens of nv_gemm_i8 and nv_gemm_i8_silu where a launch of its own makes them.
// No counterpart in the reference, whose weights and products are bf16
// (kernels/kernels.cu:98-106). The arithmetic is in nvr_int8.h.
#include "../../include/nano_hip.h"
#include "nvr_int8.h"
#include "nvr_internal.h"

namespace {

using nvr::kWave;
using nvr::Tokens;

// The waves of a row exchange through LDS.
template <int WAVES>
struct BlockJoin {
    float* sum;
    uint32_t* top;
    int lane, wave;
    __device__ void operator()(float* s, uint32_t& t) const {
        constexpr int MINE = nvr::kClasses / WAVES;
        if (lane == 0) {
#pragma unroll
            for (int i = 0; i < MINE; ++i) sum[i * WAVES + wave] = s[i];
            top[wave] = t;
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < nvr::kClasses; ++i) s[i] = sum[i];
#pragma unroll
        for (int i = 0; i < WAVES; ++i) t = max(t, top[i]);
    }
};

// CH chunks a lane of WAVES waves hold a row; 0: a row of any length, read twice.
template <int WAVES>
constexpr int kThreads = WAVES == 16 ? 1024 : 256;
template <Tokens T, bool WHOLE, int CH, int WAVES>
__global__ __launch_bounds__(kThreads<WAVES>) void quantize_rows(nvr::TokenArgs t, uint8_t* __restrict__ q,
                                                                 float* __restrict__ scales, int pitch) {
    __shared__ float sum[nvr::kClasses];
    __shared__ uint32_t top[WAVES];
    constexpr int kRows = kThreads<WAVES> / kWave / WAVES;  // rows of a block at a time
    const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave, of_row = WAVES == 1 ? 0 : wave;
    const int64_t first = int64_t(blockIdx.x) * kRows + (WAVES == 1 ? wave : 0), step = int64_t(gridDim.x) * kRows;
    const bool keep_sum = t.residual_out != nullptr;
    using Join = std::conditional_t<WAVES == 1, nvr::NoJoin, BlockJoin<WAVES>>;
    Join join;
    if constexpr (WAVES != 1) join = {sum, top, lane, wave};
    nvr::NormChunks<CH == 0 ? 1 : CH> norm;
    if constexpr (CH != 0) norm = nvr::load_norm<T, WHOLE, CH, WAVES>(t, lane, of_row);
    for (int64_t row = first; row < t.rows; row += step) {
        uint8_t* out = q + row * pitch;
        auto put = [&](int j, uint2 eight) { *reinterpret_cast<uint2*>(out + j) = eight; };
        nvr::RowStep made;
        if constexpr (CH != 0)
            made = nvr::quantize_row<T, WHOLE, CH, WAVES>(t, row, nvr::load_row<T, WHOLE, CH, WAVES>(t, row, lane, of_row),
                                                          norm, pitch, keep_sum, lane, of_row, join, put);
        else
            made = nvr::quantize_long_row<T, WHOLE>(t, row, pitch, keep_sum, lane, wave, join, put);
        if (lane == 0 && of_row == 0) scales[row] = made.scale;
        if constexpr (WAVES != 1) __syncthreads();  // sum and top are read
    }
}

// Bound by memory: 3 bytes an element move (7 with a residual): 8192 rows of 4096 in 17.7 us of a graph, inputs cold, 5.7
// TB/s, with sum and norm 4096 rows in 28 us, 4.2 TB/s. A row is read once and stays in registers. With many rows one wave
// takes up to 4096 values, so that it waits for no barrier, four up to 16384. With few, latency counts: 4 waves take up to
// 2048, 16 up to 16384, in as little code as that gives (it is read anew by each launch: 3 odd rows of 8989 by 4 waves of 8
// chunks 10 us). Longer rows are read twice. Inputs cold, in us, as for few rows and as for many, 256, 1024, 2048, 8192
// rows: k 1024 2.3, 3.1, 3.7, 9.6 and 2.1, 2.8, 3.4, 6.5; k 2048 2.7, 3.6, 4.6, 11.7 and 3.5, 3.8, 5.2, 11.0; k 4096 3.0,
// 5.9, 10.3, 30.9 and 3.3, 4.7, 6.8, 17.7; k 4090 3.2, 6.3, 11.2, 33.8 and 4.9, 6.6, 8.7, 20.7; k 16384 4.6, 11.2, 18.4,
// 71.1 and 4.8, 10.8, 17.3, 72.8. With sum and norm and a product of 16 channels behind it, 1024 and 8192 rows: k 1024 7.4,
// 19.2 and 6.8, 15.7; k 4096 15.0, 53.4 and 14.0, 45.8; but k 1111 8.3, 22.9 and 9.9, 27.3, k 8192 21.4, 103 and 22.0, 107.
template <Tokens T, bool WHOLE>
void launch(nv_context* c, const nvr::TokenArgs& t, uint8_t* q, float* scales, int pitch) {
    const int cus = c->cu_count > 0 ? c->cu_count : 256;
    const int64_t rows = t.rows;
    auto run = [&](auto chunks, auto waves) {
        constexpr int CH = decltype(chunks)::value, WAVES = decltype(waves)::value;
        constexpr int kRows = kThreads<WAVES> / kWave / WAVES;
        const int64_t blocks = std::min<int64_t>((rows + kRows - 1) / kRows, 1 << 20);  // further rows are taken in turn
        hipLaunchKernelGGL((quantize_rows<T, WHOLE, CH, WAVES>), dim3(unsigned(blocks)), dim3(kThreads<WAVES>), 0, c->stream,
                           t, q, scales, pitch);
    };
    using std::integral_constant;
    const integral_constant<int, 0> any;
    const integral_constant<int, 1> one;
    const integral_constant<int, 2> two;
    const integral_constant<int, 4> four;
    const integral_constant<int, 8> eight;
    const integral_constant<int, 16> sixteen;
    const int chunks = (pitch + nvr::kWaveChunk - 1) / nvr::kWaveChunk;
    if (rows >= 4 * cus && chunks <= 32) {
        if (chunks <= 2) run(two, one);
        else if (chunks <= 4) run(four, one);
        else if (chunks <= 8) run(eight, one);
        else if (chunks <= 16) run(four, four);
        else run(eight, four);
    } else {
        if (chunks <= 4) run(one, four);
        else if (chunks <= 16) run(one, sixteen);
        else if (chunks <= 32) run(two, sixteen);
        else run(any, sixteen);
    }
}

}  // namespace

namespace nvr {

void launch_quantize(nv_context* c, const TokenArgs& t, uint8_t* q, float* scales, int pitch) {
    auto run = [&](auto tokens) {
        constexpr Tokens T = decltype(tokens)::value;
        t.k % kChunk == 0 ? launch<T, true>(c, t, q, scales, pitch) : launch<T, false>(c, t, q, scales, pitch);
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
    if (nvr::overlap({{q, rows * nvr::i8_pitch(k)}, {scales, int64_t(rows) * 4}}, {{x, int64_t(rows) * k * 2}}))
        return nvr::fail(-2, "quantize_rows: q or scales overlap another argument");
    const nvr::TokenArgs t{static_cast<const uint16_t*>(x), nullptr, nullptr, nullptr, rows, k, 0.0f};
    nvr::launch_quantize(c, t, static_cast<uint8_t*>(q), static_cast<float*>(scales), int(nvr::i8_pitch(k)));
    return nvr::launch_status();
}
