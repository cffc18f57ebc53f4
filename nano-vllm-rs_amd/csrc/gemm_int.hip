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
typedef int i32x4_t __attribute__((ext_vector_type(4)));
typedef int i32x16_t __attribute__((ext_vector_type(16)));

// Any size: a wave forms 32 channels of 32 tokens, its operands read from memory in the matrix
// instruction's layout (lane l: row l % 32, 16 bytes at 16 (l / 32) of each 32).
template <bool GATED>
__global__ __launch_bounds__(256) void gemm_direct(nvr::ProductArgs p) {
    const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
    const int i = lane % 32, half = lane / 32;
    const int n0 = (blockIdx.x * 4 + wave) * 32;
    if (n0 >= p.n) return;
    for (int64_t m0 = int64_t(blockIdx.y) * 32; m0 < p.m; m0 += int64_t(gridDim.y) * 32) {
        const int64_t token = min(m0 + i, int64_t(p.m) - 1);
        const int channel = min(n0 + i, p.n - 1);
        const uint8_t* x = p.xq + token * p.x_pitch;
        const uint8_t* w = p.wq + int64_t(channel) * p.w_pitch;
        i32x16_t acc = {}, up = {};
        for (int k = 0; k < p.x_pitch; k += 32) {
            const int kx = k + 16 * half, kw = min(kx, p.w_pitch - 16);  // x is zero from w's pitch on
            const i32x4_t b = *reinterpret_cast<const i32x4_t*>(x + kx);
            acc = __builtin_amdgcn_mfma_i32_32x32x32_i8(*reinterpret_cast<const i32x4_t*>(w + kw), b, acc, 0, 0, 0);
            if constexpr (GATED)
                up = __builtin_amdgcn_mfma_i32_32x32x32_i8(
                    *reinterpret_cast<const i32x4_t*>(w + int64_t(p.n) * p.w_pitch + kw), b, up, 0, 0, 0);
        }
        if (m0 + i >= p.m) continue;
        const Scale xs = nvr::split_scale(p.xs[token]);
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            const int j = n0 + 8 * (r / 4) + 4 * half + r % 4;
            if (j >= p.n) continue;
            float y = nvr::scaled(acc[r], xs, nvr::split_scale(p.ws[j]));
            if constexpr (GATED) y = nvr::silu_mul(y, nvr::scaled(up[r], xs, nvr::split_scale(p.ws[int64_t(p.n) + j])));
            p.y[token * p.n + j] = nvr::f32_to_bf16(y);
        }
    }
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
    nvr::launch_quantize(c, t, xq, xs, pitch);
    const nvr::ProductArgs p{xq, xs, static_cast<const uint8_t*>(w), static_cast<const float*>(w_scales),
                             static_cast<uint16_t*>(y), m, n, pitch, int(nvr::i8_pitch(k))};
    if (m >= 64) {
        nvr::launch_product_tiles(c, p, GATED);
        return nvr::launch_status();
    }
    const dim3 grid(unsigned((int64_t(n) + 127) / 128), unsigned(std::min<int64_t>((int64_t(m) + 31) / 32, 65535)));
    hipLaunchKernelGGL(gemm_direct<GATED>, grid, dim3(256), 0, c->stream, p);
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
