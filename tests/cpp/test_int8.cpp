// The C++ host API's operators in 8-bit integers: sizes on the CPU; on a GPU each
// refusal by its Fault kind, and a norm, a gated product and a product of small
// whole numbers, exact in bf16, in a captured graph.
//
// Usage: test_int8 cpu|gpu   -> runs that suite, exit status 0 when all pass.
#include <cmath>
#include <cstdint>
#include <cstring>
#include <vector>

#include "gpu.hpp"
#include "harness.hpp"

namespace {

uint16_t bf16(float x) {
    uint32_t b;
    std::memcpy(&b, &x, 4);
    return uint16_t((b + 0x7fffu + ((b >> 16) & 1u)) >> 16);
}
float value(uint16_t h) {
    const uint32_t b = uint32_t(h) << 16;
    float x;
    std::memcpy(&x, &b, 4);
    return x;
}

// -------------------------------------------------------------- CPU suite --
TEST(i8_rows_lie_at_multiples_of_16, "cpu") {
    CHECK(nvr::i8_pitch(1) == 16 && nvr::i8_pitch(16) == 16 && nvr::i8_pitch(17) == 32 && nvr::i8_pitch(131071) == 131072);
    size_t bytes = 0;
    CHECK(nv_gemm_i8_workspace(4, 8, 131071, &bytes) == 0);
    CHECK(nv_gemm_i8_workspace(4, 8, 131072, &bytes) == -2);
    CHECK(nv_gemm_i8_silu_workspace(4, 0, 16, &bytes) == -2);
}

// -------------------------------------------------------------- GPU suite --
struct Step {
    nvr::Gpu gpu{0};
    std::size_t m = 3, n = 20, k = 24;
    nvr::Buffer x = gpu.alloc(m * k * 2), res = gpu.alloc(m * k * 2), out = gpu.alloc(m * k * 2), nw = gpu.alloc(k * 2);
    nvr::Buffer bits = gpu.alloc(2 * n * k * 2), w = gpu.alloc(2 * n * nvr::i8_pitch(k)), ws = gpu.alloc(2 * n * 4);
    nvr::Buffer y = gpu.alloc(m * n * 2), act = gpu.alloc(m * n * 2), none;
    nvr::Buffer work = gpu.alloc(gpu.gemm_i8_workspace(m, n, k) + gpu.gemm_i8_silu_workspace(m, n, k) + 16);
    void run(const nvr::Buffer& r, const nvr::Buffer& ro, const nvr::Buffer& norm, const nvr::Buffer& to, std::size_t kk) const {
        gpu.gemm_i8(x, r, ro, norm, w, ws, to, work, m, n, kk, 1e-6f);
    }
};

TEST(i8_calls_refuse_by_fault, "gpu") {
    Step s;
    CHECK_FAULT(s.run(s.res, s.none, s.none, s.y, s.k), nvr::Fault::Value);
    CHECK_FAULT(s.run(s.none, s.out, s.nw, s.y, s.k), nvr::Fault::Value);
    CHECK_FAULT(s.run(s.none, s.none, s.none, s.y, 131072), nvr::Fault::Value);
    CHECK_FAULT(s.run(s.none, s.none, s.none, s.y.slice(0, 100), s.k), nvr::Fault::Extent);
    CHECK_FAULT(s.run(s.none, s.none, s.none, s.x, s.k), nvr::Fault::Overlap);
    CHECK_FAULT(s.run(s.res, s.res, s.nw, s.y, s.k), nvr::Fault::Overlap);
    CHECK_FAULT(s.gpu.gemm_i8(s.x, s.none, s.none, s.nw, s.w, s.ws, s.y, s.work, s.m, s.n, s.k, 0.0f), nvr::Fault::Value);
    CHECK_FAULT(s.gpu.gemm_i8_silu(s.x, s.none, s.none, s.none, s.w, s.ws.slice(0, s.n * 4), s.act, s.work, s.m, s.n, s.k, 0.0f),
                nvr::Fault::Extent);
    CHECK_FAULT(s.gpu.quantize_rows(s.bits, s.w.slice(8, 32), s.ws, 1, s.k), nvr::Fault::Alignment);
    CHECK_FAULT(s.gpu.quantize_rows(s.bits, s.w, s.ws, 2 * s.n + 1, s.k), nvr::Fault::Extent);
    nvr::Gpu other(0);
    CHECK_FAULT(s.run(s.none, s.none, s.none, other.alloc(s.m * s.n * 2), s.k), nvr::Fault::Foreign);
}

TEST(i8_products_in_a_graph, "gpu") {
    Step s;
    // Rows with 127 among whole numbers below: scales of 1, integers that are the values.
    std::vector<uint16_t> w(2 * s.n * s.k), x(s.m * s.k);
    for (std::size_t j = 0; j < 2 * s.n; ++j)
        for (std::size_t l = 0; l < s.k; ++l) w[j * s.k + l] = bf16(l == j % s.k ? 127.0f : float(int(l * 5 + j * 3) % 7) - 3.0f);
    s.bits.upload_u16(w);
    const nvr::Graph graph = s.gpu.capture([&] {
        s.gpu.quantize_rows(s.bits, s.w, s.ws, 2 * s.n, s.k);
        s.run(s.none, s.none, s.none, s.y, s.k);
        s.gpu.gemm_i8_silu(s.x, s.none, s.none, s.none, s.w, s.ws, s.act, s.work, s.m, s.n, s.k, 0.0f);
    });
    for (int replay = 0; replay < 3; ++replay) {
        for (std::size_t i = 0; i < s.m; ++i)
            for (std::size_t l = 0; l < s.k; ++l) x[i * s.k + l] = bf16(l == i ? -127.0f : float(int(l * 3 + i + replay) % 5) - 2.0f);
        s.x.upload_u16(x);
        graph.replay();
        const std::vector<uint16_t> y = s.y.download_u16(s.m * s.n), act = s.act.download_u16(s.m * s.n);
        for (std::size_t i = 0; i < s.m; ++i)
            for (std::size_t j = 0; j < s.n; ++j) {
                double g = 0.0, u = 0.0;
                for (std::size_t l = 0; l < s.k; ++l) {
                    g += double(value(x[i * s.k + l])) * value(w[j * s.k + l]);
                    u += double(value(x[i * s.k + l])) * value(w[(s.n + j) * s.k + l]);
                }
                CHECK(y[i * s.n + j] == bf16(float(g)));  // a whole number below 2^24
                // Half a step of bf16, and of fp32: arguments up to 2^14, so the exponential is off by 2^-8 of e^-g at
                // most, which moves g / (1 + e^-g) by |g| e^-|g| 2^-8 < 2^-9.
                const double want = g / (1.0 + std::exp(-g)) * u;
                CHECK(std::fabs(value(act[i * s.n + j]) - want) <= std::fabs(want) * (0x1p-8 + 0x1p-20) + std::fabs(u) * 0x1p-9 + 0x1p-100);
            }
    }
}

}  // namespace
