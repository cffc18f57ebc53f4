// What the operators in 8-bit integers share: rows of values as whole numbers of
// a step (quantize.hip, gemm_int.hip), and the products' scales.
//
// A row u of k values has a = max |u_j|, the scale a / 127 and the whole numbers
// q_j = round(127 u_j / a), half to even, so |q_j| <= 127. All are 0 where a is;
// with a NaN or an infinity in the row the scale is NaN, and q_j is 0.
//
// 127 u_j / a is formed from u_j and a at the power of two that brings a into
// [1/2, 1), so nothing leaves the range of fp32 on the way, by one step of
// Markstein's division (P. Markstein, IBM J. Res. Dev. 34, 1990): with y the
// rounded reciprocal of a, q = t y, r = t - q a (exact), q + r y. Where t = 127
// u_j is exact, as for bf16 (15 bits), a quotient half way between two whole
// numbers is one of fp32 and comes out as it is. No other quotient of such t and a
// lies within 2^-17 of such a point, and fp32 is within 2^-18 of it below 128: the
// row's numbers are those of exact arithmetic.
//
// A norm's values are those of fp32, not rounded to bf16 in between: the norm's
// output feeds one product only, and 8 bits of a step keep more of them.
// Its sum of squares has one order, whoever computes it: element j belongs to
// lane (j / 8) % 64 and class (j / 512) % 4; a lane sums each class in order of
// j, the 64 lanes by a butterfly, the classes as (0 + 1) + (2 + 3). A wave that
// holds all of a row and four waves that hold a class each give the same bits, so
// a token's outputs do not depend on the call's other tokens.
#pragma once

#include <algorithm>
#include <type_traits>

#include "nvr_device.h"

struct nv_context;

namespace nvr {

constexpr int kChunk = 8;                      // elements of a lane's load (16 bytes of bf16)
constexpr int kWaveChunk = kChunk * kWave;     // elements a wave covers with one load a lane
constexpr int kClasses = 4;

// Rows of 8-bit integers start at multiples of 16 bytes.
__host__ __device__ constexpr int64_t i8_pitch(int64_t k) { return (k + 15) / 16 * 16; }

// The longest row of a product: its sums stay below 2^31, weights of -128 among them.
constexpr int kMostSummed = 131071;

enum class Tokens { kPlain, kNorm, kAddNorm };

// Tokens of a call: x, or RMSNorm(x) weight, or RMSNorm(x + residual) weight with
// residual_out <- bf16(x + residual). VEC: k is a multiple of 8 and every pointer of 16 bytes.
struct TokenArgs {
    const uint16_t* x;
    const uint16_t* residual;
    uint16_t* residual_out;  // may be null
    const uint16_t* norm_weight;
    int rows, k;
    float eps;
};

// The tokens' integers (rows at `pitch` bytes, zeros behind k) and scales (quantize.hip).
bool tokens_aligned(const TokenArgs& t);
void launch_quantize(nv_context* c, const TokenArgs& t, uint8_t* q, float* scales, int pitch);

// A product of m tokens and n channels (gated: n of gate, then n of up). Tokens' rows are zero from k to x_pitch.
struct ProductArgs {
    const uint8_t* xq;
    const float* xs;
    const uint8_t* wq;
    const float* ws;
    uint16_t* y;
    int m, n, x_pitch, w_pitch;
};

// Products of whole tiles (gemm_int_tiles.hip).
void launch_product_tiles(nv_context* c, const ProductArgs& p, bool gated);

// Elements j .. j + 7 of a row, +0 from k on.
template <bool VEC>
__device__ __forceinline__ void load_chunk(const uint16_t* row, int j, int k, float* f) {
    if constexpr (VEC) {
        unpack8(j < k ? *reinterpret_cast<const uint4*>(row + j) : make_uint4(0, 0, 0, 0), f);
    } else {
#pragma unroll
        for (int i = 0; i < kChunk; ++i) f[i] = j + i < k ? bf16_to_f32(row[j + i]) : 0.0f;
    }
}

template <bool VEC>
__device__ __forceinline__ void store_chunk(uint16_t* row, int j, int k, const float* f) {
    if constexpr (VEC) {
        if (j < k) *reinterpret_cast<uint4*>(row + j) = pack8_split(f);
    } else {
#pragma unroll
        for (int i = 0; i < kChunk; ++i)
            if (j + i < k) row[j + i] = f32_to_bf16(f[i]);
    }
}

__device__ __forceinline__ float wave_sum(float s) {
#pragma unroll
    for (int w = 1; w < kWave; w <<= 1) s = s + xor_lane(s, w);
    return s;
}
// The largest |u| of values as bits: a NaN's are above those of infinity, which are above all others.
__device__ __forceinline__ uint32_t magnitude(float u) { return __float_as_uint(u) & 0x7fffffffu; }
__device__ __forceinline__ uint32_t wave_max(uint32_t a) {
#pragma unroll
    for (int w = 1; w < kWave; w <<= 1) a = max(a, xor_lane_bits(a, w));
    return a;
}

// The step of a row whose largest magnitude has the bits `top`.
struct RowStep {
    float scale;           // top / 127; NaN, 0
    float mantissa, recip;  // of top = mantissa 2^exponent, 1 / mantissa
    int exponent;
};
__device__ __forceinline__ RowStep row_step(uint32_t top) {
    const float a = __uint_as_float(top);
    if (top == 0 || top >= 0x7f800000u) return {top == 0 ? 0.0f : __builtin_nanf(""), 1.0f, 0.0f, 0};
    const float m = __builtin_amdgcn_frexp_mantf(a);
    return {a / 127.0f, m, 1.0f / m, __builtin_amdgcn_frexp_expf(a)};
}
// A value's whole number in the low byte (two's complement): the sum with 3 * 2^22 rounds to one, half to even.
__device__ __forceinline__ uint32_t whole_number(float u, const RowStep& s) {
    const float t = __builtin_amdgcn_ldexpf(u, -s.exponent) * 127.0f;
    const float q = t * s.recip;
    const float r = __builtin_fmaf(-q, s.mantissa, t);
    return __float_as_uint(__builtin_fmaf(r, s.recip, q) + 12582912.0f);
}
// Eight values as 8 bytes.
__device__ __forceinline__ uint2 whole_numbers(const float* u, const RowStep& s) {
    if (s.recip == 0.0f) return make_uint2(0, 0);  // a row of zeros, or one with a NaN or an infinity
    uint32_t b[kChunk];
#pragma unroll
    for (int i = 0; i < kChunk; ++i) b[i] = whole_number(u[i], s);
    auto four = [](uint32_t b0, uint32_t b1, uint32_t b2, uint32_t b3) {
        const uint32_t low = __builtin_amdgcn_perm(b1, b0, 0x0c0c0400u), high = __builtin_amdgcn_perm(b3, b2, 0x0c0c0400u);
        return low | high << 16;
    };
    return make_uint2(four(b[0], b[1], b[2], b[3]), four(b[4], b[5], b[6], b[7]));
}

// A row of tokens by one wave: its step (in every lane), and put(j, eight numbers) for each chunk j < width that the lane
// holds, from k on zeros. KEEP: the row stays in registers, CH chunks a lane (width <= CH * 512); else it is read again.
// WAVES 1: this wave has the whole row. WAVES 4: four do, this one class `wave`, and join(sum or bits, ...) gathers.
template <Tokens T, bool VEC, bool KEEP, int CH, int WAVES, class Join, class Put>
__device__ __forceinline__ RowStep quantize_row(const TokenArgs& t, int64_t row, int width, bool keep_sum, int lane,
                                                int wave, Join join, Put put) {
    static_assert(WAVES == 1 || WAVES == kClasses, "a wave has all classes of a row, or one");
    const uint16_t* x = t.x + row * t.k;
    const uint16_t* res = T == Tokens::kAddNorm ? t.residual + row * t.k : nullptr;
    const int stride = WAVES * kWaveChunk, first = wave * kWaveChunk + lane * kChunk;
    const int chunks = (width + stride - 1) / stride;  // uniform in the block
    float v[KEEP ? CH : 1][kChunk];
    auto load = [&](int c, float* f) {
        const int j = first + c * stride;
        load_chunk<VEC>(x, j, t.k, f);
        if constexpr (T == Tokens::kAddNorm) {
            float r[kChunk];
            load_chunk<VEC>(res, j, t.k, r);
#pragma unroll
            for (int i = 0; i < kChunk; ++i) f[i] = f[i] + r[i];
        }
    };
    auto each = [&](auto&& f) {  // f(c, values as loaded)
        if constexpr (KEEP) {
#pragma unroll
            for (int c = 0; c < CH; ++c)
                if (c < chunks) f(c, v[c]);
        } else {
            for (int c = 0; c < chunks; ++c) {
                load(c, v[0]);
                f(c, v[0]);
            }
        }
    };
    if constexpr (KEEP) {
#pragma unroll
        for (int c = 0; c < CH; ++c)
            if (c < chunks) load(c, v[c]);
    }
    float inv = 1.0f;
    if constexpr (T != Tokens::kPlain) {
        float s[kClasses] = {};
        each([&](int c, const float* f) {
            float& sum = s[WAVES == 1 ? c % kClasses : 0];
#pragma unroll
            for (int i = 0; i < kChunk; ++i) sum = __builtin_fmaf(f[i], f[i], sum);
        });
#pragma unroll
        for (int i = 0; i < (WAVES == 1 ? kClasses : 1); ++i) s[i] = wave_sum(s[i]);
        if constexpr (WAVES != 1) join.sums(s);
        inv = inv_sqrt_rn(((s[0] + s[1]) + (s[2] + s[3])) / float(t.k) + t.eps);
    }
    auto normed = [&](int c, float* f) {
        if constexpr (T != Tokens::kPlain) {
            float g[kChunk];
            load_chunk<VEC>(t.norm_weight, first + c * stride, t.k, g);
#pragma unroll
            for (int i = 0; i < kChunk; ++i) f[i] = (f[i] * inv) * g[i];
        }
    };
    uint32_t top = 0;
    each([&](int c, float* f) {
        if (T == Tokens::kAddNorm && keep_sum) store_chunk<VEC>(t.residual_out + row * t.k, first + c * stride, t.k, f);
        normed(c, f);
#pragma unroll
        for (int i = 0; i < kChunk; ++i) top = max(top, magnitude(f[i]));
    });
    top = wave_max(top);
    if constexpr (WAVES != 1) join.most(top);
    const RowStep step = row_step(top);
    each([&](int c, float* f) {
        if constexpr (!KEEP) normed(c, f);
        if (first + c * stride < width) put(first + c * stride, whole_numbers(f, step));
    });
    return step;
}

struct NoJoin {};

// acc xs ws with both scales as mantissa and exponent: no product of two of the three leaves the range of fp32
// where the result does not.
struct Scale {
    float mantissa;
    int exponent;
};
__device__ __forceinline__ Scale split_scale(float s) {
    return {__builtin_amdgcn_frexp_mantf(s), __builtin_amdgcn_frexp_expf(s)};
}
__device__ __forceinline__ float scaled(int acc, Scale x, Scale w) {
    return __builtin_amdgcn_ldexpf(float(acc) * x.mantissa * w.mantissa, x.exponent + w.exponent);
}
// Whether float(acc) s t is the same bits as scaled's for all such scales s, t and any sum: nothing on the way overflows
// or becomes subnormal, and powers of two change no rounding.
__device__ __forceinline__ bool middling(float s) { return s == 0.0f || (s >= 0x1.0p-60f && s <= 0x1.0p40f); }

}  // namespace nvr
