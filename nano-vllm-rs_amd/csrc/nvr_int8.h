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
// So are RMSNorm(x)'s, of products of two bf16 (16 bits; t 23): a quotient that is
// not half way is further from such a point than half a step of fp32, which rounds
// none to it. A sum of two bf16 times a weight has more bits and is rounded to fp32
// first, so a quotient within 2^-15 of such a point may take either number.
//
// Of a norm, u_j = v_j g_j / rms(v), the whole numbers need the products v_j g_j alone: their common factor leaves 127 u_j /
// a as it is, and goes into the scale. So a row's sum of squares and its largest product are found in one pass, and the
// norm's values are never rounded, to bf16 or otherwise: they feed one product only, and 8 bits of a step keep more.
// The sum of squares has one order, whoever computes it: element j belongs to lane (j / 8) % 64 and class (j / 512) % 16; a
// lane sums each class in order of j, then come the 64 lanes, in wave_sum's order, and the classes in pairs. A wave that
// holds all of a row, 4 that hold 4 classes each and 16 that hold one give the same bits, so a token's outputs do not
// depend on the call's other tokens.
#pragma once

#include <algorithm>
#include <initializer_list>
#include <type_traits>

#include "nvr_device.h"

struct nv_context;

namespace nvr {

constexpr int kChunk = 8;                      // elements of a lane's load (16 bytes of bf16)
constexpr int kWaveChunk = kChunk * kWave;     // elements a wave covers with one load a lane
constexpr int kClasses = 16;

constexpr int kXcds = 8;

// Rows of 8-bit integers start at multiples of 16 bytes.
__host__ __device__ constexpr int64_t i8_pitch(int64_t k) { return (k + 15) / 16 * 16; }

// The longest row of a product: its sums stay below 2^31, weights of -128 among them.
constexpr int kMostSummed = 131071;

enum class Tokens { kPlain, kNorm, kAddNorm };

// Tokens of a call: x, or RMSNorm(x) weight, or RMSNorm(x + residual) weight with
// residual_out <- bf16(x + residual).
struct TokenArgs {
    const uint16_t* x;
    const uint16_t* residual;
    uint16_t* residual_out;  // may be null
    const uint16_t* norm_weight;
    int rows, k;
    float eps;
};

// A tensor's bytes; one that is absent has none.
struct Span {
    const void* at;
    int64_t bytes;
};
// Whether one of the tensors that a call writes has a byte in common with another of them, or with one that it reads.
inline bool overlap(std::initializer_list<Span> written, std::initializer_list<Span> read) {
    auto common = [](const Span& a, const Span& b) {
        const auto at = reinterpret_cast<uintptr_t>(a.at), bt = reinterpret_cast<uintptr_t>(b.at);
        return a.at != nullptr && b.at != nullptr && at < bt + uint64_t(b.bytes) && bt < at + uint64_t(a.bytes);
    };
    for (const Span* w = written.begin(); w != written.end(); ++w) {
        for (const Span& r : read)
            if (common(*w, r)) return true;
        for (const Span* other = written.begin(); other != w; ++other)
            if (common(*w, *other)) return true;
    }
    return false;
}

// The tokens' integers (rows at `pitch` bytes, zeros behind k) and scales (quantize.hip).
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

// Products of whole tiles (gemm_int_tiles.hip): the launch's status; with `check`, whether one launch holds them.
int launch_product_tiles(nv_context* c, const ProductArgs& p, bool gated, bool check);

__device__ __forceinline__ void store8(uint16_t* to, uint4 v);

// Elements j .. j + 7 of a row (bf16 from any even address on), +0 from k on; nothing outside the row is read. WHOLE: k is
// a multiple of 8.
template <bool WHOLE>
__device__ __forceinline__ uint4 load_chunk(const uint16_t* row, int j, int k) {
    struct __attribute__((packed, aligned(2))) Eight { uint64_t lo, hi; };
    if (!WHOLE && k < kChunk) {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
            w[i] = (j + 2 * i < k ? row[j + 2 * i] : 0) | (j + 2 * i + 1 < k ? uint32_t(row[j + 2 * i + 1]) << 16 : 0);
        return make_uint4(w[0], w[1], w[2], w[3]);
    }
    const int at = min(j, k - kChunk), past = min(j - at, kChunk);  // the row's last eight, of which `past` are before j
    const Eight e = *reinterpret_cast<const Eight*>(row + at);
    uint64_t lo = e.lo, hi = e.hi;
    if constexpr (WHOLE) {
        if (past != 0) lo = hi = 0;
    } else {
        if (past & 4) { lo = hi; hi = 0; }
        const int bits = past & 3 ? 16 * (past & 3) : 0;
        lo = lo >> bits | (bits ? hi << (64 - bits) : 0);
        hi >>= bits;
        if (past == kChunk) lo = hi = 0;
    }
    return make_uint4(uint32_t(lo), uint32_t(lo >> 32), uint32_t(hi), uint32_t(hi >> 32));
}

template <bool WHOLE>
__device__ __forceinline__ void store_chunk(uint16_t* row, int j, int k, const float* f) {
    if (j + kChunk <= k) {
        store8(row + j, pack8_split(f));
    } else if constexpr (!WHOLE) {
#pragma unroll
        for (int i = 0; i < kChunk; ++i)
            if (j + i < k) row[j + i] = f32_to_bf16(f[i]);
    }
}

// Sums over a wave by shifts inside each row of 16 lanes, then of rows' last lanes into the rows behind them: no LDS
// crossbar. Every lane gets lane 63's value.
constexpr int kDppRowShr = 0x110, kDppRowBcast15 = 0x142, kDppRowBcast31 = 0x143;
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t dpp_or_zero(uint32_t v) {
    return uint32_t(__builtin_amdgcn_update_dpp(0, int(v), CTRL, ROWS, 0xF, false));
}
template <class Op>
__device__ __forceinline__ uint32_t wave_fold(uint32_t v, Op op) {
    v = op(v, dpp_or_zero<kDppRowShr + 1, 0xF>(v));
    v = op(v, dpp_or_zero<kDppRowShr + 2, 0xF>(v));
    v = op(v, dpp_or_zero<kDppRowShr + 4, 0xF>(v));
    v = op(v, dpp_or_zero<kDppRowShr + 8, 0xF>(v));
    v = op(v, dpp_or_zero<kDppRowBcast15, 0xA>(v));
    v = op(v, dpp_or_zero<kDppRowBcast31, 0xC>(v));
    return uint32_t(__builtin_amdgcn_readlane(int(v), 63));
}
__device__ __forceinline__ float wave_sum(float s) {
    return __uint_as_float(wave_fold(__float_as_uint(s), [](uint32_t a, uint32_t b) {
        return __float_as_uint(__uint_as_float(a) + __uint_as_float(b));
    }));
}
// The largest |u| of values as bits: a NaN's are above those of infinity, which are above all others.
__device__ __forceinline__ uint32_t magnitude(float u) { return __float_as_uint(u) & 0x7fffffffu; }
__device__ __forceinline__ uint32_t wave_max(uint32_t a) {
    return wave_fold(a, [](uint32_t x, uint32_t y) { return max(x, y); });
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

// A row of tokens by WAVES waves (1, 4 or 16), CH chunks a lane: what a lane loads of it, always as many loads, so that
// later ones can stay in flight while the row is worked on.
template <Tokens T, int CH>
struct RowChunks {
    uint4 x[CH], residual[T == Tokens::kAddNorm ? CH : 1];
};
template <int CH>
struct NormChunks {
    uint4 g[CH];
};
template <int WAVES>
__device__ __forceinline__ int chunk_at(int c, int lane, int wave) {
    return (c * WAVES + wave) * kWaveChunk + lane * kChunk;
}
template <Tokens T, bool WHOLE, int CH, int WAVES>
__device__ __forceinline__ RowChunks<T, CH> load_row(const TokenArgs& t, int64_t row, int lane, int wave) {
    RowChunks<T, CH> r;
#pragma unroll
    for (int c = 0; c < CH; ++c) r.x[c] = load_chunk<WHOLE>(t.x + row * t.k, chunk_at<WAVES>(c, lane, wave), t.k);
    if constexpr (T == Tokens::kAddNorm) {
#pragma unroll
        for (int c = 0; c < CH; ++c)
            r.residual[c] = load_chunk<WHOLE>(t.residual + row * t.k, chunk_at<WAVES>(c, lane, wave), t.k);
    }
    return r;
}
template <Tokens T, bool WHOLE, int CH, int WAVES>
__device__ __forceinline__ NormChunks<CH> load_norm(const TokenArgs& t, int lane, int wave) {
    NormChunks<CH> n;
    if constexpr (T != Tokens::kPlain) {
#pragma unroll
        for (int c = 0; c < CH; ++c) n.g[c] = load_chunk<WHOLE>(t.norm_weight, chunk_at<WAVES>(c, lane, wave), t.k);
    }
    return n;
}

template <Tokens T>
__device__ __forceinline__ void row_values(const uint4& x, const uint4& residual, float* v) {
    unpack8(x, v);
    if constexpr (T == Tokens::kAddNorm) {
        float r[kChunk];
        unpack8(residual, r);
#pragma unroll
        for (int i = 0; i < kChunk; ++i) v[i] = v[i] + r[i];
    }
}
// A chunk's squares onto its class's sum.
__device__ __forceinline__ float add_squares(float sum, const float* v) {
#pragma unroll
    for (int i = 0; i < kChunk; ++i) sum = __builtin_fmaf(v[i], v[i], sum);
    return sum;
}
// A row's scale with 1 / rms in it, s its classes' sums. Where the squares leave fp32 the row is read once more, by each of
// its waves, and summed in 64 bits, in little code, which every launch has to fetch; 1 / rms is then formed at 2^80 and eps
// put in at 2^-160 (it does not count beside a mean square of 2^111 and more unless it is as large).
template <Tokens T>
__device__ __forceinline__ float normed_scale(float scale, const float* s, const TokenArgs& t, int64_t row, int lane) {
    float total[kClasses];
#pragma unroll
    for (int i = 0; i < kClasses; ++i) total[i] = s[i];
#pragma unroll
    for (int w = 1; w < kClasses; w *= 2)
#pragma unroll
        for (int i = 0; i < kClasses; i += 2 * w) total[i] = total[i] + total[i + w];
    if (__builtin_expect(total[0] != __builtin_inff(), 1)) return scale * inv_sqrt_rn(total[0] / float(t.k) + t.eps);
    double squares = 0.0;
#pragma unroll 1
    for (int j = lane; j < t.k; j += kWave) {
        float v = bf16_to_f32(t.x[row * t.k + j]);
        if constexpr (T == Tokens::kAddNorm) v = v + bf16_to_f32(t.residual[row * t.k + j]);
        squares = __builtin_fma(double(v), double(v), squares);
    }
    const float sum = wave_sum(float(squares * 0x1.0p-160));
    const float inverse = inv_sqrt_rn(sum / float(t.k) + __builtin_amdgcn_ldexpf(t.eps, -160));
    return __builtin_amdgcn_ldexpf(scale, -40) * __builtin_amdgcn_ldexpf(inverse, -40);
}
__device__ __forceinline__ void times(float* v, const uint4& weight) {
    float g[kChunk];
    unpack8(weight, g);
#pragma unroll
    for (int i = 0; i < kChunk; ++i) v[i] = v[i] * g[i];
}
__device__ __forceinline__ uint32_t most_of(uint32_t top, const float* v) {
#pragma unroll
    for (int i = 0; i < kChunk; ++i) top = max(top, magnitude(v[i]));
    return top;
}

struct NoJoin {
    __device__ void operator()(float*, uint32_t&) const {}
};

// The row's step (in every lane), and put(j, eight numbers) for each chunk j < width that the lane holds: zeros from k on.
// With more than one wave, join brings their sums and largest bits together.
template <Tokens T, bool WHOLE, int CH, int WAVES, class Join, class Put>
__device__ __forceinline__ RowStep quantize_row(const TokenArgs& t, int64_t row, const RowChunks<T, CH>& r,
                                                const NormChunks<CH>& norm, int width, bool keep_sum, int lane,
                                                int wave, Join join, Put put) {
    constexpr int MINE = kClasses / WAVES, SUMS = CH < MINE ? CH : MINE;  // a wave's classes, and those that it has chunks of
    static_assert(WAVES * MINE == kClasses, "whole classes");
    float v[CH][kChunk];
#pragma unroll
    for (int c = 0; c < CH; ++c) row_values<T>(r.x[c], r.residual[T == Tokens::kAddNorm ? c : 0], v[c]);
    float s[kClasses] = {};
    if constexpr (T != Tokens::kPlain) {
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            float& sum = s[c % MINE];
            sum = add_squares(sum, v[c]);
        }
        if (T == Tokens::kAddNorm && keep_sum) {
#pragma unroll
            for (int c = 0; c < CH; ++c)
                store_chunk<WHOLE>(t.residual_out + row * t.k, chunk_at<WAVES>(c, lane, wave), t.k, v[c]);
        }
#pragma unroll
        for (int c = 0; c < CH; ++c) times(v[c], norm.g[c]);
    }
    uint32_t top = 0;
#pragma unroll
    for (int c = 0; c < CH; ++c) top = most_of(top, v[c]);
    top = wave_max(top);
    if constexpr (T != Tokens::kPlain) {
#pragma unroll
        for (int i = 0; i < SUMS; ++i) s[i] = wave_sum(s[i]);
    }
    join(s, top);
    RowStep step = row_step(top);
    if constexpr (T != Tokens::kPlain) step.scale = normed_scale<T>(step.scale, s, t, row, lane);
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        const int j = chunk_at<WAVES>(c, lane, wave);
        if (j < width) put(j, whole_numbers(v[c], step));
    }
    return step;
}

// The same for a row of any length by 16 waves, which read it twice.
template <Tokens T, bool WHOLE, class Join, class Put>
__device__ __forceinline__ RowStep quantize_long_row(const TokenArgs& t, int64_t row, int width, bool keep_sum, int lane,
                                                     int wave, Join join, Put put) {
    const int chunks = (width + kClasses * kWaveChunk - 1) / (kClasses * kWaveChunk);
    auto load = [&](int c, float* v) {
        const int j = chunk_at<kClasses>(c, lane, wave);
        const uint4 x = load_chunk<WHOLE>(t.x + row * t.k, j, t.k);
        row_values<T>(x, T == Tokens::kAddNorm ? load_chunk<WHOLE>(t.residual + row * t.k, j, t.k) : x, v);
        return j;
    };
    float v[kChunk], s[kClasses] = {};
    uint32_t top = 0;
    for (int c = 0; c < chunks; ++c) {
        const int j = load(c, v);
        if constexpr (T != Tokens::kPlain) {
            s[0] = add_squares(s[0], v);
            if (T == Tokens::kAddNorm && keep_sum) store_chunk<WHOLE>(t.residual_out + row * t.k, j, t.k, v);
            times(v, load_chunk<WHOLE>(t.norm_weight, j, t.k));
        }
        top = most_of(top, v);
    }
    top = wave_max(top);
    if constexpr (T != Tokens::kPlain) s[0] = wave_sum(s[0]);
    join(s, top);
    RowStep step = row_step(top);
    if constexpr (T != Tokens::kPlain) step.scale = normed_scale<T>(step.scale, s, t, row, lane);
    for (int c = 0; c < chunks; ++c) {
        const int j = load(c, v);
        if constexpr (T != Tokens::kPlain) times(v, load_chunk<WHOLE>(t.norm_weight, j, t.k));
        if (j < width) put(j, whole_numbers(v, step));
    }
    return step;
}

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
// silu(g) u = g u / (1 + e^-g). Far below zero, where the 1 no longer counts, it is g e^g u with e^g in three equal factors
// and u between them: nothing on the way is flushed or overflows while the result is one of fp32, though e^g alone may be far
// below. At -512 that is 0 for any u, and so it is for all gates below, -inf among them. Hardware exponential and reciprocal,
// each within a step; without the division that nv_silu takes there, whose instructions every lane would run. A branch, since
// few waves meet such a gate (selects instead: gated 2244 tokens over 8001 x 1024 58.2 us for 55.8, 4096 over 8192 x 512 73.0 for
// 66.9).
__device__ __forceinline__ float gated(float g, float u) {
    const float t = g * -1.44269504088896340736f;
    float y = g * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(t)) * u;
    if (__builtin_expect(t > 64.0f, 0)) {
        const float at = fmaxf(g, -512.0f), e = __builtin_amdgcn_exp2f(at * 0x1.ec709ep-2f);
        y = at * e * u * e * e;
    }
    return y;
}

// Stores of four and eight bf16 to any even address.
__device__ __forceinline__ void store4(uint16_t* to, uint2 v) {
    struct __attribute__((packed, aligned(2))) Four { uint32_t w[2]; };
    *reinterpret_cast<Four*>(to) = Four{{v.x, v.y}};
}
__device__ __forceinline__ void store8(uint16_t* to, uint4 v) {
    struct __attribute__((packed, aligned(2))) Eight { uint32_t w[4]; };
    *reinterpret_cast<Eight*>(to) = Eight{{v.x, v.y, v.z, v.w}};
}
// Four outputs of a row from `channel` on, those below n.
__device__ __forceinline__ void store_outputs(uint16_t* to, const float* y, int channel, int n) {
    if (channel + 4 <= n) {
        store4(to, make_uint2(pack_bf16x2(y[0], y[1]), pack_bf16x2(y[2], y[3])));
    } else {
#pragma unroll
        for (int r = 0; r < 4; ++r)
            if (channel + r < n) to[r] = f32_to_bf16(y[r]);
    }
}

// Whether float(acc) s t is the same bits as scaled's for all such scales s, t and any sum: nothing on the way overflows
// or becomes subnormal, and powers of two change no rounding.
__device__ __forceinline__ bool middling(float s) { return s == 0.0f || (s >= 0x1.0p-60f && s <= 0x1.0p40f); }

}  // namespace nvr
