// Attention of trees of drafted tokens over the paged KV cache
// (nv_attention_tree). No counterpart in the reference, whose attention
// (kernels/kernels.cu:226-346) sees positions only.
//
// Semantics. Sequence s has n = row_starts[s + 1] - row_starts[s] drafted
// tokens, its nodes: node i is row row_starts[s] + i of q and out, and its K and
// V lie at position contexts[s] + i of the sequence. Row r = (s, i), q head h
// (kv head h / (qh / kvh)) sees the positions t < contexts[s], and node j's
// where bit j of masks[r] is set:
//   out[r, h] = sum_t p_t v_t / sum_t p_t,  p_t = exp(score_t - max score),
//   score_t = q . k_t / sqrt(dim).
// As in nv_attention, a position in a block outside [0, blocks) is not seen, and
// a row that sees nothing, or whose maximum is not finite or whose sum is not
// positive, is +0. What lies at positions that a row does not see never reaches
// it, NaN and Inf included. Sequences whose rows do not lie in [0, rows) are
// passed over; with more than max_nodes nodes, a negative context, or more than
// min(max_context, stride * bs) positions their rows are +0. Rows of no sequence
// are left as they were.
//
// Scores, maxima, sums and outputs are fp32, and the outputs rounded to bf16 once
// at the end. The tile form hands each weight p_t to the matrix instructions as the
// sum of two bf16 (within 2^-15 of it).
#include "../../include/nano_hip.h"
#include "nvr_device.h"
#include "nvr_internal.h"

#include <algorithm>
#include <type_traits>

namespace {

using nvr::kWave;
constexpr int kMaxNodes = 64;  // a row's mask is one 64-bit word
constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kInf = __builtin_inff();
struct TreeArgs {
    const uint16_t* q;
    const uint16_t* kc;
    const uint16_t* vc;
    const int* contexts;
    const int* row_starts;
    const uint64_t* masks;
    const int* tables;
    uint16_t* out;
    int rows, qh, kvh, dim, bs, blocks, stride, batch, max_nodes;
    int64_t limit;  // positions a sequence may have
    float scale;    // log2(e) / sqrt(dim)
};

struct TreeSpan {
    int start, nodes, context;  // nodes 0: nothing to write; context -1: +0 rows
};

__device__ __forceinline__ TreeSpan tree_span(const TreeArgs& a, int s) {
    TreeSpan t{a.row_starts[s], 0, a.contexts[s]};
    const int end = a.row_starts[s + 1];
    if (t.start < 0 || end > a.rows || t.start >= end) return t;
    t.nodes = end - t.start;
    if (t.context < 0 || t.nodes > a.max_nodes || int64_t(t.context) + t.nodes > a.limit) t.context = -1;
    return t;
}

// Any head dim, block size and alignment: a block per (node, q head), its four
// waves over every fourth position, lanes over the head's elements. Bound by the
// chain of one position's load, dot product and 64-lane sum after the other: with
// heads of 128, 8 trees of 25 nodes at 1030 positions in blocks of 8 take 785 us (the
// tile form in blocks of 256 22), as many as with fp32 sums.
__global__ __launch_bounds__(256) void attention_tree_direct(TreeArgs a) {
    constexpr int kWaves = 4, kElems = 4;  // 64 lanes x 4 elements: head dims up to 256
    __shared__ float part_m[kWaves];
    __shared__ double part_l[kWaves], part_o[kWaves][256];  // as the sums: of V of any size
    const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
    const int head = int(blockIdx.x % unsigned(a.qh));
    const int item = int(blockIdx.x / unsigned(a.qh));
    const int s = item / a.max_nodes, node = item % a.max_nodes;
    const TreeSpan t = tree_span(a, s);
    if (node >= t.nodes) return;
    if (t.context < 0) {
        for (int i = node; i < t.nodes; i += a.max_nodes) {
            uint16_t* o = a.out + (int64_t(t.start + i) * a.qh + head) * a.dim;
            for (int d = int(threadIdx.x); d < a.dim; d += 256) o[d] = 0;
        }
        return;
    }
    const int64_t row = int64_t(t.start + node) * a.qh + head;
    const uint64_t mask = a.masks[t.start + node];
    const int64_t pitch = int64_t(a.kvh) * a.dim, column = int64_t(head / (a.qh / a.kvh)) * a.dim;
    float q[kElems];
    double o[kElems] = {}, l = 0.0;
#pragma unroll
    for (int e = 0; e < kElems; ++e) {
        const int d = lane + e * kWave;
        q[e] = d < a.dim ? nvr::bf16_to_f32(a.q[row * a.dim + d]) : 0.0f;
    }
    float m = -kInf;
    const int keys = t.context + t.nodes;
    for (int pos = wave; pos < keys; pos += kWaves) {
        if (pos >= t.context && (mask >> (pos - t.context) & 1) == 0) continue;
        const int entry = a.tables[int64_t(s) * a.stride + pos / a.bs];
        if (entry < 0 || entry >= a.blocks) continue;
        const int64_t at = (int64_t(entry) * a.bs + pos % a.bs) * pitch + column;
        float dot = 0.0f;
#pragma unroll
        for (int e = 0; e < kElems; ++e) {
            const int d = lane + e * kWave;
            if (d < a.dim) dot = __builtin_fmaf(q[e], nvr::bf16_to_f32(a.kc[at + d]), dot);
        }
#pragma unroll
        for (int w = 1; w < kWave; w <<= 1) dot += nvr::xor_lane(dot, w);
        if (dot == -kInf) continue;
        const float top = fmaxf(m, dot);  // a NaN leaves m, and makes l NaN
        // Of the scores' distances, which are exact to their own 2^-24 however large both are.
        const float old = m == -kInf ? 0.0f : __builtin_amdgcn_exp2f((m - top) * a.scale);
        const float p = __builtin_amdgcn_exp2f((dot - top) * a.scale);
        m = top;
        l = __builtin_fma(l, double(old), double(p));
#pragma unroll
        for (int e = 0; e < kElems; ++e) {
            const int d = lane + e * kWave;
            if (d < a.dim) o[e] = __builtin_fma(double(p), double(nvr::bf16_to_f32(a.vc[at + d])), o[e] * double(old));
        }
    }
    if (lane == 0) { part_m[wave] = m; part_l[wave] = l; }
#pragma unroll
    for (int e = 0; e < kElems; ++e) part_o[wave][lane + e * kWave] = o[e];
    __syncthreads();
    float top = -kInf;
    double den = 0.0, num = 0.0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) top = fmaxf(top, part_m[w]);
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
        if (part_m[w] == -kInf && part_l[w] == 0.0) continue;  // saw nothing
        const double f = double(__builtin_amdgcn_exp2f((part_m[w] - top) * a.scale));
        den = __builtin_fma(part_l[w], f, den);
        num = __builtin_fma(part_o[w][threadIdx.x], f, num);
    }
    if (int(threadIdx.x) < a.dim)
        a.out[row * a.dim + threadIdx.x] = nvr::f32_to_bf16(den > 0.0 ? float(num / den) : 0.0f);
}

// ------------------------------------------------------------- tile form ----
typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef short s16x4_t __attribute__((ext_vector_type(4)));

__device__ __forceinline__ f32x4_t mfma(bf16x8_t a, bf16x8_t b, f32x4_t c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4_t mfma(s16x4_t a, s16x4_t b, f32x4_t c) {
    return __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ bf16x8_t operand(const uint4& w) { return __builtin_bit_cast(bf16x8_t, w); }

// At most N of this wave's vector memory operations outstanding.
template <int N>
__device__ __forceinline__ void wait_copies() {
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

constexpr int kPage = 16;  // positions that lie together in the cache: block sizes are multiples

// A weight is 2^(d - bias) of its score's distance d, in powers of two, from a scale m, which is exact to its own 2^-24
// however large both are. m follows the maximum, and the bias the weights' sum, so that a wave's sum stays below 1: fp32
// sums of the largest V are finite, over any number of positions. The maximum may outgrow m by 2^kLag before o and l are
// scaled again; where a lane's sum has passed kFull, they shrink by 2^kShrink, which the bias gives back as the maximum
// grows. So the sum is 2^-kBias at least (11 to 13), and what fp32 rounds of a sum over 32 positions, 2^-150 at most, is
// 2^-137 of the smallest V's outputs, whose last bit is 2^-133. A lag of 2 with 2^-10 would keep three bits more (8 trees
// of 25 at 1030 24.2 us against 23.1, 16 of 33 at 2000 39.5, 37.0), one of 8 with 2^-15 two less (22.9, 37.0). At the end
// the waves' and the splits' outputs meet by their shares of 1.
constexpr float kLag = 6.0f, kFull = 0x1p-5f, kShrink = 4.0f;
constexpr float kAbove = 1.0f + 0x1p-18f;

// Compile-time geometry. DIM: head dim rounded up; W: waves; QT: tiles of 16
// query rows a wave; WQ of the waves hold query rows of their own, the other
// factor WK splits each tile's T positions; NS: tiles in LDS.
template <int DIM_, int W_, int QT_, int WQ_, int T_, int NS_>
struct Shape {
    static constexpr int DIM = DIM_, W = W_, QT = QT_, WQ = WQ_, WK = W_ / WQ_, T = T_, NS = NS_;
    static constexpr int KW = T / WK;                // a wave's positions of a tile
    static constexpr int KT = KW / 16;               // 16-position tiles of those
    static constexpr float kBias = 11 + KT / 2;      // a lane's 4 KT weights of a tile, up to 2^(kLag - kBias), are 2^-3 at most
    static constexpr int DT = DIM / 16;              // 16-element tiles of a head
    static constexpr int KS = DIM / 32;              // products of 32 elements a score
    static constexpr int CH = DIM / 8;               // 16-byte chunks a row
    static constexpr int R = kWave / CH;             // rows a copy instruction
    static constexpr int OWN = T / W;                // rows that a wave copies
    static constexpr int COPIES = OWN / R;           // copy instructions a wave, tile and operand
    static constexpr int ROWS = 16 * QT * WQ;        // query rows a block
    static constexpr int kTile = T * DIM * 2;        // bytes of K or V
    static constexpr int kStage = 2 * kTile;
    static constexpr int kMerge = WK / 2 * WQ * QT * kWave * (16 * DT + 8);  // of half the waves that split positions
    static constexpr int kLds = NS * kStage > kMerge ? NS * kStage : kMerge;
    static constexpr int kFit = 160 * 1024 / (kLds + 64), kBlocks = kFit < 16 / W ? kFit : 16 / W;  // a CU (16 waves)
    static constexpr bool kAlone = WQ == 1;          // a wave reads only the rows that it copied
    static_assert(KT == 1 || KT == 2 || KT == 4, "kBias");
    static_assert((COPIES == 1 || COPIES == 2 || COPIES == 4) && T <= 64 && kPage % OWN == 0 && KW % 16 == 0 && (!kAlone || KW == OWN), "tiles");
};

// Where chunk c of a row lies in its LDS row: sixteen rows' same chunk (a K
// operand) and eight rows' same pair of chunks (a transposed V read) are on all banks.
template <int CH>
__device__ __forceinline__ int k_chunk(int row, int c) {
    return c ^ (CH == 8 ? row >> 1 & 7 : row & 15);
}
template <int CH>
__device__ __forceinline__ int v_chunk(int row, int c) {
    return c ^ (CH == 8 ? (row >> 1 & 3) << 1 : (row & 7) << 1);
}

// Two bf16, an Inf or NaN as 0.
__device__ __forceinline__ uint32_t numbers(uint32_t w) {
    return ((w & 0x7f80u) == 0x7f80u ? 0u : w & 0xffffu) | ((w & 0x7f800000u) == 0x7f800000u ? 0u : w & 0xffff0000u);
}

// Partial results of a split: its outputs by themselves, then (m, sum of 2^d) pairs.
struct Partials {
    float* out;   // [splits, rows * qh, dim]
    float2* sum;  // [splits, rows * qh]
    int splits;
};

// The fewest positions of a split. One chain of 4 at 180 whole 9.4 us, in two 11.1;
// parts of 128 against 256: 4 trees of 13 at 500 15.7, 17.0, one chain of 8 at 1000 12.1,
// 13.1, 8 of 9 at 700 with heads of 64 14.2, 17.3, one tree of 25 at 4000 21.3, 21.7. (One
// number of splits for all sequences of a call: where one is far longer than the others,
// the call lasts as long as that one's parts.)
constexpr int kWhole = 256, kShort = 1024;  // positions that are not split, that are split finely

// Tiles (of 2^shift positions) a split: the same for every split but the last.
__device__ __forceinline__ int split_tiles(int tiles, int splits, int shift) {
    const int least = tiles <= kWhole >> shift ? tiles : (tiles <= kShort >> shift ? 128 : 256) >> shift;
    const int per = max((tiles + splits - 1) / splits, least), used = (tiles + per - 1) / per;
    return (tiles + used - 1) / used;
}

// A block a (sequence, KV head, chunk of its query rows, split of its positions).
// The query rows of a KV head are its tree's nodes times the q heads over it: all
// of a chunk share one read of K and V, whose tiles of T positions come into a ring
// of NS stages by copies that bypass the registers, each wave its own rows of every
// tile. One pass, with each row's running maximum and sum:
//  - scores transposed, K q^T: a lane then holds four positions of one query row for
//    each 16, just as the second product wants its weights, which therefore never
//    leave registers; the row's maximum needs two exchanges, and only where it grew.
//  - outputs transposed, V^T p: V is read from LDS transposed by the hardware.
// Chunks lie swizzled in LDS, so that neither read has bank conflicts. Sequences are
// split, in parts of at least 128 or 256 positions, until the blocks fill the CUs; the parts
// meet in attention_tree_join.
//
// What bounds it, on MI355X (times with the join's): with few rows the read of the
// cache, 64 chains of 6 nodes at 4090 positions 155 us, 5.4 TB/s; with many each tile's
// chain of copies, LDS reads, products and exponentials, which the waves of a block go
// through in step: 4 trees of 64 at 16000 76 us, 3.6 TB/s, the matrix instructions busy
// for 27% of it, and with eight q heads a KV head 16 trees of 33 at 2000 35 us; small
// calls the launch (3 us), the tables and the first tiles, one chain of 4 at 180 9 us.
template <typename S>
__global__ __launch_bounds__(kWave* S::W, S::kBlocks* S::W / 4) void attention_tree_tiles(TreeArgs a, Partials part, int chunks,
                                                                        int page_shift, int spread) {
    constexpr int DIM = S::DIM, QT = S::QT, WQ = S::WQ, WK = S::WK, T = S::T, KT = S::KT, DT = S::DT, KS = S::KS;
    constexpr int CH = S::CH, R = S::R, COPIES = S::COPIES, NS = S::NS, kThreads = kWave * S::W;
    extern __shared__ __align__(16) unsigned char smem[];  // NS stages of K, then V
    __shared__ int poison[2];
    const int lane = threadIdx.x & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int n16 = lane & 15, g = lane >> 4;
    const int wq = wave % WQ, wk = wave / WQ;
    // spread 3: blocks go round the eight XCDs, so the chunks of one part of the cache follow each other on one, whose L2 they share.
    const unsigned turn = blockIdx.x >> spread;
    const int chunk = int(turn % unsigned(chunks));
    unsigned item = turn / unsigned(chunks) << spread | (blockIdx.x & ((1u << spread) - 1));
    const int kvhead = int(item % unsigned(a.kvh));
    item /= unsigned(a.kvh);
    const int split = int(item % unsigned(part.splits)), s = int(item / unsigned(part.splits));
    const TreeSpan span = tree_span(a, s);
    const int group = a.qh / a.kvh;
    if (span.context < 0) {
        if (split != 0) return;
        for (int64_t i = chunk * (kThreads / 16) + int(threadIdx.x) / 16; i < int64_t(span.nodes) * group;
             i += int64_t(chunks) * (kThreads / 16)) {
            uint16_t* o = a.out + ((span.start + i / group) * a.qh + kvhead * group + i % group) * a.dim;
            for (int d = 8 * n16; d < a.dim; d += 128) *reinterpret_cast<uint4*>(o + d) = make_uint4(0, 0, 0, 0);
        }
        return;
    }
    // A sequence's query rows are dealt evenly to as many blocks as they need.
    const int all = span.nodes * group, shares = (all + S::ROWS - 1) / S::ROWS;
    const int share = ((all + shares - 1) / max(shares, 1) + 16 * QT - 1) / (16 * QT) * (16 * QT);
    const int q0 = chunk * share, queries = min(all, q0 + share);
    if (chunk >= shares || q0 >= queries) return;
    const int keys = span.context + span.nodes, tiles = (keys + T - 1) / T;
    const int per = split_tiles(tiles, part.splits, __builtin_ctz(T)), used = (tiles + per - 1) / per;
    if (split >= used) return;
    const int tile0 = split * per, tile1 = min(tiles, tile0 + per);

    // ---- this wave's query rows: the B operand of the scores ----
    const bool working = q0 + wq * QT * 16 < queries;
    bf16x8_t q[QT][KS];
    uint64_t mask[QT];
#pragma unroll
    for (int t = 0; t < QT; ++t) {
        const int i = q0 + (wq * QT + t) * 16 + n16;
        const bool real = i < queries;
        const int node = real ? i / group : 0;
        const uint16_t* row = a.q + (int64_t(span.start + node) * a.qh + kvhead * group + (real ? i % group : 0)) * a.dim;
#pragma unroll
        for (int k = 0; k < KS; ++k) {
            const int d = 32 * k + 8 * g;
            q[t][k] = operand(real && d < a.dim ? *reinterpret_cast<const uint4*>(row + d) : make_uint4(0, 0, 0, 0));
        }
        mask[t] = real ? a.masks[span.start + node] : 0;
    }

    // ---- positions' places in the cache, by pages of 16 positions ----
    using Table = const __attribute__((address_space(4))) int*;  // scalar loads: they do not count with the copies
    const Table table = (Table)(a.tables + int64_t(s) * a.stride);
    const int pages = a.bs / kPage, last_page = (keys - 1) / kPage;
    auto entry_of = [&](int page) { return page_shift >= 0 ? page >> page_shift : page / pages; };
    // The cache row of a page's first position, or -1.
    auto place = [&](int page) {
        const int at = entry_of(page), entry = table[at];
        return entry >= 0 && entry < a.blocks ? entry * a.bs + (page - at * pages) * kPage : -1;
    };
    bool holes = false;
    for (int i = entry_of(tile0 * T / kPage) + lane; i <= entry_of(min(tile1 * T / kPage - 1, last_page)); i += kWave) {
        const int entry = a.tables[int64_t(s) * a.stride + i];
        holes |= entry < 0 || entry >= a.blocks;
    }
    const bool any_holes = __ballot(holes) != 0;

    const int64_t pitch = int64_t(a.kvh) * a.dim;
    const uint16_t* kcol = a.kc + int64_t(kvhead) * a.dim;
    const uint16_t* vcol = a.vc + int64_t(kvhead) * a.dim;
    const uint32_t lds = __builtin_amdgcn_readfirstlane(nvr::lds_address(smem));
    const int crow = wave * S::OWN + lane / CH, cslot = lane % CH;  // this lane's row and slot of copy 0
    // Bytes from the page's row. A copy's offset field moves both sides by its 1 KB of LDS (whole heads only:
    // there a row is at least as long in the cache).
    const bool whole = a.dim == DIM;
    uint32_t koff[COPIES], voff[COPIES];
#pragma unroll
    for (int u = 0; u < COPIES; ++u) {
        const int row = crow + u * R;
        koff[u] = uint32_t((row % kPage) * int(pitch) + 8 * k_chunk<CH>(row, cslot)) * 2 - (whole ? u * 1024 : 0);
        voff[u] = uint32_t((row % kPage) * int(pitch) + 8 * v_chunk<CH>(row, cslot)) * 2 - (whole ? u * 1024 : 0);
    }
    // M0 holds the LDS address and is restored after the copies.
#define NVR_COPY(n) "global_load_lds_dwordx4 %" #n ", %1 offset:"
#define NVR_WITH_M0(loads) "s_mov_b32 %0, m0\n\ts_mov_b32 m0, %2\n\ts_nop 0\n\t" loads "s_mov_b32 m0, %0"
    auto copy_one = [&](uint32_t offset, const uint16_t* base, uint32_t dst) {
        uint32_t saved;
        asm volatile(NVR_WITH_M0(NVR_COPY(3) "0\n\t") : "=&s"(saved) : "s"(base), "s"(dst), "v"(offset) : "memory");
    };
    auto copy_all = [&](const uint32_t (&offset)[COPIES], const uint16_t* base, uint32_t dst) {
        uint32_t saved;
        if constexpr (COPIES == 4)
            asm volatile(NVR_WITH_M0(NVR_COPY(3) "0\n\t" NVR_COPY(4) "0x400\n\t" NVR_COPY(5) "0x800\n\t" NVR_COPY(6) "0xc00\n\t")
                         : "=&s"(saved)
                         : "s"(base), "s"(dst), "v"(offset[0]), "v"(offset[1]), "v"(offset[2]), "v"(offset[3])
                         : "memory");
        else if constexpr (COPIES == 1)
            asm volatile(NVR_WITH_M0(NVR_COPY(3) "0\n\t") : "=&s"(saved) : "s"(base), "s"(dst), "v"(offset[0]) : "memory");
        else
            asm volatile(NVR_WITH_M0(NVR_COPY(3) "0\n\t" NVR_COPY(4) "0x400\n\t")
                         : "=&s"(saved)
                         : "s"(base), "s"(dst), "v"(offset[0]), "v"(offset[1])
                         : "memory");
    };
#undef NVR_COPY
#undef NVR_WITH_M0
    auto copy = [&](int tile, int row0) {  // row0: the cache row of this wave's page
        const int64_t at = int64_t(max(row0, 0)) * pitch;
        const uint16_t* kbase = kcol + at;
        const uint16_t* vbase = vcol + at;
        const uint32_t dst = __builtin_amdgcn_readfirstlane(lds + uint32_t((tile - tile0) % NS * S::kStage + wave * S::OWN * DIM * 2));
        if (whole) {
            copy_all(koff, kbase, dst);
            copy_all(voff, vbase, dst + S::kTile);
        } else {
#pragma unroll
            for (int u = 0; u < COPIES; ++u) {
                if (k_chunk<CH>(crow + u * R, cslot) * 8 < a.dim) copy_one(koff[u], kbase, dst + u * 1024);
                if (v_chunk<CH>(crow + u * R, cslot) * 8 < a.dim) copy_one(voff[u], vbase, dst + S::kTile + u * 1024);
            }
        }
    };
    auto own_page = [&](int tile) {
        return __builtin_amdgcn_readfirstlane(place(min((tile * T + wave * S::OWN) / kPage, last_page)));
    };
    int rows0[NS - 1];
#pragma unroll
    for (int i = 0; i < NS - 1; ++i) rows0[i] = own_page(min(tile0 + i, tile1 - 1));
    if (a.dim < DIM) {  // chunks past the head are never copied
        for (int i = int(threadIdx.x); i < NS * S::kStage / 16; i += kThreads)
            *reinterpret_cast<uint4*>(smem + 16 * i) = make_uint4(0, 0, 0, 0);
    }
    if (threadIdx.x < 2) poison[threadIdx.x] = -1;
    __syncthreads();
    // Every register load is awaited here, so that none is where the copies are counted.
#pragma unroll
    for (int t = 0; t < QT; ++t) {
#pragma unroll
        for (int k = 0; k < KS; ++k) asm volatile("" : "+v"(q[t][k]));
        asm volatile("" : "+v"(mask[t]));
    }
#pragma unroll
    for (int i = 0; i < NS - 1; ++i)
        if (tile0 + i < tile1) copy(tile0 + i, rows0[i]);
    int next_row = own_page(min(tile0 + NS - 1, tile1 - 1));

    f32x4_t o[QT][DT];
    float m[QT], l[QT], bias[QT];  // l: the weights' sum, of this lane's positions
#pragma unroll
    for (int t = 0; t < QT; ++t) {
        m[t] = -kInf;
        l[t] = 0.0f;
        bias[t] = S::kBias;
#pragma unroll
        for (int d = 0; d < DT; ++d) o[t][d] = f32x4_t{0, 0, 0, 0};
    }

    // One tile; `masked`: some of its positions are not seen by every row.
    auto step = [&](int tile, auto masked) {
        constexpr bool kMasked = decltype(masked)::value;
        const int stage = (tile - tile0) % NS, first = tile * T;
        const unsigned char* kt = smem + stage * S::kStage;
        unsigned char* vt = smem + stage * S::kStage + S::kTile;
        if (tile + NS - 2 < tile1) wait_copies<(NS - 2) * 2 * COPIES>();  // this wave's rows of the tile
        else wait_copies<0>();
        const bool drafted = kMasked && first + T > span.context;
        uint64_t mapped = T == 64 ? ~uint64_t(0) : (uint64_t(1) << (T & 63)) - 1;
        if constexpr (kMasked) {
            if (keys - first < T) mapped = (uint64_t(1) << (keys - first)) - 1;
#pragma unroll
            for (int i = 0; i < T / kPage; ++i)
                if (first + i * kPage < keys && place(first / kPage + i) < 0) mapped &= ~(uint64_t(0xffff) << (i * kPage));
        }
        if constexpr (kMasked) {
            bool found = false;
#pragma unroll
            for (int u = 0; u < COPIES; ++u) {
                const int row = crow + u * R;
                uint4* v = reinterpret_cast<uint4*>(vt + (row * CH + cslot) * 16);
                if ((mapped >> row & 1) == 0) {
                    *v = make_uint4(0, 0, 0, 0);  // weighs nothing, and must be a number for that
                } else if (first + row >= span.context) {
                    // What some rows do not see must be a number for their weight of 0.
                    const uint4 w = *v;
                    const uint4 whole = make_uint4(numbers(w.x), numbers(w.y), numbers(w.z), numbers(w.w));
                    if (whole.x != w.x || whole.y != w.y || whole.z != w.z || whole.w != w.w) {
                        found = true;
                        *v = whole;
                    }
                }
            }
            if (__ballot(found) != 0 && lane == 0) poison[tile & 1] = tile;
        }
        // The tile is whole, and every read of the stage that the next copies fill is done.
        if (!S::kAlone || drafted) asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
        else asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        if (tile + NS - 1 < tile1) {
            copy(tile + NS - 1, next_row);
            next_row = own_page(min(tile + NS, tile1 - 1));
        }
        if (!working) return;

        // ---- scores, transposed: positions x query rows ----
        f32x4_t x[QT][KT];
#pragma unroll
        for (int t = 0; t < QT; ++t)
#pragma unroll
            for (int j = 0; j < KT; ++j) x[t][j] = f32x4_t{0, 0, 0, 0};
#pragma unroll
        for (int j = 0; j < KT; ++j) {
            const int row = wk * S::KW + 16 * j + n16;
#pragma unroll
            for (int k = 0; k < KS; ++k) {
                const bf16x8_t kv = operand(
                    *reinterpret_cast<const uint4*>(kt + (row * CH + k_chunk<CH>(row, 4 * k + g)) * 16));
#pragma unroll
                for (int t = 0; t < QT; ++t) x[t][j] = mfma(kv, q[t][k], x[t][j]);
            }
        }
        auto seen = [&](int t) -> uint64_t {  // of this wave's positions, by row t
            const int past = span.context - first;  // positions of the context in the tile
            const uint64_t sees = past >= 64 ? ~uint64_t(0)
                                  : past > 0 ? ((uint64_t(1) << past) - 1) | mask[t] << past
                                  : past > -64 ? mask[t] >> -past : 0;
            return (sees & mapped) >> (wk * S::KW);
        };
#pragma unroll
        for (int t = 0; t < QT; ++t) {
            if constexpr (kMasked) {
                const uint64_t sees = seen(t);
#pragma unroll
                for (int j = 0; j < KT; ++j)
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        x[t][j][r] = (sees >> (16 * j + 4 * g + r) & 1) != 0 ? x[t][j][r] : -kInf;
            }
            float top = -kInf;
#pragma unroll
            for (int j = 0; j < KT; ++j)
#pragma unroll
                for (int r = 0; r < 4; ++r) top = fmaxf(top, x[t][j][r]);
            if (__ballot((top - m[t]) * a.scale > kLag || l[t] > kFull) != 0) {
                top = fmaxf(top, m[t]);
                top = fmaxf(top, nvr::xor_lane(top, 16));
                top = fmaxf(top, nvr::xor_lane(top, 32));
                float shrink = 0.0f;
                if (__ballot(l[t] > kFull) != 0) {
                    shrink = l[t] > kFull ? kShrink : 0.0f;
                    shrink = fmaxf(shrink, nvr::xor_lane(shrink, 16));
                    shrink = fmaxf(shrink, nvr::xor_lane(shrink, 32));
                }
                // Where the maximum grew, the bias comes back by as much, to a multiple of 2^-8: it stays exact.
                const float grown = (top - m[t]) * a.scale, back = fminf(bias[t] - S::kBias, __builtin_floorf(grown * 256.0f) * (1.0f / 256.0f));
                const float old = m[t] == -kInf ? 0.0f : __builtin_amdgcn_exp2f(back - shrink - grown);
                bias[t] += shrink - back;
                l[t] *= old;
#pragma unroll
                for (int d = 0; d < DT; ++d)
#pragma unroll
                    for (int r = 0; r < 4; ++r) o[t][d][r] *= old;
                m[t] = top;
            }
            const float base = m[t] == -kInf ? 0.0f : m[t];
#pragma unroll
            for (int j = 0; j < KT; ++j) {
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    x[t][j][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(x[t][j][r] - base, a.scale, -bias[t]));
                l[t] += (x[t][j][0] + x[t][j][1]) + (x[t][j][2] + x[t][j][3]);
            }
        }

        // ---- outputs, transposed: head elements x query rows ----
        const int vrow = wk * S::KW + 4 * g + (n16 >> 2);
        auto read = [&](int row, int d) {
            const int c = 2 * d + (n16 >> 1 & 1);
            auto* at = (__attribute__((address_space(3))) s16x4_t*)(vt + (row * CH + v_chunk<CH>(row, c)) * 16 + 8 * (n16 & 1));
            return __builtin_amdgcn_ds_read_tr16_b64_v4i16(at);
        };
        // Four weights, times kAbove, as two bf16 each: their upper halves and what those leave, rounded (up to 2^-15 of
        // the weight). Both are positive where the weight is, so that an Inf in V stays one.
        auto halves = [&](const f32x4_t& w, uint2& hi, uint2& lo) {
            auto upper = [](float a, float b) { return __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302u); };
            auto left = [](float f) { return __builtin_fmaf(f, kAbove, -__uint_as_float(__float_as_uint(f) & 0xffff0000u)); };
            hi = make_uint2(upper(w[0], w[1]), upper(w[2], w[3]));
            lo = make_uint2(nvr::pack_bf16x2(left(w[0]), left(w[1])), nvr::pack_bf16x2(left(w[2]), left(w[3])));
        };
        if constexpr (KT == 1) {
            s16x4_t p[QT], rest[QT];
#pragma unroll
            for (int t = 0; t < QT; ++t) {
                uint2 hi, lo;
                halves(x[t][0], hi, lo);
                p[t] = __builtin_bit_cast(s16x4_t, hi);
                rest[t] = __builtin_bit_cast(s16x4_t, lo);
            }
#pragma unroll
            for (int d = 0; d < DT; ++d) {
                const s16x4_t v = read(vrow, d);
#pragma unroll
                for (int t = 0; t < QT; ++t) o[t][d] = mfma(v, p[t], o[t][d]);
#pragma unroll
                for (int t = 0; t < QT; ++t) o[t][d] = mfma(v, rest[t], o[t][d]);
            }
        } else {
            // Positions 4 g .. 4 g + 3 of two tiles: with V read in the same order, a product's 32 positions.
            bf16x8_t p[QT][KT / 2], rest[QT][KT / 2];
#pragma unroll
            for (int t = 0; t < QT; ++t)
#pragma unroll
                for (int j = 0; j < KT / 2; ++j) {
                    uint2 hi[2], lo[2];
                    halves(x[t][2 * j], hi[0], lo[0]);
                    halves(x[t][2 * j + 1], hi[1], lo[1]);
                    p[t][j] = operand(make_uint4(hi[0].x, hi[0].y, hi[1].x, hi[1].y));
                    rest[t][j] = operand(make_uint4(lo[0].x, lo[0].y, lo[1].x, lo[1].y));
                }
#pragma unroll
            for (int d = 0; d < DT; ++d)
#pragma unroll
                for (int j = 0; j < KT / 2; ++j) {
                    const s16x4_t lo = read(vrow + 32 * j, d), hi = read(vrow + 32 * j + 16, d);
                    const bf16x8_t v = __builtin_bit_cast(bf16x8_t, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
#pragma unroll
                    for (int t = 0; t < QT; ++t) o[t][d] = mfma(v, p[t][j], o[t][d]);
#pragma unroll
                    for (int t = 0; t < QT; ++t) o[t][d] = mfma(v, rest[t][j], o[t][d]);
                }
        }
        if (drafted && poison[tile & 1] == tile) {
            // Nodes with an Inf or NaN in V, which went into the products as 0: added for the rows that see them.
#pragma unroll 1
            for (int i = 0; i < S::KW; ++i) {
                const int row = wk * S::KW + i;
                if ((mapped >> row & 1) == 0 || first + row < span.context) continue;
                const uint16_t* from = vcol + int64_t(place((first + row) / kPage) + row % kPage) * pitch;
                bool sees[QT];
#pragma unroll
                for (int t = 0; t < QT; ++t) sees[t] = (seen(t) >> i & 1) != 0;
#pragma unroll
                for (int d = 0; d < DT; ++d)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int element = 16 * d + 4 * g + e;
                        const float v = element < a.dim ? nvr::bf16_to_f32(from[element]) : 0.0f;
                        const float add = __builtin_isfinite(v) ? 0.0f : v;
#pragma unroll
                        for (int t = 0; t < QT; ++t) o[t][d][e] += sees[t] ? add : 0.0f;
                    }
            }
        }
    };
    const int plain = any_holes ? tile0 : max(tile0, min(tile1, span.context / T));  // tiles that every row sees whole
    for (int tile = tile0; tile < plain; ++tile) step(tile, std::false_type{});
#pragma unroll 1
    for (int tile = plain; tile < tile1; ++tile) step(tile, std::true_type{});

    // ---- the waves' shares, then the output or the split's partial ----
    // From here on outputs are by themselves, of whatever share of 1, and sums of 2^d.
    float sum[QT];
#pragma unroll
    for (int t = 0; t < QT; ++t) {
        float all = l[t] + nvr::xor_lane(l[t], 16);
        all += nvr::xor_lane(all, 32);
        const float inv = all > 0.0f ? 1.0f / (all * kAbove) : 0.0f;
        sum[t] = all * __builtin_amdgcn_exp2f(bias[t]);
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int r = 0; r < 4; ++r) o[t][d][r] *= inv;
    }
    // The upper half of the waves hand theirs to the lower half, until one holds all.
    f32x4_t* merge = reinterpret_cast<f32x4_t*>(smem);
    float2* merge_sums = reinterpret_cast<float2*>(smem + (WK / 2 * WQ * QT * DT * kWave) * 16);
#pragma unroll
    for (int half = WK / 2; half > 0; half /= 2) {
        __syncthreads();  // the tiles, or the round before, are read
        const int from = (wk % max(half, 1) * WQ + wq) * QT;
        if (wk >= half && wk < 2 * half) {
#pragma unroll
            for (int t = 0; t < QT; ++t) {
#pragma unroll
                for (int d = 0; d < DT; ++d) merge[((from + t) * DT + d) * kWave + lane] = o[t][d];
                merge_sums[(from + t) * kWave + lane] = make_float2(m[t], sum[t]);
            }
        }
        __syncthreads();
        if (wk < half) {
#pragma unroll
            for (int t = 0; t < QT; ++t) {
                const float2 other = merge_sums[(from + t) * kWave + lane];
                const float top = fmaxf(m[t], other.x), base = top == -kInf ? 0.0f : top;
                const float mine = sum[t] * __builtin_amdgcn_exp2f((m[t] - base) * a.scale);
                const float its = other.y * __builtin_amdgcn_exp2f((other.x - base) * a.scale);
                m[t] = top;
                sum[t] = mine + its;
                const float inv = sum[t] > 0.0f ? 1.0f / sum[t] : 0.0f, f = mine * inv, h = its * inv;
#pragma unroll
                for (int d = 0; d < DT; ++d) {
                    const f32x4_t v = merge[((from + t) * DT + d) * kWave + lane];
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[t][d][e] = __builtin_fmaf(v[e], h, o[t][d][e] * f);
                }
            }
        }
    }
    if (wk != 0) return;
#pragma unroll
    for (int t = 0; t < QT; ++t) {
        const int qi = q0 + (wq * QT + t) * 16 + n16;
        if (qi >= queries) continue;
        const int64_t out_row = int64_t(span.start + qi / group) * a.qh + kvhead * group + qi % group;
        const int64_t at = int64_t(split) * a.rows * a.qh + out_row;
#pragma unroll
        for (int d = 0; d < DT; ++d) {
            const int e = 16 * d + 4 * g;
            if (e >= a.dim) continue;
            f32x4_t y;
#pragma unroll
            for (int r = 0; r < 4; ++r) y[r] = sum[t] > 0.0f ? o[t][d][r] : 0.0f;
            if (used == 1) {
                *reinterpret_cast<uint2*>(a.out + out_row * a.dim + e) =
                    make_uint2(nvr::pack_bf16x2(y[0], y[1]), nvr::pack_bf16x2(y[2], y[3]));
            } else {
                *reinterpret_cast<f32x4_t*>(part.out + at * a.dim + e) = y;
            }
        }
        if (used != 1 && g == 0) part.sum[at] = make_float2(m[t], sum[t]);
    }
}

// The splits of each row, where there was more than one: a thread four elements
// of one (node, head), its splits' loads in flight together. Bound by its launch and
// one memory round trip: 4.3 us for 168 rows of 16 heads in up to 8 splits (10 MB of
// partial outputs), 5.1 for 226 rows in 8 (15 MB).
__global__ __launch_bounds__(256) void attention_tree_join(TreeArgs a, Partials part, int shift, int parts) {
    constexpr int kBatch = 8;
    const int item = int(blockIdx.x / unsigned(parts));
    const int s = item / a.max_nodes, node = item % a.max_nodes;
    const TreeSpan span = tree_span(a, s);
    if (node >= span.nodes || span.context < 0) return;
    const int tiles = (span.context + span.nodes + (1 << shift) - 1) >> shift;
    const int per = split_tiles(tiles, part.splits, shift), used = (tiles + per - 1) / per;
    const int quads = a.dim / 4, i = int(blockIdx.x % unsigned(parts)) * 256 + int(threadIdx.x);
    if (used == 1 || i >= a.qh * quads) return;
    const int64_t at = int64_t(span.start + node) * a.qh + i / quads, plane = int64_t(a.rows) * a.qh;
    float2 ml[kBatch];
    f32x4_t v[kBatch];
    auto sums = [&](int w0) {
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
            ml[u] = part.sum[min(w0 + u, used - 1) * plane + at];
            if (w0 + u >= used) ml[u] = make_float2(-kInf, 0.0f);
        }
    };
    auto outs = [&](int w0) {
#pragma unroll
        for (int u = 0; u < kBatch; ++u)
            v[u] = *reinterpret_cast<const f32x4_t*>(part.out + (min(w0 + u, used - 1) * plane + at) * a.dim + 4 * (i % quads));
    };
    // The splits' shares of 1 first, so that no sum of theirs passes the outputs' own range.
    sums(0);
    outs(0);
    float top = -kInf, den = 0.0f;
    for (int w0 = 0;;) {
        float high = top;
#pragma unroll
        for (int u = 0; u < kBatch; ++u) high = fmaxf(high, ml[u].x);
        const float base = high == -kInf ? 0.0f : high;
        den *= __builtin_amdgcn_exp2f((top - base) * a.scale);
#pragma unroll
        for (int u = 0; u < kBatch; ++u) den = __builtin_fmaf(ml[u].y, __builtin_amdgcn_exp2f((ml[u].x - base) * a.scale), den);
        top = high;
        if ((w0 += kBatch) >= used) break;
        sums(w0);
    }
    if (used > kBatch) sums(0);
    const float base = top == -kInf ? 0.0f : top, inv = den > 0.0f ? 1.0f / den : 0.0f;
    f32x4_t num = {0, 0, 0, 0};
    for (int w0 = 0;;) {
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
            if (w0 + u >= used) continue;
            const float f = ml[u].y * __builtin_amdgcn_exp2f((ml[u].x - base) * a.scale) * inv;
#pragma unroll
            for (int r = 0; r < 4; ++r) num[r] = __builtin_fmaf(v[u][r], f, num[r]);
        }
        if ((w0 += kBatch) >= used) break;
        sums(w0);
        outs(w0);
    }
    float y[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) y[r] = den > 0.0f ? num[r] : 0.0f;
    *reinterpret_cast<uint2*>(a.out + at * a.dim + 4 * (i % quads)) =
        make_uint2(nvr::pack_bf16x2(y[0], y[1]), nvr::pack_bf16x2(y[2], y[3]));
}

// The launch's shape: the same for the workspace's size and the launch.
struct Plan {
    int dim;              // the head dim, rounded up
    int64_t queries, pairs;  // query rows a KV head; (sequence, KV head) pairs
    int tile, chunks, splits;  // positions a tile; blocks a KV head's rows; splits of the longest sequence
};
// The shape for `queries` query rows a KV head, of sequences and KV heads in
// `pairs`. Microseconds on MI355X, 16 q heads over 8 KV heads of 128, blocks of 256:
//  - up to 32 rows four waves split each tile's positions and read only what they
//    copied themselves, so they need no barrier. Two stages and two blocks a CU beat
//    four stages and one: 64 sequences of 6 nodes at 200 positions 16.4 against 24.4,
//    at 1000 44.1, 52.6, at 4090 155, 165.
//  - up to 64 rows, four waves over stages of 32 positions, two blocks a CU, against
//    eight waves over stages of 64: 64 of 30 at 300 29.2, 40.1, 8 of 25 at 1030 23.6, 24.5.
//  - above, the same four waves where there are more pairs than CUs (64 of 60 at 300
//    35.1 against 46.7, at 1000 77, 84); else eight waves, which need half the splits
//    to fill a CU (8 of 64 at 8000 86.5 against 82.9, 4 of 64 at 16000 86.1, 84.6).
//  - heads of 64, 16 of 33 nodes at 2000 with 8 heads a KV head: three blocks of four
//    waves a CU 37.5, one of eight over stages of 64 46.9, the same with twice the rows,
//    which spills, 155. Heads of 256 with two stages: 16 of 40 at 1000 33.0, with four 40.3.
//    (256 in these rules is the CUs of an MI355X; on another number they cost time only.)
template <typename F>
void with_shape(int dim, int64_t queries, int64_t pairs, F&& f) {
    if (dim == 256) {
        queries <= 32 ? f(Shape<256, 4, 1, 2, 32, 2>{}) : f(Shape<256, 4, 1, 4, 32, 2>{});
    } else if (dim == 128) {
        queries <= 16   ? f(Shape<128, 4, 1, 1, 64, 2>{})
        : queries <= 32 ? f(Shape<128, 4, 2, 1, 64, 2>{})
        : queries <= 64 ? f(Shape<128, 4, 2, 2, 32, 4>{})
        : pairs > 256   ? f(Shape<128, 4, 2, 4, 32, 4>{}) : f(Shape<128, 8, 2, 4, 64, 4>{});
    } else {
        queries <= 16   ? f(Shape<64, 4, 1, 1, 64, 3>{})
        : queries <= 32 ? f(Shape<64, 4, 2, 1, 64, 3>{})
        : queries <= 64 ? f(Shape<64, 8, 2, 2, 64, 4>{}) : f(Shape<64, 4, 2, 4, 32, 6>{});
    }
}
Plan plan_tiles(int qh, int kvh, int dim, int batch, int max_nodes, int max_context) {
    Plan p;
    p.dim = dim <= 64 ? 64 : dim <= 128 ? 128 : 256;
    p.queries = int64_t(max_nodes) * (qh / kvh);
    p.pairs = int64_t(batch) * kvh;
    with_shape(p.dim, p.queries, p.pairs, [&](auto shape) {
        using S = decltype(shape);
        p.tile = S::T;
        p.chunks = int((p.queries + S::ROWS - 1) / S::ROWS);
        const int64_t blocks = p.pairs * p.chunks, context = max_context;
        const int64_t fine = (std::min<int64_t>(context, kShort) + 127) / 128;
        const int64_t most = context <= kWhole ? 1 : std::max(fine, (context + 255) / 256);
        p.splits = int(std::max<int64_t>(1, std::min(most, 256 * S::kBlocks / blocks)));
    });
    return p;
}

// A multiple of 16 bytes.
int64_t workspace_bytes(const Plan& p, int rows, int qh, int dim) {
    const int64_t bytes = int64_t(p.splits) * rows * qh * (4 * int64_t(dim) + int64_t(sizeof(float2)));
    return p.splits == 1 ? 0 : (bytes + 15) / 16 * 16;
}

bool too_many(int rows, int qh, int batch, int kvh) {
    return int64_t(rows) * qh > 0x7fffffff || int64_t(batch) * kvh > 0x7fffffff;
}

}  // namespace

extern "C" {

int nv_attention_tree_workspace(int rows, int qh, int kvh, int dim, int batch, int max_nodes, int max_context,
                                size_t* bytes) {
    if (rows <= 0 || qh <= 0 || kvh <= 0 || dim <= 0 || batch <= 0 || max_nodes <= 0 || max_context <= 0 || qh % kvh)
        return nvr::fail(-2, "attention_tree_workspace: dimensions must be positive, q heads a multiple of KV heads");
    if (too_many(rows, qh, batch, kvh)) return nvr::fail(-2, "attention_tree_workspace: rows * qh or batch * kvh exceed int32");
    if (max_nodes > kMaxNodes || dim > 256) return nvr::fail(-2, "attention_tree_workspace: max_nodes %d, head dim %d", max_nodes, dim);
    *bytes = dim % 8 ? 0 : size_t(workspace_bytes(plan_tiles(qh, kvh, dim, batch, max_nodes, max_context), rows, qh, dim));
    return 0;
}

int nv_attention_tree(nv_context* c, const void* q, const void* kc, const void* vc, const void* contexts,
                      const void* row_starts, const void* masks, const void* tables, void* out, void* workspace,
                      int rows, int qh, int kvh, int dim, int bs, int blocks, int stride, int batch, int max_nodes,
                      int max_context) {
    NVR_ACTIVATE(c);
    if (rows <= 0 || qh <= 0 || kvh <= 0 || dim <= 0 || bs <= 0 || blocks <= 0 || stride <= 0 || batch <= 0)
        return nvr::fail(-2, "attention_tree: dimensions must be positive");
    if (qh % kvh != 0 || dim % 2 != 0 || dim > 256)
        return nvr::fail(-2, "attention_tree: %d q heads over %d KV heads of %d (a multiple; even, at most 256)", qh, kvh, dim);
    if (max_nodes < 1 || max_nodes > kMaxNodes)
        return nvr::fail(-2, "attention_tree: max_nodes %d outside [1, %d]", max_nodes, kMaxNodes);
    if (max_context < 1) return nvr::fail(-2, "attention_tree: max_context %d is not positive", max_context);
    if (too_many(rows, qh, batch, kvh)) return nvr::fail(-2, "attention_tree: rows * qh or batch * kvh exceed int32");
    const int64_t span = std::min(int64_t(stride) * bs, int64_t(0x7fff0000));  // tiles past the end stay below 2^31
    const TreeArgs a{static_cast<const uint16_t*>(q), static_cast<const uint16_t*>(kc), static_cast<const uint16_t*>(vc),
                     static_cast<const int*>(contexts), static_cast<const int*>(row_starts),
                     static_cast<const uint64_t*>(masks), static_cast<const int*>(tables), static_cast<uint16_t*>(out),
                     rows, qh, kvh, dim, bs, blocks, stride, batch, max_nodes,
                     span < max_context ? span : int64_t(max_context), kLog2e / sqrtf(float(dim))};
    const bool fits = dim % 8 == 0 && bs % kPage == 0 && int64_t(kvh) * dim <= 0x1000000 && nvr::aligned(q, 16) &&
                      nvr::aligned(kc, 16) && nvr::aligned(vc, 16) && nvr::aligned(out, 16) &&
                      int64_t(blocks) * bs <= 0x7fffffff;
    // A launch has fewer than 2^32 threads.
    constexpr int64_t kLaunch = 0xffffffff;
    const char* const exceeded = "attention_tree: %d sequences of %d nodes and %d heads exceed one launch";
    if (fits) {
        const Plan p = plan_tiles(qh, kvh, dim, batch, max_nodes, max_context);
        const int64_t grid = p.pairs * p.chunks * p.splits, parts = (int64_t(qh) * dim / 4 + 255) / 256;
        const int64_t joins = int64_t(batch) * max_nodes * parts;
        if (grid > kLaunch / 512 || (p.splits > 1 && joins > kLaunch / 256))
            return nvr::fail(-2, exceeded, batch, max_nodes, qh);
        if (p.splits > 1 && (workspace == nullptr || !nvr::aligned(workspace, 16)))
            return nvr::fail(-2, "attention_tree: needs a workspace at a multiple of 16 bytes");
        float* partial = static_cast<float*>(workspace);
        const Partials part{partial, reinterpret_cast<float2*>(partial + int64_t(p.splits) * rows * qh * dim), p.splits};
        const int pages = bs / kPage, shift = (pages & (pages - 1)) == 0 ? __builtin_ctz(unsigned(pages)) : -1;
        // Chunks on one XCD: 32 trees of 24 at 2000 with 8 heads a KV head of 64 46.5 us against 47.3, 16 of 33 37.5, 38.5.
        const int spread = p.chunks > 1 && p.pairs * p.splits % 8 == 0 ? 3 : 0;
        with_shape(p.dim, p.queries, p.pairs, [&](auto shape) {
            using S = decltype(shape);
            hipLaunchKernelGGL(attention_tree_tiles<S>, dim3(unsigned(grid)), dim3(kWave * S::W), S::kLds, c->stream, a,
                               part, p.chunks, shift, spread);
        });
        if (p.splits > 1) {
            NVR_HIP(hipGetLastError());
            hipLaunchKernelGGL(attention_tree_join, dim3(unsigned(joins)), dim3(256), 0, c->stream, a, part,
                               __builtin_ctz(unsigned(p.tile)), int(parts));
        }
        return nvr::launch_status();
    }
    const int64_t grid = int64_t(batch) * max_nodes * qh;
    if (grid > kLaunch / 256) return nvr::fail(-2, exceeded, batch, max_nodes, qh);
    hipLaunchKernelGGL(attention_tree_direct, dim3(unsigned(grid)), dim3(256), 0, c->stream, a);
    return nvr::launch_status();
}

}  // extern "C"
