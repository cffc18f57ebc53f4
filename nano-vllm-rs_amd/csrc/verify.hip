// Verification of trees of drafted tokens (nv_verify_tree): which path of a tree
// the target model accepts, and the token that follows it, by rejection sampling
// from given random numbers. No counterpart in the reference, which samples one
// token a sequence and step (kernels/kernels.cu:372-466).
//
// Semantics. Sequence s has n = row_starts[s + 1] - row_starts[s] rows: node 0 is
// its last committed token, the others are drafted, parents[r] < their own index
// the node that each continues. logits[r] are the target's after node r; T =
// temps[s]; p_v = softmax(logits[v] / T). From v = 0, node v's children are
// tried in index order, each with its token x and its uniform number u:
//   - T > 0, no draft logits (drafted tokens were picked, not sampled):
//     accepted if p_v(x) > 0 and u * (1 - sum of p_v of the tokens rejected here)
//     < p_v(x); a token rejected here before has no chance again. After all are
//     rejected, the rest is p_v without their tokens.
//   - T > 0, draft logits (children drawn independently from q_v =
//     softmax(draft_logits[v] / T)): accepted if p > 0 and u * Z * q_v(x) < p with
//     p = max(p_v(x) - c q_v(x), 0), where c = 0 and Z = 1 at first, and after each
//     rejection c += Z and then Z = sum over x of max(p_v - c q_v, 0). (A rejection
//     leaves max(r - Z q, 0) of the rest r before it, Z its sum; and max(max(p - c q,
//     0) - Z q, 0) = max(p - (c + Z) q, 0), so one number says what all of them took.)
//     After all are rejected, the rest is max(p_v - c q_v, 0).
//   - T <= 0 (or NaN): accepted if x is v's argmax.
// The first accepted child is the next v. Where none is, the path ends and its
// last token is the argmax of ln(rest) + Gumbel noise, which nv_sample adds from
// seeds[s] and the token (for T <= 0 of the logits alone): with nothing rejected
// at v it is nv_sample's token of that row. Where the rest is nothing, it is v's
// argmax. Drafted tokens outside [0, vocab) are passed over, as are nodes whose
// parent does not come before them. NaN logits have probability 0, a logit / T
// beyond fp32 counts as infinite, and infinite ones share the probability; ties go
// to the lower index; an argmax of nothing is 0.
//
// For T > 0 the emitted tokens are distributed as the target's own samples are.
// What decides is held in fp64 sums of fp32 exponentials (added by eights first),
// and in fp64 from there on: a comparison or an argmax goes the other way than exact
// arithmetic has it only where both sides agree to about 1e-6 of the p and c q that
// they are made of, over any vocabulary. The largest exponential of a row is the same
// number wherever it is taken, so that where one token has nearly all of p, what is
// left of 1 is that exact as well.
//
// Launches: 1. verify_stats: for each row that has children, the sum of the
// exponentials (T > 0; both models') or the argmax, by shares of the rows.
// 2. verify_walk: a block a sequence folds them and walks the tree; with draft
// logits several blocks a sequence, in two launches, first sum the rests that the
// second and third child of a node need. 3. verify_sample: partitions of the last
// rows; the last block of a sequence stores the token. Small calls without draft
// logits walk in 3.
#include "../../include/nano_hip.h"
#include "nvr_device.h"
#include "nvr_internal.h"

#include <algorithm>
#include <type_traits>

namespace {

using nvr::kWave;
constexpr int kMaxNodes = 64;
constexpr int kMaxVocab = 1 << 26;
constexpr int kThreads = 256;
constexpr int kLoads = 2;             // 16-byte loads a thread and step of launch 1, the next step's in flight
constexpr int kShare = 4 * kThreads;  // 16-byte chunks a block of launch 1, at least
constexpr int kResident = 5;          // its blocks a CU
constexpr int kSampled = kThreads * 8;               // tokens a block of launch 3
constexpr int kSlices = 16;                          // blocks a sequence of the walk, with draft logits
constexpr float kLog2e = 1.44269504088896340736f, kLn2 = 0.693147180559945309417f;
constexpr float kInf = __builtin_inff();

// Part of a row's logits, or the fold of its parts. T > 0: sum of 2^(x log2(e) / T -
// offset), the offset a whole number, so that it is subtracted without an error of
// its own and sums are brought to another one exactly; -inf where there is nothing.
// An offset that is not below 2^24 (infinite, or the type's lowest value as a mask)
// is the scaled maximum itself and the sum counts the logits that have it: others
// are at least 2^15 below. Else: the maximum and its token.
struct Stats {
    float offset;
    int best;
    double sum;
};

// Where a sequence's walk ended.
struct Path {
    int row;    // its last row, or -1: an invalid sequence
    int node;   // its tokens but the last one
    int tried;  // tokens to leave out (no draft logits)
    double c;   // what rejections took (draft logits)
    double inv_sum, draft_inv_sum;  // of the last row, where c > 0
    float offset, draft_offset;
};
// The same for launch 3, and its search for the last token.
struct Ending {
    Path path;
    int token[kMaxNodes];
    uint64_t best;  // the best (score, token) of the blocks so far, as keys that compare as they do
    int blocks;     // that are done
};

struct VerifyArgs {
    const uint16_t* logits;
    const uint16_t* draft;
    const int* tokens;
    const int* parents;
    const int* row_starts;
    const float* temps;
    const float* uniforms;
    const uint64_t* seeds;
    int* out_tokens;
    int* out_nodes;
    int* out_counts;
    Stats* stats;        // [rows, parts]
    Stats* draft_stats;  // [rows, parts]
    Ending* endings;     // [batch]
    double* rests;       // [2][rows, kSlices]: of the sums of the rests after one and two rejections
    int* arrived;        // [batch]: blocks of the walk that are done
    int rows, batch, max_nodes, vocab;
    int parts, blocks;  // stats a row has room for; blocks a sequence and model of launch 1
};

// 16-byte chunks that may hold tokens of a row: its first may lie up to 7 tokens behind a boundary.
__host__ __device__ inline int64_t row_chunks(int vocab) { return (int64_t(vocab) + 7 + 7) / 8; }
inline int most_parts(int vocab) { return int((row_chunks(vocab) + kShare - 1) / kShare) + 1; }
inline int sample_blocks(int vocab) { return int((row_chunks(vocab) * 8 + kSampled - 1) / kSampled); }

// Rows of sequence s: the first and how many; none for an invalid sequence.
__device__ __forceinline__ int tree_rows(const VerifyArgs& a, int s, int* start) {
    const int first = a.row_starts[s], end = a.row_starts[s + 1];
    *start = first;
    return first < 0 || end > a.rows || end <= first || int64_t(end) - first > a.max_nodes ? 0 : end - first;
}

// Eight logits of one row as its 16-byte chunk holds them: tokens t .. t + 7, NaN
// for those outside [0, vocab): it never wins and weighs nothing. kKeep: for rows
// that are read again, through the caches.
template <bool kKeep = false>
__device__ __forceinline__ void load_chunk(const uint16_t* row, int64_t t, int vocab, float (&f)[8]) {
    if (t >= 0 && t + 8 <= vocab) {
        nvr::unpack8(kKeep ? *reinterpret_cast<const uint4*>(row + t) : nvr::load_stream(row + t), f);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = t + i >= 0 && t + i < vocab ? nvr::bf16_to_f32(row[t + i]) : __builtin_nanf("");
    }
}
// The same as it lies there, for a later unpack8; `whole`: the row's chunks are at multiples of 16 bytes.
__device__ __forceinline__ uint4 packed_chunk(const uint16_t* row, int64_t t, int vocab, bool whole) {
    if (whole && t >= 0 && t + 8 <= vocab) return nvr::load_stream(row + t);
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int64_t lo = t + 2 * i, hi = lo + 1;
        w[i] = (lo >= 0 && lo < vocab ? row[lo] : 0x7fc0u) | (hi >= 0 && hi < vocab ? row[hi] : 0x7fc0u) << 16;
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ int lead_of(const uint16_t* row) { return int(reinterpret_cast<uintptr_t>(row) >> 1 & 7); }

// log2(e) / T, finite, so that a logit of 0 stays 0.
__device__ __forceinline__ float scale_of(float temperature) { return fminf(kLog2e / temperature, 0x1.fffffep127f); }
__device__ __forceinline__ bool vast(float offset) { return !(fabsf(offset) < 0x1p24f); }
__device__ __forceinline__ double inverse(double sum) { return sum > 0.0 ? 1.0 / sum : 0.0; }
// A sum at one offset, at another that is no smaller.
__device__ __forceinline__ double at_offset(double sum, float offset, float other) {
    if (!(sum > 0.0)) return 0.0;
    return offset == other ? sum : ldexp(sum, int(fmaxf(offset - other, -1000.0f)));
}

struct Best {
    float score;
    int index;
};
__device__ __forceinline__ void consider(Best& b, float s, int i) {
    if (nvr::better(s, i, b.score, b.index)) { b.score = s; b.index = i; }
}
__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
    for (int mask = 1; mask < kWave; mask <<= 1) v = fmaxf(v, nvr::xor_lane(v, mask));
    return v;
}
// The wave's best: its top score, and of the lanes that have it the lowest index.
__device__ __forceinline__ Best wave_best(Best b) {
    const float top = wave_max(b.score);
    int index = b.score == top ? b.index : nvr::kNoIndex;
    const uint64_t holds = __ballot(index != nvr::kNoIndex);
    if ((holds & (holds - 1)) == 0) return Best{top, holds != 0 ? __builtin_amdgcn_readlane(index, __builtin_ctzll(holds)) : nvr::kNoIndex};
#pragma unroll
    for (int mask = 1; mask < kWave; mask <<= 1) index = min(index, nvr::xor_lane(index, mask));
    return Best{top, index};
}
__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
    for (int mask = 1; mask < kWave; mask <<= 1) v += __shfl_xor(v, mask);
    return v;
}

// Nodes that have children: bit v for node v, the same in every lane. Lane i holds node i's parent, or -1.
__device__ __forceinline__ uint64_t inner_nodes(int parent) {
    const uint64_t mine = parent >= 0 ? uint64_t(1) << parent : 0;
    uint32_t lo = uint32_t(mine), hi = uint32_t(mine >> 32);
#pragma unroll
    for (int mask = 1; mask < kWave; mask <<= 1) {
        lo |= nvr::xor_lane_bits(lo, mask);
        hi |= nvr::xor_lane_bits(hi, mask);
    }
    return uint64_t(uint32_t(__builtin_amdgcn_readfirstlane(int(hi)))) << 32 | uint32_t(__builtin_amdgcn_readfirstlane(int(lo)));
}

// How the rows of a sequence's nodes with children are shared by launch 1's
// blocks: one after the other they are rows * chunks 16-byte chunks, cut evenly,
// so that every block has as much to do whatever the tree. A row's parts are the
// blocks that have some of it.
struct Shares {
    uint32_t chunks, per;  // of a row; of a block (64 rows of 2^26 tokens: 2^29)
    __device__ __forceinline__ Shares(int vocab, int rows, int blocks) {
        chunks = uint32_t(row_chunks(vocab));
        per = max((chunks * rows + blocks - 1) / blocks, uint32_t(kShare));
    }
    __device__ __forceinline__ int first_block(int i) const { return int(i * chunks / per); }
    __device__ __forceinline__ int last_block(int i) const { return int(((i + 1) * chunks - 1) / per); }
};

// A thread's chunks begin, begin + kThreads, ... < end of a row and one more value,
// with their NaN, infinite and huge values looked at one by one.
__device__ __forceinline__ void careful_sum(const uint16_t* x, int lead, int begin, int end, float edge, int vocab,
                                            float scale, float* offset, double* sum) {
    float top = fmaxf(edge * scale, -kInf);
    for (int k = begin; k < end; k += kThreads) {
        float f[8];
        load_chunk(x, 8 * int64_t(k) - lead, vocab, f);
#pragma unroll
        for (int j = 0; j < 8; ++j) top = fmaxf(top, f[j] * scale);
    }
    const float at = __builtin_rintf(top);
    auto weight = [&](float v) {
        if (vast(top)) return v * scale == top ? 1.0f : 0.0f;
        const float w = __builtin_amdgcn_exp2f(__builtin_fmaf(v, scale, -at));
        return w == w ? w : 0.0f;  // nor has an infinite logit a weight where T is infinite
    };
    double total = top > -kInf ? double(weight(edge)) : 0.0;
    for (int k = begin; k < end && top > -kInf; k += kThreads) {
        float f[8], eight = 0.0f;
        load_chunk(x, 8 * int64_t(k) - lead, vocab, f);
#pragma unroll
        for (int j = 0; j < 8; ++j) eight += weight(f[j]);
        total += double(eight);
    }
    *offset = at;
    *sum = total;
}

// A block a (sequence, share, model). T > 0: one pass with an offset that follows
// each thread's maximum; a sum that comes near the ends of fp32's range, or a NaN, is
// taken again with care. Bound by the read of the logits (48 chains of 6 with draft
// logits, 117 MB, in 22 us, 5.2 TB/s) and, at five instructions and an exponential a
// token, nearly as much by its issue (24 trees of 25, 55 MB, in 15 us, 3.6 TB/s). Five
// resident blocks a CU, with the next two loads in flight: whole calls, vocabulary
// 151936, 24 trees of 25 31.8 us, 128 chains of 4 61.0; six blocks 31.9, 62.6, four 31.6,
// 61.7, eight 32.7, 64.3.
__global__ __launch_bounds__(kThreads, kResident) void verify_stats(VerifyArgs a) {
    constexpr int kWaves = kThreads / kWave;
    __shared__ float tops[kWaves];
    __shared__ double sums[kWaves];
    __shared__ int first;
    const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
    const int block = int(blockIdx.x % unsigned(a.blocks)), item = int(blockIdx.x / unsigned(a.blocks));
    const int side = item >= a.batch ? 1 : 0, s = item - side * a.batch;
    if (block == 0 && side == 0 && threadIdx.x == 0) {
        a.arrived[s] = 0;
        a.endings[s].best = 0;
        a.endings[s].blocks = 0;
    }
    int start;
    const int n = tree_rows(a, s, &start);
    if (n < 2) return;
    const float temperature = a.temps[s];
    const bool sampled = temperature > 0.0f;
    if (side == 1 && !sampled) return;
    int parent = lane > 0 && lane < n ? a.parents[start + lane] : -1;
    if (parent >= lane) parent = -1;
    uint64_t inner = inner_nodes(parent);
    const uint32_t count = uint32_t(__popcll(inner));
    const Shares shares(a.vocab, count, a.blocks);
    uint32_t at = block * shares.per;
    const uint32_t stop = min(at + shares.per, count * shares.chunks);
    if (at >= stop) return;
    const float scale = scale_of(temperature);
    int i = int(at / shares.chunks);
    for (int skip = 0; skip < i; ++skip) inner &= inner - 1;
    for (; at < stop; ++i, inner &= inner - 1) {
        const int row = start + __builtin_ctzll(inner);
        const uint16_t* x = (side ? a.draft : a.logits) + int64_t(row) * a.vocab;
        const int lead = lead_of(x);
        const uint32_t base = i * shares.chunks;
        const int begin = int(at - base), end = int(min(stop - base, shares.chunks));
        at = base + end;
        // Whole chunks, and at either end of a row the tokens of one that is not: one each of the first 16 threads'. A
        // row in one chunk has one such end.
        const int whole = (a.vocab + lead) / 8, lo = max(begin, lead != 0 ? 1 : 0), hi = min(end, whole);
        const bool head = begin == 0 && lead != 0, tail = begin <= whole && end > whole && (whole > 0 || lead == 0);
        const int lone = threadIdx.x < 8 ? (head ? int(threadIdx.x) - lead : -1)
                                         : tail && threadIdx.x < 16 ? 8 * whole - lead + int(threadIdx.x) - 8 : -1;
        float edge = -kInf;
        if (lone >= 0 && lone < a.vocab) edge = nvr::bf16_to_f32(x[lone]);
        auto load = [&](int k, uint4 (&packed)[kLoads]) {
#pragma unroll
            for (int u = 0; u < kLoads; ++u) packed[u] = nvr::load_stream(x + 8 * int64_t(min(k + u * kThreads, hi - 1)) - lead);
        };
        auto take = [&](int k, uint4 (&packed)[kLoads], uint4 (&now)[kLoads]) {  // step k, the next one's loads under way
#pragma unroll
            for (int u = 0; u < kLoads; ++u) now[u] = packed[u];
            if (k + kLoads * kThreads < hi) load(k + kLoads * kThreads, packed);
        };
        auto loaded = [&](int c, const uint4& packed, float (&f)[8]) {
            const uint32_t none = 0xff80ff80u;  // -inf: weighs nothing
            const bool in = c < hi;
            nvr::unpack8(make_uint4(in ? packed.x : none, in ? packed.y : none, in ? packed.z : none, in ? packed.w : none), f);
        };
        auto highest = [&](int k, const uint4 (&packed)[kLoads]) {
            float high = -kInf;
#pragma unroll
            for (int u = 0; u < kLoads; ++u) {
                float f[8];
                loaded(k + u * kThreads, packed[u], f);
#pragma unroll
                for (int j = 0; j < 8; ++j) high = fmaxf(high, f[j]);  // passes over NaN
            }
            return high;
        };
        const int begin_k = lo + int(threadIdx.x);
        uint4 packed[kLoads];
        if (begin_k < hi) load(begin_k, packed);
        float offset = -kInf;
        double total = 0.0;
        int where = -2;  // the chunk whose load has the maximum; -1: the edge
        if (sampled) {
            float high = edge;
            if (begin_k < hi) high = fmaxf(high, highest(begin_k, packed));
            high *= scale;
            offset = vast(high) ? 0.0f : __builtin_rintf(high);
            total = double(__builtin_amdgcn_exp2f(__builtin_fmaf(edge, scale, -offset)));
            for (int k = begin_k; k < hi; k += kLoads * kThreads) {
                uint4 now[kLoads];
                take(k, packed, now);
                const float grown = highest(k, now) * scale;
                if (grown > offset + 0.5f && !vast(grown)) {
                    const float to = __builtin_rintf(grown);
                    total = at_offset(total, offset, to);
                    offset = to;
                }
#pragma unroll
                for (int u = 0; u < kLoads; ++u) {
                    float f[8], eight = 0.0f;
                    loaded(k + u * kThreads, now[u], f);
#pragma unroll
                    for (int j = 0; j < 8; ++j) eight += __builtin_amdgcn_exp2f(__builtin_fmaf(f[j], scale, -offset));
                    total += double(eight);
                }
            }
            if (!(total >= 0x1p-20 && total < 0x1p100))
                careful_sum(x, lead, begin_k, hi, edge, a.vocab, scale, &offset, &total);
            if (!(total > 0.0)) offset = -kInf;
        } else {
            if (edge == edge && lone >= 0 && lone < a.vocab) { offset = edge; where = -1; }
            for (int k = begin_k; k < hi; k += kLoads * kThreads) {
                uint4 now[kLoads];
                take(k, packed, now);
                const float high = highest(k, now);
                if (high > offset || (where < 0 && high == offset)) {
                    offset = high;
                    where = k;
                }
            }
        }
        const float high = wave_max(offset);
        if (lane == 0) tops[wave] = high;
        if (threadIdx.x == 0) first = nvr::kNoIndex;
        __syncthreads();
        float all = tops[0];
#pragma unroll
        for (int w = 1; w < kWaves; ++w) all = fmaxf(all, tops[w]);
        if (where > -2 && offset == all) {
            // The lowest of this thread's tokens with that logit.
            int lowest = lone >= 0 && lone < a.vocab && edge == all ? lone : nvr::kNoIndex;
            // Where that is -inf, loads of NaN alone had it too: all of the thread's are looked at.
            const int from = all == -kInf ? begin_k : where, until = all == -kInf ? hi : min(hi, from + kLoads * kThreads);
#pragma unroll 1
            for (int c = from; c < until && where >= 0; c += kThreads) {
                float f[8];
                load_chunk(x, 8 * int64_t(c) - lead, a.vocab, f);
#pragma unroll
                for (int j = 7; j >= 0; --j)
                    if (f[j] == all) lowest = min(lowest, int(8 * int64_t(c) - lead) + j);
            }
            atomicMin(&first, lowest);
        }
        const double sum = wave_sum(at_offset(total, offset, all));
        if (lane == 0) sums[wave] = sum;
        __syncthreads();
        if (threadIdx.x == 0) {
            double parts = 0.0;
#pragma unroll
            for (int w = 0; w < kWaves; ++w) parts += sums[w];
            (side ? a.draft_stats : a.stats)[int64_t(row) * a.parts + block - shares.first_block(i)] = Stats{all, first, parts};
        }
    }
}

// Parts folded over a wave, a part a lane (of more than 64 some).
__device__ __forceinline__ Stats fold(const Stats& mine, double sum) {
    const Best b = wave_best(Best{mine.offset, mine.best});
    const double scaled = sum > 0.0 ? ldexp(sum, mine.offset == b.score ? 0 : int(fmaxf(mine.offset - b.score, -1000.0f))) : 0.0;
    return Stats{b.score, b.index, wave_sum(scaled)};
}
__device__ __forceinline__ void add_part(Stats& mine, double& sum, const Stats& t) {
    Best b{mine.offset, mine.best};
    consider(b, t.offset, t.best);
    sum = ldexp(sum, sum > 0.0 && mine.offset != b.score ? int(fmaxf(mine.offset - b.score, -1000.0f)) : 0) +
          at_offset(t.sum, t.offset, b.score);
    mine.offset = b.score;
    mine.best = b.index;
}

// The target's and the draft model's probabilities of a row's tokens.
struct Rows {
    const uint16_t* target;
    const uint16_t* draft;
    float offset, draft_offset;
    double inv_sum, draft_inv_sum;
};

// p - c q of one token, in fp64, since both may be near 1 and agree; NaN where p is.
struct RestTerm {
    const Rows& r;
    float scale;
    double cq;
    bool any_vast;
    __device__ __forceinline__ RestTerm(const Rows& rows, double c, float s)
        : r(rows), scale(s), cq(c * rows.draft_inv_sum), any_vast(vast(rows.offset) || vast(rows.draft_offset)) {}
    __device__ __forceinline__ float weight(float x, float offset) const {
        if (any_vast && vast(offset)) return x * scale == offset ? 1.0f : 0.0f;
        return __builtin_amdgcn_exp2f(__builtin_fmaf(x, scale, -offset));
    }
    __device__ __forceinline__ double operator()(float x, float y) const {
        const float wy = fmaxf(weight(y, r.draft_offset), 0.0f);  // a NaN is no token of q
        return __builtin_fma(double(weight(x, r.offset)), r.inv_sum, -(double(wy) * cq));
    }
};

// sum of max(p - c q, 0) over 16-byte chunks [first, end) of a row, this thread's share.
template <int kBatch>  // chunks in flight a thread
__device__ __forceinline__ double rest_sum(const Rows& r, int vocab, double c, float scale, int64_t first, int64_t end,
                                           int threads) {
    const int lead = lead_of(r.target);
    const bool alike = lead == lead_of(r.draft);
    const RestTerm term(r, c, scale);
    double sum = 0.0;
    for (int64_t k = first + int(threadIdx.x); k < end; k += kBatch * threads) {
        float x[kBatch][8], y[kBatch][8];
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
            const int64_t t = 8 * min(k + u * threads, end - 1) - lead;
            load_chunk<true>(r.target, t, vocab, x[u]);
            if (alike) {
                load_chunk<true>(r.draft, t, vocab, y[u]);
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    y[u][i] = t + i >= 0 && t + i < vocab ? nvr::bf16_to_f32(r.draft[t + i]) : __builtin_nanf("");
            }
        }
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
            double eight = 0.0;
#pragma unroll
            for (int i = 0; i < 8; ++i) eight += fmax(term(x[u][i], y[u][i]), 0.0);
            sum += k + u * threads < end ? eight : 0.0;
        }
    }
    return sum;
}

// Blocks of one launch hand values over by atomics alone, so that no cache has to
// be written back or dropped for it (a release and an acquire a block do that:
// 3600 blocks of launch 3 took 102 us with them, 22 without). An atomic that
// returns a value has been performed when the value is there; the next one is
// issued after that.
__device__ __forceinline__ void performed() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }
__device__ __forceinline__ void publish(double* to, double v) {
    const uint64_t old = __hip_atomic_exchange(reinterpret_cast<uint64_t*>(to), __builtin_bit_cast(uint64_t, v), __ATOMIC_RELAXED,
                                               __HIP_MEMORY_SCOPE_AGENT);
    asm volatile("" ::"v"(old));  // the returning form
    performed();
}
__device__ __forceinline__ int arrive(int* count) {
    performed();
    return __hip_atomic_fetch_add(count, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

constexpr int kWalkThreads = 512;
constexpr int kWalkWaves = kWalkThreads / kWave;

// A lane's value, for every lane.
__device__ __forceinline__ double lane_value(double v, int i) {
    const uint64_t bits = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = uint32_t(__builtin_amdgcn_readlane(int(uint32_t(bits)), i)), hi = uint32_t(__builtin_amdgcn_readlane(int(uint32_t(bits >> 32)), i));
    return __builtin_bit_cast(double, uint64_t(hi) << 32 | lo);
}

// A child's trial against the rest max(p - c q, 0), whose sum is z.
__device__ __forceinline__ bool accepted(double p, double q, double u, double c, double z) {
    const double rest = fmax(p - c * q, 0.0);
    return rest > 0.0 && u * z * q < rest;
}

// A sequence's tree: lane i of every wave holds node i.
struct Tree {
    int start, n;      // n 0: an invalid sequence
    int parent, token;
    double u;
    bool known;        // a drafted node that can be followed
    uint64_t inner;    // nodes with children
};
__device__ __forceinline__ Tree tree_of(const VerifyArgs& a, int s, int lane) {
    Tree t;
    t.n = tree_rows(a, s, &t.start);
    const bool mine = lane > 0 && lane < t.n;
    t.parent = mine ? a.parents[t.start + lane] : -1;
    t.token = mine ? a.tokens[t.start + lane] : -1;
    t.u = mine ? double(a.uniforms[t.start + lane]) : 0.0;
    if (t.parent < 0 || t.parent >= lane) t.parent = -1;
    t.known = t.parent >= 0 && t.token >= 0 && t.token < a.vocab;
    t.inner = inner_nodes(t.parent);
    return t;
}
// Whether no rests have to be summed: picked or greedy, or no node has a second child to try.
__device__ __forceinline__ bool no_rests(const VerifyArgs& a, const Tree& t, bool sampled) {
    return a.draft == nullptr || !sampled || __popcll(__ballot(t.known)) == __popcll(inner_nodes(t.known ? t.parent : -1));
}

// The stats of the nodes with children, a wave a node and model, kBatch of them in flight together.
template <int kWaves>
__device__ __forceinline__ void fold_nodes(const VerifyArgs& a, const Tree& t, bool drafted, int wave, int lane, Stats* target,
                                           Stats* draft) {
    constexpr int kBatch = 4;
    const int count = __popcll(t.inner), items = count * (drafted ? 2 : 1);
    const Shares shares(a.vocab, max(count, 1), a.blocks);
    uint64_t left = t.inner;
    int at = 0;  // nodes taken off left
    for (int first = wave; first < items; first += kBatch * kWaves) {
        int node[kBatch], parts[kBatch];
        const Stats* from[kBatch];
        Stats part[kBatch];
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
            const int item = min(first + u * kWaves, items - 1), side = item >= count ? 1 : 0, i = item - side * count;
            if (i < at) { left = t.inner; at = 0; }
            for (; at < i; ++at) left &= left - 1;
            node[u] = __builtin_ctzll(left);
            parts[u] = shares.last_block(i) - shares.first_block(i) + 1;
            from[u] = (side ? a.draft_stats : a.stats) + int64_t(t.start + node[u]) * a.parts;
            part[u] = from[u][min(lane, parts[u] - 1)];
        }
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
            if (first + u * kWaves >= items) continue;
            Stats mine{-kInf, nvr::kNoIndex, 0.0};
            double sum = 0.0;
            if (lane < parts[u]) add_part(mine, sum, part[u]);
            for (int i = lane + kWave; i < parts[u]; i += kWave) add_part(mine, sum, from[u][i]);
            const Stats all = fold(mine, sum);
            if (lane == 0) (first + u * kWaves >= count ? draft : target)[node[u]] = all;
        }
    }
}
__device__ __forceinline__ Rows rows_of(const VerifyArgs& a, int row, const Stats& t, const Stats& d) {
    const int64_t at = int64_t(row) * a.vocab;
    return Rows{a.logits + at, a.draft + at, t.sum > 0.0 ? t.offset : 0.0f, d.sum > 0.0 ? d.offset : 0.0f, inverse(t.sum),
                inverse(d.sum)};
}
// The probability of a logit of a row: 2^y, y = k + f, |f| <= 1/2, in fp64 but for 2^f.
__device__ __forceinline__ double chance(float x, float scale, const Stats& r) {
    if (!(r.sum > 0.0) || x != x) return 0.0;
    if (vast(r.offset)) return x * scale == r.offset ? 1.0 / r.sum : 0.0;
    const double y = double(x) * double(scale) - double(r.offset), k = rint(y);
    return y > -1000.0 ? ldexp(double(__builtin_amdgcn_exp2f(float(y - k))), int(k)) / r.sum : 0.0;
}

// A path's nodes and tokens, and their number; all but its last token, which launch 3 stores.
__device__ __forceinline__ void write_path(const VerifyArgs& a, int s, int start, const int* path, int length) {
    const int step = int(threadIdx.x);
    if (step < a.max_nodes) {
        a.out_nodes[int64_t(s) * a.max_nodes + step] = step < length ? path[step] : -1;
        if (step != length - 1) a.out_tokens[int64_t(s) * a.max_nodes + step] = step < length ? a.tokens[start + path[step + 1]] : -1;
    }
    if (step == 0) a.out_counts[s] = length;
}
__device__ __forceinline__ void write_nothing(const VerifyArgs& a, int s) {
    if (int(threadIdx.x) < a.max_nodes)
        a.out_tokens[int64_t(s) * a.max_nodes + threadIdx.x] = a.out_nodes[int64_t(s) * a.max_nodes + threadIdx.x] = -1;
    if (threadIdx.x == 0) a.out_counts[s] = 0;
}

// The walk of a block of kWaves where no rests have to be summed.
template <int kWaves>
struct SimpleWalk {
    Stats target[kMaxNodes], draft[kMaxNodes];
    int path[kMaxNodes], tried[kMaxNodes];
    __device__ __forceinline__ Path operator()(const VerifyArgs& a, const Tree& t, float temperature, int wave, int lane) {
        const bool sampled = temperature > 0.0f, drafted = sampled && a.draft != nullptr;
        const float scale = scale_of(temperature);
        const int parent = t.parent;
        float xt = 0.0f, xd = 0.0f;
        if (sampled && t.known) {
            const int64_t at = int64_t(t.start + parent) * a.vocab + t.token;
            xt = nvr::bf16_to_f32(a.logits[at]);
            if (drafted) xd = nvr::bf16_to_f32(a.draft[at]);
        }
        fold_nodes<kWaves>(a, t, drafted, wave, lane, target, draft);
        __syncthreads();
        const double p = sampled && t.known ? chance(xt, scale, target[parent]) : 0.0;
        const double q = drafted && t.known ? chance(xd, scale, draft[parent]) : 0.0;
        // Every wave walks alike.
        Path end{};
        int v = 0;
        uint64_t rejected = 0;
        for (;; ++end.node) {
            if (threadIdx.x == 0) path[end.node] = v;
            uint64_t children = __ballot(t.known && parent == v);
            const int best = children != 0 && target[v].best != nvr::kNoIndex ? target[v].best : 0;
            int next = -1;
            rejected = 0;
            for (double z = 1.0; children != 0; children &= children - 1) {
                const int i = __builtin_ctzll(children), x = __builtin_amdgcn_readlane(t.token, i);
                if (!sampled) {
                    if (x == best) { next = i; break; }
                    continue;
                }
                const double px = lane_value(p, i), ux = lane_value(t.u, i);
                if (drafted) {  // the only child
                    if (accepted(px, lane_value(q, i), ux, 0.0, 1.0)) next = i;
                    else end.c = 1.0;
                    break;
                }
                if (__ballot((rejected >> lane & 1) != 0 && t.token == x) != 0) continue;
                if (px > 0.0 && ux * z < px) { next = i; break; }
                rejected |= uint64_t(1) << i;
                z -= px;
            }
            if (next < 0) break;
            v = next;
        }
        if (wave == 0 && (rejected >> lane & 1) != 0) tried[__popcll(rejected & ((uint64_t(1) << lane) - 1))] = t.token;
        __syncthreads();  // path, tried
        end.row = t.start + v;
        end.tried = __popcll(rejected);
        if (end.c > 0.0) {
            const Rows r = rows_of(a, end.row, target[v], draft[v]);
            end.offset = r.offset;
            end.inv_sum = r.inv_sum;
            end.draft_offset = r.draft_offset;
            end.draft_inv_sum = r.draft_inv_sum;
        }
        return end;
    }
};

// The walk. One block a sequence where no rests are summed. Where drafted siblings
// were sampled, kSlices blocks: a node's second child needs the sum of the rest
// after one rejection, its third that after two, a pass over the vocabulary, which
// one block does at the rate of one CU (50257 tokens 7 us). So a first launch
// (kFirst) sums, slice by slice, the first rests that the walk may come to need, and
// the second launch the second rests; there the last block of a sequence to finish
// walks. Later rests are summed during the walk. Bound by the chain of memory round
// trips (nodes, their logits, the stats' parts, the rests' parts, the hand-over): 6.4
// us without draft logits, 4.4 + 7.0 with them where every node has one child (the first
// launch finds nothing to sum there), 9 + 12 for 8 trees of 13 with up to three over
// 50257 tokens. Fourth children cost a pass by one block each, which 16 slices whatever the
// batch leave far from a bound: 8 trees of 40 with up to four over 151936 tokens take 93 us.
template <bool kFirst>
__global__ __launch_bounds__(kWalkThreads) void verify_walk(VerifyArgs a) {
    __shared__ Stats target[kMaxNodes], draft[kMaxNodes];
    __shared__ double parts[kMaxNodes][kWalkWaves], rests[2][kMaxNodes];
    __shared__ int path[kMaxNodes];
    __shared__ int last;
    const int lane = threadIdx.x & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int s = int(blockIdx.x), slice = int(blockIdx.y), slices = int(gridDim.y);
    const Tree t = tree_of(a, s, lane);
    Ending* ending = a.endings + s;
    const float temperature = a.temps[s];
    if (t.n == 0 || no_rests(a, t, temperature > 0.0f)) {
        if constexpr (!kFirst) {
            if (slice != 0) return;
            if (t.n == 0) {
                write_nothing(a, s);
                if (threadIdx.x == 0) ending->path.row = -1;
                return;
            }
            __shared__ SimpleWalk<kWalkWaves> walk;
            const Path end = walk(a, t, temperature, wave, lane);
            write_path(a, s, t.start, walk.path, end.node + 1);
            if (int(threadIdx.x) < end.tried) ending->token[threadIdx.x] = walk.tried[threadIdx.x];
            if (threadIdx.x == 0) ending->path = end;
        }
        return;
    }
    const float scale = scale_of(temperature);
    const int start = t.start, n = t.n, parent = t.parent;
    const bool known = t.known;
    const double u = t.u;
    // The logits of each node's token, under its parent.
    float xt = 0.0f, xd = 0.0f;
    if (known) {
        const int64_t at = int64_t(start + parent) * a.vocab + t.token;
        xt = nvr::bf16_to_f32(a.logits[at]);
        xd = nvr::bf16_to_f32(a.draft[at]);
    }
    fold_nodes<kWalkWaves>(a, t, true, wave, lane, target, draft);
    __syncthreads();
    // Each node's probabilities under its parent's rows.
    const double p = known ? chance(xt, scale, target[parent]) : 0.0, q = known ? chance(xd, scale, draft[parent]) : 0.0;
    auto rows_at = [&](int v) { return rows_of(a, start + v, target[v], draft[v]); };
    const int64_t chunks = row_chunks(a.vocab);
    // This block's share of the sums of the nodes' rests, for all slices to see.
    auto sum_rests = [&](uint64_t which, double* to, auto taken) {
        const int64_t share = (chunks + slices - 1) / slices, begin = slice * share;
        for (uint64_t left = which; left != 0; left &= left - 1) {
            const int v = __builtin_ctzll(left);
            const double sum = wave_sum(rest_sum<1>(rows_at(v), a.vocab, taken(v), scale, begin, min(chunks, begin + share), kWalkThreads));
            if (lane == 0) parts[v][wave] = sum;
        }
        __syncthreads();
        if (threadIdx.x < kMaxNodes && (which >> threadIdx.x & 1) != 0) {
            double sum = 0.0;
            for (int w = 0; w < kWalkWaves; ++w) sum += parts[threadIdx.x][w];
            publish(to + int64_t(start + threadIdx.x) * kSlices + slice, sum);
        }
    };
    auto read_rests = [&](uint64_t which, const double* from, double* to) {
        for (int first = 0; first < n; first += kWalkThreads / kSlices) {  // a thread a node and slice
            const int v = first + int(threadIdx.x) / kSlices, w = int(threadIdx.x) % kSlices;
            const bool there = v < kMaxNodes && (which >> (v & 63) & 1) != 0;
            double sum = there && w < slices ? __hip_atomic_load(from + int64_t(start + v) * kSlices + w, __ATOMIC_RELAXED,
                                                                 __HIP_MEMORY_SCOPE_AGENT) : 0.0;
#pragma unroll
            for (int mask = 1; mask < kSlices; mask <<= 1) sum += __shfl_xor(sum, mask);
            if (there && w == 0) to[v] = sum;
        }
        __syncthreads();
    };
    // Nodes that the walk may come to (open) and have it reject a first child and try a second: those need the first
    // rest's sum; and those where it rejects a second and tries a third, the second's.
    uint64_t once = 0;
    auto look = [&](bool second) {
        uint64_t open = 1, found = 0;
        for (int v = 0; v < n - 1; ++v) {
            uint64_t children = __ballot(known && parent == v);
            if (children == 0 || (open >> v & 1) == 0) continue;
            int i = __builtin_ctzll(children);
            bool taken = accepted(lane_value(p, i), lane_value(q, i), lane_value(u, i), 0.0, 1.0);
            if (!taken && second && (children & (children - 1)) != 0) {
                children &= children - 1;
                i = __builtin_ctzll(children);
                taken = accepted(lane_value(p, i), lane_value(q, i), lane_value(u, i), 1.0, rests[0][v]);
            }
            children &= children - 1;
            open |= taken ? uint64_t(1) << i : children;
            // (children: none left where there was no second)
            if (!taken && children != 0 && (second ? (once >> v & 1) != 0 : true)) found |= uint64_t(1) << v;
        }
        return found;
    };
    once = look(false);
    if constexpr (kFirst) {
        if (once != 0) sum_rests(once, a.rests, [](int) { return 1.0; });
        return;
    }
    read_rests(once, a.rests, rests[0]);
    const uint64_t twice = look(true);
    if (twice == 0 && slice != 0) return;
    if (twice != 0) {
        sum_rests(twice, a.rests + int64_t(a.rows) * kSlices, [&](int v) { return 1.0 + rests[0][v]; });
        __syncthreads();
        if (threadIdx.x == 0) last = arrive(a.arrived + s) == slices - 1;
        __syncthreads();
        if (!last) return;
        read_rests(twice, a.rests + int64_t(a.rows) * kSlices, rests[1]);
    }
    // Every wave walks alike.
    int v = 0, length = 0;
    double c = 0.0;
    while (true) {
        if (threadIdx.x == 0) path[length] = v;
        ++length;
        uint64_t children = __ballot(known && parent == v);
        double z = 1.0;
        c = 0.0;
        int next = -1;
        for (int tried = 0; children != 0; ++tried) {
            const int i = __builtin_ctzll(children);
            children &= children - 1;
            if (accepted(lane_value(p, i), lane_value(q, i), lane_value(u, i), c, z)) { next = i; break; }
            c += z;
            if (children == 0) break;
            if (tried < 2) {
                z = rests[tried][v];
            } else {
                const double sum = wave_sum(rest_sum<4>(rows_at(v), a.vocab, c, scale, 0, chunks, kWalkThreads));
                if (lane == 0) parts[0][wave] = sum;
                __syncthreads();
                z = 0.0;
                for (int w = 0; w < kWalkWaves; ++w) z += parts[0][w];
                __syncthreads();
            }
        }
        if (next < 0) break;
        v = next;
    }
    __syncthreads();  // path
    write_path(a, s, start, path, length);
    if (threadIdx.x == 0) {
        const Rows r = rows_at(v);
        ending->path = Path{start + v, length - 1, 0, c, r.inv_sum, r.draft_inv_sum, r.offset, r.draft_offset};
    }
}

// (score, token) as a number that is larger for what nvr::better prefers; 0: nothing.
__device__ __forceinline__ uint64_t key_of(const Best& b) {
    if (b.index == nvr::kNoIndex) return 0;
    const uint32_t bits = __float_as_uint(b.score + 0.0f);  // -0 as +0: they are equal scores
    return uint64_t(bits & 0x80000000u ? ~bits : bits | 0x80000000u) << 32 | uint32_t(~b.index);
}

// A block a (sequence, partition of its last row). A Gumbel score is an integer
// hash and two logarithms; the noise is at most -ln(1 - u), so one hardware
// logarithm bounds it, and only a lane's best bound and the bounds that reach
// the wave's best score are scored in full. Bound by the hash: about 60 instructions
// a token, six of them multiplications at a quarter of the rate, also for tokens whose
// rest is nothing; 48 rows of 151936 tokens take 22 us, 24 rows 11. Blocks of two or four
// times the tokens gained 1 us in 49 there and lost as much at 24 rows (with fp32 rests).
// kWalks: every block walks its tree by itself, which saves launch 2.
template <bool kWalks>
__global__ __launch_bounds__(kThreads) void verify_sample(VerifyArgs a) {
    constexpr int kWaves = kThreads / kWave;
    __shared__ Best tops[kWaves];
    __shared__ std::conditional_t<kWalks, SimpleWalk<kWaves>, int> walk;
    __shared__ int tried[kMaxNodes];
    const int lane = threadIdx.x & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int s = int(blockIdx.x), part = int(blockIdx.y), parts = int(gridDim.y);
    Ending* e = a.endings + s;
    const float temperature = a.temps[s], scale = scale_of(temperature);
    const uint64_t seed = a.seeds[s];
    Path path;
    if constexpr (kWalks) {
        const Tree tree = tree_of(a, s, lane);
        if (tree.n == 0) {
            if (part == 0) write_nothing(a, s);
            return;
        }
        path = walk(a, tree, temperature, wave, lane);
        if (part == 0) write_path(a, s, tree.start, walk.path, path.node + 1);
    } else {
        path = e->path;
    }
    const int row = path.row, node = path.node, count = path.tried;
    if (row < 0) return;
    const double c = path.c;
    const uint16_t* x = a.logits + int64_t(row) * a.vocab;
    const int64_t t = int64_t(part) * kSampled + 8 * int(threadIdx.x) - lead_of(x);
    const Rows rest{x, c > 0.0 ? a.draft + int64_t(row) * a.vocab : x, path.offset, path.draft_offset, path.inv_sum, path.draft_inv_sum};
    uint4 packed_q = {};
    if (c > 0.0) packed_q = packed_chunk(rest.draft, t, a.vocab, lead_of(rest.draft) == lead_of(x));
    float f[8];
    load_chunk(x, t, a.vocab, f);
    if constexpr (!kWalks) {
        if (int(threadIdx.x) < count) tried[threadIdx.x] = e->token[threadIdx.x];
        __syncthreads();
    }
    const int* out = tried;
    if constexpr (kWalks) out = walk.tried;
    Best b{-kInf, nvr::kNoIndex};
    if (!(temperature > 0.0f)) {
#pragma unroll
        for (int i = 0; i < 8; ++i) consider(b, f[i], int(t) + i);
    } else {
        if (c > 0.0) {  // ln(p - c q) in place of the logits
            const RestTerm term(rest, c, scale);
            float q[8];
            nvr::unpack8(packed_q, q);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float w = float(term(f[i], q[i]));
                f[i] = w >= 0x1p-126f ? w : __builtin_nanf("");
            }
        }
        for (int k = 0; k < count; ++k) {
            const int64_t at = out[k] - t;
            if (at >= 0 && at < 8) {
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if (at == i) f[i] = __builtin_nanf("");
            }
        }
        auto uniform = [&](int i) { return nvr::hash_uniform(nvr::splitmix64(seed ^ (uint64_t(t + i) * nvr::kTokenMix))); };
        auto score = [&](float v, float u) {
            return (c > 0.0 ? nvr::nvr_logf(v) : v / temperature) - nvr::nvr_logf(-nvr::nvr_logf(u));
        };
        const float inverse_t = 1.0f / temperature;
        float bound[8], us[8], high = -kInf;
        if (c > 0.0) {
#pragma unroll
            for (int i = 0; i < 8; ++i) bound[i] = __builtin_amdgcn_logf(f[i]) * kLn2;
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) bound[i] = f[i] * inverse_t;
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            us[i] = uniform(i);
            // Bounds with 2^-20 of the value and 1e-4 to spare: many times what their few roundings can take.
            const float g = __builtin_fmaf(__builtin_amdgcn_logf(1.0f - us[i]), -kLn2, 1e-4f);
            bound[i] = __builtin_fmaf(bound[i], bound[i] > 0.0f ? 1.0f + 0x1p-20f : 1.0f - 0x1p-20f, g);
        }
        if (!(inverse_t < kInf)) {
#pragma unroll
            for (int i = 0; i < 8; ++i) bound[i] = f[i] == f[i] ? kInf : f[i];
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) high = fmaxf(high, bound[i]);  // passes over NaN
        int own = -1;
#pragma unroll
        for (int i = 7; i >= 0; --i) own = bound[i] == high ? i : own;
        if (own >= 0) {
            float v = f[0], u = us[0];
#pragma unroll
            for (int i = 1; i < 8; ++i)
                if (own == i) { v = f[i]; u = us[i]; }
            consider(b, score(v, u), int(t) + own);
        }
        const float reach = wave_max(b.score);
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i != own && bound[i] >= reach) consider(b, score(f[i], us[i]), int(t) + i);
        if (b.score == -kInf && (count > 0 || c > 0.0)) b.index = nvr::kNoIndex;  // the rest is nothing here
    }
    auto block_best = [&] {  // in thread 0
        b = wave_best(b);
        if (lane == 0) tops[wave] = b;
        __syncthreads();
#pragma unroll
        for (int w = 1; w < kWaves; ++w) consider(b, tops[w].score, tops[w].index);
    };
    __shared__ bool nothing;
    block_best();
    if (threadIdx.x == 0) {
        nothing = false;
        const uint64_t old = __hip_atomic_fetch_max(&e->best, key_of(b), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        asm volatile("" ::"v"(old));  // the returning form
        if (arrive(&e->blocks) == parts - 1) {
            const uint64_t key = __hip_atomic_load(&e->best, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            if (key != 0) a.out_tokens[int64_t(s) * a.max_nodes + node] = int(~uint32_t(key));
            else nothing = true;
        }
    }
    __syncthreads();
    if (!nothing) return;
    // Nothing is left: the row's argmax, or 0 where that is nothing either.
    b = Best{-kInf, nvr::kNoIndex};
    for (int64_t k = threadIdx.x; k < row_chunks(a.vocab); k += kThreads) {
        const int64_t t = 8 * k - lead_of(x);
        load_chunk(x, t, a.vocab, f);
#pragma unroll
        for (int i = 0; i < 8; ++i) consider(b, f[i], int(t) + i);
    }
    block_best();
    if (threadIdx.x == 0) a.out_tokens[int64_t(s) * a.max_nodes + node] = b.index == nvr::kNoIndex ? 0 : b.index;
}

// The workspace's parts, each at a multiple of 16 bytes.
struct Workspace {
    int64_t stats, draft_stats, endings, rests, arrived, bytes;
};
Workspace layout(int rows, int batch, int vocab) {
    const int64_t parts = most_parts(vocab);
    auto up = [](int64_t b) { return (b + 15) & ~int64_t(15); };
    Workspace w;
    w.stats = 0;
    w.draft_stats = w.stats + up(int64_t(sizeof(Stats)) * rows * parts);
    w.endings = w.draft_stats + up(int64_t(sizeof(Stats)) * rows * parts);
    w.rests = w.endings + up(int64_t(sizeof(Ending)) * batch);
    w.arrived = w.rests + up(2 * int64_t(sizeof(double)) * kSlices * rows);
    w.bytes = w.arrived + up(int64_t(sizeof(int)) * batch);
    return w;
}

}  // namespace

extern "C" {

int nv_verify_tree_workspace(int rows, int batch, int vocab, size_t* bytes) {
    if (rows <= 0 || batch <= 0 || vocab <= 0) return nvr::fail(-2, "verify_tree_workspace: dimensions must be positive");
    *bytes = size_t(layout(rows, batch, vocab).bytes);
    return 0;
}

int nv_verify_tree(nv_context* c, const void* logits, const void* draft_logits, const void* tokens,
                   const void* parents, const void* row_starts, const void* temps, const void* uniforms,
                   const void* seeds, void* out_tokens, void* out_nodes, void* out_counts, void* workspace, int rows,
                   int batch, int max_nodes, int vocab) {
    NVR_ACTIVATE(c);
    if (rows <= 0 || batch <= 0 || vocab <= 0) return nvr::fail(-2, "verify_tree: dimensions must be positive");
    if (max_nodes < 1 || max_nodes > kMaxNodes)
        return nvr::fail(-2, "verify_tree: max_nodes %d outside [1, %d]", max_nodes, kMaxNodes);
    if (vocab > kMaxVocab) return nvr::fail(-2, "verify_tree: vocab %d above %d", vocab, kMaxVocab);
    if (workspace == nullptr || !nvr::aligned(workspace, 16))
        return nvr::fail(-2, "verify_tree: needs a workspace at a multiple of 16 bytes");
    // A launch has fewer than 2^32 threads.
    const int sampled = sample_blocks(vocab);
    if (batch > 0x3fffff || int64_t(batch) * sampled > 0xffffff)
        return nvr::fail(-2, "verify_tree: %d sequences over %d tokens exceed one launch", batch, vocab);
    // As many blocks as are resident, so that none has to wait for another's end.
    const int sides = draft_logits ? 2 : 1;
    const int64_t cus = c->cu_count > 0 ? c->cu_count : 256;
    const int blocks = int(std::min<int64_t>(std::max<int64_t>(kResident * cus / (int64_t(batch) * sides), 1),
                                             int64_t(most_parts(vocab)) * std::max(max_nodes - 1, 1)));
    const Workspace w = layout(rows, batch, vocab);
    char* base = static_cast<char*>(workspace);
    const VerifyArgs a{static_cast<const uint16_t*>(logits), static_cast<const uint16_t*>(draft_logits),
                       static_cast<const int*>(tokens), static_cast<const int*>(parents),
                       static_cast<const int*>(row_starts), static_cast<const float*>(temps),
                       static_cast<const float*>(uniforms), static_cast<const uint64_t*>(seeds),
                       static_cast<int*>(out_tokens), static_cast<int*>(out_nodes), static_cast<int*>(out_counts),
                       reinterpret_cast<Stats*>(base + w.stats), reinterpret_cast<Stats*>(base + w.draft_stats),
                       reinterpret_cast<Ending*>(base + w.endings), reinterpret_cast<double*>(base + w.rests),
                       reinterpret_cast<int*>(base + w.arrived), rows, batch, max_nodes, vocab, most_parts(vocab), blocks};
    hipLaunchKernelGGL(verify_stats, dim3(unsigned(int64_t(batch) * blocks * sides)), dim3(kThreads), 0, c->stream, a);
    NVR_HIP(hipGetLastError());
    // Up to a block a CU, launch 3 walks by itself (one chain of 5 14.5 us against 16.8, 4 trees of 60 with more
    // blocks 25.2 against 25.5, 24 of 25 36.2, 31.8).
    const dim3 sample{unsigned(batch), unsigned(sampled)};
    if (!draft_logits && int64_t(batch) * sampled <= cus) {
        hipLaunchKernelGGL(verify_sample<true>, sample, dim3(kThreads), 0, c->stream, a);
        return nvr::launch_status();
    }
    const dim3 walk{unsigned(batch), unsigned(draft_logits && max_nodes > 2 ? kSlices : 1)};
    if (walk.y > 1) {
        hipLaunchKernelGGL(verify_walk<true>, walk, dim3(kWalkThreads), 0, c->stream, a);
        NVR_HIP(hipGetLastError());
    }
    hipLaunchKernelGGL(verify_walk<false>, walk, dim3(kWalkThreads), 0, c->stream, a);
    NVR_HIP(hipGetLastError());
    hipLaunchKernelGGL(verify_sample<false>, sample, dim3(kThreads), 0, c->stream, a);
    return nvr::launch_status();
}

}  // extern "C"
