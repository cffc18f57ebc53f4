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
//     rejection c += Z and then Z = sum over x of max(p_v - c q_v, 0). (The rest after a
//     rejection is max(r - Z q, 0) of the rest r before, Z its sum; and
//     max(max(p - c q, 0) - Z q, 0) = max(p - (c + Z) q, 0), so one number says what every rejection took.) After all are
//     rejected, the rest is max(p_v - c q_v, 0).
//   - T <= 0 (or NaN): accepted if x is v's argmax.
// The first accepted child is the next v. Where none is, the path ends and its
// last token is the argmax of ln(rest) + Gumbel noise, which nv_sample adds from
// seeds[s] and the token (for T <= 0 of the logits alone): with nothing rejected
// at v it is nv_sample's token of that row. Where the rest is nothing, it is v's
// argmax. Drafted tokens outside [0, vocab) are passed over, as are nodes whose
// parent does not come before them. NaN logits have probability 0; ties go to the lower index; an argmax of nothing is 0.
//
// For T > 0 the emitted tokens are distributed as the target's own samples are.
// What decides is held in fp32 sums of fp32 exponentials, and in fp64 from there
// on: a comparison or an argmax goes the other way than exact arithmetic has it
// only where both sides agree to about 1e-6.
//
// Launches: 1. verify_stats: maximum, its index and the sum of exponentials over
// partitions of each row that has children (both models'). 2. verify_walk: a
// block a sequence folds them and walks the tree. 3. verify_sample: partitions
// of the last rows. 4. verify_finish: folds those into the last token.
#include "../../include/nano_hip.h"
#include "nvr_device.h"
#include "nvr_internal.h"

namespace {

using nvr::kWave;
constexpr int kMaxNodes = 64;
constexpr int kPartition = 2048;  // tokens a block of launches 1 and 3
constexpr int kThreads = kPartition / 8;
constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kInf = __builtin_inff();

// A partition of a row's logits, or the fold of a row's partitions.
struct Stats {
    float max, sum;  // sum of exp((logit - max) / T)
    int best;        // the maximum's token
    int pad;
};

// Where a sequence's walk ended.
struct Ending {
    int row;             // the path's last row, or -1: an invalid sequence
    int node;            // the path's tokens but the last one
    int fallback;        // the row's argmax where it has children, else 0
    int tried;           // tokens to leave out (no draft logits)
    float c;             // what rejections took (draft logits)
    float max, inv_sum;  // of the target's row, where c > 0
    float draft_max, draft_inv_sum;
    int token[kMaxNodes];
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
    float* scores;       // [batch, parts]
    int* ids;            // [batch, parts]
    int rows, batch, max_nodes, vocab, parts;
};

__host__ __device__ inline int partitions(int vocab) {
    // A row's first token may lie up to 7 tokens behind a 16-byte boundary.
    return int((int64_t(vocab) + 7 + kPartition - 1) / kPartition);
}

// Rows of sequence s: the first and how many; none for an invalid sequence.
__device__ __forceinline__ int tree_rows(const VerifyArgs& a, int s, int* start) {
    const int first = a.row_starts[s], end = a.row_starts[s + 1];
    *start = first;
    return first < 0 || end > a.rows || end <= first || int64_t(end) - first > a.max_nodes ? 0 : end - first;
}

// Eight logits of one row as its 16-byte chunk holds them: tokens t .. t + 7,
// those outside [0, vocab) NaN, which never wins and weighs nothing.
__device__ __forceinline__ void load_chunk(const uint16_t* row, int64_t t, int vocab, float (&f)[8]) {
    if (t >= 0 && t + 8 <= vocab) {
        nvr::unpack8(nvr::load_stream(row + t), f);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = t + i >= 0 && t + i < vocab ? nvr::bf16_to_f32(row[t + i]) : __builtin_nanf("");
    }
}
__device__ __forceinline__ int lead_of(const uint16_t* row) { return int(reinterpret_cast<uintptr_t>(row) >> 1 & 7); }

// exp((x - top) / T) with scale = log2(e) / T; 1 at an infinite maximum, 0 for NaN.
__device__ __forceinline__ float weight(float x, float top, float scale) {
    if (x == top) return 1.0f;
    return x == x ? __builtin_amdgcn_exp2f((x - top) * scale) : 0.0f;
}

__device__ __forceinline__ float inverse(float sum) { return sum > 0.0f ? 1.0f / sum : 0.0f; }

struct Best {
    float score;
    int index;
};
__device__ __forceinline__ void consider(Best& b, float s, int i) {
    if (nvr::better(s, i, b.score, b.index)) { b.score = s; b.index = i; }
}
__device__ __forceinline__ Best wave_best(Best b) {
#pragma unroll
    for (int mask = 1; mask < kWave; mask <<= 1) {
        const float s = nvr::xor_lane(b.score, mask);
        const int i = nvr::xor_lane(b.index, mask);
        consider(b, s, i);
    }
    return b;
}
__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
    for (int mask = 1; mask < kWave; mask <<= 1) v += nvr::xor_lane(v, mask);
    return v;
}

// A block a (sequence, node, partition); nodes without children have nothing to do.
__global__ __launch_bounds__(kThreads) void verify_stats(VerifyArgs a) {
    __shared__ Best tops[kThreads / kWave];
    __shared__ float sums[kThreads / kWave];
    const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
    const int part = int(blockIdx.x % unsigned(a.parts));
    const int item = int(blockIdx.x / unsigned(a.parts));
    const int s = item / a.max_nodes, node = item % a.max_nodes;
    int start;
    const int n = tree_rows(a, s, &start);
    if (node >= n) return;
    const bool child = lane > node && lane < n && a.parents[start + lane] == node;
    if (__ballot(child) == 0) return;
    const float temperature = a.temps[s];
    const bool sampled = temperature > 0.0f;
    const float scale = kLog2e / temperature;
    const int row = start + node;
    for (int side = 0; side < (sampled && a.draft ? 2 : 1); ++side) {
        const uint16_t* x = (side ? a.draft : a.logits) + int64_t(row) * a.vocab;
        const int64_t t = int64_t(part) * kPartition + 8 * int(threadIdx.x) - lead_of(x);
        float f[8];
        load_chunk(x, t, a.vocab, f);
        Best b{-kInf, nvr::kNoIndex};
#pragma unroll
        for (int i = 0; i < 8; ++i) consider(b, f[i], int(t) + i);
        b = wave_best(b);
        if (lane == 0) tops[wave] = b;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < kThreads / kWave; ++w) consider(b, tops[w].score, tops[w].index);
        float sum = 0.0f;
        if (sampled && b.score > -kInf) {
#pragma unroll
            for (int i = 0; i < 8; ++i) sum += weight(f[i], b.score, scale);
        }
        sum = wave_sum(sum);
        if (lane == 0) sums[wave] = sum;
        __syncthreads();
        if (threadIdx.x == 0) {
            sum = 0.0f;
#pragma unroll
            for (int w = 0; w < kThreads / kWave; ++w) sum += sums[w];
            (side ? a.draft_stats : a.stats)[int64_t(row) * a.parts + part] = Stats{b.score, sum, b.index, 0};
        }
        __syncthreads();
    }
}

// A row's partitions folded, by one wave.
__device__ __forceinline__ Stats fold(const Stats* part, int parts, float scale, int lane) {
    Best b{-kInf, nvr::kNoIndex};
    for (int i = lane; i < parts; i += kWave) consider(b, part[i].max, part[i].best);
    b = wave_best(b);
    double sum = 0.0;
    for (int i = lane; i < parts; i += kWave)
        if (part[i].max > -kInf) sum += double(part[i].sum) * double(weight(part[i].max, b.score, scale));
#pragma unroll
    for (int mask = 1; mask < kWave; mask <<= 1) sum += __shfl_xor(sum, mask);
    return Stats{b.score, float(sum), b.index, 0};
}

constexpr int kWalkThreads = 1024;
constexpr int kWalkWaves = kWalkThreads / kWave;

__global__ __launch_bounds__(kWalkThreads) void verify_walk(VerifyArgs a) {
    __shared__ Stats target[kMaxNodes], draft[kMaxNodes];
    __shared__ double parts[kWalkWaves];
    __shared__ int path[kMaxNodes];
    const int lane = threadIdx.x & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int s = int(blockIdx.x);
    Ending* ending = a.endings + s;
    int start;
    const int n = tree_rows(a, s, &start);
    int* tokens = a.out_tokens + int64_t(s) * a.max_nodes;
    int* nodes = a.out_nodes + int64_t(s) * a.max_nodes;
    if (n == 0) {
        for (int i = int(threadIdx.x); i < a.max_nodes; i += kWalkThreads) tokens[i] = nodes[i] = -1;
        if (threadIdx.x == 0) { a.out_counts[s] = 0; ending->row = -1; }
        return;
    }
    const float temperature = a.temps[s];
    const bool sampled = temperature > 0.0f, drafted = sampled && a.draft != nullptr;
    const float scale = kLog2e / temperature;
    // Lane i of every wave holds node i.
    const bool mine = lane > 0 && lane < n;
    int parent = mine ? a.parents[start + lane] : -1;
    if (parent < 0 || parent >= lane) parent = -1;
    const int token = mine ? a.tokens[start + lane] : -1;
    const bool known = parent >= 0 && token >= 0 && token < a.vocab;
    const float u = mine ? a.uniforms[start + lane] : 0.0f;
    for (int v = wave; v < n; v += kWalkWaves) {
        if (__ballot(parent == v) == 0) continue;
        const int64_t at = int64_t(start + v) * a.parts;
        const Stats t = fold(a.stats + at, a.parts, scale, lane);
        if (lane == 0) target[v] = t;
        if (drafted) {
            const Stats d = fold(a.draft_stats + at, a.parts, scale, lane);
            if (lane == 0) draft[v] = d;
        }
    }
    __syncthreads();
    // Each node's probabilities under its parent's rows.
    auto chance = [&](const uint16_t* logits, const Stats& r) -> double {
        const float x = nvr::bf16_to_f32(logits[int64_t(start + parent) * a.vocab + token]);
        if (!(r.max > -kInf) || x != x) return 0.0;
        if (x == r.max) return 1.0 / double(r.sum);
        const double y = (double(x) - double(r.max)) / double(temperature);
        return y > -700.0 ? nvr::d_exp(y) / double(r.sum) : 0.0;
    };
    double p = 0.0, q = 0.0;
    if (sampled && known) {
        p = chance(a.logits, target[parent]);
        if (drafted) q = chance(a.draft, draft[parent]);
    }
    // Every wave walks alike.
    int v = 0, length = 0, tried = 0;
    double c = 0.0, z = 1.0;
    uint64_t rejected = 0;
    while (true) {
        if (threadIdx.x == 0) path[length] = v;
        ++length;
        uint64_t children = __ballot(known && parent == v);
        const int best = children != 0 && target[v].best != nvr::kNoIndex ? target[v].best : 0;
        c = 0.0; z = 1.0; rejected = 0;
        int next = -1;
        while (children != 0) {
            const int i = __builtin_ctzll(children);
            children &= children - 1;
            const int x = __builtin_amdgcn_readlane(token, i);
            if (!sampled) {
                if (x == best) { next = i; break; }
                continue;
            }
            const double px = __shfl(p, i), ux = double(__shfl(u, i));
            if (drafted) {
                const double qx = __shfl(q, i), r = fmax(px - c * qx, 0.0);
                if (r > 0.0 && ux * z * qx < r) { next = i; break; }
                c += z;
                if (children == 0) break;
                // The rest's sum, for the next child.
                const uint16_t* xt = a.logits + int64_t(start + v) * a.vocab;
                const uint16_t* xd = a.draft + int64_t(start + v) * a.vocab;
                const Stats t = target[v], d = draft[v];
                const float it = inverse(t.sum), id = float(c) * inverse(d.sum);
                double sum = 0.0;
                for (int64_t k = threadIdx.x; k < a.vocab; k += kWalkThreads) {
                    const float wt = weight(nvr::bf16_to_f32(xt[k]), t.max, scale) * it;
                    const float wd = weight(nvr::bf16_to_f32(xd[k]), d.max, scale) * id;
                    sum += double(fmaxf(wt - wd, 0.0f));
                }
#pragma unroll
                for (int mask = 1; mask < kWave; mask <<= 1) sum += __shfl_xor(sum, mask);
                if (lane == 0) parts[wave] = sum;
                __syncthreads();
                z = 0.0;
                for (int w = 0; w < kWalkWaves; ++w) z += parts[w];
                __syncthreads();
            } else {
                if (__ballot((rejected >> lane & 1) != 0 && token == x) != 0) continue;
                if (px > 0.0 && ux * z < px) { next = i; break; }
                rejected |= uint64_t(1) << i;
                z -= px;
            }
        }
        if (next < 0) break;
        v = next;
    }
    __syncthreads();  // path
    const int step = int(threadIdx.x);
    if (step < a.max_nodes) {
        nodes[step] = step < length ? path[step] : -1;
        tokens[step] = step + 1 < length ? a.tokens[start + path[step + 1]] : -1;
    }
    if (wave == 0) {
        const bool out = (rejected >> lane & 1) != 0;
        const uint64_t all = __ballot(out);
        tried = __popcll(all);
        if (out) ending->token[__popcll(all & ((uint64_t(1) << lane) - 1))] = token;
        if (lane == 0) {
            const bool inner = c > 0.0;
            a.out_counts[s] = length;
            ending->row = start + v;
            ending->node = length - 1;
            ending->tried = tried;
            ending->c = float(c);
            ending->fallback = 0;
            ending->max = inner ? target[v].max : 0.0f;
            ending->inv_sum = inner ? inverse(target[v].sum) : 0.0f;
            ending->draft_max = inner ? draft[v].max : 0.0f;
            ending->draft_inv_sum = inner ? inverse(draft[v].sum) : 0.0f;
        }
        if (__ballot(parent == v) != 0 && lane == 0 && target[v].best != nvr::kNoIndex) ending->fallback = target[v].best;
    }
}

// A block a (sequence, partition of its last row).
__global__ __launch_bounds__(kThreads) void verify_sample(VerifyArgs a) {
    __shared__ Best tops[kThreads / kWave];
    __shared__ int tried[kMaxNodes];
    const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
    const int part = int(blockIdx.x % unsigned(a.parts));
    const int s = int(blockIdx.x / unsigned(a.parts));
    const Ending* e = a.endings + s;
    const int row = e->row;
    if (row < 0) return;
    const int count = e->tried;
    if (int(threadIdx.x) < count) tried[threadIdx.x] = e->token[threadIdx.x];
    __syncthreads();
    const float temperature = a.temps[s];
    const uint64_t seed = a.seeds[s];
    const uint16_t* x = a.logits + int64_t(row) * a.vocab;
    const int64_t t = int64_t(part) * kPartition + 8 * int(threadIdx.x) - lead_of(x);
    float f[8];
    load_chunk(x, t, a.vocab, f);
    Best b{-kInf, nvr::kNoIndex};
    if (!(temperature > 0.0f)) {
#pragma unroll
        for (int i = 0; i < 8; ++i) consider(b, f[i], int(t) + i);
    } else if (e->c > 0.0f) {
        const uint16_t* y = a.draft + int64_t(row) * a.vocab;
        const float scale = kLog2e / temperature, cq = e->c * e->draft_inv_sum;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if (t + i < 0 || t + i >= a.vocab) continue;
            const float wt = weight(f[i], e->max, scale) * e->inv_sum;
            const float wd = weight(nvr::bf16_to_f32(y[t + i]), e->draft_max, scale) * cq;
            const float w = wt - wd;
            if (!(w >= 0x1p-126f)) continue;
            const float g = nvr::hash_uniform(nvr::splitmix64(seed ^ (uint64_t(t + i) * nvr::kTokenMix)));
            consider(b, nvr::nvr_logf(w) - nvr::nvr_logf(-nvr::nvr_logf(g)), int(t) + i);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float score = nvr::gumbel_score(f[i], temperature, seed, uint32_t(t + i));
            if (!nvr::better(score, int(t) + i, b.score, b.index) || (count > 0 && score == -kInf)) continue;
            bool out = false;
            for (int k = 0; k < count; ++k) out |= tried[k] == int(t) + i;
            if (!out) b = Best{score, int(t) + i};
        }
    }
    b = wave_best(b);
    if (lane == 0) tops[wave] = b;
    __syncthreads();
    if (threadIdx.x == 0) {
#pragma unroll
        for (int w = 0; w < kThreads / kWave; ++w) consider(b, tops[w].score, tops[w].index);
        a.scores[int64_t(s) * a.parts + part] = b.score;
        a.ids[int64_t(s) * a.parts + part] = b.index;
    }
}

__global__ __launch_bounds__(kWave) void verify_finish(VerifyArgs a) {
    const int s = int(blockIdx.x), lane = int(threadIdx.x);
    const Ending* e = a.endings + s;
    if (e->row < 0) return;
    Best b{-kInf, nvr::kNoIndex};
    for (int i = lane; i < a.parts; i += kWave)
        consider(b, a.scores[int64_t(s) * a.parts + i], a.ids[int64_t(s) * a.parts + i]);
    b = wave_best(b);
    if (lane == 0) a.out_tokens[int64_t(s) * a.max_nodes + e->node] = b.index == nvr::kNoIndex ? e->fallback : b.index;
}

// The workspace's parts, each at a multiple of 16 bytes.
struct Workspace {
    int64_t stats, draft_stats, endings, scores, ids, bytes;
};
Workspace layout(int rows, int batch, int vocab) {
    const int64_t parts = partitions(vocab);
    auto up = [](int64_t b) { return (b + 15) & ~int64_t(15); };
    Workspace w;
    w.stats = 0;
    w.draft_stats = w.stats + up(int64_t(sizeof(Stats)) * rows * parts);
    w.endings = w.draft_stats + up(int64_t(sizeof(Stats)) * rows * parts);
    w.scores = w.endings + up(int64_t(sizeof(Ending)) * batch);
    w.ids = w.scores + up(4 * int64_t(batch) * parts);
    w.bytes = w.ids + up(4 * int64_t(batch) * parts);
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
    if (!nvr::aligned(workspace, 16)) return nvr::fail(-2, "verify_tree: the workspace needs 16-byte alignment");
    const int parts = partitions(vocab);
    if (int64_t(batch) * max_nodes > 0x7fffffff / parts)
        return nvr::fail(-2, "verify_tree: %d sequences of %d nodes over %d tokens exceed one launch", batch, max_nodes, vocab);
    const Workspace w = layout(rows, batch, vocab);
    char* base = static_cast<char*>(workspace);
    const VerifyArgs a{static_cast<const uint16_t*>(logits), static_cast<const uint16_t*>(draft_logits),
                       static_cast<const int*>(tokens), static_cast<const int*>(parents),
                       static_cast<const int*>(row_starts), static_cast<const float*>(temps),
                       static_cast<const float*>(uniforms), static_cast<const uint64_t*>(seeds),
                       static_cast<int*>(out_tokens), static_cast<int*>(out_nodes), static_cast<int*>(out_counts),
                       reinterpret_cast<Stats*>(base + w.stats), reinterpret_cast<Stats*>(base + w.draft_stats),
                       reinterpret_cast<Ending*>(base + w.endings), reinterpret_cast<float*>(base + w.scores),
                       reinterpret_cast<int*>(base + w.ids), rows, batch, max_nodes, vocab, parts};
    hipLaunchKernelGGL(verify_stats, dim3(unsigned(int64_t(batch) * max_nodes * parts)), dim3(kThreads), 0, c->stream, a);
    NVR_HIP(hipGetLastError());
    hipLaunchKernelGGL(verify_walk, dim3(unsigned(batch)), dim3(kWalkThreads), 0, c->stream, a);
    NVR_HIP(hipGetLastError());
    hipLaunchKernelGGL(verify_sample, dim3(unsigned(int64_t(batch) * parts)), dim3(kThreads), 0, c->stream, a);
    NVR_HIP(hipGetLastError());
    hipLaunchKernelGGL(verify_finish, dim3(unsigned(batch)), dim3(kWave), 0, c->stream, a);
    return nvr::launch_status();
}

}  // extern "C"
