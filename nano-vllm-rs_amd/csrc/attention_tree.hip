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
// Scores, maxima, sums and outputs are fp32, rounded to bf16 once at the end.
#include "../../include/nano_hip.h"
#include "nvr_device.h"
#include "nvr_internal.h"

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

// Any head dim and alignment: a block per (node, q head), its four waves over
// every fourth position, lanes over the head's elements.
__global__ __launch_bounds__(256) void attention_tree_direct(TreeArgs a) {
    constexpr int kWaves = 4, kElems = 4;  // 64 lanes x 4 elements: head dims up to 256
    __shared__ float part_m[kWaves], part_l[kWaves], part_o[kWaves][256];
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
    float q[kElems], o[kElems] = {};
#pragma unroll
    for (int e = 0; e < kElems; ++e) {
        const int d = lane + e * kWave;
        q[e] = d < a.dim ? nvr::bf16_to_f32(a.q[row * a.dim + d]) : 0.0f;
    }
    float m = -kInf, l = 0.0f;
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
        const float x = dot * a.scale;
        if (x == -kInf) continue;
        const float top = fmaxf(m, x);  // a NaN leaves m, and makes l NaN
        const float old = m == -kInf ? 0.0f : __builtin_amdgcn_exp2f(m - top);
        const float p = __builtin_amdgcn_exp2f(x - top);
        m = top;
        l = __builtin_fmaf(l, old, p);
#pragma unroll
        for (int e = 0; e < kElems; ++e) {
            const int d = lane + e * kWave;
            if (d < a.dim) o[e] = __builtin_fmaf(p, nvr::bf16_to_f32(a.vc[at + d]), o[e] * old);
        }
    }
    if (lane == 0) { part_m[wave] = m; part_l[wave] = l; }
#pragma unroll
    for (int e = 0; e < kElems; ++e) part_o[wave][lane + e * kWave] = o[e];
    __syncthreads();
    float top = -kInf, den = 0.0f, num = 0.0f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) top = fmaxf(top, part_m[w]);
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
        if (part_m[w] == -kInf && part_l[w] == 0.0f) continue;  // saw nothing
        const float f = __builtin_amdgcn_exp2f(part_m[w] - top);
        den = __builtin_fmaf(part_l[w], f, den);
        num = __builtin_fmaf(part_o[w][threadIdx.x], f, num);
    }
    if (int(threadIdx.x) < a.dim) a.out[row * a.dim + threadIdx.x] = nvr::f32_to_bf16(den > 0.0f ? num / den : 0.0f);
}

}  // namespace

extern "C" {

int nv_attention_tree_workspace(int rows, int qh, int kvh, int dim, int batch, int max_nodes, int max_context,
                                size_t* bytes) {
    if (rows <= 0 || qh <= 0 || kvh <= 0 || dim <= 0 || batch <= 0 || max_nodes <= 0 || max_context <= 0 || qh % kvh)
        return nvr::fail(-2, "attention_tree_workspace: dimensions must be positive, q heads a multiple of KV heads");
    *bytes = 0;
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
    const int64_t span = int64_t(stride) * bs;
    const TreeArgs a{static_cast<const uint16_t*>(q), static_cast<const uint16_t*>(kc), static_cast<const uint16_t*>(vc),
                     static_cast<const int*>(contexts), static_cast<const int*>(row_starts),
                     static_cast<const uint64_t*>(masks), static_cast<const int*>(tables), static_cast<uint16_t*>(out),
                     rows, qh, kvh, dim, bs, blocks, stride, batch, max_nodes,
                     span < max_context ? span : int64_t(max_context), kLog2e / sqrtf(float(dim))};
    const int64_t grid = int64_t(batch) * max_nodes * qh;
    if (grid > 0x7fffffff) return nvr::fail(-2, "attention_tree: %d sequences of %d nodes exceed one launch", batch, max_nodes);
    hipLaunchKernelGGL(attention_tree_direct, dim3(unsigned(grid)), dim3(256), 0, c->stream, a);
    return nvr::launch_status();
}

}  // extern "C"
