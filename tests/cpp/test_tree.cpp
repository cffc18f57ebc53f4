// The C++ host API's operators on trees of drafted tokens: masks and size checks
// on the CPU; on a GPU each refusal by its Fault kind, and one step of
// attention, verification, compaction and a block copy in a captured graph.
//
// Usage: test_tree cpu|gpu   -> runs that suite, exit status 0 when all pass.
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
// Reproducible bf16 values in [-1, 1).
std::vector<uint16_t> noise(std::size_t n, uint64_t seed) {
    std::vector<uint16_t> out(n);
    for (std::size_t i = 0; i < n; ++i)
        out[i] = bf16(float(int64_t(nvr::sampling_seed(seed, i, 0) >> 40)) / float(1 << 23) - 1.0f);
    return out;
}

constexpr std::size_t kQh = 4, kKvh = 2, kDim = 64, kBs = 16, kBlocks = 4, kStride = 2, kLayers = 2;
constexpr std::size_t kSpan = kBlocks * kBs * kKvh * kDim * 2;  // bytes of one layer's cache

// -------------------------------------------------------------- CPU suite --
TEST(tree_masks_hold_ancestors, "cpu") {
    CHECK((nvr::tree_masks({-1, 0, 0, 1, 3, 2}) == std::vector<uint64_t>{1, 3, 5, 11, 27, 37}));
    CHECK_FAULT(nvr::tree_masks({}), nvr::Fault::Value);
    CHECK_FAULT(nvr::tree_masks({-1, 1}), nvr::Fault::Value);
    CHECK_FAULT(nvr::tree_masks({-1, -1}), nvr::Fault::Value);
    CHECK_FAULT(nvr::tree_masks(std::vector<int32_t>(65, 0)), nvr::Fault::Value);
}

// -------------------------------------------------------------- GPU suite --
struct Step {
    nvr::Gpu gpu{0};
    std::size_t rows = 5, batch = 1, width = 5, vocab = 300;
    std::vector<int32_t> parents{-1, 0, 0, 2, 3};
    nvr::Buffer q = gpu.alloc(rows * kQh * kDim * 2), out = gpu.alloc(rows * kQh * kDim * 2);
    nvr::Buffer kc = gpu.alloc(kLayers * kSpan), vc = gpu.alloc(kLayers * kSpan);
    nvr::Buffer contexts = gpu.alloc(4), starts = gpu.alloc(8), masks = gpu.alloc(rows * 8), tables = gpu.alloc(8);
    nvr::Buffer logits = gpu.alloc(rows * vocab * 2), tokens = gpu.alloc(rows * 4), up = gpu.alloc(rows * 4);
    nvr::Buffer temps = gpu.alloc(4), uniforms = gpu.alloc(rows * 4), seeds = gpu.alloc(8);
    nvr::Buffer out_tokens = gpu.alloc(width * 4), out_nodes = gpu.alloc(width * 4), counts = gpu.alloc(4);
    nvr::Buffer work = gpu.alloc(1 << 20), verify_work = gpu.alloc(gpu.verify_tree_workspace(rows, batch, vocab) + 64);

    void attention(std::size_t max_nodes, std::size_t max_context, const nvr::Buffer& to) const {
        gpu.attention_tree(q, kc, vc, contexts, starts, masks, tables, to, work, rows, kQh, kKvh, kDim, kBs, kBlocks,
                           kStride, batch, max_nodes, max_context);
    }
    void verify(std::size_t max_nodes, const nvr::Buffer& scratch) const {
        gpu.verify_tree(logits, nvr::Buffer(), tokens, up, starts, temps, uniforms, seeds, out_tokens, out_nodes,
                        counts, scratch, rows, batch, max_nodes, vocab);
    }
    void compact(std::size_t max_nodes, const nvr::Buffer& v, std::size_t layers) const {
        gpu.kv_compact(kc, v, contexts, out_nodes, counts, tables, batch, max_nodes, layers, kKvh, kDim, kBs, kBlocks,
                       kStride);
    }
};

TEST(tree_calls_refuse_by_fault, "gpu") {
    Step s;
    CHECK_FAULT(s.attention(0, 32, s.out), nvr::Fault::Value);
    CHECK_FAULT(s.attention(65, 32, s.out), nvr::Fault::Value);
    CHECK_FAULT(s.attention(5, 0, s.out), nvr::Fault::Dimension);
    CHECK_FAULT(s.attention(5, 32, s.q), nvr::Fault::Overlap);
    CHECK_FAULT(s.attention(5, 32, s.out.slice(0, 64)), nvr::Fault::Extent);
    CHECK_FAULT(s.verify(65, s.verify_work), nvr::Fault::Value);
    CHECK_FAULT(s.verify(6, s.verify_work), nvr::Fault::Extent);  // outputs of five
    CHECK_FAULT(s.verify(5, s.verify_work.slice(0, 64)), nvr::Fault::Extent);
    CHECK_FAULT(s.verify(5, s.verify_work.slice(8, s.verify_work.len() - 8)), nvr::Fault::Alignment);
    CHECK_FAULT(s.compact(0, s.vc, kLayers), nvr::Fault::Value);
    CHECK_FAULT(s.compact(5, s.vc, kLayers + 1), nvr::Fault::Extent);
    CHECK_FAULT(s.compact(5, s.kc, kLayers), nvr::Fault::Overlap);
    nvr::Gpu other(0);
    CHECK_FAULT(s.compact(5, other.alloc(kLayers * kSpan), kLayers), nvr::Fault::Foreign);
    CHECK_FAULT(s.gpu.kv_copy_blocks(s.kc, s.vc, s.contexts, s.contexts, s.contexts, 1, kLayers, kKvh, std::size_t(1) << 31, kBs,
                                     kBlocks),
                nvr::Fault::Dimension);
    CHECK_FAULT(s.gpu.kv_copy_blocks(s.kc, s.vc, s.contexts, s.contexts, s.contexts, 2, kLayers, kKvh, kDim, kBs,
                                     kBlocks),
                nvr::Fault::Extent);
}

TEST(tree_step_in_a_graph, "gpu") {
    Step s;
    const int32_t context = 9;
    const std::vector<uint16_t> q = noise(s.rows * kQh * kDim, 1), k = noise(kLayers * kSpan / 2, 2),
                                v = noise(kLayers * kSpan / 2, 3);
    s.q.upload_u16(q);
    s.contexts.upload_i32({context});
    s.starts.upload_i32({0, 5});
    s.masks.upload_u64(nvr::tree_masks(s.parents));
    s.tables.upload_i32({3, 1});
    s.up.upload_i32(s.parents);
    s.tokens.upload_i32({0, 11, 22, 33, 44});
    // Greedy: node 0 goes to 22 (node 2), node 2 to 33 (node 3), node 3 to 7, which is not drafted.
    std::vector<uint16_t> logits(s.rows * s.vocab, bf16(0.0f));
    logits[0 * s.vocab + 22] = logits[2 * s.vocab + 33] = logits[3 * s.vocab + 7] = bf16(5.0f);
    s.logits.upload_u16(logits);
    auto run = [&] {
        s.attention(5, 32, s.out);
        s.verify(5, s.verify_work);
        s.compact(5, s.vc, kLayers);
        // The block of the last positions, copied whole to block 0.
        s.gpu.kv_copy_blocks(s.kc, s.vc, s.tables.slice(0, 4), s.starts.slice(0, 4), s.starts.slice(4, 4), 1, kLayers,
                             kKvh, kDim, kBs, kBlocks);
    };
    const nvr::Graph graph = s.gpu.capture(run);
    for (int replay = 0; replay < 3; ++replay) {
        s.kc.upload_u16(k);
        s.vc.upload_u16(v);
        graph.replay();
        CHECK((s.out_tokens.download_i32(5) == std::vector<int32_t>{22, 33, 7, -1, -1}));
        CHECK((s.out_nodes.download_i32(5) == std::vector<int32_t>{0, 2, 3, -1, -1}));
        CHECK(s.counts.download_i32(1)[0] == 3);
        // Attention in fp64 over the caches as they were (layer 0).
        const std::vector<uint16_t> out = s.out.download_u16(s.rows * kQh * kDim);
        const std::vector<uint64_t> masks = nvr::tree_masks(s.parents);
        for (std::size_t r = 0; r < s.rows; ++r)
            for (std::size_t h = 0; h < kQh; ++h) {
                std::vector<double> o(kDim, 0.0);
                double sum = 0.0;
                for (std::size_t t = 0; t < std::size_t(context) + s.rows; ++t) {
                    if (t >= std::size_t(context) && (masks[r] >> (t - context) & 1) == 0) continue;
                    const std::size_t at = (3 * kBs + t) * kKvh + h / (kQh / kKvh);  // all in block 3
                    double dot = 0.0;
                    for (std::size_t d = 0; d < kDim; ++d)
                        dot += double(value(q[(r * kQh + h) * kDim + d])) * value(k[at * kDim + d]);
                    const double p = std::exp(dot / std::sqrt(double(kDim)));
                    sum += p;
                    for (std::size_t d = 0; d < kDim; ++d) o[d] += p * value(v[at * kDim + d]);
                }
                // |v| <= 1: a bf16 weight is off by 2^-8 of itself at most, the output's rounding by as much; 2^-14
                // covers the fp32 scores (64 products below 1, each rounded).
                for (std::size_t d = 0; d < kDim; ++d)
                    CHECK(std::fabs(value(out[(r * kQh + h) * kDim + d]) - o[d] / sum) <= 0x1p-8 + 0x1p-8 + 0x1p-14);
            }
        // Node 2 moved to position 10, node 3 to 11; then five slots of block 3 are block 0's too.
        const std::vector<uint16_t> kc = s.kc.download_u16(kLayers * kSpan / 2), vc = s.vc.download_u16(kLayers * kSpan / 2);
        const std::size_t slot = kKvh * kDim;
        for (std::size_t layer = 0; layer < kLayers; ++layer)
            for (std::size_t t = 0; t < kBlocks * kBs; ++t) {
                const std::size_t base = layer * kBlocks * kBs;
                std::size_t from = t;
                if (t < 5) from = 3 * kBs + t;
                if (t == 3 * kBs + 10) from = 3 * kBs + 11;
                if (t == 3 * kBs + 11) from = 3 * kBs + 12;
                for (std::size_t e = 0; e < slot; ++e) {
                    CHECK(kc[(base + t) * slot + e] == k[(base + from) * slot + e]);
                    CHECK(vc[(base + t) * slot + e] == v[(base + from) * slot + e]);
                }
            }
    }
}

}  // namespace
