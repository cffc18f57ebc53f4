// Moves inside the paged KV cache: a forked sequence's block (nv_kv_copy_blocks)
// and the nodes that a tree of drafted tokens keeps (nv_kv_compact). No
// counterpart in the reference, whose sequences only append (src/runtime.rs:747-755).
//
// Caches are [layers, blocks, bs, kvh, dim]: one launch moves K and V of every
// layer. Both are copies of bits, bound by HBM (copy_blocks) or by their chain of
// memory round trips (compact).
#include "../../include/nano_hip.h"
#include "nvr_device.h"
#include "nvr_internal.h"

namespace {

using nvr::kWave;
constexpr int kMaxNodes = 64;

// The first min(tokens[i], bs) slots of block src[i] to block dst[i]: they are
// contiguous, so a copy is cut into segments of kSegment chunks whatever the
// slot size, one a block, all loads of a thread in flight before its stores.
// Bound by HBM: 12 copies of partly filled blocks of 256 positions from 4 sources in
// 28 layers (280 MB written, 385 MB with each source read once) take 63 us, the call 67:
// 5.7 to 6.2 TB/s; a source's second and third read hit the caches. Writes bypass them, or
// they would be in the way of sources read again (98 us); reads do not (80), nor do more
// loads a thread hide more (eight 78, two 66).
constexpr int kCopyLoads = 4;
constexpr int kSegment = 256 * kCopyLoads;

template <typename Chunk>  // uint4, or uint16_t where sizes or addresses are no multiples of 16 bytes
__global__ __launch_bounds__(256) void copy_blocks(Chunk* __restrict__ kc, Chunk* __restrict__ vc,
                                                   const int* __restrict__ src, const int* __restrict__ dst,
                                                   const int* __restrict__ tokens, int copies, int bs, int blocks,
                                                   int64_t slot_chunks, int64_t segments) {
    const int64_t segment = int64_t(blockIdx.x) % segments;
    const int64_t item = int64_t(blockIdx.x) / segments;
    const int i = int(item % copies);
    const int64_t plane = item / copies;  // 2 * layer + (K: 0, V: 1)
    const int from = src[i], to = dst[i], n = min(tokens[i], bs);
    if (from < 0 || from >= blocks || to < 0 || to >= blocks || from == to || n <= 0) return;
    const int64_t block_chunks = slot_chunks * bs, end = slot_chunks * n;
    Chunk* cache = (plane & 1 ? vc : kc) + (plane >> 1) * blocks * block_chunks;
    const Chunk* s = cache + from * block_chunks;
    Chunk* d = cache + to * block_chunks;
    const int64_t first = segment * kSegment + threadIdx.x;
    Chunk v[kCopyLoads];
#pragma unroll
    for (int u = 0; u < kCopyLoads; ++u) {
        const int64_t at = first + u * 256;
        if (at < end) v[u] = s[at];
    }
#pragma unroll
    for (int u = 0; u < kCopyLoads; ++u) {
        const int64_t at = first + u * 256;
        if (at < end) {
            if constexpr (sizeof(Chunk) == 16) nvr::store_stream(d + at, v[u]);
            else d[at] = v[u];
        }
    }
}

// Position contexts[s] + nodes[s, j] to contexts[s] + j, for j < counts[s] in
// order. The nodes rise, so nodes[j] >= j: a move's target is no later move's
// source, and a thread that takes one column of the slots through all moves,
// reading kBatch of them before it writes, needs no second buffer. A block a
// (sequence, layer): its time is the chain nodes, table, slots, store: 3.6 us for 8
// sequences in 28 layers (2.5 MB), 5.3 for 64 (16 MB). Stores bypass the caches: 10
// us for the 64 with plain ones.
template <typename Chunk>
__global__ __launch_bounds__(256) void compact(Chunk* __restrict__ kc, Chunk* __restrict__ vc,
                                               const int* __restrict__ contexts, const int* __restrict__ nodes,
                                               const int* __restrict__ counts, const int* __restrict__ tables,
                                               int max_nodes, int bs, int blocks, int stride, int64_t slot_chunks) {
    constexpr int kBatch = 8;
    __shared__ int64_t from[kMaxNodes], to[kMaxNodes];
    __shared__ int moves;
    const int s = int(blockIdx.x);
    if (threadIdx.x < kWave) {
        const int j = int(threadIdx.x), count = counts[s], context = contexts[s];
        const bool named = j < max_nodes && j < count;
        const int node = named ? nodes[int64_t(s) * max_nodes + j] : 0;
        const int before = __shfl_up(node, 1);
        // Valid up to the first node that is out of range or does not rise.
        const bool bad = !named || node < j || node >= max_nodes || (j > 0 && node <= before);
        const uint64_t bads = __ballot(bad);
        const int valid = context < 0 || count > max_nodes ? 0 : bads == 0 ? kWave : __builtin_ctzll(bads);
        auto slot = [&](int64_t pos) -> int64_t {
            if (pos >= int64_t(stride) * bs) return -1;
            const int entry = tables[int64_t(s) * stride + uint32_t(pos) / uint32_t(bs)];
            return entry >= 0 && entry < blocks ? int64_t(entry) * bs + uint32_t(pos) % uint32_t(bs) : int64_t(-1);
        };
        int64_t a = -1, b = -1;
        if (j < valid && node != j) {
            a = slot(int64_t(context) + node);
            b = slot(int64_t(context) + j);
        }
        const bool moved = a >= 0 && b >= 0;
        const uint64_t all = __ballot(moved);
        const int at = __popcll(all & ((uint64_t(1) << j) - 1));
        if (moved) { from[at] = a; to[at] = b; }
        if (j == 0) moves = __popcll(all);
    }
    __syncthreads();
    if (moves == 0) return;
    // Each half of the block takes K or V of one layer.
    const int64_t layer = blockIdx.y;
    Chunk* cache = (threadIdx.x & 128 ? vc : kc) + layer * blocks * bs * slot_chunks;
    for (int64_t column = threadIdx.x & 127; column < slot_chunks; column += 128) {
        for (int j0 = 0; j0 < moves; j0 += kBatch) {
            Chunk v[kBatch];
#pragma unroll
            for (int u = 0; u < kBatch; ++u)
                if (j0 + u < moves) v[u] = cache[from[j0 + u] * slot_chunks + column];
#pragma unroll
            for (int u = 0; u < kBatch; ++u)
                if (j0 + u < moves) {
                    Chunk* at = cache + to[j0 + u] * slot_chunks + column;
                    if constexpr (sizeof(Chunk) == 16) nvr::store_stream(at, v[u]);
                    else *at = v[u];
                }
        }
    }
}

// Whether slots can be moved in 16-byte chunks.
bool chunked(const void* kc, const void* vc, int64_t width) {
    return width % 8 == 0 && nvr::aligned(kc, 16) && nvr::aligned(vc, 16);
}

}  // namespace

extern "C" {

int nv_kv_copy_blocks(nv_context* c, void* kc, void* vc, const void* src, const void* dst, const void* tokens,
                      int copies, int layers, int kvh, int dim, int bs, int blocks) {
    NVR_ACTIVATE(c);
    if (copies <= 0 || layers <= 0 || kvh <= 0 || dim <= 0 || bs <= 0 || blocks <= 0)
        return nvr::fail(-2, "kv_copy_blocks: dimensions must be positive");
    const int64_t width = int64_t(kvh) * dim;
    if (width > 0x7fffffff) return nvr::fail(-2, "kv_copy_blocks: kvh * dim exceeds int32");
    auto s = static_cast<const int*>(src), d = static_cast<const int*>(dst), t = static_cast<const int*>(tokens);
    const bool wide = chunked(kc, vc, width);
    const int64_t slot_chunks = wide ? width / 8 : width;
    const int64_t segments = (slot_chunks * bs + kSegment - 1) / kSegment;
    if (segments > 0xffffff / (2 * int64_t(layers)) / copies)  // a launch has fewer than 2^32 threads
        return nvr::fail(-2, "kv_copy_blocks: %d copies in %d layers exceed one launch", copies, layers);
    const dim3 grid(unsigned(2 * int64_t(layers) * copies * segments));
    if (wide)
        hipLaunchKernelGGL(copy_blocks<uint4>, grid, dim3(256), 0, c->stream, static_cast<uint4*>(kc),
                           static_cast<uint4*>(vc), s, d, t, copies, bs, blocks, slot_chunks, segments);
    else
        hipLaunchKernelGGL(copy_blocks<uint16_t>, grid, dim3(256), 0, c->stream, static_cast<uint16_t*>(kc),
                           static_cast<uint16_t*>(vc), s, d, t, copies, bs, blocks, slot_chunks, segments);
    return nvr::launch_status();
}

int nv_kv_compact(nv_context* c, void* kc, void* vc, const void* contexts, const void* nodes, const void* counts,
                  const void* tables, int batch, int max_nodes, int layers, int kvh, int dim, int bs, int blocks,
                  int stride) {
    NVR_ACTIVATE(c);
    if (batch <= 0 || layers <= 0 || kvh <= 0 || dim <= 0 || bs <= 0 || blocks <= 0 || stride <= 0)
        return nvr::fail(-2, "kv_compact: dimensions must be positive");
    if (max_nodes < 1 || max_nodes > kMaxNodes)
        return nvr::fail(-2, "kv_compact: max_nodes %d outside [1, %d]", max_nodes, kMaxNodes);
    const int64_t width = int64_t(kvh) * dim;
    if (width > 0x7fffffff) return nvr::fail(-2, "kv_compact: kvh * dim exceeds int32");
    if (layers > 65535 || batch > 0xffffff)
        return nvr::fail(-2, "kv_compact: %d sequences in %d layers exceed one launch", batch, layers);
    auto x = static_cast<const int*>(contexts), n = static_cast<const int*>(nodes);
    auto k = static_cast<const int*>(counts), t = static_cast<const int*>(tables);
    const dim3 grid{unsigned(batch), unsigned(layers)};
    if (chunked(kc, vc, width))
        hipLaunchKernelGGL(compact<uint4>, grid, dim3(256), 0, c->stream, static_cast<uint4*>(kc),
                           static_cast<uint4*>(vc), x, n, k, t, max_nodes, bs, blocks, stride, width / 8);
    else
        hipLaunchKernelGGL(compact<uint16_t>, grid, dim3(256), 0, c->stream, static_cast<uint16_t*>(kc),
                           static_cast<uint16_t*>(vc), x, n, k, t, max_nodes, bs, blocks, stride, width);
    return nvr::launch_status();
}

}  // extern "C"
