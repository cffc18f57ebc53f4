/*
 * nano_hip.h — C ABI of the nano-vllm-rs fused per-layer kernels for AMD
 * Instinct MI355X (gfx950).
 *
 * Every `nv_*` entry point keeps the name, argument order and meaning of the
 * CUDA library that the nano-vllm-rs Rust host links against, so the Rust
 * declarations in src/gpu.rs:17-178 bind to this library unchanged. Each
 * declaration cites the reference definition it replaces
 * (kernels/kernels.cu:<line>) and the Rust wrapper that calls it.
 *
 * Conventions (as in the reference):
 *  - Every function returning int returns 0 on success, a HIP error code on a
 *    runtime failure, hipBLAS status + 10000 on a BLAS failure, -1 when a host
 *    allocation fails, and -2 when arguments are rejected. The message is in a
 *    thread-local buffer returned by nv_last_error().
 *  - One context = one device, one non-blocking stream, one hipBLAS handle.
 *    Kernels are asynchronous launches on that stream; they never allocate or
 *    synchronise, so every kernel entry point is safe under graph capture.
 *  - Tensor arguments are device pointers. bf16 tensors are arrays of IEEE
 *    binary32 upper halves (uint16_t); int tensors are int32; seeds are uint64.
 *  - Row-major layouts; extents and aliasing are validated by the caller
 *    (src/gpu.rs:482-509 in the reference). The kernels still guard device
 *    metadata: token ids, gather indices, KV slots and RoPE positions.
 */
#ifndef NANO_HIP_H
#define NANO_HIP_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

typedef struct nv_context nv_context;

/* ------------------------------------------------------------ runtime ---- */

/* kernels/kernels.cu:28 — thread-local text of the last failure. */
const char* nv_last_error(void);
/* kernels/kernels.cu:29-33 — the context's hipStream_t (src/gpu.rs:18). */
int nv_stream(nv_context* c, void** output);
/* kernels/kernels.cu:34-38 — compute-unit count (src/gpu.rs:19, sm_count). */
int nv_sm_count(nv_context* c, int* output);
/* kernels/kernels.cu:39-51 — device, non-blocking stream, hipBLAS handle. */
int nv_create(int device, nv_context** output);
/* kernels/kernels.cu:52-59 — synchronises the stream, then frees. */
void nv_destroy(nv_context* c);
/* kernels/kernels.cu:60-66 — device allocation, zero-filled on the stream.
 * Refused while the stream is being captured. */
int nv_alloc(nv_context* c, size_t bytes, void** output);
/* kernels/kernels.cu:67 */
void nv_free(nv_context* c, void* buffer);
/* kernels/kernels.cu:68-72 — host -> device, synchronous on return. */
int nv_upload(nv_context* c, void* dst, const void* src, size_t bytes);
/* kernels/kernels.cu:73-77 — device -> host, synchronous on return. */
int nv_download(nv_context* c, const void* src, void* dst, size_t bytes);
/* kernels/kernels.cu:78 */
int nv_sync(nv_context* c);
/* kernels/kernels.cu:79 */
int nv_mem_info(nv_context* c, size_t* free_bytes, size_t* total_bytes);
/* kernels/kernels.cu:80 — thread-local stream capture. */
int nv_capture_begin(nv_context* c);
/* kernels/kernels.cu:81-89 — ends capture and instantiates (hipGraphExec_t). */
int nv_capture_end(nv_context* c, void** graph);
/* kernels/kernels.cu:90-95 */
void nv_capture_abort(nv_context* c);
/* kernels/kernels.cu:96 */
int nv_graph_replay(nv_context* c, void* graph);
/* kernels/kernels.cu:97 */
void nv_graph_destroy(nv_context* c, void* graph);

/* ---------------------------------------------------------------- GEMM ---- */

/* kernels/kernels.cu:98-106 — row-major Y[m,n] = X[m,k] * W[n,k]^T, bf16 in and
 * out, fp32 accumulation (src/gpu.rs:535-560). hipBLAS, except for products of
 * at most 32 rows whose n, k and 16-byte aligned x and w one of this library's
 * own kernels serves faster: there the order of the fp32 sums is that kernel's,
 * and two calls of one shape at other alignments may differ by fp32 rounding.
 * Every call repeats its bits. A null operand is refused (-2). */
int nv_gemm(nv_context* c, const void* x, const void* w, void* y, int m, int n, int k);

/* ------------------------------------------------ fused per-layer kernels ---- */

/* kernels/kernels.cu:139-144,469 — out[r,:] = weight[tokens[r],:], or +0 when
 * the token is outside [0, vocab) (src/gpu.rs:561-585). */
int nv_embedding(nv_context* c, const void* tokens, const void* weight, void* out,
                 int rows, int hidden, int vocab);

/* kernels/kernels.cu:145-164,470 — out = RMSNorm(x) * weight (src/gpu.rs:586-611). */
int nv_rms(nv_context* c, const void* x, const void* weight, void* out,
           int rows, int hidden, float eps);

/* kernels/kernels.cu:145-164,471 — v = x + residual (fp32); residual <- bf16(v);
 * out = RMSNorm(v) * weight, normalising the unrounded v (src/gpu.rs:612-642). */
int nv_add_rms(nv_context* c, const void* x, void* residual, const void* weight, void* out,
               int rows, int hidden, float eps);

/* The final add-RMSNorm and the last-token gather of src/model.rs:781-797 in
 * one launch (no single reference entry point: nv_add_rms, kernels/kernels.cu:471,
 * followed by nv_gather, :487). For output row r with i = indices[r] in
 * [0, input_rows): out[r] = nv_add_rms's output row i; other indices give a
 * +0 row. Only gathered rows are computed, and the residual is read, not
 * updated (nothing reads it after the final norm), so rows may repeat.
 * x and residual are [input_rows, hidden], out is [rows, hidden]. */
int nv_add_rms_gather(nv_context* c, const void* x, const void* residual, const void* weight,
                      const void* indices, void* out, int rows, int hidden, int input_rows,
                      float eps);

/* No single counterpart in the reference: nv_rms / nv_add_rms
 * (kernels/kernels.cu:145-164,470-471) followed by nv_gemm (:98-106) on the
 * normalised rows, in one launch for decode-sized batches
 * (src/model.rs:659-678 and :753-770). With residual == NULL, X = RMSNorm(x);
 * otherwise v = x + residual, residual_out <- bf16(v) (a different buffer from
 * residual; may be NULL) and X = RMSNorm(v), both exactly as nv_add_rms.
 * Then y[m, n] = bf16(X W^T) with fp32 accumulation in a fixed order (its own:
 * equal to nv_gemm to fp32 rounding). normed (may be NULL) receives
 * X. Limits (else -2): 1 <= m <= 32, n a multiple of 16, k in {512, 1024, 2048},
 * 16-byte aligned tensors. x, residual, residual_out, normed: [m, k];
 * w: [n, k]; y: [m, n]. */
int nv_rms_gemm(nv_context* c, const void* x, const void* residual, void* residual_out,
                const void* norm_weight, const void* w, void* y, void* normed, int m, int n, int k,
                float eps);

/* nv_gemm for decode-sized batches without hipBLAS (kernels/kernels.cu:98-106's
 * Y[m, n] = X[m, k] W[n, k]^T, bf16 in and out, fp32 accumulation in a fixed
 * order — on MFMA, or with dot2 instructions for outputs narrower than one
 * 16-column tile per CU at m <= 16: equal to nv_gemm to fp32 rounding, the
 * same bits on every launch of a shape). Limits (else -2): 1 <= m <= 32, n a multiple of 16,
 * k in {1024, 2048, 3072, 4096}, 16-byte aligned x and w. */
int nv_gemm_rows(nv_context* c, const void* x, const void* w, void* y, int m, int n, int k);

/* nv_rms_gemm for the gate_up projection with SiLU·up (kernels/kernels.cu:356-365,
 * nv_silu) as its epilogue: no single counterpart in the reference
 * (src/model.rs:753-770). w_tiled is the [2 * intermediate, k] gate_up weight
 * with its rows in tile order — tile t holds gate rows 8t..8t+7, then up rows
 * 8t..8t+7 — and act[m, i] = bf16(silu(gate) * up) of the bf16-rounded GEMM
 * outputs, with nv_silu's arithmetic (the same bits). gate_up (may be NULL)
 * receives the GEMM output in the reference's [m, gate | up] layout.
 * Limits as nv_rms_gemm, and intermediate a multiple of 8. */
int nv_rms_gemm_silu(nv_context* c, const void* x, const void* residual, void* residual_out,
                     const void* norm_weight, const void* w_tiled, void* gate_up, void* act, void* normed,
                     int m, int intermediate, int k, float eps);

/* kernels/kernels.cu:166-211,472 — per-head q/k RMSNorm, NeoX RoPE with the
 * angle computed inline, q -> qout, k/v -> paged caches at slots[r]
 * (src/gpu.rs:661-706). qkv is [rows, qh + 2*kvh, dim]; caches are
 * [blocks, bs, kvh, dim]. */
int nv_qkv_rope(nv_context* c, const void* qkv, const void* qw, const void* kw,
                const void* positions, const void* slots, void* qout, void* kc, void* vc,
                int rows, int qh, int kvh, int dim, int bs, int blocks, float eps, float theta);

/* kernels/kernels.cu:213-224,473 — fp32 table [positions, cos(dim/2) | sin(dim/2)]
 * (src/gpu.rs:753-773). */
int nv_rope_cache(nv_context* c, void* cache, int positions, int dim, float theta);

/* kernels/kernels.cu:166-211,474 — as nv_qkv_rope with cos/sin read from the
 * table; positions outside [0, max_positions) rotate by angle 0
 * (src/gpu.rs:774-825). */
int nv_qkv_rope_cached(nv_context* c, const void* qkv, const void* qw, const void* kw,
                       const void* positions, const void* slots, void* qout, void* kc, void* vc,
                       int rows, int qh, int kvh, int dim, int bs, int blocks, float eps,
                       const void* rope_cache, int max_positions);

/* kernels/kernels.cu:475-485 — causal paged GQA attention over flattened
 * ragged prefill and decode rows (src/gpu.rs:826-887). q, out: [rows, qh, dim]
 * bf16; kc, vc: [blocks, bs, kvh, dim] bf16; positions, seqs: [rows] i32;
 * tables: [batch, stride] i32. Row r attends to positions[r] + 1 keys of
 * sequence seqs[r] in the fp32 order of kernels/kernels.cu:226-346. Returns -2
 * for qh % kvh != 0, an odd head dim or one above 256, or max_context outside
 * [1, 4096]. */
int nv_attention(nv_context* c, const void* q, const void* kc, const void* vc,
                 const void* positions, const void* seqs, const void* tables, void* out,
                 int rows, int qh, int kvh, int dim, int bs, int blocks, int stride, int batch,
                 int max_context);

/* No single counterpart in the reference: nv_qkv_rope_cached followed by
 * nv_attention (kernels/kernels.cu:166-211,474 then 475-485) in one launch for
 * decode batches, with the same outputs (out; K and V at slots[r]) bit for bit
 * and without writing the rotated q to memory. Head dim 128 and 16-byte
 * aligned tensors only (else -2). No row may read a KV slot that another row
 * of the call writes: rows do not wait for each other's cache writes. */
int nv_attention_qkv_rope(nv_context* c, const void* qkv, const void* qw, const void* kw,
                          const void* positions, const void* slots, void* kc, void* vc,
                          const void* seqs, const void* tables, void* out, int rows, int qh, int kvh,
                          int dim, int bs, int blocks, int stride, int batch, int max_context, float eps,
                          const void* rope_cache, int max_positions);

/* kernels/kernels.cu:356-365,486 — out[r,i] = bf16(silu(gate) * up) with
 * packed = [rows, 2, intermediate] (src/gpu.rs:996-1019). */
int nv_silu(nv_context* c, const void* packed, void* out, int rows, int intermediate);

/* kernels/kernels.cu:366-371,487 — out[r,:] = x[indices[r],:], or +0 when the
 * index is outside [0, input_rows) (src/gpu.rs:1020-1043). */
int nv_gather(nv_context* c, const void* x, const void* indices, void* out,
              int rows, int hidden, int input_rows);

/* kernels/kernels.cu:372-407,488 — one token per row: greedy argmax when
 * temps[r] <= 0, else Gumbel-max with SplitMix64 noise keyed by seeds[r]
 * (src/gpu.rs:1045-1072). */
int nv_sample(nv_context* c, const void* logits, const void* temps, const void* seeds, void* out,
              int batch, int vocab);

/* kernels/kernels.cu:409-466,489-501 — same result as nv_sample through a
 * vocabulary-partitioned reduction. partial_scores (f32) and partial_ids (i32)
 * are caller scratch of batch * ceil(vocab / 2048) entries each
 * (src/gpu.rs:1073-1111). */
int nv_sample_parallel(nv_context* c, const void* logits, const void* temps, const void* seeds,
                       void* out, void* partial_scores, void* partial_ids, int batch, int vocab);

/* ------------------------------------------------- additions (no Rust caller) ---- */

/* Standalone paged KV-cache slot write: the K/V half of
 * kernels/kernels.cu:188-190,206-209 without the norm and rotation.
 * k, v are [rows, kvh, dim]; for each row with 0 <= slots[r] < bs*blocks,
 * kc[slots[r]] = k[r] and vc[slots[r]] = v[r] (bit-exact copies); other rows
 * are skipped. Slot derivation follows src/runtime.rs:747-755. */
int nv_kv_write(nv_context* c, const void* k, const void* v, const void* slots, void* kc, void* vc,
                int rows, int kvh, int dim, int bs, int blocks);

/* No counterpart in the reference: nv_sample_parallel without the caller's
 * scratch, for callers that cannot allocate device memory (code under HIP graph
 * capture, tight serving loops, harnesses that forbid hipMalloc). The partials
 * live in a static 1 MiB device array per GPU (131072 entries of f32 score +
 * i32 id), bound at nv_create; it calls no allocator. Returns -2 when
 * batch * ceil(vocab / 2048) exceeds 131072. Every call on one GPU shares that
 * array: calls that overlap on one GPU (two streams or contexts at once) race. */
int nv_sample_parallel_static(nv_context* c, const void* logits, const void* temps, const void* seeds,
                              void* out, int batch, int vocab);

/* Serving with trees of drafted tokens (no counterpart in the reference). A tree
 * has 1 to max_nodes <= 64 nodes, node 0 the sequence's last committed token, the
 * others drafted, each after its parent. Sequence s's nodes are the rows
 * row_starts[s] .. row_starts[s + 1] - 1 (row_starts: [batch + 1] i32) of the step,
 * and node i's K and V lie at position contexts[s] + i of the sequence
 * (contexts: [batch] i32, positions committed before node 0), wherever in the
 * tree it stands. Node i's RoPE position is contexts[s] + its depth. */

/* Bytes of workspace that nv_attention_tree needs for these arguments, the call's
 * own (0: none, and NULL will do); a host function, no device work. A workspace
 * starts at a multiple of 16 bytes (else -2), its contents do not matter before a
 * call and are unspecified after; calls that may overlap need one each. */
int nv_attention_tree_workspace(int rows, int qh, int kvh, int dim, int batch, int max_nodes, int max_context,
                                size_t* bytes);

/* Attention of the trees' nodes over the paged cache. q, out: [rows, qh, dim] bf16;
 * kc, vc: [blocks, bs, kvh, dim] bf16; masks: [rows] u64; tables: [batch, stride]
 * i32. Row (s, i) attends to the positions before contexts[s] and to node j's for
 * each bit j of its mask, its own among them if set. Softmax of q . k / sqrt(dim);
 * sums and statistics of 32 bits or more, finite for any finite V. Rows that see nothing are +0, as are those of
 * sequences with more than max_nodes nodes or more than min(max_context, stride *
 * bs) positions, a negative context, or a score that is not finite at the maximum;
 * positions in blocks outside [0, blocks) are not seen. Rows of no sequence are
 * left as they were. max_context is any positive bound on a sequence's positions
 * (contexts[s] + nodes) and, like max_nodes, sizes the launch. Head dims that are
 * multiples of 8 in blocks of multiples of 16 positions, with q, kc, vc and out at
 * multiples of 16 bytes, take the matrix instructions, with each weight as two bf16
 * (within 2^-15 of it); others a kernel for any layout, many times slower. Returns -2 for
 * qh % kvh != 0, an odd head dim or one above 256, max_nodes outside [1, 64], and
 * sizes past one launch (2^32 threads) or past int32 (rows * qh, batch * kvh). */
int nv_attention_tree(nv_context* c, const void* q, const void* kc, const void* vc, const void* contexts,
                      const void* row_starts, const void* masks, const void* tables, void* out, void* workspace,
                      int rows, int qh, int kvh, int dim, int bs, int blocks, int stride, int batch, int max_nodes,
                      int max_context);

/* Bytes of workspace that nv_verify_tree needs, under the same rules as nv_attention_tree's. */
int nv_verify_tree_workspace(int rows, int batch, int vocab, size_t* bytes);

/* Rejection sampling of the trees' drafted tokens: the path that the target
 * accepts, and the token after it. logits: [rows, vocab] bf16, the target's after
 * each node; draft_logits: the same of the model that drafted, whose distribution
 * at a node its children were drawn from independently, or NULL for children that
 * were picked (the most likely, looked up); tokens, parents: [rows] i32 (parents:
 * node indices below the node's own; node 0's is not read); temps: [batch] f32, <= 0
 * greedy; uniforms: [rows] f32 in [0, 1), one a drafted token; seeds: [batch] u64,
 * the Gumbel noise of the last token as nv_sample's. out_tokens: [batch, max_nodes]
 * i32, the accepted tokens, then the token after them, then -1; out_nodes: [batch,
 * max_nodes] i32, the path's nodes from 0 on, then -1; out_counts: [batch] i32, how
 * many of either (0 for a sequence without rows, or with more than max_nodes, or
 * with rows outside [0, rows)). For temps > 0 the tokens are distributed as the
 * target's samples; for temps <= 0 they are its argmaxes. With nothing rejected at
 * the path's last node, the token after it is nv_sample's for that row. Drafted
 * tokens outside [0, vocab) and nodes whose parent does not come before them are
 * passed over. Returns -2 for max_nodes outside [1, 64], vocab above 2^26, and sizes
 * past one launch (batch above 2^22 - 1, or 2^32 threads over the vocabularies). */
int nv_verify_tree(nv_context* c, const void* logits, const void* draft_logits, const void* tokens,
                   const void* parents, const void* row_starts, const void* temps, const void* uniforms,
                   const void* seeds, void* out_tokens, void* out_nodes, void* out_counts, void* workspace, int rows,
                   int batch, int max_nodes, int vocab);

/* After verification: K and V at position contexts[s] + nodes[s, j] move to contexts[s]
 * + j for j < counts[s], in every layer. nodes ([batch, max_nodes] i32) and counts
 * ([batch] i32) are nv_verify_tree's out_nodes and out_counts; a sequence's nodes
 * must rise from nodes[s, 0] >= 0 (moves stop at the first that does not, or that
 * is not below max_nodes; a count above max_nodes moves nothing). kc, vc: [layers,
 * blocks, bs, kvh, dim] bf16 (layers 1 for a layer by itself). Moves that touch a
 * block outside [0, blocks) or a position past the table are left out; no sequence
 * may read a slot that another writes. */
int nv_kv_compact(nv_context* c, void* kc, void* vc, const void* contexts, const void* nodes, const void* counts,
                  const void* tables, int batch, int max_nodes, int layers, int kvh, int dim, int bs, int blocks,
                  int stride);

/* The first min(tokens[i], bs) slots of block src[i] are copied to block dst[i], in
 * every layer (src, dst, tokens: [copies] i32): the block that a forked sequence
 * and its origin would both write, or any blocks that are to move. Copies of
 * blocks outside [0, blocks) and onto themselves are left out. No block may be
 * written twice, or read and written, by one call. */
int nv_kv_copy_blocks(nv_context* c, void* kc, void* vc, const void* src, const void* dst, const void* tokens,
                      int copies, int layers, int kvh, int dim, int bs, int blocks);

/* Serving with weights in 8-bit integers (no counterpart in the reference, whose
 * projections are bf16). A weight [n, k] is kept as rows of k int8 at multiples of
 * 16 bytes (k rounded up to a multiple of 16 is a row's pitch, and w starts at a
 * multiple of 16 bytes) and a scale (f32) a row, its channel. k is at most 131071,
 * so that sums of products are exact in 32 bits; a longer one is refused (-2).
 *
 * Rows of bf16 as 8-bit integers: x [rows, k] bf16; q [rows, pitch] i8, zeros
 * behind k; scales [rows] f32. With a = max |x_j| of a row, its scale is a / 127 and
 * q_j = 127 x_j / a to the nearest whole number, half to even; 0 where a is 0. A
 * row that holds a NaN or an infinity has a scale of NaN and integers 0. Neither q nor
 * scales overlaps another argument (else -2). */
int nv_quantize_rows(nv_context* c, const void* x, void* q, void* scales, int rows, int k);

/* Bytes of workspace that nv_gemm_i8 needs; a host function, no device work. A
 * workspace starts at a multiple of 16 bytes (else -2), its contents do not matter
 * before a call and are unspecified after; calls that may overlap need one each.
 * Every call takes one, a small one too that makes its tokens without it. */
int nv_gemm_i8_workspace(int m, int n, int k, size_t* bytes);

/* y[m, n] = bf16(sum_l xq[i, l] w[j, l] * xs[i] * w_scales[j]), where xq and xs are
 * the tokens as nv_quantize_rows makes them of
 *   x                            norm_weight NULL (residual and residual_out too),
 *   RMSNorm(x)                   residual NULL (residual_out too),
 *   RMSNorm(x + residual)        with residual_out <- bf16(x + residual), unless NULL;
 * the norm in fp32 (as nv_rms but for roundings, its values not rounded to bf16).
 * x, residual, residual_out: [m, k] bf16; residual_out, y and the workspace overlap
 * neither each other nor any other argument (else -2); norm_weight: [k] bf16;
 * w, w_scales as nv_quantize_rows' q and scales (integers of any source; -128 too);
 * y: [m, n] bf16. Sums of products are exact, so a token's outputs are the same bits
 * in any batch. A token with a NaN or an infinity (or whose product with the norm's
 * weight leaves fp32) has NaN in its row of y, and no other has where the scales are
 * finite: a channel of scale NaN, as nv_quantize_rows makes it of a row with a NaN,
 * is NaN for every token. eps is read with a norm_weight only. Any m and n that one
 * launch holds (2^32 threads; else -2) and any k; tensors of bf16 start at any even
 * address, scales at multiples of 4 bytes. */
int nv_gemm_i8(nv_context* c, const void* x, const void* residual, void* residual_out, const void* norm_weight,
               const void* w, const void* w_scales, void* y, void* workspace, int m, int n, int k, float eps);

int nv_gemm_i8_silu_workspace(int m, int intermediate, int k, size_t* bytes);

/* The gated feed-forward block's first half, both projections and SiLU·up in one
 * product: w is [2 * intermediate, k], the gate's rows, then the up projection's
 * (as a bf16 gate_up weight has them), and act[m, intermediate] =
 * bf16(g / (1 + e^-g) * u) with g and u the products of nv_gemm_i8 before its
 * rounding, in fp32: one past its range is an infinity, and a gate of -inf gives 0
 * for any finite u (an infinity times 0 is NaN). Everything else as nv_gemm_i8. */
int nv_gemm_i8_silu(nv_context* c, const void* x, const void* residual, void* residual_out, const void* norm_weight,
                    const void* w, const void* w_scales, void* act, void* workspace, int m, int intermediate, int k,
                    float eps);

/* Per-row Gumbel seed of src/runtime.rs:780-790 (host function, no device
 * work): mix(mix(base) ^ mix(request_id) ^ mix(generated)). */
uint64_t nv_sampling_seed(uint64_t base, uint64_t request_id, uint64_t generated);

#ifdef __cplusplus
}
#endif

#endif /* NANO_HIP_H */
