"""The operators on trees of drafted tokens (nv_attention_tree, nv_verify_tree, nv_kv_compact, nv_kv_copy_blocks)
on the GPU against their definitions in 64 bits (tree_reference.py)."""
import numpy as np
import pytest

import nvr
import oracle as ora
import tree_reference as ref

pytestmark = pytest.mark.gpu


def put(gpu, array):
    return gpu.upload_array(np.ascontiguousarray(array))


# ---------------------------------------------------------------- attention ----
class Trees:
    """A batch of trees over a paged cache: `sizes` nodes over `contexts` committed positions."""

    def __init__(self, sizes, contexts, qh, kvh, dim, bs, seed, fan=3, pad=0, spread=1.0, spare=1):
        rng = np.random.default_rng(seed)
        self.sizes, self.contexts = sizes, np.array(contexts, np.int32)
        self.qh, self.kvh, self.dim, self.bs, self.batch = qh, kvh, dim, bs, len(sizes)
        self.row_starts = np.concatenate([[0], np.cumsum(sizes)]).astype(np.int32)
        self.rows = int(self.row_starts[-1]) + pad
        need = [-(-(c + n) // bs) if n else 0 for c, n in zip(contexts, sizes)]
        self.stride, self.blocks = max(need + [1]), sum(need) + spare
        ids, at = rng.permutation(self.blocks), 0
        self.tables = np.full((self.batch, self.stride), -1, np.int32)
        for s, n in enumerate(need):
            self.tables[s, :n] = ids[at:at + n]
            at += n
        self.parents = [ref.random_tree(rng, n, fan) if n else [] for n in sizes]
        masks = [nvr.tree_masks(p) for p in self.parents if p] + [np.zeros(pad, np.uint64)]
        self.masks = np.concatenate(masks)
        self.q = ora.normal_bf16((self.rows, qh, dim), seed + 1, 0.0, 2.0 * spread)
        self.kc = ora.normal_bf16((self.blocks * bs, kvh, dim), seed + 2)
        self.vc = ora.normal_bf16((self.blocks * bs, kvh, dim), seed + 3)
        self.max_nodes, self.max_context = max(list(sizes) + [1]), self.stride * bs
        self.out = np.full((self.rows, qh, dim), 0x4049, np.uint16)  # what no row's kernel writes stays

    def upload(self, gpu):
        need = gpu.attention_tree_workspace(self.rows, self.qh, self.kvh, self.dim, self.batch, self.max_nodes,
                                            self.max_context)
        self.buffers = [put(gpu, a) for a in (self.q, self.kc, self.vc, self.contexts, self.row_starts, self.masks,
                                              self.tables, self.out)]
        self.workspace = put(gpu, np.full(max(need, 4), 0xFF, np.uint8))  # NaN wherever it is read unwritten
        return self

    def launch(self, gpu):
        gpu.attention_tree(*self.buffers, self.workspace, self.rows, self.qh, self.kvh, self.dim, self.bs, self.blocks,
                           self.stride, self.batch, self.max_nodes, self.max_context)

    def result(self):
        return self.buffers[7].download(np.uint16, self.out.size).reshape(self.out.shape)

    def check(self, got):
        values = [nvr.bf16_values(a).astype(np.float64) for a in (self.q, self.kc, self.vc, self.out)]
        want, bound = ref.attention(*values[:3], self.contexts, self.row_starts, self.masks, self.tables, self.kvh,
                                    self.bs, self.blocks, self.max_nodes, self.max_context, values[3])
        got = nvr.bf16_values(got).astype(np.float64)
        with np.errstate(invalid="ignore"):
            off = np.abs(got - want)
            bad = ~((off <= bound) | (got == want) | (np.isnan(want) & np.isnan(got)))
        assert not bad.any(), (f"{int(bad.sum())} of {bad.size} elements off; first {np.argwhere(bad)[0]}, worst "
                               f"{np.nanmax(off):.3g}")

    def run(self, gpu):
        self.upload(gpu).launch(gpu)
        got = self.result()
        self.check(got)
        return got


@pytest.mark.parametrize("sizes,contexts,qh,kvh,dim,bs", [
    ([1], [0], 16, 8, 128, 256),                      # the smallest: one token, no context
    ([1], [1], 16, 8, 128, 16),
    ([5], [200], 16, 8, 128, 256),
    ([7], [0], 16, 8, 128, 16),                       # only drafted tokens
    ([64], [63], 16, 8, 128, 16),                     # the largest tree; tiles end inside pages
    ([64], [1], 8, 1, 128, 32),                       # 512 rows a KV head
    ([8, 1, 0, 13, 64, 3], [100, 5, 7, 0, 333, 1030], 16, 8, 128, 16),  # ragged, one without rows
    ([25] * 8, [1000 - 37 * i for i in range(8)], 16, 8, 128, 256),
    ([6, 3], [4090, 2047], 16, 8, 128, 256),
    ([4], [9000], 16, 8, 128, 256),                   # past nv_attention's 4096
    ([33, 9], [500, 64], 32, 4, 64, 16),
    ([17, 30], [129, 300], 12, 6, 80, 32),            # a head dim that is no multiple of 32
    ([5, 21], [77, 190], 8, 4, 256, 16),
    ([9, 2], [70, 31], 6, 2, 96, 16),
    ([3, 12], [40, 77], 4, 4, 10, 16),                # rows of 20 bytes
    ([11], [50], 3, 1, 6, 5),
    ([4, 40], [33, 260], 64, 2, 32, 8),
    ([2], [60], 5, 5, 128, 7),                        # odd block size
    ([50, 7], [333, 95], 16, 8, 128, 48),             # three pages a block
    ([60] * 34, [17 * i % 90 for i in range(34)], 16, 8, 128, 16),  # more pairs than CUs, wide
    ([20, 7], [100, 90], 8, 4, 64, 16),
    ([3], [40], 8, 4, 64, 32),
    ([14, 5], [1000, 129], 16, 8, 128, 16),
    ([16] * 40, [17 * i for i in range(40)], 2, 1, 64, 16),
])
def test_attention_of_trees(gpu, sizes, contexts, qh, kvh, dim, bs):
    Trees(sizes, contexts, qh, kvh, dim, bs, 100 + len(sizes)).run(gpu)


def test_attention_takes_any_masks_and_leaves_padded_rows(gpu):
    """Masks that are no trees, one that leaves a row without a context empty, and one of bits past the tree."""
    t = Trees([9, 6, 3], [70, 0, 0], 16, 8, 128, 16, 200, pad=5)
    rng = np.random.default_rng(201)
    t.masks[:18] = rng.integers(0, 2 ** 63, 18, dtype=np.uint64) * np.uint64(2) + np.uint64(1)
    t.masks[9 + 2] = 0               # no context: sees nothing
    t.masks[15] = ~np.uint64(7)      # only bits past its tree's three nodes
    t.masks[4] = 0                   # sees its context alone
    got = t.run(gpu)
    assert not got[11].any() and not got[15].any()
    assert (got[18:] == 0x4049).all()


@pytest.mark.parametrize("dim", [128, 64, 80, 10])
@pytest.mark.parametrize("poison", [0x7FC0, 0x7F80, 0xFF80])
def test_attention_never_sees_masked_values(gpu, poison, dim):
    """NaN and Inf in K and V of masked nodes, of slots past the tree, of unmapped pages and of other sequences."""
    t = Trees([20, 5, 40], [37, 150, 64], 8, 4, dim, 16, 300, spare=3)
    clean = t.run(gpu)
    used = np.zeros(t.blocks * t.bs, bool)
    for s, (n, c) in enumerate(zip(t.sizes, t.contexts)):
        pos = np.arange(c + n)
        used[t.tables[s][pos // t.bs] * t.bs + pos % t.bs] = True
    t.kc[~used] = poison
    t.vc[~used] = poison
    t.upload(gpu).launch(gpu)
    assert np.array_equal(t.result(), clean)
    # A node that only it and its descendants see.
    seen = t.masks[:20] >> np.uint64(7) & np.uint64(1)
    at = t.tables[0][44 // 16] * 16 + 44 % 16
    for cache in (t.vc, t.kc):
        cache[at] = poison
        t.upload(gpu).launch(gpu)
        assert np.array_equal(t.result()[:20][seen == 0], clean[:20][seen == 0])
        t.check(t.result())


def test_attention_passes_over_unmapped_blocks(gpu):
    """Positions in blocks outside [0, blocks) are not seen, in the context and among the nodes."""
    t = Trees([20, 8], [300, 40], 16, 8, 128, 16, 400)
    t.tables[0, 3], t.tables[0, 7], t.tables[1, 2] = -1, t.blocks, 2 ** 31 - 1
    t.run(gpu)
    t.tables[1, :] = -1  # nothing is mapped
    assert not t.run(gpu)[20:].any()


def test_attention_of_invalid_sequences(gpu):
    """+0 rows for a negative context, too long a sequence or too large a tree; ranges outside the rows are passed
    over, and the other sequences are as they were."""
    t = Trees([4, 5, 6, 7, 3], [30, 20, 10, 0, 50], 16, 8, 128, 16, 500)
    t.contexts[0], t.contexts[1], t.max_nodes = -1, t.stride * t.bs - 4, 6
    got = t.run(gpu)
    assert not got[:9].any() and not got[15:22].any() and got[9:15].any() and got[22:].any()
    t = Trees([4, 5, 6], [30, 20, 10], 16, 8, 128, 16, 501)
    t.max_context = 25
    got = t.run(gpu)
    assert not got[:4].any() and got[4:].any()
    for starts in ([0, 4, 2, 15], [-3, 4, 9, 15], [0, 4, 9, 16], [0, 0, 0, 0], [15, 15, 15, 15]):
        t = Trees([4, 5, 6], [30, 20, 10], 16, 8, 128, 16, 502)
        t.row_starts = np.array(starts, np.int32)
        if starts == [0, 4, 2, 15]:
            t.max_nodes = 5  # rows 2 .. 14 are a tree too large; 2 and 3 belong to two sequences
            t.upload(gpu).launch(gpu)
            got = t.result()
            assert not got[4:].any() and got[:2].any()
        else:
            t.run(gpu)


@pytest.mark.parametrize("what", ["q", "kc", "vc"])
def test_attention_of_infinite_and_nan_operands(gpu, what):
    """As nv_attention: a maximum or sum that is not finite gives +0; an Inf among seen values stays."""
    for value in (0x7F80, 0xFF80, 0x7FC0):
        t = Trees([5], [70], 4, 2, 128, 16, 600)
        if what == "q":
            t.q[2, 1, 9] = value
        else:
            getattr(t, what)[t.tables[0][1] * 16 + 5, 0, 9] = value
        t.upload(gpu).launch(gpu)
        got = nvr.bf16_values(t.result())
        if what == "vc":
            assert not np.isfinite(got[:, :2, 9]).any() and np.isfinite(got[:, 2:]).all()
            assert np.isfinite(np.delete(got, 9, 2)).all()
        elif what == "q":
            assert not got[2, 1].any() and np.isfinite(got).all()
        elif value == 0x7FC0:
            assert not got[:, :2].any() and got[:, 2:].any()
        else:
            assert np.isfinite(got).all()


@pytest.mark.parametrize("dim", [128, 64, 256, 10])
@pytest.mark.parametrize("size", [1e4, 3e8, 5e12, -3e8, -5e12])
def test_attention_of_vast_scores(gpu, dim, size):
    """Scores of up to 2^80, and as far below 0: the positions with the largest one share the weight. The mean of their
    V to the sums' roundings (2^-16 of their magnitudes) and the output's (2^-8 of it)."""
    t = Trees([9, 3], [700, 35], 8, 4, dim, 16, 650)
    q = np.zeros(t.q.shape, np.float32)
    q[..., 0] = abs(size)
    k = nvr.bf16_values(t.kc).copy()
    k[..., 0] = np.where(np.arange(len(k)) % 7 == 3, 1.0, 0.5 if size > 0 else 2.0)[:, None] * size
    t.q, t.kc = nvr.bf16_bits(q), nvr.bf16_bits(k)
    t.upload(gpu).launch(gpu)
    got, v = nvr.bf16_values(t.result()), nvr.bf16_values(t.vc).astype(np.float64)
    for s, (n, c) in enumerate(zip(t.sizes, t.contexts)):
        for i in range(n):
            row = int(t.row_starts[s]) + i
            seen = [p for p in range(c + n) if p < c or int(t.masks[row]) >> (p - c) & 1]
            at = np.array([t.tables[s, p // 16] * 16 + p % 16 for p in seen])
            if (at % 7 == 3).any():
                at = at[at % 7 == 3]
            want = np.repeat(v[at].mean(0), 2, 0)
            bound = 2.0 ** -8 * np.abs(want) + 2.0 ** -16 * np.repeat(np.abs(v[at]).mean(0), 2, 0)
            assert (np.abs(got[row] - want) <= bound).all(), (s, i)


@pytest.mark.parametrize("dim,size", [(128, 3.2e38), (64, 3.2e38), (256, 3.2e38), (10, 3.2e38), (128, 1e-30), (10, 1e-30)])
def test_attention_of_the_largest_and_smallest_values(gpu, dim, size):
    """V of one magnitude, with a sign a head element: the outputs are that, to the weights' sums' roundings (2^-16)
    and the output's (2^-8), however many positions share the weight."""
    t = Trees([9, 3], [2100, 35], 8, 4, dim, 16, 660, spread=0.01)
    signs = np.where(np.arange(dim) % 3 == 0, -size, size)
    t.vc = nvr.bf16_bits(np.broadcast_to(signs, t.vc.shape))
    t.upload(gpu).launch(gpu)
    got, want = nvr.bf16_values(t.result()).astype(np.float64), nvr.bf16_values(t.vc)[0, 0].astype(np.float64)
    assert (np.abs(got - want) <= (2.0 ** -8 + 2.0 ** -16) * np.abs(want)).all()


def test_attention_of_one_node_trees_is_the_decode_attention(gpu):
    """A tree of one node is a decode row: nv_attention's result to both kernels' roundings."""
    t = Trees([1] * 12, [0, 1, 15, 16, 31, 100, 255, 256, 700, 1023, 64, 3], 16, 8, 128, 16, 700)
    got = t.run(gpu)
    out = gpu.alloc(t.out.nbytes)
    gpu.paged_attention(t.buffers[0], t.buffers[1], t.buffers[2], t.buffers[3], put(gpu, np.arange(12, dtype=np.int32)),
                        t.buffers[6], out, 12, 16, 8, 128, 16, t.blocks, t.stride, 12, t.max_context)
    t.check(out.download(np.uint16, t.out.size).reshape(t.out.shape))
    assert got.any()


def test_attention_with_offsets_past_32_bits(gpu):
    """A cache of more than 2^32 elements, whose used blocks lie at both ends."""
    kvh, dim, bs = 8, 128, 256
    blocks = 2 ** 32 // (kvh * dim * bs) + 40
    t = Trees([7, 12], [700, 300], 16, kvh, dim, bs, 800)
    kc, vc = gpu.alloc(blocks * bs * kvh * dim * 2), gpu.alloc(blocks * bs * kvh * dim * 2)
    width, moved = bs * kvh * dim * 2, {}
    for i, b in enumerate(sorted(set(t.tables[t.tables >= 0].tolist()))):
        moved[b] = blocks - 1 - i if i % 2 == 0 else i
        for cache, host in ((kc, t.kc), (vc, t.vc)):
            cache.slice(moved[b] * width, width).upload(host[b * bs:(b + 1) * bs])
    want = t.run(gpu)
    t.buffers[1], t.buffers[2], t.blocks = kc, vc, blocks
    t.buffers[6] = put(gpu, np.vectorize(lambda b: moved.get(b, -1), otypes=[np.int32])(t.tables))
    t.buffers[7].upload(t.out)
    t.launch(gpu)
    assert np.array_equal(t.result(), want)


def test_attention_of_unaligned_operands(gpu):
    """Views that start at any multiple of their element's width."""
    t = Trees([9, 30], [100, 45], 8, 2, 128, 16, 900)
    want = t.run(gpu)
    for i in (0, 1, 2, 7):
        size = t.buffers[i].bytes
        view = gpu.alloc(size + 16).slice(2, size)
        view.upload(t.buffers[i].download(np.uint16, size // 2))
        kept, t.buffers[i] = t.buffers[i], view
        t.buffers[7].upload(t.out)
        t.launch(gpu)
        t.check(t.result())
        t.buffers[i] = kept
    t.buffers[7].upload(t.out)
    t.launch(gpu)
    assert np.array_equal(t.result(), want)


# ------------------------------------------------------------- verification ----
class Drafts:
    """A batch of drafted trees with the target's (and a draft model's) logits after each node."""

    def __init__(self, sizes, vocab, seed, draft, fan=3, temps=(0.7, 0.0, 1.2), pad=0, likely=8):
        rng = np.random.default_rng(seed)
        self.sizes, self.vocab, self.batch = sizes, vocab, len(sizes)
        self.row_starts = np.concatenate([[0], np.cumsum(sizes)]).astype(np.int32)
        self.rows, self.max_nodes = max(1, int(self.row_starts[-1]) + pad), max(list(sizes) + [1])
        parents = [ref.random_tree(rng, n, fan) if n else [] for n in sizes]
        self.parents = np.array([p for t in parents for p in t] + [0] * (self.rows - int(self.row_starts[-1])), np.int32)
        x = rng.normal(size=(self.rows, vocab))
        peaks = rng.integers(0, vocab, (self.rows, min(likely, vocab)))
        # A few tokens share about as much as all the others.
        np.put_along_axis(x, peaks, np.log(vocab) + 0.5 + rng.normal(size=peaks.shape), 1)
        self.logits = nvr.bf16_bits(x)
        self.draft = nvr.bf16_bits(x + rng.normal(size=x.shape) * 0.7) if draft else None
        self.temps = np.array([temps[s % len(temps)] for s in range(self.batch)], np.float32)
        self.uniforms = rng.random(self.rows, dtype=np.float32)
        self.seeds = rng.integers(0, 2 ** 64, self.batch, dtype=np.uint64)
        self.tokens = np.zeros(self.rows, np.int32)
        for s, tree in enumerate(parents):
            rank = [0] * len(tree)
            for i in range(1, len(tree)):
                row = int(self.row_starts[s]) + tree[i]
                if draft:
                    q = ref.softmax(nvr.bf16_values(self.draft[row]).astype(np.float64), max(float(self.temps[s]), 0.5))
                    token = rng.choice(vocab, p=q)
                else:
                    token = peaks[row, rank[tree[i]] % peaks.shape[1]]
                self.tokens[int(self.row_starts[s]) + i] = token
                rank[tree[i]] += 1

    def upload(self, gpu):
        self.inputs = [put(gpu, self.logits), None if self.draft is None else put(gpu, self.draft)]
        self.inputs += [put(gpu, a) for a in (self.tokens, self.parents, self.row_starts, self.temps, self.uniforms,
                                              self.seeds)]
        junk = np.full(self.batch * self.max_nodes, 12345, np.int32)
        self.outputs = [put(gpu, junk), put(gpu, junk), put(gpu, junk[:self.batch])]
        self.workspace = put(gpu, np.full(gpu.verify_tree_workspace(self.rows, self.batch, self.vocab), 0xFF, np.uint8))
        return self

    def launch(self, gpu):
        gpu.verify_tree(*self.inputs, *self.outputs, self.workspace, self.rows, self.batch, self.max_nodes, self.vocab)

    def result(self):
        tokens, nodes = (b.download(np.int32, self.batch * self.max_nodes).reshape(self.batch, -1)
                         for b in self.outputs[:2])
        return tokens, nodes, self.outputs[2].download(np.int32, self.batch)

    def want(self):
        draft = None if self.draft is None else nvr.bf16_values(self.draft).astype(np.float64)
        return ref.verify(nvr.bf16_values(self.logits).astype(np.float64), draft, self.tokens, self.parents,
                          self.row_starts, self.temps, self.uniforms, self.seeds, self.max_nodes)

    def check(self):
        tokens, nodes, counts = self.result()
        for s, (emitted, path) in enumerate(self.want()):
            fill = [-1] * (self.max_nodes - len(emitted))
            assert counts[s] == len(emitted), (s, counts[s], emitted, path)
            assert nodes[s].tolist() == path + fill, s
            assert tokens[s].tolist() == emitted + fill, s
        return counts

    def run(self, gpu):
        self.upload(gpu).launch(gpu)
        return self.check()


@pytest.mark.parametrize("draft", [False, True])
@pytest.mark.parametrize("sizes,vocab,fan", [
    ([1], 1, 1), ([1, 1, 1], 151936, 1), ([5], 151936, 1), ([2, 3, 2], 2, 2), ([6, 1, 0, 9, 13, 25], 2048, 3),
    ([64, 40, 7], 2049, 4), ([8] * 30, 509, 1), ([13] * 12, 50257, 3), ([9, 17, 4], 32000, 4), ([20] * 9, 7, 3),
    ([63, 64], 4096, 2), ([33, 5], 20011, 4), ([3], (1 << 22) + 5, 2),
])
def test_verification_of_trees(gpu, sizes, vocab, fan, draft):
    Drafts(sizes, vocab, 1000 + len(sizes) + vocab % 97, draft, fan).run(gpu)


@pytest.mark.parametrize("draft", [False, True])
@pytest.mark.parametrize("vocab", [1, 2, 3, 4, 5, 6, 7, 8, 9, 15, 16, 17])
def test_verification_over_few_tokens(gpu, vocab, draft):
    """Rows that begin and end inside 16 bytes, at every offset."""
    Drafts([5, 9, 2, 13] * 8, vocab, 1150 + vocab, draft, fan=3, temps=(0.7, 1.0, 0.0, 1.4), likely=2).run(gpu)


@pytest.mark.parametrize("draft", [False, True])
def test_verification_accepts_and_rejects(gpu, draft):
    """Over many sequences every length of path occurs."""
    d = Drafts([6] * 400, 61, 1100, draft, fan=2, temps=(0.7, 1.0, 1.4), likely=3)
    counts = d.run(gpu)
    assert set(range(1, 4)) <= set(counts.tolist())


@pytest.mark.parametrize("draft", [False, True])
def test_verified_tokens_have_the_targets_distribution(gpu, draft):
    """The first emitted token of 20000 sequences with the same logits: each token's share of N is within five
    standard deviations, sqrt(p (1 - p) / N), of its probability (a false alarm in 6 tokens: 4e-6)."""
    n, vocab = 20000, 6
    rng = np.random.default_rng(1200)
    target, drafts = nvr.bf16_bits(rng.normal(size=vocab) * 1.5), nvr.bf16_bits(rng.normal(size=vocab))
    d = Drafts([3] * n, vocab, 1201, draft, fan=2, temps=(0.8,))
    d.logits[:] = target
    d.parents = np.tile(np.array([-1, 0, 0], np.int32), n)
    if draft:
        d.draft[:] = drafts
        q = ref.softmax(nvr.bf16_values(drafts).astype(np.float64), 0.8)
        d.tokens = rng.choice(vocab, size=3 * n, p=q).astype(np.int32)
    else:
        d.tokens = np.tile(np.array([0, 4, 2], np.int32), n)
    d.upload(gpu).launch(gpu)
    first = d.result()[0][:, 0]
    p = ref.softmax(nvr.bf16_values(target).astype(np.float64), 0.8)
    share = np.bincount(first, minlength=vocab) / n
    assert (np.abs(share - p) <= 5 * np.sqrt(p * (1 - p) / n)).all(), (share, p)


def test_one_row_verification_is_the_sampler(gpu):
    """A tree of one node: nv_sample's token, whatever the logits hold."""
    batch, vocab = 24, 5000
    logits = ora.normal_bf16((batch, vocab), 1300, 0.0, 3.0)
    logits[3] = 0xFF80                       # -inf everywhere
    logits[4] = 0x7FC0                       # NaN everywhere
    logits[5, ::2], logits[6, :4000] = 0x7FC0, 0xFF80
    logits[7, 77] = logits[7, 4100] = 0x7F80  # +inf
    logits[8], logits[9] = 0xFF7F, 0x3F80     # the lowest value everywhere; all equal
    logits[10, 5:] = 0xFF7F
    d = Drafts([1] * batch, vocab, 1301, False, temps=(0.6, 0.0, 1.3, -1.0))
    d.logits = logits
    d.upload(gpu).launch(gpu)
    out = gpu.alloc(4 * batch)
    gpu.sample(d.inputs[0], d.inputs[5], d.inputs[7], out, batch, vocab)
    assert d.result()[0][:, 0].tolist() == out.download(np.int32, batch).tolist()


@pytest.mark.parametrize("draft", [False, True])
def test_verification_of_masked_logits(gpu, draft):
    """-inf, the lowest value and NaN among the logits: drafted tokens there are never accepted, nor emitted."""
    d = Drafts([7] * 24, 3000, 1400, draft, fan=3, temps=(0.7, 1.0))
    rng = np.random.default_rng(1401)
    for s in range(24):
        rows = slice(7 * s, 7 * s + 7)
        keep = rng.random(3000) < (0.5, 0.01, 0.002)[s % 3]
        keep[rng.integers(0, 3000)] = True
        d.logits[rows][:, ~keep] = (0xFF80, 0xFF7F, 0x7FC0)[s % 3]
    d.uniforms[::5] = 0.0  # the smallest uniform accepts no token of probability 0
    d.run(gpu)
    tokens, _, counts = d.result()
    for s in range(24):
        assert np.isfinite(nvr.bf16_values(d.logits[7 * s, tokens[s, 0]])) and d.logits[7 * s, tokens[s, 0]] != 0xFF7F


def test_verification_leaves_out_what_was_rejected(gpu):
    """Where the drafted siblings hold all but one token of the vocabulary, a path that ends there ends with that
    one; a token drafted twice is tried once."""
    d = Drafts([5] * 60, 4, 1500, False, fan=4, temps=(1.0,))
    d.logits[:] = nvr.bf16_bits(np.array([0.0, 0.2, -0.3, 0.1]))
    d.parents = np.tile(np.array([-1, 0, 0, 0, 0], np.int32), 60)
    d.tokens = np.tile(np.array([0, 3, 1, 3, 0], np.int32), 60)
    d.run(gpu)
    tokens, nodes, counts = d.result()
    ended = counts == 1
    assert ended.any() and (tokens[ended, 0] == 2).all()
    assert (nodes[~ended, 1] != 3).all()
    d.uniforms[:] = np.nextafter(np.float32(1), np.float32(0))  # rejects whatever can be
    d.run(gpu)


@pytest.mark.parametrize("draft", [False, True])
@pytest.mark.parametrize("mask", [0xFF80, 0xFF7F, 0x7FC0])
def test_verification_of_masks_at_any_level(gpu, draft, mask):
    """Most tokens masked by -inf, the lowest value or NaN, whole stretches among them, the others far below or above
    0, at temperatures at which the lowest value's scaled products round up and down; rows of -inf or NaN alone."""
    rng = np.random.default_rng(1470 + mask)
    d = Drafts([6] * 40, 9001, 1471, draft, fan=3, temps=(0.3, 0.7, 1.0, 1.5, 0.9))
    for s in range(40):
        rows = slice(6 * s, 6 * s + 6)
        keep = rng.random(9001) < (0.3, 0.003)[s % 2]
        keep[:4096 * (s % 3)] = False
        keep[rng.integers(0, 9001, 2)] = True
        level = (0.0, -300.0, 250.0, -500.0)[s % 4]
        for x in ([d.logits] if d.draft is None else [d.logits, d.draft]):
            x[rows] = nvr.bf16_bits(nvr.bf16_values(x[rows]).astype(np.float64) + level)
            x[rows][:, ~keep] = mask
        if s % 8 == 5 and mask != 0xFF7F:
            d.logits[rows] = mask
        allowed = np.flatnonzero(keep)
        d.tokens[rows] = rng.choice(allowed, 6)
    d.run(gpu)


@pytest.mark.parametrize("vocab", [1000, 120011])  # walks in the last launch, and in one of its own
def test_verification_at_extreme_temperatures(gpu, vocab):
    """T infinite: the tokens that are not masked are equally likely. T below the smallest normal number: the largest
    logits share, zeros among them. Two such tokens have 1/2 each, so u decides, and a rejected one leaves the other."""
    cases = [(np.inf, -np.inf, 1.0, 0.4, [3, 5]), (np.inf, -np.inf, 1.0, 0.6, [5]), (np.inf, -np.inf, -2.0, 0.6, [5]),
             (1e-40, -1.0, 0.0, 0.4, [3, 5]), (1e-40, -1.0, 0.0, 0.6, [5]),
             (1e-40, -1.0, 2.0, 0.4, [3, 5]), (1e-40, -1.0, 2.0, 0.6, [5])]
    for draft in (False, True):
        d = Drafts([2] * len(cases), vocab, 1450, draft, fan=1)
        for s, (t, low, high, u, want) in enumerate(cases):
            x = np.full((2, vocab), low)
            x[0, [3, 5]] = high
            x[1, 5] = high
            d.logits[2 * s:2 * s + 2] = nvr.bf16_bits(x)
            if draft:  # every sample is of token 3, which the target accepts with 1/2
                x[:] = low
                x[:, 3] = high
                d.draft[2 * s:2 * s + 2] = nvr.bf16_bits(x)
            d.temps[s], d.uniforms[2 * s + 1], d.tokens[2 * s + 1] = t, u, 3
        d.upload(gpu).launch(gpu)
        tokens, _, counts = d.result()
        for s, case in enumerate(cases):
            assert tokens[s, :counts[s]].tolist() == case[4], (draft, s)


def test_verification_of_invalid_nodes_and_sequences(gpu):
    """Tokens outside the vocabulary, parents that do not come before their node, sequences without rows, with too
    many, or outside the rows: none is followed, and what is not a sequence gives no tokens."""
    for draft in (False, True):
        d = Drafts([6, 6, 0, 6, 9, 6], 300, 1600, draft, fan=2, temps=(0.9, 0.0))
        d.max_nodes = 6
        d.tokens[1], d.tokens[2], d.tokens[8] = -1, 300, 2 ** 31 - 1
        d.parents[3], d.parents[4], d.parents[9], d.parents[15] = 3, 5, -7, 64
        d.run(gpu)
        assert d.result()[2][2] == 0 and d.result()[2][4] == 0
        d.row_starts = np.array([0, 6, 3, 12, -1, 20, 34], np.int32)
        d.run(gpu)


def test_verification_of_invalid_sequences_in_large_calls(gpu):
    """The same where the call has more blocks than a GPU has CUs, so that the walk is a launch of its own."""
    d = Drafts([6, 6, 0, 6, 9, 6], 120011, 1650, False, fan=4, temps=(0.9, 0.0, 1.1))
    d.max_nodes = 6
    d.tokens[1], d.tokens[8], d.parents[9], d.parents[15] = -1, 120011, -7, 64
    d.tokens[20] = d.tokens[19]
    d.uniforms[18:24] = 0.999
    d.run(gpu)
    assert d.result()[2][2] == 0 and d.result()[2][4] == 0
    d.row_starts = np.array([0, 6, 3, 12, -1, 20, 34], np.int32)
    d.run(gpu)


def test_verification_of_unaligned_rows(gpu):
    """Logits whose rows start at every alignment, in a view that starts at any."""
    for draft in (False, True):
        d = Drafts([5, 4], 2047, 1700, draft, fan=2)
        d.upload(gpu)
        for i in range(2 if draft else 1):
            view = gpu.alloc(d.inputs[i].bytes + 16).slice(6, d.inputs[i].bytes)
            view.upload(d.inputs[i].download(np.uint16, d.inputs[i].bytes // 2))
            d.inputs[i] = view
        d.launch(gpu)
        d.check()


@pytest.mark.parametrize("draft", [False, True])
def test_verification_with_offsets_past_32_bits(gpu, draft):
    """Logits of more than 2^32 elements, with a tree at either end (between them a sequence with too many rows)."""
    vocab = (1 << 20) + 3
    d = Drafts([5, 5], vocab, 1800, draft, fan=2, temps=(0.8, 1.1))
    d.run(gpu)
    want = d.result()
    rows = 2 ** 32 // vocab + 20
    place = np.concatenate([np.arange(5), np.arange(rows - 5, rows)])
    for i in range(2 if draft else 1):
        big = gpu.alloc(rows * vocab * 2)
        for row, values in zip(place, (d.logits, d.draft)[i]):
            big.slice(int(row) * vocab * 2, vocab * 2).upload(values)
        d.inputs[i] = big
    for i, a in ((2, d.tokens), (3, d.parents), (6, d.uniforms)):
        wide = np.zeros(rows, a.dtype)
        wide[place] = a
        d.inputs[i] = put(gpu, wide)
    d.inputs[4] = put(gpu, np.array([0, 5, rows - 5, rows], np.int32))
    d.inputs[5], d.inputs[7] = put(gpu, d.temps[[0, 0, 1]]), put(gpu, d.seeds[[0, 0, 1]])
    outputs = [gpu.alloc(3 * 5 * 4), gpu.alloc(3 * 5 * 4), gpu.alloc(12)]
    gpu.verify_tree(*d.inputs, *outputs, gpu.alloc(gpu.verify_tree_workspace(rows, 3, vocab)), rows, 3, 5, vocab)
    got = [b.download(np.int32, n).reshape(3, -1) for b, n in zip(outputs, (15, 15, 3))]
    for a, b in zip(got, want):
        assert np.array_equal(a[[0, 2]].reshape(b.shape), b)
    assert got[2][1] == 0


# -------------------------------------------------------------------- pages ----
@pytest.mark.parametrize("layers,kvh,dim,bs", [(1, 8, 128, 256), (28, 8, 128, 16), (3, 4, 80, 16), (2, 3, 10, 5),
                                               (2, 1, 7, 1), (1, 16, 256, 32)])
def test_compaction_of_paths(gpu, layers, kvh, dim, bs):
    rng = np.random.default_rng(2000 + dim)
    batch, width = 7, 24
    contexts = np.array([0, 1, 15, 16, 33, 60, 100], np.int32)
    need = [-(-(c + width) // bs) for c in contexts]
    stride, blocks = max(need), sum(need) + 2
    ids, at = rng.permutation(blocks), 0
    tables = np.full((batch, stride), -1, np.int32)
    for s, n in enumerate(need):
        tables[s, :n] = ids[at:at + n]
        at += n
    nodes, counts = np.full((batch, width), -1, np.int32), np.zeros(batch, np.int32)
    for s in range(batch):
        counts[s] = (24, 1, 0, 9, 12, 2, 20)[s]
        nodes[s, :counts[s]] = np.sort(rng.choice(width, counts[s], replace=False))
    _compact_both(gpu, layers, kvh, dim, bs, blocks, contexts, nodes, counts, tables)


def _compact_both(gpu, layers, kvh, dim, bs, blocks, contexts, nodes, counts, tables, offset=0):
    batch, width = nodes.shape
    shape = (layers, blocks * bs, kvh * dim)
    rng = np.random.default_rng(2001)
    kc, vc = (rng.integers(0, 2 ** 16, shape, dtype=np.uint16) for _ in range(2))
    buffers = []
    for cache in (kc, vc):
        view = gpu.alloc(cache.nbytes + 16).slice(offset, cache.nbytes)
        view.upload(cache)
        buffers.append(view)
    gpu.kv_compact(*buffers, put(gpu, contexts), put(gpu, nodes), put(gpu, counts), put(gpu, tables), batch, width,
                   layers, kvh, dim, bs, blocks, tables.shape[1])
    for cache, buffer in zip((kc, vc), buffers):
        before = cache.copy()
        ref.compact(cache, contexts, nodes, counts, tables, bs, blocks, width)
        got = buffer.download(np.uint16, cache.size).reshape(shape)
        assert np.array_equal(got, cache)
        if counts.max() > 1 and offset == 0 and not (nodes >= blocks * bs).any():
            assert not np.array_equal(cache, before)


def test_compaction_of_invalid_paths(gpu):
    """Counts and contexts out of range, nodes that do not rise or are too large, unmapped blocks and positions past
    the table: such moves are left out."""
    width, bs, blocks = 8, 4, 40
    tables = np.arange(40, dtype=np.int32).reshape(10, 4)
    contexts = np.array([0, -1, 3, 3, 3, 3, 12, 3, 2 ** 31 - 1, 3], np.int32)
    nodes = np.tile(np.array([1, 3, 4, 6, 7, -1, -1, -1], np.int32), (10, 1))
    counts = np.full(10, 5, np.int32)
    counts[2], counts[3] = -4, 9
    nodes[4, 2] = 3            # does not rise
    nodes[5, 3] = 8            # too large
    nodes[7, 0] = -1
    tables[9, 1], tables[0, 0] = -1, blocks
    _compact_both(gpu, 2, 2, 16, bs, blocks, contexts, nodes, counts, tables)


def test_compaction_of_unaligned_caches(gpu):
    tables = np.arange(12, dtype=np.int32).reshape(2, 6)
    nodes = np.array([[0, 2, 5, 7], [1, 2, 3, 11]], np.int32)
    nodes = np.concatenate([nodes, np.full((2, 8), -1, np.int32)], 1)
    _compact_both(gpu, 2, 2, 64, 4, 12, np.array([5, 9], np.int32), nodes, np.array([4, 4], np.int32), tables, offset=2)


def test_moves_with_offsets_past_32_bits(gpu):
    """Caches of more than 2^32 elements in three layers: moves in the first block and in the last ones."""
    layers, kvh, dim, bs = 3, 8, 128, 16
    width, slots = kvh * dim, 2 ** 32 // (3 * kvh * dim) + 64 * bs
    blocks = slots // bs
    rng = np.random.default_rng(2050)
    used = [0, blocks - 3, blocks - 2, blocks - 1]
    buffers, hosts = [], []
    for _ in range(2):
        cache = gpu.alloc(layers * blocks * bs * width * 2)
        host = rng.integers(0, 2 ** 16, (layers, len(used) * bs, width), dtype=np.uint16)
        for layer in range(layers):
            for i, b in enumerate(used):
                cache.slice((layer * blocks + b) * bs * width * 2, bs * width * 2).upload(host[layer, i * bs:(i + 1) * bs])
        buffers.append(cache)
        hosts.append(host)

    def check():
        for cache, host in zip(buffers, hosts):
            for layer in range(layers):
                for i, b in enumerate(used):
                    got = cache.slice((layer * blocks + b) * bs * width * 2, bs * width * 2).download(np.uint16, bs * width)
                    assert np.array_equal(got, host[layer, i * bs:(i + 1) * bs].reshape(-1)), (layer, b)

    contexts, counts = np.array([2, 9], np.int32), np.array([4, 5], np.int32)
    nodes = np.array([[0, 3, 4, 9, -1], [1, 2, 7, 12, 19]], np.int32)
    nodes = np.concatenate([nodes, np.full((2, 20), -1, np.int32)], 1)
    small = np.array([[0, 2], [1, 3]], np.int32)
    gpu.kv_compact(*buffers, put(gpu, contexts), put(gpu, nodes), put(gpu, counts),
                   put(gpu, np.array(used, np.int32)[small]), 2, 25, layers, kvh, dim, bs, blocks, 2)
    for host in hosts:
        ref.compact(host, contexts, nodes, counts, small, bs, len(used), 25)
    check()
    gpu.kv_copy_blocks(*buffers, *(put(gpu, np.array(a, np.int32)) for a in ([0, blocks - 1], [blocks - 2, blocks - 3], [16, 7])),
                       2, layers, kvh, dim, bs, blocks)
    for host in hosts:
        host[:, 2 * bs:3 * bs] = host[:, :bs]
        host[:, bs:bs + 7] = host[:, 3 * bs:3 * bs + 7]
    check()


@pytest.mark.parametrize("layers,kvh,dim,bs,offset", [(1, 8, 128, 256, 0), (28, 8, 128, 16, 0), (3, 4, 80, 16, 0),
                                                      (2, 3, 10, 5, 0), (2, 1, 7, 1, 0), (2, 8, 64, 16, 2)])
def test_copies_of_blocks(gpu, layers, kvh, dim, bs, offset):
    """Whole and partly filled blocks, one source of several copies; blocks out of range and copies of nothing or
    onto themselves are left out."""
    rng = np.random.default_rng(2100 + dim)
    blocks = 14
    src = np.array([3, 3, 3, 0, 13, -1, 5, 14, 2, 9], np.int32)
    dst = np.array([4, 6, 7, 1, 8, 10, -2, 11, 14, 9], np.int32)
    tokens = np.array([bs, 1, bs - 1, bs + 9, (bs + 1) // 2, bs, bs, bs, bs, bs], np.int32)
    src, dst, tokens = np.append(src, 5), np.append(dst, 12), np.append(tokens, np.int32(-3))
    shape = (layers, blocks, bs, kvh * dim)
    caches = [rng.integers(0, 2 ** 16, shape, dtype=np.uint16) for _ in range(2)]
    buffers = []
    for cache in caches:
        view = gpu.alloc(cache.nbytes + 16).slice(offset, cache.nbytes)
        view.upload(cache)
        buffers.append(view)
    gpu.kv_copy_blocks(*buffers, put(gpu, src.astype(np.int32)), put(gpu, dst.astype(np.int32)),
                       put(gpu, tokens.astype(np.int32)), len(src), layers, kvh, dim, bs, blocks)
    for cache, buffer in zip(caches, buffers):
        want = cache.copy()
        for a, b, n in zip(src, dst, tokens):
            if 0 <= a < blocks and 0 <= b < blocks and a != b and n > 0:
                want[:, b, :n] = cache[:, a, :n]
        assert np.array_equal(buffer.download(np.uint16, cache.size).reshape(shape), want)


# ------------------------------------------------------------------- graphs ----
def test_tree_operators_replay_in_a_graph(gpu):
    """Captured once and replayed with other values in the same buffers, eager work and synchronisations between;
    two graphs share the workspaces."""
    t = Trees([12, 5, 30], [300, 77, 1000], 16, 8, 128, 16, 3000).upload(gpu)
    d = Drafts([12, 5, 30], 3001, 3001, True).upload(gpu)
    t.launch(gpu), d.launch(gpu)
    gpu.sync()
    graphs = [gpu.capture(lambda: (t.launch(gpu), d.launch(gpu))), gpu.capture(lambda: (d.launch(gpu), t.launch(gpu)))]
    for step in range(5):
        t.q = ora.normal_bf16(t.q.shape, 3100 + step, 0.0, 2.0)
        t.contexts = np.array([300 - step * 31, 77 + step, step], np.int32)
        d.logits = ora.normal_bf16(d.logits.shape, 3200 + step, 0.0, 2.0)
        t.buffers[0].upload(t.q), t.buffers[3].upload(t.contexts), d.inputs[0].upload(d.logits)
        graphs[step % 2].replay()
        gpu.sync()
        replayed = t.result()
        t.check(replayed)
        d.check()
        t.buffers[7].upload(t.out)
        t.launch(gpu)
        assert np.array_equal(t.result(), replayed)


def test_contexts_run_at_once(gpu):
    """Two contexts, each with its stream, its buffers and its workspaces: calls of both in flight together give what
    each gives alone."""
    other = nvr.Gpu()
    sides = []
    for i, g in enumerate((gpu, other)):
        t = Trees([25, 9, 33], [2000, 700 + i, 90], 16, 8, 128, 16, 3300 + i).upload(g)
        sides.append((g, t, Drafts([25, 9, 33], 20011, 3310 + i, True).upload(g)))
        g.sync()
    for _ in range(20):
        for g, t, d in sides:
            t.launch(g)
            d.launch(g)
    for g, t, d in sides:
        g.sync()
        t.check(t.result())
        d.check()
        first = t.result()
        t.buffers[7].upload(t.out)
        t.launch(g)
        assert np.array_equal(t.result(), first)


def test_c_entries_refuse_what_does_not_fit(gpu):
    """Workspaces that are missing or unaligned, vocabularies and launches past the limits: the C entries return -2
    before they launch anything, whatever the other arguments."""
    lib, h = gpu.lib, gpu.handle
    tree = lambda work, rows, qh, kvh, batch, nodes, context, dim=128, bs=16: lib.nv_attention_tree(  # noqa: E731
        h, *[None] * 8, work, rows, qh, kvh, dim, bs, 4, 4, batch, nodes, context)
    verify = lambda work, rows, batch, vocab: lib.nv_verify_tree(  # noqa: E731
        h, *[None] * 11, work, rows, batch, 4, vocab)
    some = gpu.alloc(64)
    for status in (tree(None, 25, 16, 8, 1, 25, 4000), tree(some.ptr + 8, 25, 16, 8, 1, 25, 4000),
                   tree(some.ptr, 2 ** 28, 16, 8, 4, 8, 64), tree(some.ptr, 8, 2 ** 16, 2 ** 16, 2 ** 16, 8, 64),
                   tree(some.ptr, 8, 8, 8, 2 ** 22, 8, 64), tree(some.ptr, 8, 8, 8, 2 ** 20, 64, 64, bs=5),
                   verify(None, 8, 2, 100), verify(some.ptr + 8, 8, 2, 100), verify(some.ptr, 8, 2, 2 ** 26 + 1),
                   verify(some.ptr, 8, 2 ** 22, 100), verify(some.ptr, 8, 2 ** 20, 2 ** 20),
                   lib.nv_kv_compact(h, *[None] * 6, 2 ** 24, 4, 1, 8, 128, 16, 4, 4),
                   lib.nv_kv_compact(h, *[None] * 6, 4, 4, 65536, 8, 128, 16, 4, 4),
                   lib.nv_kv_copy_blocks(h, *[None] * 5, 2 ** 20, 28, 8, 128, 16, 4)):
        assert status == -2


# -------------------------------------------------------- a step as a whole ----
class Model:
    """Two decoder layers with random weights, its steps over one paged cache of both layers."""

    H, QH, KVH, D, I, V, BS, BLOCKS, STRIDE, LAYERS = 256, 4, 2, 64, 512, 1000, 16, 40, 8, 2

    def __init__(self, gpu, seed):
        self.gpu = g = gpu
        normal = lambda i, *s: put(g, ora.normal_bf16(s, seed + i, 0.0, s[-1] ** -0.5))  # noqa: E731
        ones = lambda n: put(g, nvr.bf16_bits(np.ones(n, np.float32)))  # noqa: E731
        heads = self.QH + 2 * self.KVH
        self.table = put(g, ora.normal_bf16((self.V, self.H), seed))
        self.head = put(g, ora.normal_bf16((self.V, self.H), seed + 50, 0.0, 3.0 * self.H ** -0.5))
        self.layers = [dict(qkv=normal(10 * i + 1, heads * self.D, self.H), o=normal(10 * i + 2, self.H, self.QH * self.D),
                            gu=normal(10 * i + 3, 2 * self.I, self.H), down=normal(10 * i + 4, self.H, self.I))
                       for i in range(self.LAYERS)]
        self.norm, self.headnorm = ones(self.H), ones(self.D)
        self.rope = g.alloc(512 * self.D * 4)
        g.rope_cache(self.rope, 512, self.D, 1e6)
        self.span = self.BLOCKS * self.BS * self.KVH * self.D * 2
        self.kc, self.vc = g.alloc(self.LAYERS * self.span), g.alloc(self.LAYERS * self.span)

    def forward(self, tokens, positions, slots, attention):
        """Logits [rows, V] of the rows; attention(q, kc, vc, out) runs each layer's."""
        g, n, heads = self.gpu, len(tokens), self.QH + 2 * self.KVH
        new = lambda *s: g.alloc(int(np.prod(s)) * 2)  # noqa: E731
        pos, slot = put(g, np.asarray(positions, np.int32)), put(g, np.asarray(slots, np.int32))
        residual, hidden, normed = new(n, self.H), new(n, self.H), new(n, self.H)
        g.embedding(put(g, np.asarray(tokens, np.int32)), self.table, residual, n, self.H, self.V)
        g.rms_norm(residual, self.norm, normed, n, self.H, 1e-6)
        for i, w in enumerate(self.layers):
            kc, vc = self.kc.slice(i * self.span, self.span), self.vc.slice(i * self.span, self.span)
            qkv, q, out, gu, act = (new(n, heads * self.D), new(n, self.QH * self.D), new(n, self.QH * self.D),
                                    new(n, 2 * self.I), new(n, self.I))
            g.gemm(normed, w["qkv"], qkv, n, heads * self.D, self.H)
            g.qkv_rope_cached(qkv, self.headnorm, self.headnorm, pos, slot, q, kc, vc, n, self.QH, self.KVH, self.D,
                              self.BS, self.BLOCKS, 1e-6, self.rope, 512)
            attention(q, kc, vc, out)
            g.gemm(out, w["o"], hidden, n, self.H, self.QH * self.D)
            g.add_rms_norm(hidden, residual, self.norm, normed, n, self.H, 1e-6)
            g.gemm(normed, w["gu"], gu, n, 2 * self.I, self.H)
            g.silu_mul(gu, act, n, self.I)
            g.gemm(act, w["down"], hidden, n, self.H, self.I)
            g.add_rms_norm(hidden, residual, self.norm, normed, n, self.H, 1e-6)
        logits = new(n, self.V)
        g.gemm(normed, self.head, logits, n, self.V, self.H)
        return logits

    def slots(self, table, positions):
        p = np.asarray(positions)
        return np.asarray(table)[p // self.BS] * self.BS + p % self.BS

    def prefill(self, table, tokens):
        """The logits of every position of one sequence, by nv_attention."""
        g, n = self.gpu, len(tokens)
        pos = np.arange(n, dtype=np.int32)
        ids, tables, at = put(g, np.zeros(n, np.int32)), put(g, np.asarray(table, np.int32)), put(g, pos)
        logits = self.forward(tokens, pos, self.slots(table, pos), lambda q, kc, vc, out: g.paged_attention(
            q, kc, vc, at, ids, tables, out, n, self.QH, self.KVH, self.D, self.BS, self.BLOCKS, self.STRIDE, 1, 128))
        return nvr.bf16_values(logits.download(np.uint16, n * self.V)).reshape(n, self.V)


def test_speculative_decoding_emits_the_greedy_tokens(gpu):
    """Prefill, fork, then steps of drafted trees: attention_tree in each layer, verify_tree, kv_compact. Drafted
    branches hold some of the right tokens and wrong ones. The tokens are those that plain steps of one token by
    nv_attention choose: every emitted token's logit there is the largest to what the two attentions' roundings
    change (2^-8 each of values near 1, over two layers and the head's 256 products: 0.25 of logits near 9)."""
    m = Model(gpu, 4000)
    rng = np.random.default_rng(4001)
    prompt = rng.integers(0, m.V, 21)
    first, second, plain = list(range(0, 8)), list(range(8, 16)), list(range(16, 24))
    m.prefill(first, prompt)
    # The second sequence shares the first's full block and copies the filled part of the next.
    second[0] = first[0]
    args = [put(gpu, np.array([v], np.int32)) for v in (first[1], second[1], 21 - 16)]
    gpu.kv_copy_blocks(m.kc, m.vc, *args, 1, m.LAYERS, m.KVH, m.D, m.BS, m.BLOCKS)
    tables = np.array([first, second], np.int32)
    texts = [list(prompt) + [int(rng.integers(0, m.V))] for _ in range(2)]  # each goes on with a token of its own
    contexts, emitted = [21, 21], [0, 0]
    start = [len(t) for t in texts]
    lengths = set()
    for step in range(6):
        trees, tokens, depth = [], [], []
        for s, text in enumerate(texts):
            right = list(text)
            for _ in range(step % 4):  # the tokens that follow, as a good draft would have them
                right.append(int(m.prefill(plain, right)[-1].argmax()))
            right = right[len(text):]
            parents, mine, level = [-1], [text[-1]], [0]
            at = 0
            for k, token in enumerate(right):
                for wrong in range(1 + s):
                    parents.append(at), mine.append(int(rng.integers(0, m.V))), level.append(k + 1)
                parents.append(at), mine.append(token), level.append(k + 1)
                at = len(parents) - 1
            parents.append(at), mine.append(int(rng.integers(0, m.V))), level.append(level[at] + 1)
            trees.append(parents), tokens.append(mine), depth.append(level)
        sizes = [len(t) for t in trees]
        starts, rows, width = np.concatenate([[0], np.cumsum(sizes)]).astype(np.int32), sum(sizes), max(sizes)
        cb, sb, tb = (put(gpu, np.asarray(a, np.int32)) for a in (contexts, starts, tables))
        masks = put(gpu, np.concatenate([nvr.tree_masks(t) for t in trees]))
        positions = np.concatenate([c + np.array(l) for c, l in zip(contexts, depth)])
        slots = np.concatenate([m.slots(tables[s], contexts[s] + np.arange(sizes[s])) for s in range(2)])
        work = gpu.alloc(max(1, gpu.attention_tree_workspace(rows, m.QH, m.KVH, m.D, 2, width, 128)))
        logits = m.forward(np.concatenate(tokens), positions, slots, lambda q, kc, vc, out: gpu.attention_tree(
            q, kc, vc, cb, sb, masks, tb, out, work, rows, m.QH, m.KVH, m.D, m.BS, m.BLOCKS, m.STRIDE, 2, width, 128))
        outs = [gpu.alloc(8 * width), gpu.alloc(8 * width), gpu.alloc(8)]
        scratch = gpu.alloc(gpu.verify_tree_workspace(rows, 2, m.V))
        gpu.verify_tree(logits, None, put(gpu, np.concatenate(tokens).astype(np.int32)),
                        put(gpu, np.concatenate(trees).astype(np.int32)), sb, put(gpu, np.zeros(2, np.float32)),
                        put(gpu, np.zeros(rows, np.float32)), put(gpu, np.zeros(2, np.uint64)), *outs, scratch, rows, 2,
                        width, m.V)
        gpu.kv_compact(m.kc, m.vc, cb, outs[1], outs[2], tb, 2, width, m.LAYERS, m.KVH, m.D, m.BS, m.BLOCKS, m.STRIDE)
        counts = outs[2].download(np.int32, 2)
        got = outs[0].download(np.int32, 2 * width).reshape(2, width)
        for s in range(2):
            texts[s] += got[s, :counts[s]].tolist()
            contexts[s] += int(counts[s])
            emitted[s] += int(counts[s])
            lengths.add(int(counts[s]))
    assert max(lengths) >= 3 and min(emitted) >= 9
    for s in range(2):
        want = m.prefill(plain, texts[s][:-1])
        for i in range(start[s], len(texts[s])):
            assert want[i - 1].max() - want[i - 1][texts[s][i]] <= 0.25, (s, i)
        # The first layer's K and V of every committed position, moved or not, are those of plain steps.
        at, mine = m.slots(plain, np.arange(contexts[s])), m.slots(tables[s], np.arange(contexts[s]))
        for cache in (m.kc, m.vc):
            rows = nvr.bf16_values(cache.download(np.uint16, m.span // 2)).reshape(-1, m.KVH * m.D)
            # One rounding of K or V, and of the normalised row and the rotation before it, a side.
            assert np.abs(rows[mine] - rows[at]).max() <= 2.0 ** -6 * np.abs(rows[at]).max()
