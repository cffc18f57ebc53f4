"""The operators on trees of drafted tokens where their numbers reach their types' ends, in each of the attention's
launch shapes, against the definitions in 64 bits (tree_reference.py)."""
import numpy as np
import pytest

import nvr
import tree_reference as ref
from test_gpu_tree import Drafts, Trees

pytestmark = pytest.mark.gpu

# Nodes a tree, q heads, KV heads, head dim: one of each launch shape of the tile form (by head dim, query rows a KV
# head and, at 128, (sequence, KV head) pairs), a head dim between two shapes, and the form for any layout.
SHAPES = {
    "128, 16 rows": ([8, 3], 16, 8, 128), "128, 32 rows": ([16, 5], 16, 8, 128), "128, 64 rows": ([30, 9], 16, 8, 128),
    "128, 100 rows": ([50, 20], 16, 8, 128), "128, 80 rows, 272 pairs": ([40, 3] + [2] * 32, 16, 8, 128),
    "64, 16 rows": ([2, 1], 32, 4, 64), "64, 32 rows": ([4, 3], 32, 4, 64), "64, 64 rows": ([8, 5], 32, 4, 64),
    "64, 264 rows": ([33, 9], 32, 4, 64), "256, 32 rows": ([16, 5], 8, 4, 256), "256, 42 rows": ([17, 21], 8, 4, 256),
    "80, 46 rows": ([23, 6], 12, 6, 80), "10, any layout": ([9, 4], 8, 4, 10),
}
each_shape = pytest.mark.parametrize("shape", SHAPES)


def trees(shape, first, second, seed, **more):
    """Trees of one shape, the first two over `first` and `second` committed positions, others over few."""
    sizes, qh, kvh, dim = SHAPES[shape]
    contexts = [first, second] + [7 + 3 * s for s in range(len(sizes) - 2)]
    return Trees(sizes, contexts, qh, kvh, dim, 16, seed, **more)


def values(bits):
    return nvr.bf16_values(bits).astype(np.float64)


def check_tightly(t, got):
    """As Trees.check, with weights held in more than 16 bits. Off against the formula: a weight by 2^-15 where
    it is two bf16 (the upper half leaves up to 2^-7 of it, which rounds by 2^-8 of that), by the exponential's few
    roundings (2^-18, and as much in the normaliser) and by its score (dim roundings of the sum of its products' sizes;
    twice); a sum of N weights or products by N roundings, twice; the output by its own, which is 2^-134 where it is subnormal: bf16's last bit is
    2^-133 there. Sums of subnormal products round by 2^-150, once in 32 positions, at weights of 2^-13 for the largest:
    2^-137 of the output."""
    with np.errstate(all="ignore"):
        want, _ = ref.attention(values(t.q), values(t.kc), values(t.vc), t.contexts, t.row_starts, t.masks, t.tables,
                                t.kvh, t.bs, t.blocks, t.max_nodes, t.max_context, values(t.out))
    off = np.abs(values(got) - want)
    group = t.qh // t.kvh
    q, kc, vc = values(t.q), values(t.kc), np.abs(values(t.vc))
    for s, context in enumerate(t.contexts.tolist()):
        a, n = int(t.row_starts[s]), t.sizes[s]
        for i in range(n):
            seen = [p for p in range(context + n) if p < context or int(t.masks[a + i]) >> (p - context) & 1]
            at = np.array([t.tables[s, p // t.bs] * t.bs + p % t.bs for p in seen])
            for h in range(t.qh):
                k = kc[at, h // group]
                score = k @ q[a + i, h] / np.sqrt(t.dim)
                p = np.exp(score - score.max())
                score_off = t.dim * 2.0 ** -24 * (np.abs(k) @ np.abs(q[a + i, h])).max() / np.sqrt(t.dim)
                part = 2.0 ** -15 + 2 * 2.0 ** -18 + 2 * score_off + 2 * len(at) * 2.0 ** -24
                bound = p @ vc[at, h // group] / p.sum() * part + 2.0 ** -8 * np.abs(want[a + i, h]) + 2.0 ** -134 + -(-len(at) // 32) * 2.0 ** -137
                assert (off[a + i, h] <= bound).all(), (s, i, h, float((off[a + i, h] / bound).max()))


@each_shape
def test_attention_holds_its_weights(gpu, shape):
    """Values of both signs, whose weighted sums nearly cancel here and there: what is off is what a weight of 16 bits
    may be off, not one of eight. The longer sequence lies in several blocks' parts."""
    t = trees(shape, 150, 600, 5000)
    t.upload(gpu).launch(gpu)
    check_tightly(t, t.result())


def constant_values(t, gpu, size):
    """The outputs for V of one size, with a sign a head element, and what they are: that, however many positions share
    the weight, to the roundings of two sums of up to 2^12 weights (2^-12 each) and the output's."""
    signs = np.where(np.arange(t.dim) % 3 == 0, -size, size)
    t.vc = nvr.bf16_bits(np.broadcast_to(signs, t.vc.shape))
    t.upload(gpu).launch(gpu)
    want = values(t.vc)[0, 0]
    return values(t.result()), want, (2.0 ** -8 + 2 * 2.0 ** -12) * np.abs(want)


@pytest.mark.parametrize("dim", [128, 64, 256, 10])
@pytest.mark.parametrize("level", [22.7, 24.4, 25.3, 25.9, 26.6, 27.2, 27.8, 28.5, 29.9])
def test_attention_of_the_largest_values_under_vast_scores(gpu, dim, level):
    """All scores alike, 2^level as powers of two, where a maximum's own rounding is whole powers of two: the weights
    are of a score's distance from it, and the largest V's sums stay finite."""
    t = Trees([9, 3], [2100, 35], 8, 4, dim, 16, 5100, spread=0.01)
    size = np.sqrt(2.0 ** level * np.sqrt(dim) / np.log2(np.e))
    for x in (t.q, t.kc):
        x[:] = 0
        x[..., 0] = nvr.bf16_bits(np.array([size]))[0]
    got, want, bound = constant_values(t, gpu, 3.2e38)
    assert (np.abs(got - want) <= bound).all()


@each_shape
@pytest.mark.parametrize("size", [1e-38, 3e-38, 1e-36, 1e-20, 1e20, 1e30, 3.3e38])
def test_attention_of_values_of_any_size(gpu, shape, size):
    """V of one size, from the smallest normal numbers to the largest, its weight spread over 700 positions."""
    t = trees(shape, 700, 150, 5200, spread=0.01)
    got, want, bound = constant_values(t, gpu, size)
    assert (np.abs(got - want) <= bound).all()


@each_shape
@pytest.mark.parametrize("size", [1e-37, 1e37])
def test_attention_holds_values_of_any_size(gpu, shape, size):
    """Values of both signs near either end of the type: as exact as those near 1."""
    t = trees(shape, 600, 150, 5300)
    t.vc = nvr.bf16_bits(values(t.vc) * size)
    t.upload(gpu).launch(gpu)
    check_tightly(t, t.result())


@pytest.mark.parametrize("dim", [128, 64, 256, 80, 10])
def test_attention_of_small_values_beside_large_ones(gpu, dim):
    """Head elements of the largest V, of the smallest and of subnormals in one head: each is as exact as by itself. A
    subnormal output is off by half its last bit, 2^-134."""
    t = Trees([9, 3], [2100, 35], 8, 4, dim, 16, 5400, spread=0.01)
    sizes = np.resize(np.array([3.2e38, 1e-38, 1.0, -4e-39, -3.2e38, 2e-40]), dim)
    t.vc = nvr.bf16_bits(np.broadcast_to(sizes, t.vc.shape))
    t.upload(gpu).launch(gpu)
    got, want = values(t.result()), values(t.vc)[0, 0]
    assert (np.abs(got - want) <= (2.0 ** -8 + 2 * 2.0 ** -12) * np.abs(want) + 2.0 ** -134).all()


@pytest.mark.parametrize("dim,bs", [(64, 256), (128, 256), (256, 64), (64, 7)])
def test_attention_of_the_largest_values_at_many_positions(gpu, dim, bs):
    """More than 2^17 positions that share the weight: two sums of n weights are off by n roundings each at most, which
    is 2^-5.9 for the 137000 of them."""
    positions = 137000
    t = Trees([4], [positions], 1, 1, dim, bs, 5500, spread=0.01)
    t.vc = nvr.bf16_bits(np.broadcast_to(np.where(np.arange(dim) % 3 == 0, -3.2e38, 3.2e38), t.vc.shape))
    t.upload(gpu).launch(gpu)
    got, want = values(t.result()), values(t.vc)[0, 0]
    bound = (2.0 ** -8 + 2 * positions * 2.0 ** -24) * np.abs(want)
    assert (np.abs(got - want) <= bound).all()


@each_shape
@pytest.mark.parametrize("value", [0x7F80, 0xFF80, 0x7FC0])
def test_attention_of_infinite_values_in_the_context(gpu, shape, value):
    """An Inf or NaN in V at a committed position stays in its head element of every row of its KV head, and changes no
    other."""
    t = trees(shape, 300, 700, 5600)
    clean = t.run(gpu)
    group = t.qh // t.kvh
    t.vc[t.tables[0][100 // 16] * 16 + 100 % 16, 1 % t.kvh, 5] = value
    t.upload(gpu).launch(gpu)
    got, heads = t.result(), slice(1 % t.kvh * group, (1 % t.kvh + 1) * group)
    assert not np.isfinite(values(got[:t.sizes[0], heads, 5])).any()
    got[:t.sizes[0], heads, 5] = clean[:t.sizes[0], heads, 5]
    assert np.array_equal(got, clean)


@pytest.mark.parametrize("masked", [False, True])
def test_verification_sums_large_vocabularies(gpu, masked):
    """Rows of about a million equal logits (with `masked`, every other one a NaN), each summed by one block: drafted
    tokens of probability 1 / n are accepted by a uniform 3e-6 below that and rejected by one 3e-6 above it. The sum is
    within 1e-6: additions of eight exponentials and their own roundings (2^-21), the parts' to fp32 (2^-23)."""
    batch, nodes, vocab = 20, 64, 1_000_003
    rng = np.random.default_rng(6000)
    levels = nvr.bf16_bits(rng.normal(size=batch * nodes) * 3.0)
    logits = gpu.alloc(batch * nodes * vocab * 2)
    row = np.empty(vocab, np.uint16)
    for i, level in enumerate(levels):
        row[:] = level
        if masked:
            row[1::2] = 0x7FC0
        logits.slice(i * vocab * 2, vocab * 2).upload(row)
    p = 1.0 / (vocab - vocab // 2 if masked else vocab)
    uniforms = np.full((batch, nodes), p * (1 - 3e-6), np.float32)
    ends = rng.integers(1, nodes, batch)  # the node that is rejected
    uniforms[np.arange(batch), ends] = p * (1 + 3e-6)
    tokens = (2 * rng.integers(0, vocab // 2, batch * nodes)).astype(np.int32)
    inputs = [gpu.upload_array(a) for a in (
        tokens, np.tile(np.arange(-1, nodes - 1, dtype=np.int32), batch), np.arange(batch + 1, dtype=np.int32) * nodes,
        rng.uniform(0.5, 1.5, batch).astype(np.float32), uniforms, rng.integers(0, 2 ** 64, batch, dtype=np.uint64))]
    outputs = [gpu.alloc(batch * nodes * 4), gpu.alloc(batch * nodes * 4), gpu.alloc(batch * 4)]
    gpu.verify_tree(logits, None, *inputs, *outputs, gpu.alloc(gpu.verify_tree_workspace(batch * nodes, batch, vocab)),
                    batch * nodes, batch, nodes, vocab)
    assert outputs[2].download(np.int32, batch).tolist() == ends.tolist()


@pytest.mark.parametrize("draft", [False, True])
@pytest.mark.parametrize("vocab", [9001, 50257])
def test_verification_of_what_one_token_leaves(gpu, vocab, draft):
    """One token has all but 1e-5 (picked) or 1e-9 (drawn) of both models' probabilities, somewhere in the row, and the
    drafted ones are others, but the first of the picked ones it: what is left of 1 and the rest's sum are differences
    of numbers near 1, and the path and its last token those of the 64-bit walk all the same."""
    d = Drafts([4] * 150, vocab, 6100 + vocab % 7, draft, fan=3, temps=(0.3, 0.7, 1.0))
    rng = np.random.default_rng(6101)
    d.parents = np.tile(np.array([-1, 0, 0, 0], np.int32), 150)
    scale = np.repeat(np.resize(np.array([0.3, 0.7, 1.0]), 150), 4)[:, None]
    x = rng.normal(size=(600, vocab)) * scale  # a mass of about vocab * exp(1/2) without the one token
    at = rng.integers(0, vocab, 600)
    high = np.log(vocab) + 0.5 + (9 if draft else 5) * np.log(10)
    for logits in [d.logits] + ([d.draft] if draft else []):
        y = x if logits is d.logits else x + 0.5 * rng.normal(size=x.shape) * scale
        y[np.arange(600), at] = (high + 0.3 * rng.normal(size=600)) * scale[:, 0]
        logits[:] = nvr.bf16_bits(y)
    d.tokens = rng.integers(0, vocab, 600).astype(np.int32)
    d.uniforms = rng.random(600, dtype=np.float32)
    if not draft:
        d.tokens[1::4] = at[0::4]
        d.uniforms[1::4] = np.nextafter(np.float32(1), np.float32(0))
    counts = d.run(gpu)
    assert (d.result()[0][counts == 1, 0] != at[0::4][counts == 1]).any()


@pytest.mark.parametrize("vocab", [30011, 120011])  # walks in the last launch, and in one of its own
def test_greedy_verification_of_rows_without_numbers(gpu, vocab):
    """Rows of NaN and some -inf: their argmax is the first -inf, wherever it lies; of NaN alone, token 0."""
    d = Drafts([3] * 6, vocab, 6200, False, fan=1, temps=(0.0,))
    d.logits[:] = 0x7FC0
    firsts = [6000, vocab - 1, 4100, 0, 20007, None]
    for s, first in enumerate(firsts):
        if first is not None:
            d.logits[3 * s:3 * s + 3, [first, min(first + 4000, vocab - 1)]] = 0xFF80
        d.tokens[3 * s + 1:3 * s + 3] = first or 0
    d.run(gpu)
    tokens, _, counts = d.result()
    assert (counts == 3).all() and tokens.tolist() == [[first or 0] * 3 for first in firsts]


@each_shape
@pytest.mark.parametrize("poison", [0x7FC0, 0x7F80, 0xFF80])
def test_attention_never_sees_masked_values_in_any_shape(gpu, shape, poison):
    """NaN and Inf in K and V of slots past the trees, of no sequence and of unmapped blocks change nothing; in K or V
    of a node, a context's position of one sequence and a block's last slot, only rows that see them."""
    t = trees(shape, 70, 333, 5700, spare=3)
    clean = t.run(gpu)
    used = np.zeros(t.blocks * t.bs, bool)
    for s, (n, c) in enumerate(zip(t.sizes, t.contexts.tolist())):
        pos = np.arange(c + n)
        used[t.tables[s][pos // t.bs] * t.bs + pos % t.bs] = True
    t.kc[~used] = poison
    t.vc[~used] = poison
    t.upload(gpu).launch(gpu)
    assert np.array_equal(t.result(), clean)
    first = t.sizes[0]
    for position in {70 + first // 2, 70 + first - 1, 69, 15}:  # a node in the middle, the last, the context's last, one more
        node = position - 70
        sees = np.ones(first, bool) if node < 0 else (t.masks[:first] >> np.uint64(node) & np.uint64(1)) != 0
        at = t.tables[0][position // 16] * 16 + position % 16
        for cache in (t.vc, t.kc):
            kept = cache[at].copy()
            cache[at] = poison
            t.upload(gpu).launch(gpu)
            got = t.result()
            assert np.array_equal(got[:first][~sees], clean[:first][~sees])
            assert np.array_equal(got[first:], clean[first:])
            t.check(got)
            cache[at] = kept


@each_shape
def test_attention_passes_over_unmapped_blocks_in_any_shape(gpu, shape):
    """Holes in tiles of the context that every row would see whole, in the tile where the nodes begin and among the
    nodes; a sequence with no block at all."""
    t = trees(shape, 300, 700, 5800)
    holes = [(0, 3, -1), (0, 7, t.blocks), (1, 0, 2 ** 31 - 1), (1, 21, -1), (1, 22, -2 ** 31), (0, 300 // 16, -1)]
    for s, entry, value in holes:
        t.tables[s, entry] = value
    t.run(gpu)
    at = np.where((t.tables[1] >= 0) & (t.tables[1] < t.blocks))[0]
    unseen = np.ones(t.blocks, bool)
    for s in range(t.batch):
        unseen[t.tables[s][(t.tables[s] >= 0) & (t.tables[s] < t.blocks)]] = False
    assert len(at) and unseen.any()
    clean = t.result()
    for cache in (t.kc, t.vc):  # block 0 is read in a hole's place
        cache.reshape(t.blocks, -1)[unseen] = 0x7FC0
    t.upload(gpu).launch(gpu)
    assert np.array_equal(t.result(), clean)
    t.tables[1, :] = -1
    n = t.sizes[0]
    assert not t.run(gpu)[n:n + t.sizes[1]].any()


@each_shape
@pytest.mark.parametrize("size", [1e4, 3e8, -3e8, 5e12, -5e12])
def test_attention_of_vast_scores_in_any_shape(gpu, shape, size):
    """Scores of up to 2^80, and as far below 0, in chains: the positions with the largest one share the weight. The
    mean of their V to the sums' roundings (2^-13 of their magnitudes for up to 400) and the output's."""
    t = trees(shape, 700, 35, 5900, fan=1)
    q, k = np.zeros(t.q.shape, np.float32), nvr.bf16_values(t.kc).copy()
    q[..., 0] = abs(size)
    best = np.arange(len(k)) % 7 == 3
    k[..., 0] = np.where(best, 1.0, 0.5 if size > 0 else 2.0)[:, None] * size
    t.q, t.kc = nvr.bf16_bits(q), nvr.bf16_bits(k)
    t.upload(gpu).launch(gpu)
    got, v = values(t.result()), values(t.vc)
    for s, (n, c) in enumerate(zip(t.sizes, t.contexts.tolist())):
        for i in range(n):
            pos = np.arange(c + i + 1)
            at = t.tables[s, pos // 16] * 16 + pos % 16
            at = at[best[at]] if best[at].any() else at
            want = np.repeat(v[at].mean(0), t.qh // t.kvh, 0)
            bound = 2.0 ** -8 * np.abs(want) + 2.0 ** -13 * np.repeat(np.abs(v[at]).mean(0), t.qh // t.kvh, 0)
            assert (np.abs(got[t.row_starts[s] + i] - want) <= bound).all(), (s, i)


@pytest.mark.parametrize("dim", [64, 128])
def test_attention_of_a_late_key_after_many_positions(gpu, dim):
    """137000 positions that share the weight, V 0, in long parts (64 sequences over the same blocks), then a key whose
    score is 2^60 of theirs, with the smallest V: the outputs are that V, to the roundings of its products (2^-137) and
    the output's."""
    t = Trees([2], [137000], 8, 4, dim, 256, 6300)
    last = t.tables[0][137000 // 256] * 256 + 137000 % 256
    q, k = np.zeros(t.q.shape), np.zeros(t.kc.shape)
    q[..., 0], k[last, :, 0] = 1.0, 60 / np.log2(np.e) * np.sqrt(dim)
    t.q, t.kc = nvr.bf16_bits(q), nvr.bf16_bits(k)
    t.vc[:] = 0
    t.vc[last] = nvr.bf16_bits(np.resize(np.array([1.2e-38, -2e-38, 5e-38]), dim))
    t.batch, t.rows, t.row_starts = 64, 128, 2 * np.arange(65, dtype=np.int32)
    t.tables, t.contexts, t.masks = np.tile(t.tables, (64, 1)), np.tile(t.contexts, 64), np.tile(t.masks, 64)
    t.q, t.out = np.tile(t.q, (64, 1, 1)), np.tile(t.out, (64, 1, 1))
    t.upload(gpu).launch(gpu)
    got, want = values(t.result()), values(t.vc[last])[0]
    assert (np.abs(got - want) <= 2.0 ** -8 * np.abs(want) + 2.0 ** -136).all()
