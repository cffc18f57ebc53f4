"""The operators on trees of drafted tokens where their numbers reach their types' ends, in each of the attention's
launch shapes, against the definitions in 64 bits (tree_reference.py)."""
import numpy as np
import pytest

import nvr
import tree_reference as ref
from test_gpu_tree import Trees

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
    """As Trees.check, with weights held in more than 16 bits. Off against the formula: a weight by 2^-17 at most
    where it is two bf16 (2^-18 each, and as much in the normaliser), by the exponential's few roundings (2^-18, twice
    likewise) and by its score (dim roundings of the sum of its products' sizes; twice); a sum of N weights or
    products by N roundings, twice; the output by its own."""
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
                part = 2 * 2.0 ** -17 + 2 * score_off + 2 * len(at) * 2.0 ** -24
                bound = p @ vc[at, h // group] / p.sum() * part + 2.0 ** -8 * np.abs(want[a + i, h])
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
