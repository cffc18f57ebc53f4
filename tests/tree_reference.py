"""The operators on trees of drafted tokens, from their definitions, in 64 bits (numpy)."""
import numpy as np

GOLDEN, TOKEN_MIX = 0x9E3779B97F4A7C15, 0xD2B74407B1CE6E93


def attention(q, kc, vc, contexts, row_starts, masks, tables, kvh, bs, blocks, max_nodes, max_context, before):
    """q [rows, qh, dim], kc, vc [blocks * bs, kvh, dim] in float64. Returns the output (rows of no sequence as in
    `before`), and for each element a bound on what fp32 scores and bf16 weights may change: a weight is off by
    half a bf16 step, 2^-8 of itself, and by what its score is off. A score sums dim products, each rounded, so
    it is off by at most dim * 2^-24 of the sum of their sizes, the weight and the normaliser by that much each;
    2^-18 covers the exponential's own few roundings of arguments up to 64. The output's rounding is half a step."""
    rows, qh, dim = q.shape
    out, bound = np.array(before, np.float64), np.zeros((rows, qh, dim))
    stride = tables.shape[1]
    for s, context in enumerate(contexts):
        a, b = int(row_starts[s]), int(row_starts[s + 1])
        if not 0 <= a < b <= rows:
            continue
        n = b - a
        out[a:b], bound[a:b] = 0.0, 0.0
        if n > max_nodes or context < 0 or context + n > min(max_context, stride * bs):
            continue
        pos = np.arange(context + n)
        entry = tables[s][pos // bs]
        mapped = (entry >= 0) & (entry < blocks)
        place = np.where(mapped, entry, 0).astype(np.int64) * bs + pos % bs
        for i in range(n):
            node = pos - context
            bit = (np.uint64(masks[a + i]) >> np.clip(node, 0, 63).astype(np.uint64)) & np.uint64(1)
            at = place[mapped & ((node < 0) | (bit == 1))]
            if not at.size:
                continue
            for h in range(qh):
                k, v = kc[at, h // (qh // kvh)], vc[at, h // (qh // kvh)]
                with np.errstate(invalid="ignore", over="ignore"):
                    score = k @ q[a + i, h] / np.sqrt(dim)
                    if np.isnan(score).any() or not np.isfinite(score.max()):
                        continue
                    p = np.exp(score - score.max())
                    out[a + i, h] = p @ v / p.sum()
                    off = dim * 2.0 ** -24 * (np.abs(k) @ np.abs(q[a + i, h])).max() / np.sqrt(dim)
                    bound[a + i, h] = (p @ np.abs(v) / p.sum() * (2.0 ** -8 + 2 * off + 2.0 ** -18)
                                       + 2.0 ** -8 * np.abs(out[a + i, h]))
    return out, bound


def splitmix(x):
    with np.errstate(over="ignore"):
        x = x + np.uint64(GOLDEN)
        x = (x ^ (x >> np.uint64(30))) * np.uint64(0xBF58476D1CE4E5B9)
        x = (x ^ (x >> np.uint64(27))) * np.uint64(0x94D049BB133111EB)
    return x ^ (x >> np.uint64(31))


def gumbel(seed, vocab):
    with np.errstate(over="ignore"):
        bits = splitmix(np.uint64(seed) ^ (np.arange(vocab, dtype=np.uint64) * np.uint64(TOKEN_MIX))) >> np.uint64(41)
    return -np.log(-np.log((bits.astype(np.float64) + 0.5) * 2.0 ** -23))


def softmax(logits, temperature):
    """Probabilities; NaN logits have none, and a row of nothing has none at all."""
    x = np.where(np.isnan(logits), -np.inf, logits)
    top = x.max()
    if top == -np.inf:
        return np.zeros_like(x)
    with np.errstate(invalid="ignore"):
        w = np.where(x == top, 1.0, np.exp((x - top) / temperature))
    return w / w.sum()


def argmax(scores):
    """The lowest index of the largest score; NaN never wins; 0 where nothing does."""
    ok = ~np.isnan(scores)
    return int(np.flatnonzero(ok & (scores == scores[ok].max()))[0]) if ok.any() else 0


def verify(logits, draft, tokens, parents, row_starts, temps, uniforms, seeds, max_nodes):
    """Per sequence: emitted tokens and the accepted path's nodes."""
    rows, vocab = logits.shape
    answers = []
    for s in range(len(temps)):
        a, b = int(row_starts[s]), int(row_starts[s + 1])
        if not 0 <= a < b <= rows or b - a > max_nodes:
            answers.append(([], []))
            continue
        t, v, path, emitted = float(temps[s]), 0, [0], []
        while True:
            row = logits[a + v]
            children = [i for i in range(v + 1, b - a) if parents[a + i] == v and 0 <= tokens[a + i] < vocab]
            following = None
            if not t > 0:
                following = next((i for i in children if tokens[a + i] == argmax(row)), None)
                rest = None
            elif draft is None:
                p, rest, left, tried = softmax(row, t), softmax(row, t), 1.0, []
                for i in children:
                    x = int(tokens[a + i])
                    if x in tried:
                        continue
                    if p[x] > 0 and float(uniforms[a + i]) * left < p[x]:
                        following = i
                        break
                    left -= p[x]
                    rest[x] = 0.0
                    tried.append(x)
            else:
                p, q, c, z = softmax(row, t), softmax(draft[a + v], t), 0.0, 1.0
                rest = p
                for i in children:
                    x = int(tokens[a + i])
                    if rest[x] > 0 and float(uniforms[a + i]) * z * q[x] < rest[x]:
                        following = i
                        break
                    c += z
                    rest = np.maximum(p - c * q, 0.0)
                    z = rest.sum()
            if following is None:
                break
            emitted.append(int(tokens[a + following]))
            path.append(following)
            v = following
        if rest is None or not rest.any():
            emitted.append(argmax(row))
        else:
            with np.errstate(divide="ignore"):
                emitted.append(argmax(np.log(rest) + gumbel(seeds[s], vocab)))
        answers.append((emitted, path))
    return answers


def compact(cache, contexts, nodes, counts, tables, bs, blocks, max_nodes):
    """cache [layers, blocks * bs, width], changed in place."""
    stride = tables.shape[1]

    def slot(s, pos):
        entry = int(tables[s][pos // bs]) if pos < stride * bs else -1
        return entry * bs + pos % bs if 0 <= entry < blocks else -1

    for s, context in enumerate(contexts):
        if context < 0 or counts[s] > max_nodes:
            continue
        last = -1
        for j in range(int(counts[s])):
            node = int(nodes[s][j])
            if node <= last or node >= max_nodes:
                break
            last = node
            if node != j:
                src, dst = slot(s, int(context) + node), slot(s, int(context) + j)
                if src >= 0 and dst >= 0:
                    cache[:, dst] = cache[:, src]


def random_tree(rng, n, fan):
    """Parents of n nodes, each node's after it: at most `fan` children a node."""
    parents, children = [-1], [0] * n
    for i in range(1, n):
        choices = [j for j in range(i) if children[j] < fan]
        p = choices[min(int(rng.exponential(2.0)), len(choices) - 1)] if fan > 1 else i - 1
        children[p] += 1
        parents.append(p)
    return parents
