"""Serving with drafted token trees: what one verification step calls beside the model's layers.

A step takes every sequence's tree of drafted tokens (node 0 is its last committed token) through the model at
once. Each layer's attention reads the paged cache and, among the drafted tokens, each node's ancestors
(attention_tree). The logits of all nodes decide which path is accepted and which token follows it (verify_tree).
The accepted nodes' K and V then move to the positions that they have in the sequence (kv_compact). Sequences that
share a prompt are forked by copying the block that they will both write (kv_copy_blocks).

Shapes are those of the runner (host/model.cpp): 16 q heads over 8 KV heads of 128, vocabulary 151936, 28 layers,
blocks of 256 slots; and generic ones beside them. Caches, queries and logits are random. Queries have twice the
spread of keys, so that the softmax has some heavy keys. Logits are unit normal with eight tokens a row that share
most of the probability, as a language model's are; drafted tokens are mostly among those.

The plain forms are torch on torch tensors. With `own`, inputs lie in the library's buffers (it takes no others).
"""
import math
import os
import random
import sys

import numpy as np
import torch

own = False

QH, KVH, D, V, LAYERS, BS = 16, 8, 128, 151936, 28, 256
LIKELY = 8  # tokens a row of logits that share most of its probability

_gpu = None


def gpu():
    global _gpu
    if _gpu is None:
        path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "nano-vllm-rs_amd")
        if path not in sys.path:
            sys.path.insert(0, path)
        import nvr

        torch.cuda.init()
        _gpu = nvr.Gpu(0)
    return _gpu


# ------------------------------------------------------------------- cases --
def listed():
    return [
        # One user, a short chain found by lookup in the prompt: launches and latency are all there is.
        {"name": "attn_chain_1x4", "kind": "attn", "seqs": 1, "nodes": 4, "fan": 1, "context": 180, "qh": QH,
         "kvh": KVH, "dim": D, "bs": BS},
        # A serving batch with trees of a draft head, a thousand tokens in.
        {"name": "attn_tree_8x25", "kind": "attn", "seqs": 8, "nodes": 25, "fan": 4, "context": 1030, "qh": QH,
         "kvh": KVH, "dim": D, "bs": BS},
        # Few sequences with long contexts and the largest trees: most products a byte.
        {"name": "attn_tree_4x64", "kind": "attn", "seqs": 4, "nodes": 64, "fan": 4, "context": 16000, "qh": QH,
         "kvh": KVH, "dim": D, "bs": BS},
        # A large batch of short chains at the longest context of the runner: the cache streams from HBM.
        {"name": "attn_chain_64x6", "kind": "attn", "seqs": 64, "nodes": 6, "fan": 1, "context": 4090, "qh": QH,
         "kvh": KVH, "dim": D, "bs": BS},
        # Other heads: eight q heads a KV head of 64, small blocks.
        {"name": "attn_tree_16x33", "kind": "attn", "seqs": 16, "nodes": 33, "fan": 3, "context": 2000, "qh": 32,
         "kvh": 4, "dim": 64, "bs": 16},
        # One user's chain against the target alone (the drafts were looked up).
        {"name": "verify_chain_1x5", "kind": "verify", "seqs": 1, "nodes": 5, "fan": 1, "draft": False, "vocab": V},
        # A batch of chains that a draft model sampled: both models' logits.
        {"name": "verify_draft_48x6", "kind": "verify", "seqs": 48, "nodes": 6, "fan": 1, "draft": True, "vocab": V},
        # Trees of likely tokens, some rows greedy.
        {"name": "verify_tree_24x25", "kind": "verify", "seqs": 24, "nodes": 25, "fan": 4, "draft": False, "vocab": V},
        # Trees whose siblings a draft model sampled, odd vocabulary.
        {"name": "verify_tree_draft_8x13", "kind": "verify", "seqs": 8, "nodes": 13, "fan": 3, "draft": True,
         "vocab": 50257},
        # After a step of eight sequences: a few tokens each, in every layer.
        {"name": "compact_8", "kind": "compact", "seqs": 8, "nodes": 25, "fan": 4, "context": 90, "layers": LAYERS,
         "kvh": KVH, "dim": D, "bs": 16},
        # After a step of a large batch.
        {"name": "compact_64", "kind": "compact", "seqs": 64, "nodes": 13, "fan": 3, "context": 60, "layers": LAYERS,
         "kvh": KVH, "dim": D, "bs": 16},
        # Four prompts, each continued three ways: the partly filled last block of each is copied.
        {"name": "fork_12", "kind": "fork", "copies": 12, "layers": LAYERS, "kvh": KVH, "dim": D, "bs": BS},
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["attn", "attn", "attn", "verify", "verify", "compact", "fork"])
    heads = rng.choice([(QH, KVH, D), (QH, KVH, D), (QH, KVH, D), (32, 4, 64), (8, 1, 128), (12, 6, 80), (8, 4, 256)])
    fan = rng.choice([1, 1, 2, 3, 4])
    if kind == "attn":
        qh, kvh, dim = heads
        seqs, nodes = _log_int(rng, 1, 64), _log_int(rng, 1, 64)
        most = min(16000, 2 ** 28 // (seqs * kvh * dim), 2 ** 26 // (seqs * qh * nodes))
        return {"kind": kind, "seqs": seqs, "nodes": nodes, "fan": fan, "context": _log_int(rng, 1, max(2, most)),
                "qh": qh, "kvh": kvh, "dim": dim, "bs": rng.choice([16, 32, BS])}
    if kind == "verify":
        seqs = _log_int(rng, 1, 32)
        return {"kind": kind, "seqs": seqs, "nodes": _log_int(rng, 1, max(2, min(64, 400 // seqs))), "fan": fan,
                "draft": rng.random() < 0.5, "vocab": rng.choice([V, V, 32000, 50257])}
    if kind == "compact":
        return {"kind": kind, "seqs": _log_int(rng, 1, 64), "nodes": _log_int(rng, 3, 25), "fan": max(2, fan),
                "context": _log_int(rng, 1, 60), "layers": rng.randint(1, LAYERS), "kvh": heads[1], "dim": heads[2],
                "bs": rng.choice([16, 32])}
    return {"kind": kind, "copies": _log_int(rng, 1, 12), "layers": rng.randint(1, LAYERS), "kvh": KVH, "dim": D,
            "bs": rng.choice([16, 32, BS])}


# ---------------------------------------------------- what a case alone fixes --
def _trees(case):
    """Each sequence's parents, by node: chains (fan 1), or trees of at most `fan` children a node."""
    r = random.Random("%d %d %d" % (case["seqs"], case["nodes"], case["fan"]))
    trees = []
    for s in range(case["seqs"]):
        n = max(1, case["nodes"] - s * 5 % (case["nodes"] // 3 + 1))
        parents, children = [-1], [0]
        for i in range(1, n):
            if case["fan"] == 1:
                parent = i - 1
            else:  # early nodes first: wide near the root, as draft heads make them
                open_ = [j for j in range(i) if children[j] < case["fan"]]
                parent = open_[min(int(r.expovariate(0.4)), len(open_) - 1)]
            parents.append(parent)
            children[parent] += 1
            children.append(0)
        trees.append(parents)
    return trees


def _contexts(case):
    return [case["context"] - s * 37 % max(1, case["context"] // 2) for s in range(case["seqs"])]


def _kept(case):
    """The nodes that each sequence keeps after a step: a path from the root, of some length."""
    r = random.Random("kept %d %d" % (case["seqs"], case["nodes"]))
    kept = []
    for parents in _trees(case):
        node, path = r.randrange(len(parents)), []
        while node >= 0:
            path.append(node)
            node = parents[node]
        kept.append(path[::-1])
    return kept


def _filled(case):
    return [case["bs"] - i * 29 % max(1, case["bs"] // 2) for i in range(case["copies"])]


# ------------------------------------------------------------------- inputs --
class _Inputs:
    """Random tensors on the GPU from one seed, made in a fixed order."""

    def __init__(self, seed):
        self.g = torch.Generator(device="cuda")
        self.g.manual_seed(int(seed))
        self.r = random.Random(int(seed))

    def normal(self, *shape, std=1.0):
        return (torch.randn(shape, generator=self.g, device="cuda") * std).to(torch.bfloat16)

    def uniform(self, *shape):
        return torch.rand(shape, generator=self.g, device="cuda")

    def ints(self, low, high, *shape):
        return torch.randint(low, high, shape, generator=self.g, device="cuda")


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _tables(case, x):
    """Block tables of the case's sequences over a shuffled pool, and the pool's size."""
    need = [-(-(c + len(t)) // case["bs"]) for c, t in zip(_contexts(case), _trees(case))]
    ids = list(range(sum(need) + 1))
    x.r.shuffle(ids)
    tables, at = [], 0
    for n in need:
        tables.append(ids[at:at + n] + [-1] * (max(need) - n))
        at += n
    return tables, len(ids)


def _starts(trees):
    return [sum(len(t) for t in trees[:s]) for s in range(len(trees) + 1)]


def _ancestors(parents):
    """Each node's mask: itself and its ancestors."""
    masks = []
    for i, p in enumerate(parents):
        masks.append((masks[p] if p >= 0 else 0) | 1 << i)
    return masks


def _values(case, seed):
    """The case's inputs as torch tensors."""
    x, kind = _Inputs(seed), case["kind"]
    if kind == "fork":
        ids = list(range(2 * case["copies"]))
        x.r.shuffle(ids)
        shape = (case["layers"], len(ids), case["bs"], case["kvh"], case["dim"])
        third = -(-case["copies"] // 3)
        return {"kc": x.normal(*shape), "vc": x.normal(*shape),
                "sources": _i32([ids[i % third] for i in range(case["copies"])]),
                "targets": _i32(ids[case["copies"]:]), "filled": _i32(_filled(case))}
    trees = _trees(case)
    if kind == "verify":
        return _verify_values(case, x, trees)
    tables, blocks = _tables(case, x)
    v = {"contexts": _i32(_contexts(case)), "tables": _i32(tables)}
    if kind == "compact":
        kept, width = _kept(case), case["nodes"]
        shape = (case["layers"], blocks, case["bs"], case["kvh"], case["dim"])
        return {**v, "kc": x.normal(*shape), "vc": x.normal(*shape), "counts": _i32([len(k) for k in kept]),
                "nodes": _i32([k + [-1] * (width - len(k)) for k in kept])}
    rows, shape = sum(len(t) for t in trees), (blocks, case["bs"], case["kvh"], case["dim"])
    masks = np.array([m for t in trees for m in _ancestors(t)], np.uint64).view(np.int64)
    return {**v, "q": x.normal(rows, case["qh"], case["dim"], std=2.0), "kc": x.normal(*shape), "vc": x.normal(*shape),
            "starts": _i32(_starts(trees)), "masks": torch.from_numpy(masks).cuda()}


def _verify_values(case, x, trees):
    vocab, starts = case["vocab"], _starts(trees)
    rows = starts[-1]
    temps = torch.tensor([0.0 if s % 4 == 3 else 0.6 + 0.2 * (s % 3) for s in range(len(trees))], device="cuda")
    row_temp = torch.tensor([0.6 + 0.2 * (s % 3) for s, t in enumerate(trees) for _ in t], device="cuda")[:, None]
    logits = x.normal(rows, vocab)
    likely = x.ints(0, vocab, rows, LIKELY)
    # The likely tokens get about the rest's mass each, those earlier in the list a little more.
    rest = torch.logsumexp(logits.float() / row_temp, -1, keepdim=True)
    gain = 1.0 - 0.4 * torch.arange(LIKELY, device="cuda") + torch.randn((rows, LIKELY), generator=x.g, device="cuda")
    peaks = (rest + gain) * row_temp
    logits.scatter_(1, likely, peaks.to(torch.bfloat16))
    draft = None
    if case["draft"]:
        draft = x.normal(rows, vocab)
        noise = torch.randn((rows, LIKELY), generator=x.g, device="cuda")
        draft.scatter_(1, likely, (peaks + 0.7 * noise * row_temp).to(torch.bfloat16))
        drawn = torch.multinomial(torch.softmax(draft.float() / row_temp, -1), max(1, case["fan"]), replacement=True,
                                  generator=x.g)
    else:
        drawn = likely
    parent_row, rank = [], []
    for s, parents in enumerate(trees):
        for i, p in enumerate(parents):
            parent_row.append(starts[s] + max(p, 0))
            rank.append(sum(1 for j in range(1, i) if parents[j] == p))
    at = torch.tensor(parent_row, device="cuda"), torch.tensor(rank, device="cuda")
    return {"logits": logits, "draft": draft, "tokens": drawn[at[0], at[1]].to(torch.int32),
            "parents": _i32([p for t in trees for p in t]), "starts": _i32(starts), "temps": temps,
            "uniforms": x.uniform(rows), "seeds": x.ints(-2 ** 62, 2 ** 62, len(trees))}


# ------------------------------------------------------------------ prepare --
class _Memory:
    """A buffer of the library in the form torch takes views of."""

    def __init__(self, buffer, typestr, shape):
        self.buffer = buffer
        self.__cuda_array_interface__ = {"data": (buffer.ptr, False), "typestr": typestr, "shape": tuple(shape),
                                         "strides": None, "version": 3}


_KINDS = {torch.bfloat16: ("<i2", 2), torch.int32: ("<i4", 4), torch.int64: ("<i8", 8), torch.float32: ("<f4", 4)}


def _buffer(shape, dtype):
    """A buffer of the library and a tensor over its memory."""
    buffer = gpu().alloc(math.prod(shape) * _KINDS[dtype][1])
    t = torch.as_tensor(_Memory(buffer, _KINDS[dtype][0], shape), device="cuda")
    return buffer, t.view(dtype) if dtype == torch.bfloat16 else t


def _outputs(case, v):
    """Names, shapes and types of what the operator writes beside the caches."""
    if case["kind"] == "attn":
        return {"out": (tuple(v["q"].shape), torch.bfloat16)}
    if case["kind"] == "verify":
        shape = (case["seqs"], case["nodes"])
        return {"out_tokens": (shape, torch.int32), "out_nodes": (shape, torch.int32),
                "out_counts": (shape[:1], torch.int32)}
    return {}


def prepare(case, seed):
    v = _values(case, seed)
    state = {"case": dict(case), "tensors": v}
    if own:  # the library takes its own buffers, and a program keeps its workspace: same values, same work in run()
        g, buffers = gpu(), {}
        for name, t in v.items():
            if t is not None:
                buffers[name], v[name] = _buffer(t.shape, t.dtype)
                g.sync()  # the zero fill
                v[name].copy_(t)
        for name, (shape, dtype) in _outputs(case, v).items():
            buffers[name], v[name] = _buffer(shape, dtype)
        need = 0
        if case["kind"] == "attn":
            need = g.attention_tree_workspace(v["q"].shape[0], case["qh"], case["kvh"], case["dim"], case["seqs"],
                                              case["nodes"], _span(v, case))
        elif case["kind"] == "verify":
            need = g.verify_tree_workspace(v["logits"].shape[0], case["seqs"], case["vocab"])
        buffers["workspace"] = g.alloc(max(need, 1))
        g.sync()
        state["buffers"] = buffers
    torch.cuda.synchronize()
    return state


# ---------------------------------------------------------------------- run --
def run(state):
    case, v, kind = state["case"], state["tensors"], state["case"]["kind"]
    if own:
        return _run_own(case, v, state["buffers"])
    if kind == "attn":
        return {"out": _attention(case, v)}
    if kind == "verify":
        tokens, nodes, counts = _verify(case, v)
        return {"tokens": tokens, "nodes": nodes, "counts": counts}
    move = _compact if kind == "compact" else _fork
    move(case, v)
    return {"k": v["kc"], "v": v["vc"]}


def _run_own(case, v, b):
    g, kind = gpu(), case["kind"]
    if kind == "attn":
        g.attention_tree(b["q"], b["kc"], b["vc"], b["contexts"], b["starts"], b["masks"], b["tables"], b["out"],
                         b["workspace"], v["q"].shape[0], case["qh"], case["kvh"], case["dim"], case["bs"],
                         v["kc"].shape[0], v["tables"].shape[1], case["seqs"], case["nodes"], _span(v, case))
        return {"out": v["out"]}
    if kind == "verify":
        g.verify_tree(b["logits"], b.get("draft"), b["tokens"], b["parents"], b["starts"], b["temps"], b["uniforms"],
                      b["seeds"], b["out_tokens"], b["out_nodes"], b["out_counts"], b["workspace"],
                      v["logits"].shape[0], case["seqs"], case["nodes"], case["vocab"])
        return {"tokens": v["out_tokens"], "nodes": v["out_nodes"], "counts": v["out_counts"]}
    if kind == "compact":
        g.kv_compact(b["kc"], b["vc"], b["contexts"], b["nodes"], b["counts"], b["tables"], case["seqs"],
                     case["nodes"], case["layers"], case["kvh"], case["dim"], case["bs"], v["kc"].shape[1],
                     v["tables"].shape[1])
    else:
        g.kv_copy_blocks(b["kc"], b["vc"], b["sources"], b["targets"], b["filled"], case["copies"], case["layers"],
                         case["kvh"], case["dim"], case["bs"], v["kc"].shape[1])
    return {"k": v["kc"], "v": v["vc"]}


def _span(v, case):
    """The longest sequence that the block tables hold."""
    return v["tables"].shape[1] * case["bs"]


# -------------------------------------------------------------- plain forms --
def _attention(case, v):
    """softmax(q k / sqrt(dim)) v over the context and the nodes of each row's mask, trees padded to one size."""
    seqs, nodes, kvh, dim, bs = case["seqs"], case["nodes"], case["kvh"], case["dim"], case["bs"]
    group, rows = case["qh"] // kvh, v["q"].shape[0]
    starts, contexts = v["starts"].long(), v["contexts"].long()
    t = torch.arange(_span(v, case), device="cuda")
    place = v["tables"].long()[:, t // bs] * bs + t % bs
    mapped = place >= 0
    place = place.clamp(min=0)
    k = v["kc"].view(-1, kvh, dim)[place].float().permute(0, 2, 3, 1).contiguous()
    i = torch.arange(nodes, device="cuda")
    row = starts[:-1, None] + i
    real = row < starts[1:, None]
    row = row.clamp(max=rows - 1)
    q = v["q"][row].float().view(seqs, nodes, kvh, group, dim).permute(0, 2, 1, 3, 4).reshape(seqs, kvh, nodes * group, dim)
    scores = torch.matmul(q, k) * dim ** -0.5
    node = t[None, :] - contexts[:, None]
    drafted = (node >= 0) & (node < (starts[1:] - starts[:-1])[:, None])
    bit = (v["masks"][row][:, :, None] >> node.clamp(0, 63)[:, None, :]) & 1
    sees = ((node < 0)[:, None, :] | (drafted[:, None, :] & (bit == 1))) & mapped[:, None, :]
    scores = scores.view(seqs, kvh, nodes, group, -1).masked_fill(~sees[:, None, :, None, :], -math.inf)
    p = torch.exp(scores - scores.amax(-1, keepdim=True))
    p = (p / p.sum(-1, keepdim=True)).view(seqs, kvh, nodes * group, -1)
    values = v["vc"].view(-1, kvh, dim)[place].float().permute(0, 2, 1, 3).contiguous()
    o = torch.matmul(p, values).view(seqs, kvh, nodes, group, dim).permute(0, 2, 1, 3, 4)
    # Rows lie by sequence, then node: the real ones of the padded trees in order.
    at = torch.where(real, starts[:-1, None] + i, rows).view(-1)
    out = torch.empty((rows + 1, case["qh"], dim), device="cuda", dtype=torch.bfloat16)
    out[at] = o.reshape(seqs * nodes, case["qh"], dim).to(torch.bfloat16)
    return out[:rows]


def _shift_right(x, n):
    return (x >> n) & ((1 << (64 - n)) - 1)


def _mix(x):
    """SplitMix64's finaliser on int64, whose products wrap as unsigned ones do."""
    x = x + (0x9E3779B97F4A7C15 - (1 << 64))
    x = (x ^ _shift_right(x, 30)) * (0xBF58476D1CE4E5B9 - (1 << 64))
    x = (x ^ _shift_right(x, 27)) * (0x94D049BB133111EB - (1 << 64))
    return x ^ _shift_right(x, 31)


def _gumbel(seeds, vocab):
    """The sampler's noise of every token: -ln(-ln u), u from the seed's and the token's hash."""
    token = torch.arange(vocab, device="cuda", dtype=torch.int64)
    bits = _shift_right(_mix(seeds[:, None] ^ (token * (0xD2B74407B1CE6E93 - (1 << 64)))[None, :]), 41)
    return -torch.log(-torch.log((bits.double() + 0.5) * 2.0 ** -23))


def _first_max(x):
    """The index of each row's largest value, the lowest of equal ones."""
    index = torch.arange(x.shape[-1], device="cuda")
    return torch.where(x == x.amax(-1, keepdim=True), index, x.shape[-1]).amin(-1)


def _verify(case, v):
    """In 64 bits: a drafted token is accepted by a comparison, and the last token is an argmax."""
    seqs, width = case["seqs"], case["nodes"]
    starts, rows = v["starts"].long(), v["logits"].shape[0]
    row = torch.arange(rows, device="cuda")
    seq = torch.searchsorted(starts[1:], row, right=True)
    first = starts[seq]
    root = row == first
    up = first + v["parents"].long().clamp(min=0)  # the parent's row
    token, u = v["tokens"].long(), v["uniforms"].double()
    temp = v["temps"].double()
    greedy = temp <= 0
    scale = torch.where(greedy, 1.0, temp)[seq][:, None]
    x = v["logits"].double() / scale
    p = torch.exp(x - x.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    best = _first_max(v["logits"].float())
    # earlier[i, j]: j is an earlier sibling of i
    earlier = (up[:, None] == up[None, :]) & (row[None, :] < row[:, None]) & ~root[:, None] & ~root[None, :]
    chance = p[up, token]
    if v["draft"] is None:
        again = (earlier & (token[:, None] == token[None, :])).any(-1)
        chance = torch.where(again | root, 0.0, chance)
        accepted = u * (1.0 - (earlier * chance[None, :]).sum(-1)) < chance
        c = q = None
    else:
        y = v["draft"].double() / scale
        q = torch.exp(y - y.amax(-1, keepdim=True))
        q = q / q.sum(-1, keepdim=True)
        rank = earlier.sum(-1)
        c, z = torch.zeros(rows, device="cuda", dtype=torch.float64), torch.ones(rows, device="cuda", dtype=torch.float64)
        accepted = torch.zeros(rows, device="cuda", dtype=torch.bool)
        for j in range(case["fan"]):
            mine = ~root & (rank == j)
            accepted |= mine & (u * z[up] * q[up, token] < (chance - c[up] * q[up, token]).clamp(min=0))
            has = torch.zeros(rows + 1, device="cuda", dtype=torch.bool)
            has[torch.where(mine, up, rows)] = True
            c = torch.where(has[:rows], c + z, c)
            z = torch.where(has[:rows], (p - c[:, None] * q).clamp(min=0).sum(-1), z)
    accepted = torch.where(greedy[seq], token == best[up], accepted) & ~root
    chosen = accepted & ~(earlier & accepted[None, :]).any(-1)
    reached = root
    for _ in range(width - 1):
        reached = root | (chosen & reached[up])
    # Padded to [seqs, width]: a path's nodes rise, so sorting puts it in order.
    node = torch.arange(width, device="cuda")
    at = (starts[:-1, None] + node).clamp(max=rows - 1)
    on = reached[at] & (starts[:-1, None] + node < starts[1:, None])
    path = torch.where(on, node, width).sort(-1).values
    counts = on.sum(-1)
    last = starts[:-1] + path.gather(1, counts[:, None] - 1)[:, 0]
    noise = _gumbel(v["seeds"], case["vocab"])
    if v["draft"] is None:
        tried = torch.zeros((seqs, case["vocab"] + 1), device="cuda", dtype=torch.bool)
        children = ~root & (up == last[seq])
        tried[seq, torch.where(children, token, case["vocab"])] = True
        rest = x[last].masked_fill(tried[:, :-1], -math.inf)
    else:
        rest = torch.log((p[last] - c[last][:, None] * q[last]).clamp(min=0))
    last_token = torch.where(greedy | (rest.amax(-1) == -math.inf), best[last], _first_max(rest + noise))
    after = torch.where(path < width, starts[:-1, None] + path, 0)
    tokens = torch.cat([v["tokens"][after][:, 1:], torch.zeros((seqs, 1), device="cuda", dtype=torch.int32)], -1)
    tokens = torch.where(node < counts[:, None] - 1, tokens.long(), -1)
    tokens = torch.where(node == counts[:, None] - 1, last_token[:, None], tokens)
    nodes = torch.where(path < width, path, -1)
    return tokens.to(torch.int32), nodes.to(torch.int32), counts.to(torch.int32)


def _compact(case, v):
    """Moves each kept node's K and V to its place behind the context, in every layer."""
    bs, width = case["bs"], case["nodes"]
    j = torch.arange(width, device="cuda")
    kept = j < v["counts"][:, None]
    to = v["contexts"].long()[:, None] + torch.where(kept, j, 0)
    at = v["contexts"].long()[:, None] + torch.where(kept, v["nodes"].long(), 0)
    slot = lambda pos: (v["tables"].long().gather(1, pos // bs) * bs + pos % bs).view(-1)  # noqa: E731
    to, at = slot(to), slot(at)
    for cache in (v["kc"], v["vc"]):
        flat = cache.view(case["layers"], -1, case["kvh"] * case["dim"])
        flat[:, to] = flat[:, at]


def _fork(case, v):
    """Copies the filled slots of each source block to its target block, in every layer."""
    t = torch.arange(case["bs"], device="cuda")
    to = v["targets"].long()[:, None] * case["bs"] + t
    at = torch.where(t < v["filled"].long()[:, None], v["sources"].long()[:, None] * case["bs"] + t, to)
    for cache in (v["kc"], v["vc"]):
        flat = cache.view(case["layers"], -1, case["kvh"] * case["dim"])
        flat[:, to.view(-1)] = flat[:, at.view(-1)]


# --------------------------------------------------------------------- work --
def work(case):
    kind = case["kind"]
    if kind == "fork":
        return {"bytes": 2 * 2 * 2 * sum(_filled(case)) * case["layers"] * case["kvh"] * case["dim"], "flops": 0}
    if kind == "compact":
        moved = sum(j != n for k in _kept(case) for j, n in enumerate(k))
        small = sum(8 * len(k) for k in _kept(case))
        return {"bytes": 2 * 2 * 2 * moved * case["layers"] * case["kvh"] * case["dim"] + small, "flops": 0}
    trees = _trees(case)
    rows = sum(len(t) for t in trees)
    if kind == "verify":
        # Logits of the nodes with children, and of the last node of each path.
        inner = sum(len(set(t[1:])) for t in trees)
        last = sum(len(t) == 1 for t in trees)
        sides = 2 if case["draft"] else 1
        return {"bytes": 2 * case["vocab"] * (sides * inner + last) + 20 * rows, "flops": 4 * case["vocab"] * sides * inner}
    keys = sum(c + len(t) for c, t in zip(_contexts(case), trees))
    pairs = sum(len(t) * c + sum(bin(m).count("1") for m in _ancestors(t)) for c, t in zip(_contexts(case), trees))
    return {"bytes": 2 * (2 * keys * case["kvh"] * case["dim"] + 2 * rows * case["qh"] * case["dim"]),
            "flops": 4 * pairs * case["qh"] * case["dim"]}


# -------------------------------------------------------------------- exact --
def exact(case, seed):
    """run()'s outputs from the definitions, in 64 bits; None for tokens and nodes, which are no computed numbers."""
    if case["kind"] == "verify":
        return None
    v = _values(case, seed)
    if case["kind"] == "attn":
        return {"out": _attention64(case, v)}
    k, w = v["kc"].double(), v["vc"].double()
    for before, after in ((v["kc"], k), (v["vc"], w)):
        if case["kind"] == "fork":
            for i, n in enumerate(_filled(case)):
                after[:, int(v["targets"][i]), :n] = before[:, int(v["sources"][i]), :n].double()
        else:
            tables = v["tables"].tolist()
            for s, (context, path) in enumerate(zip(_contexts(case), _kept(case))):
                for j, n in enumerate(path):
                    (a, b), (c, d) = (divmod(context + i, case["bs"]) for i in (j, n))
                    after[:, tables[s][a], b] = before[:, tables[s][c], d].double()
    return {"k": k, "v": w}


def _attention64(case, v):
    group, trees = case["qh"] // case["kvh"], _trees(case)
    tables, out = v["tables"].long(), torch.empty(v["q"].shape, device="cuda", dtype=torch.float64)
    for s, (context, parents, start) in enumerate(zip(_contexts(case), trees, _starts(trees))):
        n = len(parents)
        sees = torch.zeros((n, context + n), dtype=torch.bool)
        sees[:, :context] = True
        for i in range(n):
            j = i
            while j >= 0:
                sees[i, context + j] = True
                j = parents[j]
        sees = sees.cuda()
        at = torch.arange(context + n, device="cuda")
        block, offset = tables[s][at // case["bs"]], at % case["bs"]
        for h in range(case["kvh"]):
            k, w = v["kc"][block, offset, h].double(), v["vc"][block, offset, h].double()
            for a in range(h * group, (h + 1) * group):
                scores = v["q"][start:start + n, a].double() @ k.T.contiguous() / math.sqrt(case["dim"])
                weight = torch.softmax(scores.masked_fill(~sees, -math.inf), -1)
                out[start:start + n, a] = weight @ w
    return out
