"""The 64-bit reference of the drafted-tree operators against what it must be, and the host's checks of their
arguments (no GPU)."""
import itertools

import numpy as np
import pytest

import nvr
import oracle as ora
import tree_reference as ref


def test_reference_noise_is_the_samplers():
    """Without a draft the last token of a one-node tree is the sampler's, for the oracle's seeds and scores."""
    logits = ora.normal_bf16((6, 5003), 31, 0.0, 3.0)
    temps = np.array([0.0, 0.6, 1.3, 0.0, 0.9, 2.0], np.float32)
    seeds = np.array([ora.sampling_seed(3, r, r) for r in range(6)], np.uint64)
    values = nvr.bf16_values(logits).astype(np.float64)
    got = ref.verify(values, None, np.zeros(6, int), -np.ones(6, int), np.arange(7), temps, np.zeros(6), seeds, 1)
    assert [t for t, _ in got] == [[int(t)] for t in ora.sample(logits, temps, seeds, 6, 5003)]


def _first_token(p, tree, q, vocab):
    """The exact distribution of the first emitted token under the acceptance rules: over the uniforms by the
    rules' own acceptance chances, over the drafted siblings (drawn from q) by enumeration."""
    total = np.zeros(vocab)
    for drawn in itertools.product(range(vocab), repeat=tree) if q is not None else [tuple(range(tree))]:
        weight = np.prod([q[x] for x in drawn]) if q is not None else 1.0
        rest, z, c, alive, tried = p.copy(), 1.0, 0.0, weight, []
        for x in drawn:
            if q is None:
                accept = min(1.0, rest[x] / z) if z > 0 else 0.0
            else:
                accept = min(1.0, rest[x] / (z * q[x])) if z > 0 else 0.0
            total[x] += alive * accept
            alive *= 1.0 - accept
            if q is None:
                z -= rest[x]
                rest[x] = 0.0
            else:
                c += z
                rest = np.maximum(p - c * q, 0.0)
                z = rest.sum()
        if alive > 1e-15:
            total += alive * rest / rest.sum()
    return total


@pytest.mark.parametrize("children", [1, 2, 3])
@pytest.mark.parametrize("drawn", [False, True])
def test_acceptance_keeps_the_targets_distribution(children, drawn):
    rng = np.random.default_rng(children)
    p, q = ref.softmax(rng.normal(size=5) * 1.5, 1.0), ref.softmax(rng.normal(size=5), 1.0)
    got = _first_token(p, children, q if drawn else None, 5)
    assert np.abs(got - p).max() < 1e-12


def test_tree_masks_hold_ancestors():
    parents = [-1, 0, 0, 1, 3, 2]
    got = nvr.tree_masks(parents)
    assert got.dtype == np.uint64
    assert [bin(int(m)) for m in got] == ["0b1", "0b11", "0b101", "0b1011", "0b11011", "0b100101"]
    assert int(nvr.tree_masks(list(range(-1, 63)))[63]) == 2 ** 64 - 1
    for bad in ([], [-1] + [0] * 64, [-1, 1], [-1, -1], [-1, 0, 5]):
        with pytest.raises(nvr.ArgumentError) as e:
            nvr.tree_masks(bad)
        assert e.value.fault == "value"


# ---------------------------------------------------------------- refusals ----
def _fake():
    gpu = object.__new__(nvr.Gpu)
    gpu._device = nvr._Device(None, 0)
    gpu.lib = None

    def buffer(nbytes):
        return nvr.Buffer(nvr._Memory(gpu._device, None, nbytes), 0, nbytes)

    return gpu, buffer


ROWS, QH, KVH, D, BS, BLOCKS, STRIDE, BATCH = 6, 4, 2, 64, 16, 4, 2, 2


def _attention_call(**change):
    gpu, buffer = _fake()
    a = dict(q=buffer(ROWS * QH * D * 2), kcache=buffer(BLOCKS * BS * KVH * D * 2),
             vcache=buffer(BLOCKS * BS * KVH * D * 2), contexts=buffer(BATCH * 4), row_starts=buffer(BATCH * 4 + 4),
             masks=buffer(ROWS * 8), block_tables=buffer(BATCH * STRIDE * 4), out=buffer(ROWS * QH * D * 2),
             workspace=buffer(1 << 24), rows=ROWS, qheads=QH, kvheads=KVH, head_dim=D, block_size=BS,
             num_blocks=BLOCKS, table_stride=STRIDE, batch_size=BATCH, max_nodes=4, max_context=32)
    a.update({k: f(buffer, a) for k, f in change.items()})
    gpu.attention_tree(**a)


def _verify_call(**change):
    gpu, buffer = _fake()
    vocab = 100
    a = dict(logits=buffer(ROWS * vocab * 2), draft_logits=buffer(ROWS * vocab * 2), tokens=buffer(ROWS * 4),
             parents=buffer(ROWS * 4), row_starts=buffer(BATCH * 4 + 4), temperatures=buffer(BATCH * 4),
             uniforms=buffer(ROWS * 4), seeds=buffer(BATCH * 8), out_tokens=buffer(BATCH * 16),
             out_nodes=buffer(BATCH * 16), out_counts=buffer(BATCH * 4), workspace=buffer(1 << 20), rows=ROWS,
             batch_size=BATCH, max_nodes=4, vocab=vocab)
    a.update({k: f(buffer, a) for k, f in change.items()})
    gpu.verify_tree(**a)


def _compact_call(**change):
    gpu, buffer = _fake()
    a = dict(kcache=buffer(3 * BLOCKS * BS * KVH * D * 2), vcache=buffer(3 * BLOCKS * BS * KVH * D * 2),
             contexts=buffer(BATCH * 4), nodes=buffer(BATCH * 16), counts=buffer(BATCH * 4),
             block_tables=buffer(BATCH * STRIDE * 4), batch_size=BATCH, max_nodes=4, layers=3, kvheads=KVH,
             head_dim=D, block_size=BS, num_blocks=BLOCKS, table_stride=STRIDE)
    a.update({k: f(buffer, a) for k, f in change.items()})
    gpu.kv_compact(**a)


def _copy_call(**change):
    gpu, buffer = _fake()
    a = dict(kcache=buffer(3 * BLOCKS * BS * KVH * D * 2), vcache=buffer(3 * BLOCKS * BS * KVH * D * 2),
             sources=buffer(8), targets=buffer(8), tokens=buffer(8), copies=2, layers=3, kvheads=KVH, head_dim=D,
             block_size=BS, num_blocks=BLOCKS)
    a.update({k: f(buffer, a) for k, f in change.items()})
    gpu.kv_copy_blocks(**a)


@pytest.mark.parametrize("call", [_attention_call, _verify_call, _compact_call, _copy_call])
def test_tree_calls_that_keep_the_contract_reach_the_library(call):
    with pytest.raises(AttributeError):  # these Gpus have no library to call
        call()


@pytest.mark.parametrize("call,fault,change", [
    (_attention_call, "value", dict(max_nodes=lambda b, a: 0)),
    (_attention_call, "value", dict(max_nodes=lambda b, a: 65)),
    (_attention_call, "value", dict(kvheads=lambda b, a: 3)),
    (_attention_call, "value", dict(head_dim=lambda b, a: 63)),
    (_attention_call, "value", dict(head_dim=lambda b, a: 258)),
    (_attention_call, "dimension", dict(max_context=lambda b, a: 0)),
    (_attention_call, "dimension", dict(rows=lambda b, a: 0)),
    (_attention_call, "dimension", dict(batch_size=lambda b, a: 0)),
    (_attention_call, "extent", dict(row_starts=lambda b, a: b(BATCH * 4))),  # batch + 1 entries
    (_attention_call, "extent", dict(masks=lambda b, a: b(ROWS * 4))),
    (_attention_call, "extent", dict(q=lambda b, a: b(ROWS * QH * D * 2 - 2))),
    (_attention_call, "alignment", dict(masks=lambda b, a: b(ROWS * 8 + 8).slice(4, ROWS * 8))),
    (_attention_call, "overlap", dict(out=lambda b, a: a["q"])),
    (_attention_call, "overlap", dict(out=lambda b, a: a["kcache"])),
    (_attention_call, "extent", dict(max_context=lambda b, a: 100000, workspace=lambda b, a: b(1024))),
    (_attention_call, "extent", dict(max_context=lambda b, a: 100000, workspace=lambda b, a: None)),
    (_attention_call, "alignment", dict(max_context=lambda b, a: 1000, workspace=lambda b, a: a["workspace"].slice(8, 1 << 20))),
    (_attention_call, "overlap", dict(max_context=lambda b, a: 1000, kcache=lambda b, a: a["workspace"])),
    (_verify_call, "value", dict(max_nodes=lambda b, a: 65)),
    (_verify_call, "dimension", dict(vocab=lambda b, a: 0)),
    (_verify_call, "extent", dict(draft_logits=lambda b, a: b(ROWS * 100 * 2 - 2))),
    (_verify_call, "extent", dict(workspace=lambda b, a: b(64))),
    (_verify_call, "extent", dict(workspace=lambda b, a: None)),
    (_verify_call, "alignment", dict(workspace=lambda b, a: b(1 << 20).slice(8, (1 << 20) - 8))),
    (_verify_call, "extent", dict(out_tokens=lambda b, a: b(BATCH * 16 - 4))),
    (_verify_call, "alignment", dict(seeds=lambda b, a: b(BATCH * 8 + 8).slice(4, BATCH * 8))),
    (_verify_call, "overlap", dict(out_nodes=lambda b, a: a["out_tokens"])),
    (_verify_call, "overlap", dict(logits=lambda b, a: a["workspace"])),
    (_compact_call, "value", dict(max_nodes=lambda b, a: 0)),
    (_compact_call, "extent", dict(layers=lambda b, a: 4)),
    (_compact_call, "overlap", dict(vcache=lambda b, a: a["kcache"])),
    (_compact_call, "extent", dict(nodes=lambda b, a: b(BATCH * 16 - 4))),
    (_copy_call, "extent", dict(layers=lambda b, a: 4)),
    (_copy_call, "dimension", dict(copies=lambda b, a: 0)),
    (_copy_call, "overlap", dict(vcache=lambda b, a: a["kcache"])),
    (_copy_call, "extent", dict(tokens=lambda b, a: b(4))),
    (_copy_call, "dimension", dict(kvheads=lambda b, a: 2 ** 31 - 1)),
])
def test_tree_calls_refuse(call, fault, change):
    with pytest.raises(nvr.ArgumentError) as e:
        call(**change)
    assert e.value.fault == fault, str(e.value)


def test_workspace_sizes_refuse_bad_dimensions():
    gpu, _ = _fake()
    assert gpu.verify_tree_workspace(1, 1, 1) > 0
    for bad in ((0, 1, 1), (1, 0, 1), (1, 1, 0), (2 ** 31, 1, 1)):
        with pytest.raises(nvr.ArgumentError) as e:
            gpu.verify_tree_workspace(*bad)
        assert e.value.fault == "dimension"
    for i in (0, 4, 6):
        args = [8, 16, 8, 128, 2, 4, 100]
        args[i] = 0
        with pytest.raises(nvr.ArgumentError):
            gpu.attention_tree_workspace(*args)
    for big in ((2 ** 28, 16, 8, 128, 2, 4, 100), (8, 16, 16, 128, 2 ** 28, 4, 100)):
        with pytest.raises(nvr.BackendError):
            gpu.attention_tree_workspace(*big)


@pytest.mark.parametrize("rows,qheads,head_dim", [(7, 5, 128), (1, 1, 8), (3, 3, 40), (64, 16, 128)])
def test_workspaces_are_as_large_as_a_call_asks(rows, qheads, head_dim):
    """A buffer of the size that is told is admitted: sizes are whole numbers of the 16 bytes that it is aligned to."""
    gpu, _ = _fake()
    for max_context in (1, 300, 700, 1280, 1800, 5000):
        assert gpu.attention_tree_workspace(rows, qheads, 1, head_dim, 1, min(rows, 64), max_context) % 16 == 0
    assert gpu.verify_tree_workspace(rows, 3, 77) % 16 == 0
