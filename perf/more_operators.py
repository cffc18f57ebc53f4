"""Serving with 8-bit weights: the projections of a decoder layer in 8-bit integers.

A weight is kept as 8-bit integers with one scale a channel (a row of it), made once when the model is loaded. A call
takes the tokens in bf16, adds the residual and takes the norm where the layer has them in front of the projection,
gives each token a scale of its own and rounds it to 8-bit integers, and forms the product of integers: exact sums,
times both scales, rounded once to bf16 (gemm_i8). The gated form has the gate's and the up projection's weights one
after the other, and returns silu(gate) * up (gemm_i8_silu).

Shapes are those of the runner (host/model.cpp): hidden size 1024, 16 q heads over 8 KV heads of 128 (q, k and v are
4096 columns, the output projection reads 2048), vocabulary 151936, prompts of 2048 tokens; and generic ones beside
them. Tokens are normal with a few channels of far larger values, as activations of language models are; weights are
normal, with another spread in each channel.

The plain forms are torch on torch tensors. With `own`, inputs lie in the library's buffers (it takes no others).
"""
import math
import os
import sys

import torch

own = False

HIDDEN, QKV, HEADS, V = 1024, 4096, 2048, 151936
EPS = 1e-6

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
# m tokens, n columns (of the gated form: n of gate and n of up), k values a token. norm: "none" (the tokens as they
# are), "rms" (their norm), "add" (the residual is added first, and returned with it).
def listed():
    return [
        # One user's token through the output projection: launches and latency are all there is.
        {"name": "linear_1x1024x2048", "gated": False, "m": 1, "n": HIDDEN, "k": HEADS, "norm": "none"},
        # A decode step's q, k and v of eight users, with the residual and the norm in front.
        {"name": "linear_8x4096x1024", "gated": False, "m": 8, "n": QKV, "k": HIDDEN, "norm": "add"},
        # The logits of 32 sequences: a wide weight that streams from HBM.
        {"name": "linear_32x151936x1024", "gated": False, "m": 32, "n": V, "k": HIDDEN, "norm": "rms"},
        # A decode step of a larger model's second feed-forward projection: long sums.
        {"name": "linear_16x4096x12288", "gated": False, "m": 16, "n": 4096, "k": 12288, "norm": "none"},
        # A step that mixes a large decode batch with a piece of a prompt.
        {"name": "linear_100x6144x4096", "gated": False, "m": 100, "n": 6144, "k": 4096, "norm": "add"},
        # Sizes that are multiples of nothing.
        {"name": "linear_333x1000x1111", "gated": False, "m": 333, "n": 1000, "k": 1111, "norm": "none"},
        # A prompt of the runner through q, k and v.
        {"name": "linear_2048x4096x1024", "gated": False, "m": 2048, "n": QKV, "k": HIDDEN, "norm": "add"},
        # Prompts of a larger model: the most products.
        {"name": "linear_8192x12288x4096", "gated": False, "m": 8192, "n": 12288, "k": 4096, "norm": "none"},
        # One user's token through the gated projections.
        {"name": "gated_1x4096x1024", "gated": True, "m": 1, "n": 4096, "k": HIDDEN, "norm": "add"},
        # A decode step of a larger model: both weights stream from HBM.
        {"name": "gated_24x11008x4096", "gated": True, "m": 24, "n": 11008, "k": 4096, "norm": "add"},
        # Odd sizes again.
        {"name": "gated_777x2730x1030", "gated": True, "m": 777, "n": 2730, "k": 1030, "norm": "rms"},
        # Prompts through the gated projections of a larger model.
        {"name": "gated_4096x12288x4096", "gated": True, "m": 4096, "n": 12288, "k": 4096, "norm": "add"},
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    gated = rng.random() < 0.4
    k = rng.choice([HIDDEN, HEADS, 4096, _log_int(rng, 16, 16384), _log_int(rng, 16, 16384)])
    m = _log_int(rng, 1, 8192)
    # At most the largest listed case's products, and 200 MB of weights.
    most = min(32768, 200_000_000 // k, 4096 * 2 ** 26 // (m * k)) // (2 if gated else 1)
    n = _log_int(rng, 16, max(17, most))
    if rng.random() < 0.5:
        n = max(16, n // 16 * 16)
    return {"gated": gated, "m": m, "n": n, "k": k, "norm": rng.choice(["none", "rms", "add"])}


# ------------------------------------------------------------------- inputs --
def _values(case, seed):
    """The case's inputs as torch tensors: tokens, weights in bf16, the norm's weight and the residual."""
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    m, k, n = case["m"], case["k"], case["n"] * (2 if case["gated"] else 1)

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda")

    # One channel in 128 is 12 times as large as the others.
    spread = torch.where(torch.rand(k, generator=g, device="cuda") < 1 / 128, 12.0, 1.0)
    v = {"x": (normal(m, k) * spread).to(torch.bfloat16),
         "w": (normal(n, k) * (0.02 * torch.exp(0.3 * normal(n, 1)))).to(torch.bfloat16)}
    if case["norm"] != "none":
        v["norm_weight"] = (1.0 + 0.2 * normal(k)).to(torch.bfloat16)
    if case["norm"] == "add":
        v["residual"] = (3.0 * normal(m, k)).to(torch.bfloat16)
    return v


def _scales(x):
    """A scale a row: its largest magnitude over 127."""
    return x.float().abs().amax(-1) / 127.0


def _round_rows(x):
    """Rows as whole numbers of their scale, in 64 bits: a value half way between two has to stay there."""
    top = x.abs().amax(-1, keepdim=True).double()
    return torch.round(x.double() * 127.0 / torch.where(top > 0, top, 1.0)).to(torch.int8)


# ------------------------------------------------------------------ prepare --
class _Memory:
    """A buffer of the library in the form torch takes views of."""

    def __init__(self, buffer, typestr, shape):
        self.buffer = buffer
        self.__cuda_array_interface__ = {"data": (buffer.ptr, False), "typestr": typestr, "shape": tuple(shape),
                                         "strides": None, "version": 3}


def _buffer(*shape):
    """A bf16 buffer of the library and a tensor over its memory."""
    buffer = gpu().alloc(math.prod(shape) * 2)
    return buffer, torch.as_tensor(_Memory(buffer, "<i2", shape), device="cuda").view(torch.bfloat16)


def prepare(case, seed):
    v = _values(case, seed)
    state = {"case": dict(case), "tensors": v}
    if not own:
        w = v.pop("w")
        v["q"], v["scales"] = _round_rows(w), _scales(w)
        torch.cuda.synchronize()
        return state
    # The library takes its own buffers; a program keeps its workspace, and its weights in 8 bits.
    g, b = gpu(), {}
    import nvr

    m, n, k = case["m"], case["n"], case["k"]
    for name, t in list(v.items()):
        b[name], mine = _buffer(*t.shape)
        g.sync()  # the zero fill
        mine.copy_(t)
    torch.cuda.synchronize()
    w, rows = b.pop("w"), v.pop("w").shape[0]
    b["q"], b["scales"] = g.alloc(rows * nvr.i8_pitch(k)), g.alloc(rows * 4)
    g.quantize_rows(w, b["q"], b["scales"], rows, k)
    b["y"], v["y"] = _buffer(m, n)
    if case["norm"] == "add":
        b["residual_out"], v["residual_out"] = _buffer(m, k)
    need = g.gemm_i8_silu_workspace(m, n, k) if case["gated"] else g.gemm_i8_workspace(m, n, k)
    b["workspace"] = g.alloc(max(need, 1))
    g.sync()
    state["buffers"] = b
    return state


# ---------------------------------------------------------------------- run --
def run(state):
    case, v = state["case"], state["tensors"]
    if own:
        b = state["buffers"]
        call = gpu().gemm_i8_silu if case["gated"] else gpu().gemm_i8
        call(b["x"], b.get("residual"), b.get("residual_out"), b.get("norm_weight"), b["q"], b["scales"], b["y"],
             b["workspace"], case["m"], case["n"], case["k"], EPS)
        return {"y": v["y"], "residual": v.get("residual_out")}
    return _plain(case, v)


# -------------------------------------------------------------- plain forms --
def _plain(case, v):
    """The tokens' norm, scales and whole numbers, the product of whole numbers, both scales, and the gate."""
    x, residual = v["x"].float(), None
    if case["norm"] == "add":
        x = x + v["residual"].float()
        residual = x.to(torch.bfloat16)
    if case["norm"] != "none":
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * v["norm_weight"].float()
    y = torch.matmul(_round_rows(x).float(), v["q"].float().t())
    y = y * _scales(x)[:, None] * v["scales"]
    if case["gated"]:
        gate, up = y[:, :case["n"]], y[:, case["n"]:]
        y = gate / (1.0 + torch.exp(-gate)) * up
    return {"y": y.to(torch.bfloat16), "residual": residual}


# --------------------------------------------------------------------- work --
def work(case):
    m, n, k = case["m"], case["n"], case["k"]
    weights = n * (2 if case["gated"] else 1)
    tokens = {"none": 2 * m * k, "rms": 2 * m * k + 2 * k, "add": 6 * m * k + 2 * k}[case["norm"]]
    return {"bytes": tokens + weights * (k + 4) + 2 * m * n, "flops": 2 * m * weights * k}


# -------------------------------------------------------------------- exact --
def exact(case, seed):
    """run()'s outputs from the definitions, in 64 bits."""
    v = _values(case, seed)
    x = v["x"].double()
    residual = None
    if "residual" in v:
        x += v["residual"].double()
        residual = x.clone()
    if "norm_weight" in v:
        x /= torch.sqrt(x.pow(2).sum(-1, keepdim=True) / case["k"] + EPS)
        x *= v["norm_weight"].double()

    def eight_bits(t):  # (whole numbers in [-127, 127], step) of each row
        step = t.abs().max(-1, keepdim=True).values
        whole = (t * 127.0).div_(step.clamp(min=1e-300)).round_()
        return whole, step / 127.0

    tokens, a = eight_bits(x)
    weight, b = eight_bits(v["w"].double())
    sums = tokens @ weight.T.contiguous()
    y = sums.mul_(a).mul_(b.T)
    if case["gated"]:
        y = torch.sigmoid(y[:, :case["n"]]) * y[:, :case["n"]] * y[:, case["n"]:]
    return {"y": y, "residual": residual}
