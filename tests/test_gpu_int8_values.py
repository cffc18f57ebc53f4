"""Values at the ends of the range in nv_gemm_i8 and nv_gemm_i8_silu, against 64 bits: gates far below zero,
rows with a norm whose squares leave fp32, NaN and infinities in them; a norm's whole numbers; the same bits again and in any
batch."""
import numpy as np
import pytest

import int8_reference as ref
from helpers import assert_bits_equal, bf16_of, f32_of
from int8_reference import HALF16, HALF32, TINY
from test_gpu_int8 import Call, f64

pytestmark = pytest.mark.gpu

# ------------------------------------------------------------------- the gate --
GATES = (-1.0, -5.0, -20.0, -44.0, -45.0, -60.0, -87.0, -100.0, -150.0, -200.0, -300.0, -1e4, -3e38)
UPS = (3.0, -1e-20, 1e20, -3e38)


def gate_call(gpu, m, n, k):
    """Tokens of one value, +1 or -1, in another place each, so a gate (an up value) is one product of 64 with a channel's
    scale: every gate of GATES with every up value of UPS, again and again over the channels."""
    x = np.zeros((m, k), np.float32)
    x[np.arange(m), np.arange(m) * 7 % k] = np.where(np.arange(m) % 3 == 2, -1.0, 1.0)
    wq = np.full((2 * n, k), 64, np.int8)
    j = np.arange(n)
    gate, up = np.array(GATES)[j % len(GATES)], np.array(UPS)[j // len(GATES) % len(UPS)]
    wq[:n] = -64
    # -64 and a positive scale make the gate; a sign of `up` goes into its integers.
    wq[n:] = np.where(up < 0, -64, 64)[:, None]
    ws = np.r_[-gate / 64, np.abs(up) / 64].astype(np.float32)
    return Call(gpu, m, n, k, gated=True, x=bf16_of(x), wq=wq, ws=ws)


def gate_values(call):
    """y and its bound. The token's scale is 1 / 127 in fp32, its sum 127 * 64; two products round g, and u, of which g moves
    g / (1 + e^-g) by (1 + |g|) times its own part. The exponential's argument is off by two roundings, and two more where it is
    taken in parts; three exponentials, a reciprocal and six products are one step each at most."""
    sign = np.where(f64(call.x).sum(1) < 0, -1.0, 1.0)
    unit = np.float64(np.float32(1.0) / np.float32(127.0)) * 127 * sign[:, None]
    ws = call.ws.astype(np.float64)
    g, u = unit * ws[:call.n] * -64, unit * ws[call.n:] * np.sign(call.wq[call.n:, 0]) * 64
    y = np.exp(np.minimum(g, 0.0)) * g * u / (1.0 + np.exp(-np.abs(g)))
    off = ((1 + np.abs(g)) * 2 + 4 * np.abs(g) + 2 * 10 + 2) * HALF32
    return y, np.abs(y) * (off + HALF16 + off * HALF16) + TINY


FORMS = [(1, 104, 40), (3, 104, 520), (8, 2100, 136), (16, 300, 1000), (13, 9001, 64),  # tokens made in the block
         (24, 9001, 264), (16, 9000, 2056),                                             # streamed, made before
         (12, 52, 4104), (20, 104, 2100), (50, 60, 72), (64, 600, 136),                  # few rows of the weight a block
         (16, 2500, 4104), (30, 2500, 1100), (64, 2200, 264), (200, 600, 136),           # more rows of the weight a block
         (63, 8300, 264), (260, 4200, 1030), (4111, 2059, 160), (4090, 2043, 1040)]      # tiles


@pytest.mark.parametrize("m,n,k", FORMS)
def test_gates_far_below_zero_and_above(gpu, m, n, k):
    call = gate_call(gpu, m, n, k)
    call.run()
    y, bound = gate_values(call)
    got = f64(call.outputs())
    fits = np.abs(y) < 3.38e38  # what bf16 holds for certain
    over = np.abs(y) > 3.41e38
    assert fits.any() and over.any() == (m > 2)  # the first two tokens have no gate above zero
    off = np.abs(np.where(fits, got - y, 0.0)) - np.where(fits, bound, 0.0)
    assert not (off > 0).any() and not np.isnan(off).any(), [(y.flat[i], got.flat[i], bound.flat[i]) for i in
                                                             np.flatnonzero(~(off.ravel() <= 0))[:5]]
    assert (got[over] == np.sign(y[over]) * np.inf).all()


@pytest.mark.parametrize("m,n,k", FORMS)
def test_a_gate_of_minus_infinity_is_closed(gpu, m, n, k):
    """A gate whose product leaves fp32 below: 0 times the up value, as of any other gate so far below zero."""
    call = gate_call(gpu, m, n, k)
    sign = np.where(f64(call.x).sum(1) < 0, -1.0, 1.0)
    call.x = bf16_of(f32_of(call.x) * np.float32(64.0))
    call.bx.upload(call.x)
    call.run()
    far = np.flatnonzero((call.ws[:n] > 4e36) & (call.ws[n:] < 1e30))
    assert far.size
    closed = f64(call.outputs())[sign > 0][:, far]
    assert closed.size and (closed == 0).all()


# ------------------------------------------------------------- rows with a norm --
KINDS = ("normal", "zeros", "nan", "infinite", "large", "largest", "one large", "product past fp32")


def norm_rows(m, k, shift, residual):
    """Row i is of kind (i + shift): x, the residual (or None), and the norm's weight, whose first value is 4."""
    rng = np.random.default_rng(100 * m + k + shift)
    v, r = rng.standard_normal((m, k)), rng.standard_normal((m, k))
    kinds = [KINDS[(i + shift) % len(KINDS)] for i in range(m)]
    for i, kind in enumerate(kinds):
        at = int(rng.integers(k))
        if kind == "zeros":
            v[i] = -f32_of(bf16_of(r[i].astype(np.float32))) if residual else 0
        elif kind == "nan":
            v[i, at] = np.nan
        elif kind == "infinite":
            v[i, at] = -np.inf
        elif kind == "large":
            v[i], r[i] = v[i] * 2.0 ** 70, r[i] * 2.0 ** 69
        elif kind == "largest":
            v[i], r[i] = rng.uniform(-1, 1, k) * 2.0 ** 124, rng.uniform(-1, 1, k) * 2.0 ** 120
        elif kind == "one large":
            v[i, at], r[i, at] = 2.0 ** 100, 0
        elif kind == "product past fp32":
            v[i, 0], r[i, 0] = 3e38, 0
    weight = bf16_of((1.0 + 0.2 * rng.standard_normal(k)).astype(np.float32))
    weight[0] = bf16_of(np.float32(4.0))
    up = lambda a: bf16_of(a.astype(np.float32))  # noqa: E731
    return kinds, up(v), up(r) if residual else None, weight


# One wave a row in the block; a launch of its own with 4 waves, 16, 16 of two chunks, 16 that read a row twice; many rows by
# one wave of 2, 4 and 8 chunks, by 4 of 4 and of 8.
NORM_FORMS = [(1, 40), (4, 1000), (4, 1111), (4, 4096), (8, 1111), (8, 2048), (16, 505), (16, 1024),
              (20, 200), (20, 2041), (40, 2500), (17, 5000), (40, 9000), (17, 16000), (40, 17000), (3, 20001),
              (1030, 200), (1030, 2000), (1030, 2041), (1030, 4000), (1030, 8000), (1030, 16001)]


@pytest.mark.parametrize("norm", ["rms", "add"])
@pytest.mark.parametrize("m,k", NORM_FORMS)
def test_rows_of_every_kind_with_a_norm(gpu, m, k, norm):
    """Rows whose sum of squares leaves fp32 have the values of any others; a NaN or an infinity, and a product with the norm's
    weight past fp32, make their row NaN and no other."""
    for shift in range(len(KINDS) if m < len(KINDS) else 1):
        kinds, x, residual, weight = norm_rows(m, k, shift, norm == "add")
        call = Call(gpu, m, 33, k, norm, seed=k, x=x, residual=residual)
        call.weight = weight
        call.bnw.upload(weight)
        call.run()
        with np.errstate(invalid="ignore", over="ignore"):
            want, bound = ref.product(f64(x), None if residual is None else f64(residual), f64(weight), 1e-6, call.wq,
                                      call.ws.astype(np.float64))
        got = f64(call.outputs())
        for i, kind in enumerate(kinds):
            if kind in ("nan", "infinite", "product past fp32"):
                assert np.isnan(got[i]).all(), (shift, i, kind)
            else:
                assert not np.isnan(got[i]).any(), (shift, i, kind)
                assert (np.abs(got[i] - want[i]) <= bound[i]).all(), (shift, i, kind, got[i][:4], want[i][:4])
            assert kind != "zeros" or not got[i].any()


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("m", [3, 40, 300])
def test_a_channel_with_a_nan_is_nan_for_every_token(gpu, m, gated):
    """quantize_rows gives such a channel a scale of NaN; no other channel has one."""
    n, k = 40, 200
    w = np.random.default_rng(m).standard_normal(((2 if gated else 1) * n, k)).astype(np.float32)
    w[7, 3], w[-1, k - 1] = np.nan, np.inf  # gated: channel 7 of the gate, the last of up
    q, s = gpu.alloc(w.shape[0] * ref.pitch(k)), gpu.alloc(w.shape[0] * 4)
    gpu.quantize_rows(gpu.upload_array(bf16_of(w)), q, s, *w.shape)
    call = Call(gpu, m, n, k, "rms", gated)
    call.bw, call.bs = q, s
    call.run()
    assert np.array_equal(np.isnan(f64(call.outputs())), np.isin(np.arange(n), (7, n - 1))[None].repeat(m, 0))


# ------------------------------------------------------- whole numbers of a norm --
@pytest.mark.parametrize("m,k", [(1, 40), (4, 1000), (4, 4096), (8, 2041), (16, 1024), (20, 200), (20, 2041), (40, 2500),
                                 (17, 5000), (17, 16000), (18, 17000), (1030, 1024), (1030, 2041), (1030, 4000), (1030, 5000)])
def test_whole_numbers_of_a_norm_are_exact(gpu, m, k):
    """Of RMSNorm(x) they are those of exact arithmetic: x_j g_j has 16 bits, 127 times that 23, so no step of fp32 rounds
    before the quotient, and none that is not half way between two numbers can round to such a point. Channels of one 1 give
    one number times the token's scale, which bf16 tells apart: 127 / (1 + 2^8) < 1/2."""
    rng = np.random.default_rng(m + k)
    x, weight = bf16_of(rng.standard_normal((m, k)).astype(np.float32)), bf16_of((1 + 0.2 * rng.standard_normal(k)).astype(np.float32))
    x[:, 0], weight[0] = bf16_of(np.float32(4.0)), bf16_of(np.float32(2.0))  # a power of two at the top: quotients end in a half
    places = np.unique(np.r_[np.arange(min(k, 300)), k - 1, rng.integers(0, k, 200)])
    wq = np.zeros((places.size, k), np.int8)
    wq[np.arange(places.size), places] = 1
    call = Call(gpu, m, places.size, k, "rms", x=x, wq=wq, ws=np.ones(places.size, np.float32))
    call.weight = weight
    call.bnw.upload(weight)
    call.run()
    products = f64(x) * f64(weight)
    want, top = ref.whole_numbers(products)
    scale = top / np.sqrt((f64(x) ** 2).mean(-1) + 1e-6) / 127
    assert_bits_equal(np.rint(f64(call.outputs()) / scale[:, None]).astype(np.int8), want[:, places])


@pytest.mark.parametrize("norm", ["rms", "add"])
@pytest.mark.parametrize("m,n,k,gated", [(8, 4096, 1024, False), (32, 20000, 1024, False), (100, 6144, 1030, False),
                                         (520, 2000, 1030, True), (2048, 4096, 512, False), (1200, 4096, 1050, True)])
def test_a_call_repeats_itself(gpu, m, n, k, gated, norm):
    call = Call(gpu, m, n, k, norm, gated)
    call.run()
    first, summed = call.outputs(), None if call.bout is None else call.bout.download(np.uint16, m * k)
    for _ in range(5):
        call.by.upload(np.full(call.by.bytes, 0xA5, np.uint8))
        call.run()
        assert_bits_equal(call.outputs(), first)
        assert summed is None or (call.bout.download(np.uint16, m * k) == summed).all()


# Every form, on both sides of the rules by tokens: made in the block, streamed, split tiles of each size, whole tiles.
@pytest.mark.parametrize("norm", ["none", "rms", "add"])
@pytest.mark.parametrize("n,k", [(150, 1024), (64, 4104), (72, 1111), (2250, 512), (9001, 264), (1100, 3000), (6000, 1050)])
def test_a_gated_token_has_the_same_bits_in_any_batch(gpu, n, k, norm):
    m = 600
    whole = Call(gpu, m, n, k, norm, True, seed=9)
    whole.run()
    want = whole.outputs()
    for rows in (1, 5, 16, 17, 32, 33, 64, 130, 300):
        part = Call(gpu, rows, n, k, norm, True, x=whole.x[m - rows:].copy(), wq=whole.wq, ws=whole.ws, seed=9,
                    residual=None if whole.residual is None else whole.residual[m - rows:].copy())
        part.run()
        assert_bits_equal(part.outputs(), want[m - rows:], f"{rows} tokens")


@pytest.mark.parametrize("n,k", [(300, 1024), (128, 4096), (72, 1111), (17000, 264), (2100, 10000)])
def test_a_token_behind_a_norm_has_the_same_bits_in_any_batch(gpu, n, k):
    m = 300
    whole = Call(gpu, m, n, k, "rms", seed=9)
    whole.run()
    want = whole.outputs()
    for rows in (1, 5, 16, 17, 32, 33, 64, 130):
        part = Call(gpu, rows, n, k, "rms", x=whole.x[m - rows:].copy(), wq=whole.wq, ws=whole.ws, seed=9)
        part.run()
        assert_bits_equal(part.outputs(), want[m - rows:], f"{rows} tokens")


# ---------------------------------------------------------------------- refusals --
def test_the_library_refuses_what_overlaps(gpu):
    """At the C entries: an output or the workspace over any other argument, the other outputs too."""
    lib, h, m, n, k = gpu.lib, gpu.handle, 3, 40, 100
    names = ("x", "residual", "residual_out", "norm_weight", "w", "w_scales", "y", "workspace")
    for call, channels, need in ((lib.nv_gemm_i8, n, gpu.gemm_i8_workspace(m, n, k)),
                                 (lib.nv_gemm_i8_silu, 2 * n, gpu.gemm_i8_silu_workspace(m, n, k))):
        sizes = dict(zip(names, (m * k * 2, m * k * 2, m * k * 2, k * 2, channels * 112, channels * 4, m * n * 2, need)))
        room = gpu.alloc(len(names) << 15)
        at = {name: room.ptr + (i << 15) + (1 << 14) for i, name in enumerate(names)}
        run = lambda **change: call(h, *{**at, **change}.values(), m, n, k, 1e-6)  # noqa: E731
        assert run() == 0 and run(x=at["residual"]) == 0
        for written in ("residual_out", "y", "workspace"):
            for other in names:
                if other == written:
                    continue
                for place in (at[other], at[other] + (sizes[other] - 1) // 16 * 16, at[other] - (sizes[written] - 1) // 16 * 16):
                    assert run(**{written: place}) == -2, (written, other, place - at[other])
                assert run(**{written: at[other] + (sizes[other] + 15) // 16 * 16}) == 0, (written, other)  # behind it
    rows = 5
    x, q, s = (room.ptr + (i << 15) for i in range(3))
    assert lib.nv_quantize_rows(h, x, q, s, rows, k) == 0
    for args in ((x, x, s), (x, x + 992, s), (x, q, x + 996), (x, q, q), (x, q, q + rows * 112 - 4)):
        assert lib.nv_quantize_rows(h, *args, rows, k) == -2, args
    assert lib.nv_quantize_rows(h, x, x + 1008, q, rows, k) == 0 and lib.nv_quantize_rows(h, x, q, q + rows * 112, rows, k) == 0
    gpu.sync()


# ------------------------------------------------------------- tokens brought to LDS --
# Made by a launch of their own, for weights that stream: more than 16 tokens over wide weights of short rows, and weights whose
# parts lie a power of two apart; and the shapes beside them, which go by tiles.
@pytest.mark.parametrize("m,n,k,gated", [
    (17, 65540, 72, False), (24, 65600, 400, False), (32, 70001, 1030, False), (29, 33000, 264, True), (32, 33001, 1000, True),
    (31, 66000, 1152, False), (20, 66008, 130, False), (24, 65504, 72, False), (24, 65500, 264, False), (18, 66000, 1160, False),
    (12, 16384, 4096, False), (16, 16390, 4090, False), (3, 16384, 8190, False), (20, 32768, 2048, False), (12, 16384, 4104, False),
    (10, 16384, 4096, True), (9, 32760, 2040, True), (17, 8192, 8192, False)])
@pytest.mark.parametrize("norm", ["none", "add"])
def test_products_over_wide_weights(gpu, m, n, k, gated, norm):
    call = Call(gpu, m, n, k, norm, gated, seed=n + k)
    call.run()
    got = f64(call.outputs())
    # The first and the last channels, and those of places in between.
    some = np.unique(np.r_[np.arange(100), np.arange(n - 100, n), np.random.default_rng(n).integers(0, n, 300)])
    rows = np.r_[some, n + some] if gated else some
    want, bound = ref.product(f64(call.x), None if call.residual is None else f64(call.residual),
                              None if call.weight is None else f64(call.weight), 1e-6, call.wq[rows],
                              call.ws[rows].astype(np.float64), gated)
    assert (np.abs(got[:, some] - want) <= bound).all()
    assert not np.isnan(got).any() and np.abs(got).max() < 1e6  # the others: no byte of 0xA5 is left
    assert (got == f64(np.uint16(0xA5A5))).mean() < 1e-3
    assert (call.by.download(np.uint8, call.by.bytes)[-256:] == 0xA5).all()
    # A token by itself has the same bits: other forms made it.
    one = Call(gpu, 1, n, k, norm, gated, x=call.x[-1:].copy(), wq=call.wq, ws=call.ws, seed=n + k,
               residual=None if call.residual is None else call.residual[-1:].copy())
    one.run()
    assert_bits_equal(one.outputs()[0], call.outputs()[-1])


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("m,k", [(1, 1024), (8, 1111), (20, 200), (40, 2500), (17, 9000), (3, 20001), (1030, 2000), (1030, 5000)])
def test_the_sum_may_stay_inside(gpu, m, k, gated):
    """A residual without residual_out: the same outputs."""
    call = Call(gpu, m, 70, k, "add", gated)
    call.run()
    want, call.bout = call.outputs(), None
    call.by.upload(np.full(call.by.bytes, 0xA5, np.uint8))
    call.run()
    assert_bits_equal(call.outputs(), want)
