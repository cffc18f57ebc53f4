"""nv_quantize_rows, nv_gemm_i8 and nv_gemm_i8_silu against their definitions in 64 bits."""
import numpy as np
import pytest

import int8_reference as ref
import nvr
import oracle as ora
from helpers import assert_bits_equal, bf16_of, f32_of

pytestmark = pytest.mark.gpu

NORMS = ("none", "rms", "add")
GUARD = 256  # bytes behind each output that have to stay as they were


def f64(bits):
    return f32_of(bits).astype(np.float64)


class Call:
    """One product's inputs on the host, and its buffers."""

    def __init__(self, gpu, m, n, k, norm="none", gated=False, seed=0, x=None, wq=None, ws=None, residual=None):
        self.gpu, self.m, self.n, self.k, self.gated = gpu, m, n, k, gated
        self.channels = 2 * n if gated else n
        rng = np.random.default_rng(seed + 7)
        self.x = ora.normal_bf16((m, k), seed + 1) if x is None else x
        if x is None and k > 8:
            self.x[:, rng.integers(0, k, max(1, k // 128))] = ora.normal_bf16((m, 1), seed + 2, 0.0, 12.0)
        self.wq = rng.integers(-127, 128, (self.channels, k), dtype=np.int8) if wq is None else wq
        self.ws = np.exp(0.3 * rng.standard_normal(self.channels)).astype(np.float32) * np.float32(1e-3) if ws is None else ws
        self.residual = (ora.normal_bf16((m, k), seed + 3, 0.0, 3.0) if residual is None else residual) if norm == "add" else None
        self.weight = ora.normal_bf16((k,), seed + 4, 1.0, 0.2) if norm != "none" else None
        padded = np.zeros((self.channels, ref.pitch(k)), np.int8)
        padded[:, :k] = self.wq
        up = lambda a: None if a is None else gpu.upload_array(a)  # noqa: E731
        self.bx, self.bw, self.bs, self.bres, self.bnw = up(self.x), up(padded), up(self.ws), up(self.residual), up(self.weight)
        fill = lambda count: gpu.upload_array(np.full(count * 2 + GUARD, 0xA5, np.uint8))  # noqa: E731
        self.by = fill(m * n)
        self.bout = fill(m * k) if norm == "add" else None
        need = gpu.gemm_i8_silu_workspace(m, n, k) if gated else gpu.gemm_i8_workspace(m, n, k)
        self.work = gpu.upload_array(np.full(need + GUARD, 0x5A, np.uint8))
        self.need = need

    def run(self):
        call = self.gpu.gemm_i8_silu if self.gated else self.gpu.gemm_i8
        call(self.bx, self.bres, self.bout, self.bnw, self.bw, self.bs, self.by, self.work, self.m, self.n, self.k, 1e-6)

    def outputs(self):
        return self.by.download(np.uint16, self.m * self.n).reshape(self.m, self.n)

    def check(self):
        y, bound = ref.product(f64(self.x), None if self.residual is None else f64(self.residual),
                               None if self.weight is None else f64(self.weight), 1e-6, self.wq,
                               self.ws.astype(np.float64), self.gated)
        got = f64(self.outputs())
        assert (np.isnan(got) == np.isnan(y)).all()
        off = np.nan_to_num(np.abs(got - y)) - np.nan_to_num(bound)
        worst = np.unravel_index(off.argmax(), off.shape)
        assert off.max() <= 0, f"at {worst}: {got[worst]} for {y[worst]} +- {bound[worst]}"
        if self.residual is not None:
            want = bf16_of(ref.residual_of(f32_of(self.x), f32_of(self.residual)))
            assert_bits_equal(self.bout.download(np.uint16, self.m * self.k).reshape(self.m, self.k), want, "residual_out")
            assert (self.bout.download(np.uint8, self.bout.bytes)[-GUARD:] == 0xA5).all()
        assert (self.by.download(np.uint8, self.by.bytes)[-GUARD:] == 0xA5).all()
        assert (self.work.download(np.uint8, self.work.bytes)[-GUARD:] == 0x5A).all()


# ------------------------------------------------------------ quantize_rows --
@pytest.mark.parametrize("rows,k", [(1, 1), (1, 2), (3, 7), (2, 8), (5, 15), (4, 16), (3, 17), (2, 40), (7, 511), (3, 512),
                                    (5, 513), (2, 1030), (3, 1111), (300, 128), (1100, 40), (1030, 1024), (1025, 2049),
                                    (2, 4096), (1027, 4096), (3, 4104), (5, 8200), (2, 16384), (3, 16385), (2, 20000),
                                    (1, 131071)])
def test_quantize_rows_bit_for_bit(gpu, rows, k):
    x = ora.normal_bf16((rows, k), rows + k, 0.0, 1.0)
    x[:, 0] = bf16_of(np.float32(4.0)) if rows % 2 else x[:, 0]  # a power of two at the top: quotients end in a half
    bx, pitch = gpu.upload_array(x), ref.pitch(k)
    q, s = gpu.upload_array(np.full(rows * pitch + GUARD, 0xA5, np.uint8)), gpu.upload_array(np.full(rows + 64, 7.0, np.float32))
    gpu.quantize_rows(bx, q, s, rows, k)
    want, top = ref.whole_numbers(f64(x))
    got = q.download(np.int8, rows * pitch).reshape(rows, pitch)
    assert_bits_equal(got[:, :k], want, "integers")
    assert not got[:, k:].any()
    assert_bits_equal(s.download(np.float32, rows), top.astype(np.float32) / np.float32(127.0), "scales")
    assert (q.download(np.uint8, q.bytes)[-GUARD:] == 0xA5).all() and (s.download(np.float32, rows + 64)[rows:] == 7.0).all()


def test_quantize_rows_of_every_magnitude(gpu):
    """Rows over all exponents, subnormal and largest ones, zeros, NaN and infinities."""
    k = 96
    rows = [np.full(k, 0.0), np.r_[np.nan, np.ones(k - 1)], np.r_[np.ones(k - 1), -np.inf], np.r_[np.full(k - 1, -0.0), 2.0 ** -133]]
    rng = np.random.default_rng(3)
    for e in range(-133, 128, 3):
        rows.append(rng.integers(-255, 256, k) * 2.0 ** max(e - 8, -133))
    rows.append(np.r_[f64(np.uint16(0x7F7F)), rng.standard_normal(k - 1) * 2.0 ** 120])
    with np.errstate(over="ignore"):
        x = bf16_of(np.array(rows).astype(np.float32))
    q, s = gpu.alloc(len(rows) * ref.pitch(k)), gpu.alloc(len(rows) * 4)
    gpu.quantize_rows(gpu.upload_array(x), q, s, len(rows), k)
    want, top = ref.whole_numbers(f64(x))
    assert_bits_equal(q.download(np.int8, want.size).reshape(want.shape), want)
    scales = s.download(np.float32, len(rows))
    assert np.isnan(scales[1:3]).all() and not np.isnan(np.delete(scales, [1, 2])).any()
    with np.errstate(invalid="ignore"):
        assert_bits_equal(np.nan_to_num(scales), np.nan_to_num(top.astype(np.float32) / np.float32(127.0)))


def test_quantize_rows_from_odd_places(gpu):
    """A view of x at an odd number of elements, and of scales at any."""
    rows, k = 6, 64
    x = ora.normal_bf16((rows * k + 3,), 5)
    q, s = gpu.alloc(rows * k), gpu.alloc(rows * 4 + 4)
    gpu.quantize_rows(gpu.upload_array(x).slice(6, rows * k * 2), q, s.slice(4, rows * 4), rows, k)
    want, _ = ref.whole_numbers(f64(x[3:].reshape(rows, k)))
    assert_bits_equal(q.download(np.int8, rows * k).reshape(rows, k), want)


# ----------------------------------------------------------------- products --
SHAPES = [(1, 1, 1), (1, 16, 16), (1, 17, 1), (2, 3, 7), (1, 100, 1024), (1, 1000, 2048), (3, 33, 130), (5, 64, 65),
          (8, 48, 128), (8, 520, 1024), (15, 31, 129), (16, 16, 64), (16, 1024, 1030), (17, 64, 256), (17, 130, 1111),
          (24, 300, 2056), (31, 77, 200), (32, 256, 1024), (33, 256, 512), (40, 100, 96), (48, 1000, 640), (63, 65, 127),
          (64, 64, 128), (65, 129, 192), (100, 256, 4096), (127, 128, 1000), (128, 130, 257), (129, 200, 136), (200, 33, 515),
          (256, 256, 128), (257, 300, 384), (300, 513, 48), (513, 257, 144), (700, 96, 72), (1030, 40, 33)]


@pytest.mark.parametrize("norm", NORMS)
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_products(gpu, m, n, k, gated, norm):
    call = Call(gpu, m, n, k, norm, gated, seed=m + n + k)
    call.run()
    call.check()


@pytest.mark.parametrize("m,n,k", [(1, 40, 9000), (2, 24, 16384), (16, 40, 12288), (20, 70, 20000), (70, 33, 5000), (200, 130, 17000)])
@pytest.mark.parametrize("norm", ["none", "add"])
def test_products_of_long_rows(gpu, m, n, k, norm):
    call = Call(gpu, m, n, k, norm, seed=k)
    call.run()
    call.check()


@pytest.mark.parametrize("m,n,k,gated", [
    # few tokens over wide weights: made in the block, several tiles a wave, lines of outputs kept and not
    (1, 40000, 136, False), (3, 20001, 264, False), (8, 70000, 72, False), (8, 12001, 520, True), (5, 9000, 2048, False),
    (2, 12000, 4096, False), (16, 33000, 1000, False), (13, 9001, 64, True), (1, 12345, 1111, False), (7, 20008, 333, True),
    # made by a launch of their own, then brought to LDS
    (9, 20000, 1032, False), (16, 18001, 2056, False), (24, 17000, 264, False), (32, 40008, 144, False), (29, 9001, 1030, True),
    (32, 8400, 2048, True),
    # tiles of 64 tokens by 128 rows of the weight, of 128 by 128 where k is short, and of 256 by 256
    (40, 17001, 72, False), (64, 16700, 400, False), (63, 8300, 264, True), (300, 4001, 500, False), (4100, 4097, 40, False),
    (260, 4200, 1030, True), (3900, 4344, 136, False), (4111, 2059, 160, True), (4090, 4089, 1050, False),
    (4090, 2043, 1040, True)])
@pytest.mark.parametrize("norm", ["none", "add"])
def test_products_in_every_form(gpu, m, n, k, gated, norm):
    call = Call(gpu, m, n, k, norm, gated, seed=n)
    call.run()
    call.check()


# The longest rows that each block makes by itself, and the ones behind them; tiles of 16 rows up to one a CU, and one more.
@pytest.mark.parametrize("m,n,k,norm", [
    (4, 50, 4096, "add"), (4, 50, 4095, "rms"), (5, 50, 4096, "add"), (3, 50, 4097, "add"), (1, 9, 2049, "rms"), (5, 50, 2048, "rms"),
    (8, 50, 2041, "add"), (6, 50, 2049, "add"), (8, 50, 4096, "none"), (7, 50, 4090, "none"), (8, 50, 4104, "none"),
    (9, 50, 2048, "none"), (16, 50, 2047, "none"), (16, 5000, 1500, "none"), (10, 50, 2049, "none"), (16, 50, 1024, "rms"),
    (11, 50, 1025, "add"), (16, 4096, 2056, "none"), (16, 4097, 2056, "none"), (32, 4090, 136, "add"), (32, 4100, 136, "add"),
    (64, 4081, 72, "none"), (64, 4112, 72, "none"), (129, 1360, 200, "none"), (1025, 200, 96, "add"), (1025, 241, 96, "add")])
@pytest.mark.parametrize("gated", [False, True])
def test_products_on_both_sides_of_each_rule(gpu, m, n, k, norm, gated):
    call = Call(gpu, m, n, k, norm, gated, seed=k + m)
    call.run()
    call.check()


@pytest.mark.parametrize("m", [1, 20, 150])
def test_sums_of_the_longest_rows_stay_exact(gpu, m):
    """The largest sums that 32 bits hold: 131071 times 127 times -128."""
    n, k = 5, 131071
    x = np.tile(bf16_of(np.float32(1.0)), (m, k))
    wq = np.full((n, k), -128, np.int8)
    wq[1], wq[2, ::2], wq[3] = 127, 127, 0
    call = Call(gpu, m, n, k, x=x, wq=wq, ws=np.ones(n, np.float32))
    call.run()
    call.check()


@pytest.mark.parametrize("m,batches", [(300, (1, 5, 16, 17, 32, 33, 64, 130))])
@pytest.mark.parametrize("norm", ["none", "add"])
@pytest.mark.parametrize("n,k", [(300, 1024), (128, 4096), (72, 1111), (4500, 512), (17000, 264), (2100, 10000)])
def test_a_token_has_the_same_bits_in_any_batch(gpu, m, batches, n, k, norm):
    whole = Call(gpu, m, n, k, norm, seed=9)
    whole.run()
    want = whole.outputs()
    for rows in batches:
        part = Call(gpu, rows, n, k, norm, x=whole.x[m - rows:].copy(), wq=whole.wq, ws=whole.ws, seed=9,
                    residual=None if whole.residual is None else whole.residual[m - rows:].copy())
        part.run()
        assert_bits_equal(part.outputs(), want[m - rows:], f"{rows} tokens")


@pytest.mark.parametrize("m", [4, 20, 140, 400])
@pytest.mark.parametrize("gated", [False, True])
def test_rows_of_nothing_nan_and_infinity(gpu, m, gated):
    """Rows of zeros are +0 (or -0), rows with a NaN or an infinity NaN, and no other row is touched by them."""
    k = 200
    x = ora.normal_bf16((m, k), 11)
    x[0], x[1, 17], x[3, k - 1] = 0, 0x7FC0, 0xFF80
    call = Call(gpu, m, 70, k, gated=gated, x=x)
    call.run()
    call.check()
    y = f64(call.outputs())
    assert (y[0] == 0).all() and np.isnan(y[[1, 3]]).all() and not np.isnan(y[2]).any()


@pytest.mark.parametrize("m", [2, 40, 300])
def test_scales_at_both_ends_of_the_range(gpu, m):
    """Small tokens with large channels' scales, and the other way round: no product on the way leaves the range."""
    n, k = 6, 64
    x = bf16_of((np.arange(m * k).reshape(m, k) % 17 - 8) * np.float32(2.0) ** np.where(np.arange(m) % 2, 110, -115)[:, None].astype(np.float32))
    ws = np.array([1e-38, 1e-30, 1.0, 1e20, 3e38, 1e-45], np.float32)
    call = Call(gpu, m, n, k, x=x, ws=ws)
    call.run()
    y, bound = ref.product(f64(x), None, None, 0.0, call.wq, ws.astype(np.float64))
    got = f64(call.outputs())
    inside = np.abs(y) < 3.38e38
    assert (np.abs(got - y)[inside] <= bound[inside]).all()
    assert (np.isinf(got) | inside | (np.abs(y) < 3.41e38)).all()
    assert inside.any() and (np.abs(y[inside]) > 1e-38).any()


@pytest.mark.parametrize("m", [1, 12, 50, 260])
def test_views_at_odd_places(gpu, m):
    """x, the residual, the norm's weight, scales and y from any element on."""
    n, k = 37, 264
    c = Call(gpu, m, n, k, "add", seed=4)

    def shift(buf, values, width):
        big = gpu.alloc(values.nbytes + width)
        big.slice(width, values.nbytes).upload(values)
        return big.slice(width, values.nbytes)

    c.bx, c.bres, c.bnw, c.bs = shift(c.bx, c.x, 2), shift(c.bres, c.residual, 2), shift(c.bnw, c.weight, 2), shift(c.bs, c.ws, 4)
    c.by, c.bout = (gpu.upload_array(np.full(count * 2 + GUARD + 2, 0xA5, np.uint8)) for count in (m * n, m * k))
    c.by, c.bout = c.by.slice(2, c.by.bytes - 2), c.bout.slice(2, c.bout.bytes - 2)
    c.run()
    c.check()


@pytest.mark.parametrize("m", [1, 9, 48, 200])
@pytest.mark.parametrize("gated", [False, True])
def test_a_captured_product_follows_its_inputs(gpu, m, gated):
    c = Call(gpu, m, 136, 1024, "add", gated, seed=2)
    graph = gpu.capture(c.run)
    for replay in range(4):
        c.x = ora.normal_bf16((m, 1024), 50 + replay)
        c.bx.upload(c.x)
        graph.replay()
        c.check()
        c.run()  # the program's own call between replays
        c.check()


@pytest.mark.parametrize("m", [3, 40, 300])
def test_two_graphs_share_a_workspace(gpu, m):
    """Captured products that use one workspace in turn on one stream, each replayed several times in changing order."""
    calls = [Call(gpu, m, 264, 2056, "add", False, seed=1), Call(gpu, m, 136, 1000, "rms", True, seed=2)]
    shared = gpu.upload_array(np.full(max(c.need for c in calls) + GUARD, 0x5A, np.uint8))
    for c in calls:
        c.work = shared
    graphs = [gpu.capture(c.run) for c in calls]
    for order in ((0, 1), (1, 0), (1, 1, 0), (0, 0, 1)):
        for i in order:
            calls[i].by.upload(np.full(calls[i].by.bytes, 0xA5, np.uint8))
            graphs[i].replay()
        for c in calls:
            c.check()


@pytest.mark.parametrize("m", [2, 14, 60, 300])
def test_x_and_the_residual_may_be_one_buffer(gpu, m):
    c = Call(gpu, m, 72, 520, "add", seed=5)
    c.residual, c.bres = c.x, c.bx
    c.run()
    c.check()


@pytest.mark.parametrize("rows,k", [(3, 700), (1200, 512)])
def test_a_captured_quantize_rows_follows_its_rows(gpu, rows, k):
    bx, q, s = gpu.alloc(rows * k * 2), gpu.alloc(rows * ref.pitch(k)), gpu.alloc(rows * 4)
    bx.upload(ora.normal_bf16((rows, k), 1))
    graph = gpu.capture(lambda: gpu.quantize_rows(bx, q, s, rows, k))
    for replay in range(3):
        x = ora.normal_bf16((rows, k), 60 + replay)
        bx.upload(x)
        graph.replay()
        want, _ = ref.whole_numbers(f64(x))
        assert_bits_equal(q.download(np.int8, rows * ref.pitch(k)).reshape(rows, -1)[:, :k], want)


def test_two_programs_at_once(gpu):
    """Calls of two contexts, each with a workspace of its own, in turns without waiting."""
    other = nvr.Gpu(0)
    calls = [Call(g, 33, 520, 1024, "add", gated, seed=s) for s, (g, gated) in
             enumerate([(gpu, False), (other, False), (gpu, True), (other, True)])]
    for _ in range(10):
        for c in calls:
            c.run()
    for c in calls:
        c.check()


def test_offsets_past_32_bits(gpu):
    """A weight of more than 2^32 bytes and outputs of more than 2^32 elements' bytes, checked at their ends."""
    n, k, m = 34000, 131056, 2
    rng = np.random.default_rng(6)
    wq, x = rng.integers(-127, 128, (16, k), dtype=np.int8), ora.normal_bf16((m, k), 8)
    w = gpu.alloc(n * k)
    for at in (0, n - 16):
        w.slice(at * k, 16 * k).upload(wq)
    ws, y = np.ones(n, np.float32), gpu.alloc(m * n * 2)
    work = gpu.alloc(gpu.gemm_i8_workspace(m, n, k))
    gpu.gemm_i8(gpu.upload_array(x), None, None, None, w, gpu.upload_array(ws), y, work, m, n, k, 1e-6)
    want, bound = ref.product(f64(x), None, None, 0.0, wq, ws[:16].astype(np.float64))
    got = f64(y.download(np.uint16, m * n).reshape(m, n))
    for at in (0, n - 16):
        assert (np.abs(got[:, at:at + 16] - want) <= bound).all()
    assert not got[:, 16:n - 16].any()
    del w
    m, n, k = 70000, 34000, 16
    x = np.tile(ora.normal_bf16((50, k), 8), (m // 50, 1))
    c_w, ws = np.tile(wq[:, :k], (n // 16, 1)), np.ones(n, np.float32)
    y, work = gpu.alloc(m * n * 2), gpu.alloc(gpu.gemm_i8_workspace(m, n, k))
    gpu.gemm_i8(gpu.upload_array(x), None, None, None, gpu.upload_array(c_w), gpu.upload_array(ws), y, work, m, n, k, 1e-6)
    want, bound = ref.product(f64(x[:50]), None, None, 0.0, c_w[:16], np.ones(16))
    for at in (0, m // 2, m - 50):
        got = f64(y.slice(at * n * 2, 50 * n * 2).download(np.uint16, 50 * n).reshape(50, n // 16, 16))
        assert (np.abs(got - want[:, None]) <= bound[:, None]).all(), at


# ------------------------------------------------------------ as a model uses --
@pytest.mark.parametrize("m", [1, 6, 40, 300])
def test_a_feed_forward_block_in_8_bits(gpu, m):
    """Weights made by quantize_rows; norm, gated projections and the way back; then the next layer's norm with its sum.
    Every call's input is the one before's output, so each is checked by itself."""
    hidden, inter = 1024, 640
    gate_up = ora.normal_bf16((2 * inter, hidden), 1, 0.0, 0.03)
    down = ora.normal_bf16((hidden, inter), 2, 0.0, 0.03)
    qkv = ora.normal_bf16((520, hidden), 3, 0.0, 0.03)
    made = []
    for w in (gate_up, down, qkv):
        q, s = gpu.alloc(w.shape[0] * ref.pitch(w.shape[1])), gpu.alloc(w.shape[0] * 4)
        gpu.quantize_rows(gpu.upload_array(w), q, s, *w.shape)
        wq, top = ref.whole_numbers(f64(w))
        made.append((q, s, wq, (top.astype(np.float32) / np.float32(127.0)).astype(np.float64)))
    x, res = ora.normal_bf16((m, hidden), 4), ora.normal_bf16((m, hidden), 5, 0.0, 2.0)
    nw = ora.normal_bf16((hidden,), 6, 1.0, 0.1)
    bx, bres, bnw = gpu.upload_array(x), gpu.upload_array(res), gpu.upload_array(nw)
    res1, act, y, res2, out = (gpu.alloc(m * c * 2) for c in (hidden, inter, hidden, hidden, 520))
    work = gpu.alloc(max(1, gpu.gemm_i8_silu_workspace(m, inter, hidden), gpu.gemm_i8_workspace(m, hidden, inter),
                         gpu.gemm_i8_workspace(m, 520, hidden)))

    def layer():
        gpu.gemm_i8_silu(bx, bres, res1, bnw, made[0][0], made[0][1], act, work, m, inter, hidden, 1e-6)
        gpu.gemm_i8(act, None, None, None, made[1][0], made[1][1], y, work, m, hidden, inter, 1e-6)
        gpu.gemm_i8(y, res1, res2, bnw, made[2][0], made[2][1], out, work, m, 520, hidden, 1e-6)

    graph = gpu.capture(layer)
    for _ in range(3):
        graph.replay()
        bits = {name: b.download(np.uint16, m * c).reshape(m, c) for name, b, c in
                (("res1", res1, hidden), ("act", act, inter), ("y", y, hidden), ("res2", res2, hidden), ("out", out, 520))}
        assert_bits_equal(bits["res1"], bf16_of(f32_of(x) + f32_of(res)))
        assert_bits_equal(bits["res2"], bf16_of(f32_of(bits["y"]) + f32_of(bits["res1"])))
        for got, (want, bound) in (
                ("act", ref.product(f64(x), f64(res), f64(nw), 1e-6, made[0][2], made[0][3], True)),
                ("y", ref.product(f64(bits["act"]), None, None, 0.0, made[1][2], made[1][3])),
                ("out", ref.product(f64(bits["y"]), f64(bits["res1"]), f64(nw), 1e-6, made[2][2], made[2][3]))):
            assert (np.abs(f64(bits[got]) - want) <= bound).all(), got


def test_the_library_refuses(gpu):
    """What reaches the C entries past the wrapper's checks."""
    lib, h = gpu.lib, gpu.handle
    b = gpu.alloc(1 << 16)
    p, far = b.ptr, b.ptr + (1 << 15)

    def product(**change):
        a = dict(x=p, residual=None, residual_out=None, norm_weight=None, w=p, w_scales=p, y=far, workspace=p + 4096, m=2,
                 n=3, k=16, eps=1e-6)
        a.update(change)
        return lib.nv_gemm_i8(h, *a.values()), lib.nv_gemm_i8_silu(h, *a.values())

    for change in (dict(m=0), dict(n=0), dict(k=0), dict(k=131072), dict(n=2 ** 31 - 1), dict(x=None), dict(w=None),
                   dict(w_scales=None), dict(y=None), dict(w=p + 8), dict(x=p + 1), dict(y=far + 1), dict(w_scales=p + 2),
                   dict(residual=p), dict(residual_out=p), dict(norm_weight=p, residual_out=p), dict(workspace=p + 4104)):
        assert product(**change) == (-2, -2), change
    # An output over the tokens or the other output: blocks read while others write.
    apart = dict(residual=p + 8192, residual_out=p + 12288, norm_weight=p)
    assert product(**apart) == (0, 0)
    for change in (dict(residual_out=p + 8192), dict(residual_out=p + 8192 + 62), dict(residual_out=p), dict(y=p + 62), dict(y=p),
                   dict(y=p + 8192), dict(y=p + 12288 - 2), dict(y=p + 12288 + 62)):
        assert product(**{**apart, **change}) == (-2, -2), change
    assert product(**{**apart, "y": p + 12288 + 64}) == (0, 0)  # right behind it
    # More tiles than one launch holds: nothing is read or written.
    assert lib.nv_gemm_i8(h, p, None, None, None, p, p, far, p + 4096, 40, 2 ** 31 - 1000, 16, 1e-6) == -2
    for args in ((None, p, p, 1, 16), (p, None, p, 1, 16), (p, p, None, 1, 16), (p, far, p, 0, 16), (p, far, p, 1, 0),
                 (p, far, p, 1, 131072), (p + 1, far, p, 1, 16), (p, far + 8, p, 1, 16), (p, far, p + 2, 1, 16)):
        assert lib.nv_quantize_rows(h, *args) == -2, args
    gpu.sync()
