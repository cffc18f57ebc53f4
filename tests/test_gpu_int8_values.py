"""Values at the ends of the range in nv_gemm_i8 and nv_gemm_i8_silu, against 64 bits: gates far below zero."""
import numpy as np
import pytest

from helpers import bf16_of, f32_of
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
