"""The 64-bit references of the operators in 8-bit integers against exact fractions, and the operators' refusals that
need no GPU."""
import ctypes
from fractions import Fraction

import numpy as np
import pytest

import int8_reference as ref
import nvr
import oracle as ora
from helpers import f32_of


def _round_half_even(f: Fraction) -> int:
    return round(f)  # Python rounds fractions half to even


def test_whole_numbers_are_those_of_exact_fractions():
    rng = np.random.default_rng(1)
    rows = [f32_of(ora.normal_bf16((64,), seed)).astype(np.float64) for seed in range(20)]
    # Magnitudes that make many quotients end in a half: powers of two over numbers of 8 bits.
    rows += [np.r_[2.0 ** rng.integers(-3, 4), rng.integers(1, 256, 63) * 2.0 ** -rng.integers(6, 12)] for _ in range(40)]
    halves = 0
    for row in rows:
        q, top = ref.whole_numbers(row[None])
        a = max(abs(Fraction(float(v))) for v in row)
        assert Fraction(float(top[0])) == a
        for v, got in zip(row, q[0]):
            exact = Fraction(float(v)) * 127 / a
            halves += exact.denominator == 2
            assert int(got) == _round_half_even(exact)
    assert halves > 50


def test_whole_numbers_of_rows_without_a_step():
    q, top = ref.whole_numbers(np.array([[0.0, -0.0], [1.0, np.nan], [-np.inf, 2.0]]))
    assert not q.any() and top[0] == 0 and np.isnan(top[1:]).all()


def test_product_of_small_integers_by_hand():
    x = np.array([[127.0, -64.0, 1.0]])
    wq = np.array([[1, 2, 3], [-128, 0, 127]], np.int8)
    y, bound = ref.product(x, None, None, 0.0, wq, np.array([0.5, 2.0]))
    assert np.array_equal(y, [[(127 - 128 + 3) * 0.5, (-128 * 127 + 127) * 2.0]])
    assert (bound <= np.abs(y) * 2.0 ** -7.9 + 2.0 ** -133).all()


def test_a_bound_covers_integers_that_may_be_the_next():
    """A norm's value half way between two integers: the other one lies within the bound."""
    x = np.array([[2.0, 1.0, 0.0, 0.0]])  # 127 / 2 is 63.5
    wq = np.array([[0, 100, 0, 0]], np.int8)
    y, bound = ref.product(x, None, np.ones(4), 1e-6, wq, np.ones(1))
    step = 2.0 / np.sqrt(1.25 + 1e-6) / 127 * 100
    assert bound[0, 0] >= step and bound[0, 0] < step + abs(y[0, 0]) * 2.0 ** -7


def test_pitch_matches():
    for k in (1, 15, 16, 17, 1111, 131071):
        assert nvr.i8_pitch(k) == ref.pitch(k)


# ---------------------------------------------------------------- refusals --
def _fake_gpu():
    g = object.__new__(nvr.Gpu)
    g._device, g.lib = nvr._Device(None, 0), None
    return g


def _buffer(g, nbytes):
    return nvr.Buffer(nvr._Memory(g._device, None, nbytes), 0, nbytes)


def _fault(fault, fn, *args):
    with pytest.raises(nvr.ArgumentError) as e:
        fn(*args)
    assert e.value.fault == fault, str(e.value)


def test_workspaces_hold_the_tokens_and_refuse_sizes():
    g = _fake_gpu()
    for m, n, k in ((1, 1, 1), (3, 5, 1111), (8192, 12288, 4096), (2, 7, 131071)):
        for need in (g.gemm_i8_workspace(m, n, k), g.gemm_i8_silu_workspace(m, n, k)):
            assert need == 0 or need >= m * (k + 4)
    for bad in (0, -1, 131072):
        _fault("value", g.gemm_i8_workspace, 1, 1, bad)
    _fault("dimension", g.gemm_i8_workspace, 0, 1, 1)
    _fault("dimension", g.gemm_i8_silu_workspace, 1, 0, 1)
    lib, need = nvr.library(), ctypes.c_size_t()
    for m, n, k in ((0, 1, 1), (1, 0, 1), (1, 1, 0), (1, 1, 131072), (1, 2 ** 31 - 1, 16), (-1, 1, 1)):
        assert lib.nv_gemm_i8_workspace(m, n, k, ctypes.byref(need)) == -2
        assert lib.nv_gemm_i8_silu_workspace(m, n, k, ctypes.byref(need)) == -2
    assert lib.nv_gemm_i8_silu_workspace(1, 2 ** 30, 16, ctypes.byref(need)) == -2


def test_quantize_rows_refuses():
    g = _fake_gpu()
    x, q, s = _buffer(g, 2 * 20 * 2), _buffer(g, 64), _buffer(g, 8)
    _fault("value", g.quantize_rows, x, q, s, 2, 131072)
    _fault("value", g.quantize_rows, x, q, s, 2, 0)
    _fault("dimension", g.quantize_rows, x, q, s, 0, 20)
    _fault("extent", g.quantize_rows, x, q.slice(0, 48), s, 2, 20)  # a row is 32 bytes
    _fault("extent", g.quantize_rows, x, q, s.slice(0, 4), 2, 20)
    _fault("overlap", g.quantize_rows, x, x, s, 1, 16)
    _fault("alignment", g.quantize_rows, x, _buffer(g, 80).slice(8, 64), s, 2, 20)
    with pytest.raises(AttributeError):  # admitted: the fake Gpu has no library to call
        g.quantize_rows(x, q, s, 2, 20)


@pytest.mark.parametrize("gated", [False, True])
def test_products_refuse(gated):
    g = _fake_gpu()
    m, n, k, rows = 3, 5, 20, 10 if gated else 5
    call = g.gemm_i8_silu if gated else g.gemm_i8
    need = g.gemm_i8_silu_workspace(m, n, k) if gated else g.gemm_i8_workspace(m, n, k)
    x, res, out = (_buffer(g, m * k * 2) for _ in range(3))
    nw, w, s, y = _buffer(g, k * 2), _buffer(g, rows * 32), _buffer(g, rows * 4), _buffer(g, m * n * 2)
    work = _buffer(g, need + 64)

    def args(**change):
        a = dict(x=x, residual=res, residual_out=out, norm_weight=nw, w=w, w_scales=s, y=y, workspace=work, m=m, n=n,
                 k=k, eps=1e-6)
        a.update(change)
        return a.values()

    _fault("value", call, *args(norm_weight=None))  # a residual without a norm
    _fault("value", call, *args(residual=None))  # a sum to return, but none to form
    _fault("value", call, *args(eps=0.0))
    _fault("value", call, *args(k=131072))
    _fault("dimension", call, *args(m=0))
    _fault("dimension", call, *args(n=2 ** 31))
    _fault("extent", call, *args(w=w.slice(0, rows * 32 - 16)))
    _fault("extent", call, *args(w_scales=s.slice(0, rows * 4 - 4)))
    _fault("extent", call, *args(y=y.slice(0, m * n * 2 - 2)))
    _fault("overlap", call, *args(residual_out=res))  # the residual is read by rows that are written later
    _fault("overlap", call, *args(y=x))
    _fault("alignment", call, *args(w=_buffer(g, rows * 32 + 16).slice(8, rows * 32)))
    _fault("foreign", call, *args(w=_buffer(_fake_gpu(), rows * 32)))
    if need:
        _fault("extent", call, *args(workspace=None))
        _fault("extent", call, *args(workspace=work.slice(0, need - 16)))
        _fault("alignment", call, *args(workspace=work.slice(8, need + 16)))
    for fine in (args(), args(residual_out=None), args(residual=None, residual_out=None),
                 args(residual=None, residual_out=None, norm_weight=None, eps=0.0)):
        with pytest.raises(AttributeError):  # admitted: the fake Gpu has no library to call
            call(*fine)
    if gated:
        _fault("dimension", call, *args(n=2 ** 30))
