"""The gated layer where products of its factors leave f32 and the gradient does not."""
import numpy as np
import pytest

import gated as gt
from test_gated import check_forward, slope_error
from test_int8 import STEP, as_type, values_of
from test_int8_tiles import ACT

gpu = pytest.mark.gpu


@pytest.fixture(scope="module")
def ag():
    import autograph_amd as ag
    ag.Device(0)
    return ag


@gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("m", [1, 40, 300])
@pytest.mark.parametrize("n", [3, 130])
def test_gradients_whose_factors_pass_f32(ag, dtype, m, n):
    """dy u beyond f32 under a slope that is 0 (relu's gate below 0) or small (silu, gelu and sigmoid far below 0): dg is a number, and so are the sums of its rows."""
    rng = np.random.default_rng(n)
    far = {"relu": -2.0, "silu": -50.0, "gelu": -7.0, "sigmoid": -50.0}
    for activation, g in far.items():
        slope = abs(float(gt.gate(g, activation)[1]))
        big = 1e25 if slope == 0 else np.sqrt(1e30 / slope)  # dy u slope of 1e30, its sums of 1e33 at most
        h = as_type(np.concatenate((np.full((m, n), g), big * rng.uniform(0.5, 1, (m, n))), 1), dtype)
        dy = as_type(big * rng.uniform(0.5, 1, (m, n)), dtype)
        assert np.all(dy[1] * h[1][:, n:] > 3.5e38)
        want = gt.input_grad(h[1], dy[1], activation)
        th, td, dh, db = ag.Tensor.from_array(h[0]), ag.Tensor.from_array(dy[0]), ag.Tensor.zeros((m, 2 * n), dtype), ag.Tensor.zeros((2 * n,), dtype)
        call = getattr(ag.lib, f"agh_gated_dense_backward_{dtype}")
        ag._ffi.check(call(m, 1, n, None, 0, 1, 1, None, 0, 1, 1, th._ptr(), td._ptr(), ACT[activation], dh._ptr(), None, None, db._ptr()))
        got = values_of(dh)
        assert np.isfinite(got).all() and np.isfinite(values_of(db)).all()
        # the slope's two terms by gate_error, of which the larger is at most 1.05 times the slope here; their sum, the products
        e = 1.1 * gt.gate_error(np.float64(g), activation) + 2.0**-21
        assert np.all(np.abs(got - want) <= (e + STEP[dtype] * 1.02) * np.abs(want))


@gpu
@pytest.mark.parametrize("m,n,k", [(300, 130, 512), (1000, 1002, 48), (40, 2050, 304), (513, 66, 64), (8, 34, 4), (700, 666, 1000)])
def test_f32_halves_off_16_bytes(ag, m, n, k):
    """Rows of the weight on 16 bytes whose second halves are not: f32 reads them in vectors all the same, a row at a time, column by column and through a view."""
    rng = np.random.default_rng(n)
    x, w, bias = rng.standard_normal((m, k)).astype(np.float32), rng.standard_normal((k, 2 * n)).astype(np.float32), rng.standard_normal(2 * n).astype(np.float32)
    layer = ag.GatedDense(ag.Tensor.from_array(w), ag.Tensor.from_array(bias), "silu")
    for tx in (ag.Tensor.from_array(x), ag.Tensor.from_array(np.ascontiguousarray(x.T)).t()):
        y, h = layer.forward_train(tx)
        check_forward(values_of(y), values_of(h), x.astype(np.float64), w.astype(np.float64), bias.astype(np.float64), "silu", "f32")
    wide = ag.Tensor.from_array(np.concatenate((w, w), 0)).slice_rows(k, 2 * k)
    y, h = ag.Tensor.from_array(x).gated_dot(wide, None, "gelu", keep=True)
    check_forward(values_of(y), values_of(h), x.astype(np.float64), w.astype(np.float64), None, "gelu", "f32")


@gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("m,n,k", [(7, 3, 20), (40, 130, 33), (65, 515, 40), (300, 259, 64), (1000, 17, 24), (33, 4099, 8)])
def test_gradients_one_by_one_and_in_place(ag, dtype, m, n, k):
    """dh in place of h, where a row's last group of columns lies beside what another workgroup writes, and each gradient alone: the bits of the call that forms them all."""
    rng = np.random.default_rng(m)
    x, w, h, dy = (ag.Tensor.from_array(as_type(rng.standard_normal(s), dtype)[0]) for s in ((m, k), (k, 2 * n), (m, 2 * n), (m, n)))
    call = getattr(ag.lib, f"agh_gated_dense_backward_{dtype}")
    z = lambda *s: ag.Tensor.zeros(s, dtype)  # noqa: E731

    def run(h, dh, dx=None, dw=None, db=None):
        at = lambda t: None if t is None else t._ptr()  # noqa: E731
        ag._ffi.check(call(m, k, n, x._ptr(), 0, k, 1, w._ptr(), 0, 2 * n, 1, h._ptr(), dy._ptr(), 2, dh._ptr(), at(dx), at(dw), at(db)))
        return [None if t is None else t.into_array() for t in (dh, dx, dw, db)]
    want = run(h, z(m, 2 * n), z(m, k), z(k, 2 * n), z(2 * n))
    check_dh = gt.input_grad(values_of(h), values_of(dy), "silu")
    assert np.all(np.abs(values_of(ag.Tensor.from_array(want[0])) - check_dh) <= slope_error(values_of(h), values_of(dy), "silu") + 1.02 * STEP[dtype] * np.abs(check_dh) + 1e-37)
    same = ag.Tensor.from_array(h.into_array())
    for got, ref in zip(run(same, same, z(m, k), z(k, 2 * n), z(2 * n)), want):
        assert np.array_equal(got, ref)
    for i, one in enumerate((z(m, k), z(k, 2 * n), z(2 * n))):
        got = run(h, z(m, 2 * n), *[one if i == j else None for j in range(3)])
        assert np.array_equal(got[0], want[0]) and np.array_equal(got[1 + i], want[1 + i])
    assert np.array_equal(run(h, z(m, 2 * n))[0], want[0])
