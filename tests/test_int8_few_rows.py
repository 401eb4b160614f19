"""8-bit integer products of few rows, which the kernel quantises itself, where its loops go round more than once and at the borders of its rule: against the definition, and
bit for bit against the quantiser's codes and the product of two operands quantised before.  Tolerances as in test_int8 and test_int8_tiles."""
import numpy as np
import pytest

import gated as gt
import int8
from test_int8 import as_type, check_product, values_of
from test_int8_tiles import ACT, Result, check_gated, operands, product

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ag():
    import autograph_amd as ag
    ag.Device(0)
    return ag


# two tiles of columns a workgroup (from 12289 columns on); a lane's share of x beyond what it holds; more blocks of a weight than two a wave; codes of more than 48 KB; both sides
# of 16384 values and, from five rows on, of 32768 bytes; and a wave without a step of its own
SIZES = [(1, 12320, 200), (3, 12305, 300), (4, 12289, 3000), (1, 13000, 1100), (4, 40, 16384), (4, 40, 16385), (2, 40, 12000), (4, 33, 9000), (1, 40, 16384), (1, 17, 16385), (5, 40, 3276),
         (5, 40, 3277), (5, 40, 1638), (5, 40, 1639), (16, 40, 1024), (16, 40, 1025), (16, 40, 512), (16, 33, 513), (9, 70, 1800), (2, 100, 65)]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("m,n,k", SIZES)
def test_dense(ag, dtype, m, n, k):
    x, w, bias = operands(np.random.default_rng(m + n + k), m, n, k, dtype)
    codes = int8.quantize(x[1])
    v = product(codes, int8.quantize(w[1].T))
    tx, tb = ag.Tensor.from_array(x[0]), ag.Tensor.from_array(np.ascontiguousarray(bias[0][:, 1]))
    qw, qx = ag.Tensor.from_array(w[0]).quantize_int8(axis=0), tx.quantize_int8()
    got = qx.into_arrays()
    assert np.array_equal(got[0], codes[0]) and np.array_equal(got[1], codes[1])
    plain, fused = ag.I8Dense(qw).forward(tx), ag.I8Dense(qw, tb).forward(tx, relu=True)
    check_product(values_of(plain), v, dtype)
    check_product(values_of(fused), v, dtype, bias[1][:, 1], True)
    assert np.array_equal(plain.into_array(), qx.dot(qw, dtype=dtype).into_array())
    assert np.array_equal(fused.into_array(), qx.dot(qw, bias=tb, relu=True, dtype=dtype).into_array())
    call, strided = getattr(ag.lib, f"agh_dense_int8_{dtype}"), ag.Tensor.from_array(bias[0])
    for by_rows in (True, False):
        c = Result(ag, m, n, dtype, by_rows)
        ag._ffi.check(call(m, k, n, tx._ptr(), 0, k, 1, qw.codes.ptr, qw.scales.ptr, c.tensor._ptr(), c.offset, c.rs, c.cs, strided._ptr(), 1, 2, 1))
        assert np.array_equal(c.values(), values_of(fused)), by_rows


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("m,n,k", SIZES)
def test_gated(ag, dtype, m, n, k):
    activation = gt.ACTIVATIONS[(m + n + k) % len(gt.ACTIVATIONS)]
    x, w, bias = operands(np.random.default_rng(m + n + k), m, 2 * n, k, dtype)
    v = product(int8.quantize(x[1]), int8.quantize(w[1].T))
    tx, tb, strided = (ag.Tensor.from_array(t) for t in (x[0], np.ascontiguousarray(bias[0][:, 1]), bias[0]))
    layer = ag.GatedDense(ag.Tensor.from_array(w[0]), tb, activation).quantize_int8()
    y = layer.forward(tx)
    check_gated(values_of(y), v, bias[1][:, 1], activation, dtype)
    call = getattr(ag.lib, f"agh_gated_dense_int8_{dtype}")
    for by_rows in (True, False):
        c = Result(ag, m, n, dtype, by_rows)
        ag._ffi.check(call(m, k, n, tx._ptr(), 0, k, 1, layer.gate.codes.ptr, layer.gate.scales.ptr, layer.up.codes.ptr, layer.up.scales.ptr, c.tensor._ptr(), c.offset, c.rs, c.cs,
                           strided._ptr(), 1, 2, ACT[activation]))
        assert np.array_equal(c.values(), values_of(y)), by_rows


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_infinities_and_nan(ag, dtype):
    """In rows whose values a lane reads twice: those rows stand for NaNs, the others are untouched."""
    rng = np.random.default_rng(8)
    clean, w, _ = operands(rng, 4, 40, 12000, dtype)
    x = clean[1].copy()
    x[1, 11999], x[3, 5000] = np.inf, np.nan
    qw = ag.Tensor.from_array(w[0]).quantize_int8(axis=0)
    got = values_of(ag.I8Dense(qw).forward(ag.Tensor.from_array(as_type(x, dtype)[0])))
    want = values_of(ag.I8Dense(qw).forward(ag.Tensor.from_array(clean[0])))
    assert np.isnan(got[[1, 3]]).all() and np.array_equal(got[[0, 2]], want[[0, 2]])
