"""Layer norm where f32 runs out: rows far from zero, rows of one value, and layers with one of their two parameters.  Formulas and bounds
of the ordinary cases are those of test_layer_norm.py."""
import numpy as np
import pytest

from test_layer_norm import ag, as_type, backward, check_backward, make, values_of  # noqa: F401

gpu = pytest.mark.gpu
U = 2.0**-24
EPS = 1e-5


@gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows,cols", [(3, 32), (300, 20), (3, 100), (200, 193), (300, 700), (5, 1001), (5, 3001), (3, 5003), (3, 7001), (3, 12345), (2, 20002), (2, 40003)])
def test_gradients_of_rows_far_from_zero(ag, dtype, rows, cols):  # noqa: F811
    """Rows of 2^122, exact in both types: every deviation is 0, while (0 - mean) * rstd, what a place behind a row's end would give, is beyond f32."""
    rng = np.random.default_rng(21)
    x = as_type(np.full((rows, cols), 2.0**122), dtype)
    _, w, _, dy = make(rng, rows, cols, dtype)
    mean, rstd = np.full(rows, 2.0**122, np.float32), np.full(rows, EPS**-0.5, np.float32)
    tx, tdy, tw, tm, tr = (ag.Tensor.from_array(v) for v in (x[0], dy[0], w[0], mean, rstd))
    got = [values_of(t) for t in tx.layer_norm_backward(tdy, tw, tm, tr)]
    assert np.isfinite(got[0]).all()
    check_backward(got, x[1], dy[1], w[1], mean.astype(np.float64), rstd.astype(np.float64), dtype)


COLS = [1, 3, 10, 100, 193, 1000, 1001, 3001, 5003, 7001, 12345, 16384, 20001, 40003]


@gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("cols", COLS)
def test_rows_of_one_value(ag, dtype, cols):  # noqa: F811
    """Their mean is that value: y is the bias, exactly, and rstd 1 / sqrt(eps) within three roundings.  A first mean off by at most L u |x| (L as in
    test_layer_norm.py) leaves deviations that are all the same, and their mean, off by L u of itself, the rest of it: less than half a step for L^2 u < 1/2, L < 2896."""
    rng = np.random.default_rng(22)
    x = as_type(np.repeat(np.array([[1000.1], [-7.3e5], [0.1], [3.0], [-1e4], [0.0], [2.0**20 + 0.1], [-65000.7], [1e-30], [1e15]]), cols, 1), dtype)
    _, w, b, _ = make(rng, 1, cols, dtype)
    tx, tw, tb = (ag.Tensor.from_array(v) for v in (x[0], w[0], b[0]))
    y, mean, rstd = tx.layer_norm(tw, tb, EPS, stats=True)
    assert np.array_equal(values_of(mean), x[1][:, 0])
    assert np.all(np.abs(values_of(rstd) - EPS**-0.5) <= 4 * U * EPS**-0.5)
    assert np.array_equal(values_of(y), np.repeat(b[1][None, :], len(x[1]), 0))
    # with eps 0 the formula divides 0 by 0, in those rows alone
    mixed = x[0].copy()
    mixed[4:8] = as_type(rng.standard_normal((4, cols)), dtype)[0]
    mixed = ag.Tensor.from_array(mixed)
    got, want = values_of(mixed.layer_norm(tw, tb, 0.0)), values_of(mixed.layer_norm(tw, tb, 1e-30))
    one = [0, 1, 2, 3, 8, 9] if cols > 1 else list(range(10))
    assert np.isnan(got[one]).all()
    rest = [r for r in range(10) if r not in one]
    assert np.array_equal(got[rest], want[rest]) and np.isfinite(got[rest]).all()


@gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_long_rows_of_one_value(ag, dtype):  # noqa: F811
    """As above at the most columns that are promised: a thread adds 2048 of them one after another and 16 sums more, 2064^2 u < 1/2."""
    cols = 2**21
    x = as_type(np.repeat(np.array([[1000.1], [-7.3e5], [0.1]]), cols, 1), dtype)
    y, mean, _ = ag.Tensor.from_array(x[0]).layer_norm(stats=True)
    assert np.array_equal(values_of(mean), x[1][:, 0]) and not values_of(y).any()


@gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("cols", COLS[2:])
def test_mean_of_rows_far_from_zero(ag, dtype, cols):  # noqa: F811
    """Where the spread is small against the mean, the mean is the rounded one: off by u |mean| and by the f32 sum of the deviations from a first one, (L + 3) u mean |d|,
    |d| larger than the true deviation by at most the first mean's L u mean |x|."""
    rng = np.random.default_rng(23)
    spread = np.array([[1.0], [20.0], [0.01], [5.0], [1e-3], [40.0], [2.0], [0.3]])
    x = as_type(1000 + spread * rng.standard_normal((8, cols)), dtype)
    mean = values_of(ag.Tensor.from_array(x[0]).layer_norm(stats=True)[1])
    m = x[1].mean(1)
    L = cols / 16 + 16
    d = np.abs(x[1] - m[:, None]).mean(1) + L * U * np.abs(x[1]).mean(1)
    assert np.all(np.abs(mean - m) <= U * np.abs(m) + (L + 3) * U * d)


@gpu
@pytest.mark.parametrize("dtype,rows,cols", [("bf16", 15, 2**22 + 8), ("f32", 15, 2**20 + 3), ("f32", 40, 2**21), ("bf16", 600, 70001)])
def test_scratch_of_long_rows(ag, dtype, rows, cols):  # noqa: F811
    """The library's own memory for the weight gradients does not grow with the rows (8 bytes for each element of 15 rows, 503 MB, were kept).  The values are ones that
    f32 sums hold exactly: mean 0, rstd 1, x and dy small integers, so dw and db are whole numbers."""
    import ctypes as C
    check = ag._ffi.check
    rng = np.random.default_rng(24)
    x, dy = (as_type(np.tile(rng.integers(-2, 3, (rows, 4099)), (1, -(-cols // 4099)))[:, :cols], dtype) for _ in range(2))
    tx, tdy, tw = ag.Tensor.from_array(x[0]), ag.Tensor.from_array(dy[0]), ag.Tensor.from_array(as_type(np.ones(cols), dtype)[0])
    mean, rstd = ag.Tensor.from_array(np.zeros(rows, np.float32)), ag.Tensor.from_array(np.ones(rows, np.float32))
    check(ag.lib.agh_sync())
    check(ag.lib.agh_cache_release())
    before, after = C.c_size_t(), C.c_size_t()
    check(ag.lib.agh_workspace_stats(C.byref(before), None))
    _, dw, db = tx.layer_norm_backward(tdy, tw, mean, rstd)
    check(ag.lib.agh_workspace_stats(C.byref(after), None))
    assert after.value - before.value <= 80 << 20  # at most 34 MB are asked for; the workspace grows by doubling
    for got, want in ((dw, (x[1][:, :4099] * dy[1][:, :4099]).sum(0)), (db, dy[1][:, :4099].sum(0))):
        want = as_type(want, dtype)[1]  # whole numbers below 2^24, rounded once
        assert np.array_equal(values_of(got), np.tile(want, -(-cols // 4099))[:cols])


@gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_no_rows_of_many_columns(ag, dtype):  # noqa: F811
    """Zeros in every column, also behind the 2^25 that one launch adds at once."""
    cols = 2**25 + 1000
    s = ag.Tensor.zeros((0,), "f32")
    x, w = ag.Tensor.zeros((0, cols), dtype), ag.Tensor.zeros((cols,), dtype)
    out = [ag.Tensor.uninit((cols,), dtype) for _ in range(2)]
    for t in out:
        ag._ffi.check(ag.lib.agh_memset(t._ptr(), 0xFF, t.buffer.nbytes))
    ag._ffi.check(getattr(ag.lib, f"agh_layer_norm_backward_{dtype}")(x._ptr(), x._ptr(), w._ptr(), s._ptr(), s._ptr(), None, out[0]._ptr(), out[1]._ptr(), 0, cols))
    assert not any(t.into_array().any() for t in out)


@gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows", [4, 5, 8, 9, 16, 17, 32, 33, 64, 65, 128, 129, 192, 193, 256, 257])
def test_gradients_of_few_rows(ag, dtype, rows):  # noqa: F811
    """On both sides of the numbers of rows at which one workgroup takes over from several and gives way to them again."""
    for cols in (30, 84, 200):
        rng = np.random.default_rng(rows + cols)
        x, w, _, dy = make(rng, rows, cols, dtype)
        tx, tdy, tw = (ag.Tensor.from_array(v[0]) for v in (x, dy, w))
        _, mean, rstd = tx.layer_norm(tw, stats=True)
        got = [values_of(t) for t in tx.layer_norm_backward(tdy, tw, mean, rstd)]
        check_backward(got, x[1], dy[1], w[1], values_of(mean), values_of(rstd), dtype)
