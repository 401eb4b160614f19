"""Layer norm, forward and backward, against the formulas in 64 bits and against differences.

Tolerances.  u = 2^-24.  A sum of n terms is formed in chains of at most L = n / 16 + 16 additions (no form has fewer than 16 chains a row; their sums
are added in at most 16 more), so it is off by at most L u sum |terms|.  mean: L u mean|x| + u |mean|.  The deviations d carry that and u |x|; rstd
is off by half of what the sum of squares is, (L + 8) u, and by the mean's error, of second order.  y: |w| rstd (|d|'s error) + |w d rstd| of (L + 8) u,
u |b|, and half a step of its type."""
import ctypes as C
import types

import numpy as np
import pytest

import oracle as orc

gpu = pytest.mark.gpu
U = 2.0**-24
STEP = {"f32": 2.0**-24, "bf16": 2.0**-8}
EPS = 1e-5


@pytest.fixture(scope="module")
def ag():
    import autograph_amd as ag
    ag.Device(0)
    return ag


def as_type(a, dtype):
    a = np.asarray(a, dtype=np.float32)
    if dtype == "f32":
        return a, a.astype(np.float64)
    b = orc.f32_to_bf16(a)
    return b, orc.bf16_to_f32(b).astype(np.float64)


def values_of(t):
    a = t.into_array()
    return (orc.bf16_to_f32(a) if t.dtype == "bf16" else a).astype(np.float64)


def forward(x, w, b, eps=EPS):
    mean = x.mean(-1, keepdims=True)
    rstd = 1 / np.sqrt(((x - mean) ** 2).mean(-1, keepdims=True) + eps)
    return (x - mean) * rstd * w + b, mean[..., 0], rstd[..., 0]


def backward(x, dy, w, mean, rstd):
    mean, rstd = mean[:, None], rstd[:, None]
    h = (x - mean) * rstd
    g = dy * w
    dx = rstd * (g - g.mean(1, keepdims=True) - h * (g * h).mean(1, keepdims=True))
    return dx, (dy * h).sum(0), dy.sum(0)


def check_forward(got, mean, rstd, x, w, b, dtype, eps=EPS):
    want, m, r = forward(x, w, b, eps)
    L = x.shape[1] / 16 + 16
    off_mean = L * U * np.abs(x).mean(1) + U * np.abs(m)
    var = 1 / r**2
    off_rstd = r * ((L + 8) * U + 2 * (U * np.abs(x).max(1)) * np.abs(x - m[:, None]).mean(1) / var + off_mean**2 / var)
    if mean is not None:
        assert np.all(np.abs(mean - m) <= off_mean + 1e-40) and np.all(np.abs(rstd - r) <= off_rstd)
    d = np.abs(x - m[:, None])
    off = np.abs(w) * (r[:, None] * (off_mean[:, None] + U * np.abs(x)) + d * (off_rstd + 4 * U * r)[:, None]) + U * (np.abs(want) + np.abs(b))
    bad = np.abs(got - want) - (1.01 * off + STEP[dtype] * np.abs(want) * (1 + STEP[dtype]) + 1e-38)
    assert np.all(bad <= 0), (bad.max(), x.shape, dtype)


def check_backward(got, x, dy, w, mean, rstd, dtype):
    """mean and rstd as they were given: the gradients' own errors alone."""
    dx, dw, db = backward(x, dy, w, mean, rstd)
    rows, cols = x.shape
    L = cols / 16 + 16
    h = np.abs((x - mean[:, None]) * rstd[:, None]) + 1e-30
    off_h = 2 * U * h + U * np.abs(x - mean[:, None]) * rstd[:, None] + 2 * U * h
    g = np.abs(dy * w)
    s1, s2 = g.mean(1, keepdims=True), (g * h).mean(1, keepdims=True)
    off = rstd[:, None] * ((L + 8) * U * (s1 + h * s2) + off_h * s2 + h * (g * off_h).mean(1, keepdims=True) + 8 * U * (g + s1 + h * s2))
    for name, a, b, o in (("dx", got[0], dx, off), ("dw", got[1], dw, (rows + 16) * U * np.abs(dy * h).sum(0) + (np.abs(dy) * off_h).sum(0)),
                          ("db", got[2], db, (rows + 16) * U * np.abs(dy).sum(0))):
        bad = np.abs(a - b) - (1.01 * o + STEP[dtype] * np.abs(b) * (1 + STEP[dtype]) + 1e-38)
        assert np.all(bad <= 0), (name, bad.max(), x.shape, dtype)


def make(rng, rows, cols, dtype):
    x = as_type(rng.standard_normal((rows, cols)) * np.exp(0.5 * rng.standard_normal(cols)) + rng.standard_normal(cols), dtype)
    return x, as_type(1 + 0.2 * rng.standard_normal(cols), dtype), as_type(0.3 * rng.standard_normal(cols), dtype), as_type(rng.standard_normal((rows, cols)), dtype)


# ---- without a GPU ----


def test_refusals_in_python(monkeypatch):
    from autograph_amd import AghError, tensor
    monkeypatch.setattr(tensor, "Buffer", lambda nbytes: types.SimpleNamespace(ptr=0, nbytes=nbytes))
    u = tensor.Tensor.uninit
    x, v, s = u((4, 8), "f32"), u((8,), "f32"), u((4,), "f32")
    for kw in ({"weight": u((4,), "f32")}, {"bias": u((1, 8), "f32")}, {"weight": u((8,), "bf16")}):
        with pytest.raises(AghError):
            x.layer_norm(**kw)
    with pytest.raises(AghError):
        u((), "f32").layer_norm()
    for args in ((u((4, 7), "f32"), v, s, s), (u((4, 8), "bf16"), v, s, s), (x, u((4,), "f32"), s, s), (x, v, u((8,), "f32"), s), (x, v, s, u((4,), "bf16")),
                 (x, v, s, u((4, 1), "f32"))):
        with pytest.raises(AghError):
            x.layer_norm_backward(*args)


def test_the_oracle():
    """The backward formula against differences of the forward one."""
    rng = np.random.default_rng(1)
    x, dy = rng.standard_normal((3, 7)), rng.standard_normal((3, 7))
    w, b = rng.standard_normal(7), rng.standard_normal(7)
    y, mean, rstd = forward(x, w, b)
    grads = backward(x, dy, w, mean, rstd)
    for which, p in enumerate((x, w, b)):
        for i in np.ndindex(p.shape):
            old = p[i]
            p[i] = old + 1e-6
            hi = (forward(x, w, b)[0] * dy).sum()
            p[i] = old - 1e-6
            lo = (forward(x, w, b)[0] * dy).sum()
            p[i] = old
            assert abs((hi - lo) / 2e-6 - grads[which][i]) < 1e-7


# ---- on the GPU ----

SHAPES = [(1, 1), (1, 4096), (3, 2), (7, 16), (5, 31), (100, 84), (33, 129), (64, 512), (19, 1000), (9, 1001), (6, 2048), (5, 2047), (4, 4097), (3, 8192), (2, 12345),
          (2, 16384), (3, 20000), (2, 70000), (1000, 10), (2500, 64), (1500, 257), (333, 700)]


@gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_layer_norm(ag, dtype, rows, cols):
    rng = np.random.default_rng(rows * 7 + cols)
    x, w, b, dy = make(rng, rows, cols, dtype)
    layer = ag.LayerNorm(ag.Tensor.from_array(w[0]), ag.Tensor.from_array(b[0]))
    tx, tdy = ag.Tensor.from_array(x[0]), ag.Tensor.from_array(dy[0])
    y, mean, rstd = layer.forward_train(tx)
    assert (y.shape, mean.shape, rstd.shape, mean.dtype) == ((rows, cols), (rows,), (rows,), "f32")
    check_forward(values_of(y), values_of(mean), values_of(rstd), x[1], w[1], b[1], dtype)
    assert np.array_equal(layer.forward(tx).into_array(), y.into_array())
    got = layer.backward(tx, tdy, mean, rstd)
    check_backward([values_of(t) for t in got], x[1], dy[1], w[1], values_of(mean), values_of(rstd), dtype)
    again = layer.backward(tx, tdy, mean, rstd)
    assert all(np.array_equal(p.into_array(), q.into_array()) for p, q in zip(got, again))  # the order of sums depends on sizes alone


@gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows,cols", [(1700, 1300), (1600, 2600), (1100, 4090), (600, 7001), (530, 10250)])
def test_layer_norm_many_wide_rows(ag, dtype, rows, cols):
    """Several rows for each workgroup, at widths that a whole workgroup shares."""
    test_layer_norm(ag, dtype, rows, cols)


@gpu
def test_more_columns_than_a_launch_adds_at_once(ag):
    """2^20 groups of 32 columns and some: the workgroups that add the shares of dw and db take a second turn."""
    rng = np.random.default_rng(3)
    cols = 2**25 + 1000
    x, w, b, dy = make(rng, 1, cols, "bf16")
    layer = ag.LayerNorm(ag.Tensor.from_array(w[0]), ag.Tensor.from_array(b[0]))
    tx, tdy = ag.Tensor.from_array(x[0]), ag.Tensor.from_array(dy[0])
    y, mean, rstd = layer.forward_train(tx)
    _, dw, db = (values_of(t) for t in layer.backward(tx, tdy, mean, rstd))
    h = (x[1] - values_of(mean)[:, None]) * values_of(rstd)[:, None]
    # one row: dy * h in f32 (three roundings) and one to bf16
    want = (dy[1] * h)[0]
    assert np.all(np.abs(dw - want) <= np.abs(want) * (2.0**-8 + 2.0**-21) + 1e-38) and np.array_equal(db, dy[1][0])
    assert np.all(np.abs(values_of(y) - (h * w[1] + b[1])) <= 2.0**-8 * 1.01 * np.abs(h * w[1] + b[1]) + 2.0**-20 * (np.abs(h * w[1]) + np.abs(b[1])))


@gpu
@pytest.mark.parametrize("rows,cols", [(140000, 16384), (70000, 32776)])
def test_rows_beyond_32_bits(ag, rows, cols):
    """4.6 GB of bf16, in rows that a workgroup holds and longer ones: rows behind 4 GiB are found, in both directions and in place.  The rows repeat with a
    period of 8, and a row's results depend on the row alone."""
    from autograph_amd._ffi import check
    rng = np.random.default_rng(5)
    x, w, b, dy = make(rng, 8, cols, "bf16")
    layer = ag.LayerNorm(ag.Tensor.from_array(w[0]), ag.Tensor.from_array(b[0]))
    few, few_dy = ag.Tensor.from_array(x[0]), ag.Tensor.from_array(dy[0])
    y, mean, rstd = layer.forward_train(few)
    dx = layer.backward(few, few_dy, mean, rstd)[0]

    def many(t):
        out, have = ag.Tensor.uninit((rows, cols), "bf16"), 8
        check(ag.lib.agh_memcpy_d2d(out.buffer.ptr, t.buffer.ptr, 8 * cols * 2))
        while have < rows:
            n = min(have, rows - have)
            check(ag.lib.agh_memcpy_d2d(out.buffer.ptr + have * cols * 2, out.buffer.ptr, n * cols * 2))
            have += n
        return out
    mx, mdy = many(few), many(few_dy)
    my, mmean, mrstd = layer.forward_train(mx)
    mdx, dw, db = layer.backward(mx, mdy, mmean, mrstd)
    tail = lambda t: t.slice_rows(rows - 8, rows).into_array()  # noqa: E731
    assert np.array_equal(tail(my), y.into_array()) and np.array_equal(mmean.into_array()[-8:], mean.into_array())
    assert np.array_equal(tail(mdx), dx.into_array()) and np.array_equal(tail(mx), x[0])
    # dw, db: 8750 or 17500 times the sum of 8 rows; a chain of f32 sums is shorter than 2000, and one rounding to bf16
    h = (x[1] - values_of(mean)[:, None]) * values_of(rstd)[:, None]
    for got, terms in ((dw, dy[1] * h), (db, dy[1])):
        want, size = terms.sum(0) * (rows // 8), np.abs(terms).sum(0) * (rows // 8)
        assert np.all(np.abs(values_of(got) - want) <= 2.0**-8 * 1.01 * np.abs(want) + 2000 * 2.0**-24 * size)
    check(ag.lib.agh_layer_norm_bf16(mx.buffer.ptr, layer.weight.buffer.ptr, layer.bias.buffer.ptr, EPS, mx.buffer.ptr, None, None, rows, cols))
    assert np.array_equal(tail(mx), y.into_array())


@gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_without_weight_or_bias(ag, dtype):
    rng = np.random.default_rng(5)
    x, w, b, dy = make(rng, 12, 100, dtype)
    tx, tw, tb, tdy = (ag.Tensor.from_array(v[0]) for v in (x, w, b, dy))
    for weight, bias in ((None, None), (tw, None), (None, tb)):
        y, mean, rstd = tx.layer_norm(weight, bias, 1e-3, stats=True)
        check_forward(values_of(y), values_of(mean), values_of(rstd), x[1], w[1] if weight else np.ones(100), b[1] if bias else np.zeros(100), dtype, 1e-3)
    dx, dw, db = tx.layer_norm_backward(tdy, None, mean, rstd)
    assert dw is None and db is None
    m, r = values_of(mean), values_of(rstd)
    check_backward([values_of(dx), *backward(x[1], dy[1], 1.0, m, r)[1:]], x[1], dy[1], np.ones(100), m, r, dtype)


@gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("cols", [40, 1000, 5000, 40000])
def test_large_mean(ag, dtype, cols):
    """Rows far from zero: the squares are taken of deviations, not of the values.  And rows of one value: var 0."""
    rng = np.random.default_rng(6)
    x = as_type(1000 + rng.standard_normal((5, cols)) * np.array([[1], [0], [4], [0], [0.5]]), dtype)
    one, zero = np.ones(cols), np.zeros(cols)
    y, mean, rstd = ag.Tensor.from_array(x[0]).layer_norm(stats=True)
    m = x[1].mean(1)
    L = cols / 16 + 16
    assert np.all(np.abs(values_of(mean) - m) <= (L + 1) * U * np.abs(m))
    # (the mean's error is not small against the deviations here: the rest is checked with the mean that was found)
    d = x[1] - values_of(mean)[:, None]
    r = 1 / np.sqrt((d**2).mean(1) + EPS)
    assert np.all(np.abs(values_of(rstd) - r) <= r * (L + 8) * U)
    want = d * values_of(rstd)[:, None] * one + zero
    assert np.all(np.abs(values_of(y) - want) <= (STEP[dtype] * 1.01 + 4 * U) * np.abs(want) + 1e-38)


@gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_infinities_and_nan_stay_in_their_rows(ag, dtype):
    rng = np.random.default_rng(7)
    for rows, cols in ((9, 100), (9, 3000), (5, 30000)):
        x, w, b, dy = make(rng, rows, cols, dtype)
        bad = x[0].copy()
        bad[1, 5], bad[3, cols - 1] = as_type([np.nan, np.inf], dtype)[0]
        layer = ag.LayerNorm(ag.Tensor.from_array(w[0]), ag.Tensor.from_array(b[0]))
        y, mean, rstd = layer.forward_train(ag.Tensor.from_array(bad))
        dx, _, db = layer.backward(ag.Tensor.from_array(bad), ag.Tensor.from_array(dy[0]), mean, rstd)
        good = [r for r in range(rows) if r not in (1, 3)]
        want, want_mean, want_rstd = layer.forward_train(ag.Tensor.from_array(x[0]))
        want_dx, _, want_db = layer.backward(ag.Tensor.from_array(x[0]), ag.Tensor.from_array(dy[0]), want_mean, want_rstd)
        assert np.array_equal(y.into_array()[good], want.into_array()[good]) and np.isnan(values_of(y)[[1, 3]]).all()
        assert np.array_equal(dx.into_array()[good], want_dx.into_array()[good]) and np.isnan(values_of(dx)[[1, 3]]).all()
        assert np.array_equal(db.into_array(), want_db.into_array())


@gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_views_and_leading_axes(ag, dtype):
    rng = np.random.default_rng(8)
    x, w, b, dy = make(rng, 60, 37, dtype)
    tx, tdy = ag.Tensor.from_array(x[0]), ag.Tensor.from_array(dy[0])
    tw, tb = ag.Tensor.from_array(w[0]), ag.Tensor.from_array(b[0])
    want, m, r = tx.layer_norm(tw, tb, stats=True)
    grads = tx.layer_norm_backward(tdy, tw, m, r)
    # a row slice starts at any element's address
    assert np.array_equal(tx.slice_rows(3, 20).layer_norm(tw, tb).into_array(), want.into_array()[3:20])
    # columns of a transposed matrix are copied
    flipped = ag.Tensor.from_array(np.ascontiguousarray(x[0].T)).t()
    assert np.array_equal(flipped.layer_norm(tw, tb).into_array(), want.into_array())
    assert all(np.array_equal(p.into_array(), q.into_array()) for p, q in zip(flipped.layer_norm_backward(tdy, tw, m, r), grads))
    # leading axes
    y, m3, r3 = tx.into_shape((3, 4, 5, 37)).layer_norm(tw, tb, stats=True)
    assert y.shape == (3, 4, 5, 37) and m3.shape == (3, 4, 5)
    assert np.array_equal(y.into_array().reshape(60, 37), want.into_array())
    got = tx.into_shape((3, 20, 37)).layer_norm_backward(tdy.into_shape((3, 20, 37)), tw, m.into_shape((3, 20)), r.into_shape((3, 20)))
    assert got[0].shape == (3, 20, 37) and all(np.array_equal(p.into_array().reshape(q.shape), q.into_array()) for p, q in zip(got, grads))
    # a vector is one row
    v, mv, rv = tx.slice_rows(2, 3).into_shape((37,)).layer_norm(tw, tb, stats=True)
    assert v.shape == (37,) and mv.shape == () and np.array_equal(v.into_array(), want.into_array()[2])


@gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows,cols", [(40, 24), (300, 1000), (7, 9000), (3, 66000)])
def test_in_place_and_single_gradients(ag, dtype, rows, cols):
    rng = np.random.default_rng(9)
    x, w, b, dy = make(rng, rows, cols, dtype)
    tx, tdy, tw, tb = (ag.Tensor.from_array(v[0]) for v in (x, dy, w, b))
    y, mean, rstd = tx.layer_norm(tw, tb, stats=True)
    grads = [t.into_array() for t in tx.layer_norm_backward(tdy, tw, mean, rstd)]
    fn = getattr(ag.lib, f"agh_layer_norm_backward_{dtype}")
    for into in ("x", "dy"):
        cx, cdy = tx.clone(), tdy.clone()
        dw, db = ag.Tensor.uninit((cols,), dtype), ag.Tensor.uninit((cols,), dtype)
        dx = cx if into == "x" else cdy
        ag._ffi.check(fn(cx._ptr(), cdy._ptr(), tw._ptr(), mean._ptr(), rstd._ptr(), dx._ptr(), dw._ptr(), db._ptr(), rows, cols))
        assert all(np.array_equal(p.into_array(), q) for p, q in zip((dx, dw, db), grads))
    for k in range(3):
        out = [ag.Tensor.uninit((rows, cols) if i == 0 else (cols,), dtype) if i == k else None for i in range(3)]
        ag._ffi.check(fn(tx._ptr(), tdy._ptr(), tw._ptr(), mean._ptr(), rstd._ptr(), *[None if t is None else t._ptr() for t in out], rows, cols))
        assert np.array_equal(out[k].into_array(), grads[k])
    cx = tx.clone()
    ag._ffi.check(getattr(ag.lib, f"agh_layer_norm_{dtype}")(cx._ptr(), tw._ptr(), tb._ptr(), EPS, cx._ptr(), None, None, rows, cols))
    assert np.array_equal(cx.into_array(), y.into_array())


@gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_empty_and_refusals(ag, dtype):
    one = as_type(np.ones(5), dtype)[0]
    x, w = ag.Tensor.zeros((0, 5), dtype), ag.Tensor.from_array(one)
    y, m, r = x.layer_norm(w, w, stats=True)
    assert y.shape == (0, 5) and m.shape == (0,)
    dx, dw, db = x.layer_norm_backward(ag.Tensor.zeros((0, 5), dtype), w, m, r)
    assert dx.shape == (0, 5) and not dw.into_array().any() and not db.into_array().any()
    f, g = getattr(ag.lib, f"agh_layer_norm_{dtype}"), getattr(ag.lib, f"agh_layer_norm_backward_{dtype}")
    t = ag.Tensor.zeros((8, 8), dtype)
    s = ag.Tensor.zeros((8,), "f32")
    p, q = t._ptr(), s._ptr()
    for args, code in (((p, None, None, EPS, p, None, None, -1, 8), -1), ((p, None, None, EPS, p, None, None, 8, 0), -1), ((p, None, None, EPS, p, None, None, 2**31, 8), -4),
                       ((None, None, None, EPS, p, None, None, 8, 8), -3), ((p, None, None, EPS, None, None, None, 8, 8), -3), ((p, None, None, -1.0, p, None, None, 8, 8), -1),
                       ((p, None, None, float("nan"), p, None, None, 8, 8), -1)):
        assert f(*args) == code
    for args, code in (((p, p, None, q, q, p, None, None, 8, 0), -1), ((None, p, None, q, q, p, None, None, 8, 8), -3), ((p, None, None, q, q, p, None, None, 8, 8), -3),
                       ((p, p, None, None, q, p, None, None, 8, 8), -3), ((p, p, None, q, None, p, None, None, 8, 8), -3)):
        assert g(*args) == code
    assert not t.into_array().any()


@gpu
def test_gradients_against_differences(ag):
    """The kernels' gradients against differences of the 64-bit forward formula (f32 tolerances as above, far above the differences' own error)."""
    rng = np.random.default_rng(10)
    x, w, b, dy = make(rng, 4, 33, "f32")
    tx, tdy, tw, tb = (ag.Tensor.from_array(v[0]) for v in (x, dy, w, b))
    _, mean, rstd = tx.layer_norm(tw, tb, stats=True)
    got = [values_of(t) for t in tx.layer_norm_backward(tdy, tw, mean, rstd)]
    for which, p in enumerate((x[1], w[1], b[1])):
        for i in list(np.ndindex(p.shape))[::3]:
            old = p[i]
            p[i] = old + 1e-5
            hi = (forward(x[1], w[1], b[1])[0] * dy[1]).sum()
            p[i] = old - 1e-5
            lo = (forward(x[1], w[1], b[1])[0] * dy[1]).sum()
            p[i] = old
            assert abs((hi - lo) / 2e-5 - got[which][i]) < 2e-5 * (1 + np.abs(dy[1]).sum())


@gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_a_block_trained_and_served(ag, dtype):
    """Layer norm, a Dense layer in 4 bits with bias and relu, and backward through both (the gradients' products in 4 bits too), step by step against
    64 bits on the operands that each step was given; the whole of it captured into a graph and replayed with other inputs."""
    import mxfp4
    from test_mx import check_product
    rng = np.random.default_rng(11)
    m, k, n = 70, 200, 96
    x, w, b, _ = make(rng, m, k, dtype)
    wd, bd, dy = as_type(rng.standard_normal((k, n)) * 0.1, dtype), as_type(rng.standard_normal(n) * 0.1, dtype), as_type(rng.standard_normal((m, n)), dtype)
    tx, tw, tb, twd, tbd, tdy = (ag.Tensor.from_array(v[0]) for v in (x, w, b, wd, bd, dy))
    norm, dense = ag.LayerNorm(tw, tb), ag.Dense(twd, tbd).quantize_mxfp4()
    h, mean, rstd = norm.forward_train(tx)
    y = dense.forward(h, relu=True)
    check_product(values_of(y), mxfp4.round_trip(values_of(h)), mxfp4.round_trip(wd[1].T), dtype, bd[1], True)
    g = y.relu_backward(tdy)
    dh = g.quantize_mxfp4(axis=1).dot(twd.quantize_mxfp4(axis=1).t(), dtype=dtype)
    check_product(values_of(dh), mxfp4.round_trip(values_of(g)), mxfp4.round_trip(wd[1]), dtype)
    dwd = h.quantize_mxfp4(axis=0).t().dot(g.quantize_mxfp4(axis=0), dtype=dtype)
    check_product(values_of(dwd), mxfp4.round_trip(values_of(h).T), mxfp4.round_trip(values_of(g).T), dtype)
    grads = norm.backward(tx, dh, mean, rstd)
    check_backward([values_of(t) for t in grads], x[1], values_of(dh), w[1], values_of(mean), values_of(rstd), dtype)

    # the same calls on buffers that stay, captured
    fn = lambda stem: getattr(ag.lib, f"{stem}_{dtype}")  # noqa: E731
    u = ag.Tensor.uninit
    check = ag._ffi.check
    o = {"h": u((m, k), dtype), "mean": u((m,), "f32"), "rstd": u((m,), "f32"), "y": u((m, n), dtype), "g": u((m, n), dtype), "dh": u((m, k), dtype), "dwd": u((k, n), dtype),
         "dx": u((m, k), dtype), "dw": u((k,), dtype), "db": u((k,), dtype)}
    q = {"g1": ag.MxTensor.uninit((m, n), 1), "w1": ag.MxTensor.uninit((k, n), 1), "h0": ag.MxTensor.uninit((m, k), 0), "g0": ag.MxTensor.uninit((m, n), 0)}
    wq = dense.weight
    P = lambda t: t._data_ptr()  # noqa: E731
    Q = lambda t: (t.codes.ptr, t.scales.ptr)  # noqa: E731

    def step():
        check(fn("agh_layer_norm")(P(tx), P(tw), P(tb), EPS, P(o["h"]), P(o["mean"]), P(o["rstd"]), m, k))
        check(fn("agh_dense_mxfp4")(m, k, n, P(o["h"]), 0, k, 1, *Q(wq), P(o["y"]), 0, n, 1, P(tbd), 0, 1, 1))
        check(fn("agh_relu_backward")(P(o["y"]), P(tdy), P(o["g"]), m * n))
        check(fn("agh_quantize_mxfp4")(P(o["g"]), 0, n, 1, m, n, *Q(q["g1"])))
        check(fn("agh_quantize_mxfp4")(P(twd), 0, n, 1, k, n, *Q(q["w1"])))
        check(fn("agh_gemm_mxfp4")(m, n, k, *Q(q["g1"]), *Q(q["w1"]), P(o["dh"]), 0, k, 1, None, 0, 0, 0))
        check(fn("agh_quantize_mxfp4")(P(o["h"]), 0, 1, k, k, m, *Q(q["h0"])))
        check(fn("agh_quantize_mxfp4")(P(o["g"]), 0, 1, n, n, m, *Q(q["g0"])))
        check(fn("agh_gemm_mxfp4")(k, m, n, *Q(q["h0"]), *Q(q["g0"]), P(o["dwd"]), 0, n, 1, None, 0, 0, 0))
        check(fn("agh_layer_norm_backward")(P(tx), P(o["dh"]), P(tw), P(o["mean"]), P(o["rstd"]), P(o["dx"]), P(o["dw"]), P(o["db"]), m, k))

    step()
    for name, t in (("h", h), ("y", y), ("dh", dh), ("dwd", dwd), ("dx", grads[0]), ("dw", grads[1]), ("db", grads[2])):
        assert np.array_equal(o[name].into_array(), t.into_array()), name
    check(ag.lib.agh_sync())
    check(ag.lib.agh_graph_begin())
    try:
        step()
    finally:
        graph = C.c_void_p()
        check(ag.lib.agh_graph_end(C.byref(graph)))
    for i in range(3):
        new = as_type(rng.standard_normal((m, k)) * (i + 1), dtype)[0]
        check(ag.lib.agh_memcpy_h2d(P(tx), new.ctypes.data, new.nbytes))
        check(ag.lib.agh_sync())
        for t in o.values():
            check(ag.lib.agh_memset(t._ptr(), 0xFF, t.buffer.nbytes))
        check(ag.lib.agh_graph_launch(graph))
        got = {name: t.into_array() for name, t in o.items()}
        step()  # eagerly, on the same buffers
        assert all(np.array_equal(t.into_array(), got[name]) for name, t in o.items()), i
    check(ag.lib.agh_graph_destroy(graph))
