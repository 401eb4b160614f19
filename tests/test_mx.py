"""MXFP4: quantisation along either axis, its inverse and the product, against the definition in 64 bits (tests/mxfp4.py).

Codes, scales and dequantised values are compared for equality.  A product's tolerance: within a block the products of two codes are multiples of
1/4 below 36 * 32, exact in f32; a step of 128 along k adds its four blocks to the running sum, each of these at most five additions off by no
more than a step of f32 (2^-23, should the hardware cut instead of round) of at most sum |a b|; bias one more, and the result half a step of
its type (2^-24, 2^-8 of its size)."""
import ctypes as C
import types

import numpy as np
import pytest

import mxfp4
import oracle as orc

gpu = pytest.mark.gpu
STEP = {"f32": 2.0**-24, "bf16": 2.0**-8}


@pytest.fixture(scope="module")
def ag():
    import autograph_amd as ag
    ag.Device(0)
    return ag


def as_type(a, dtype):
    """(what the framework takes, the same values in f64)"""
    a = np.asarray(a, dtype=np.float32)
    if dtype == "f32":
        return a, a.astype(np.float64)
    b = orc.f32_to_bf16(a)
    return b, orc.bf16_to_f32(b).astype(np.float64)


def values_of(t):
    a = t.into_array()
    return (orc.bf16_to_f32(a) if t.dtype == "bf16" else a).astype(np.float64)


def some(rng, shape):
    """Values of many sizes: blocks of different scales, zeros among them, one block of zeros where there is room."""
    x = rng.standard_normal(shape) * np.exp2(rng.integers(-20, 20, shape[:-1] + (1,)))
    x *= np.exp2(rng.integers(-3, 4, shape))
    x[rng.random(shape) < 0.1] = 0
    if shape[-1] > 64:
        x[0, 32:64] = 0
    return x


def check_product(got, a, b, dtype, bias=None, relu=False):
    """a [m, k], b [n, k]: f64 values of the operands."""
    want, size = a @ b.T, np.abs(a) @ np.abs(b).T
    if bias is not None:
        want, size = want + bias, size + np.abs(bias)
    if relu:
        want = np.maximum(want, 0)
    steps = -(-a.shape[1] // 128)
    off = np.abs(got - want)
    assert np.all(off <= (5 * steps + 2) * 2.0**-23 * size + STEP[dtype] * np.abs(want) * 1.01 + 1e-38), (off.max(), a.shape, b.shape)


# ---- without a GPU ----


def fake(monkeypatch):
    from autograph_amd import tensor
    monkeypatch.setattr(tensor, "Buffer", lambda nbytes: types.SimpleNamespace(ptr=0, nbytes=nbytes))
    return tensor


def test_buffer_sizes():
    from autograph_amd import MxTensor, _ffi
    a, b = C.c_size_t(), C.c_size_t()
    for rows, k in ((0, 0), (0, 5), (5, 0), (1, 1), (16, 128), (17, 129), (64, 32), (65, 4096), (100000, 100001)):
        assert _ffi.lib.agh_mxfp4_bytes(rows, k, C.byref(a), C.byref(b)) == 0
        steps = -(-k // 128)
        assert (a.value, b.value) == (-(-rows // 16) * steps * 1024, -(-rows // 64) * steps * 256)
    for rows, k, code in ((-1, 4, -1), (4, -1, -1), (2**31, 4, -4), (4, 2**31, -4)):
        assert _ffi.lib.agh_mxfp4_bytes(rows, k, C.byref(a), C.byref(b)) == code
    assert _ffi.lib.agh_mxfp4_bytes(1, 1, None, C.byref(b)) == -3
    assert MxTensor


def test_sizes_that_a_launch_cannot_count():
    """2^24 pieces of 64 rows x 128 values, a workgroup of 256 each, are the first that do not fit (64 x (2^31 - 513) is 2^24 - 4 of
    them); refused before memory is asked for."""
    from autograph_amd import _ffi
    a, b = C.c_size_t(), C.c_size_t()
    for rows, k, code in ((2**30 - 64, 128, 0), (2**30 - 63, 128, -4), (2**30, 128, -4), (64, 2**31 - 513, 0), (65, 2**31 - 513, -4), (64 * 4095, 128 * 4096, 0), (64 * 4096, 128 * 4096, -4)):
        assert _ffi.lib.agh_mxfp4_bytes(rows, k, C.byref(a), C.byref(b)) == code, (rows, k)


@pytest.mark.parametrize("rows,k", [(1, 1), (16, 128), (70, 300), (130, 33)])
def test_places_do_not_overlap(rows, k):
    from autograph_amd import MxTensor
    codes, scales = MxTensor._places(rows, k)
    steps = -(-k // 128)
    assert len(np.unique(codes)) == codes.size == rows * -(-k // 32) and (codes % 16 == 0).all()
    assert codes.min() >= 0 and codes.max() + 16 <= -(-rows // 16) * steps * 1024
    assert len(np.unique(scales)) == scales.size and scales.min() >= 0 and scales.max() < -(-rows // 64) * steps * 256


def test_refusals_in_python(monkeypatch):
    tensor = fake(monkeypatch)
    from autograph_amd import AghError, Dense, MxDense, MxTensor, Tensor
    t = Tensor.uninit((4, 8), "f32")
    for axis in (2, -1, None):
        with pytest.raises(AghError):
            t.quantize_mxfp4(axis)
    with pytest.raises(AghError):
        Tensor.uninit((4, 8, 2), "f32").quantize_mxfp4()
    a, b = MxTensor.uninit((4, 8), 1), MxTensor.uninit((8, 5), 0)
    for left, right in ((a, b.t()), (b, a), (a.t(), b), (a, MxTensor.uninit((9, 5), 0)), (a, MxTensor.uninit((8, 5), 1))):
        with pytest.raises(AghError):
            left.dot(right)
    for kw in ({"dtype": "f16"}, {"bias": Tensor.uninit((5,), "f32"), "dtype": "bf16"}, {"bias": Tensor.uninit((4,), "bf16")}, {"bias": Tensor.uninit((1, 5), "bf16")}):
        with pytest.raises(AghError):
            a.dot(b, **kw)
    with pytest.raises(AghError):
        a.dequantize("f16")
    with pytest.raises(AghError):
        MxDense(b.t())
    for layer, x in ((MxDense(b), Tensor.uninit((4, 9), "f32")), (MxDense(b), Tensor.uninit((8,), "f32")),
                     (MxDense(b, Tensor.uninit((5,), "bf16")), Tensor.uninit((4, 8), "f32")), (MxDense(b, Tensor.uninit((6,), "f32")), Tensor.uninit((4, 8), "f32"))):
        with pytest.raises(AghError):
            layer.forward(x)
    for codes, scales, axis in ((np.zeros((4, 40), np.uint8), np.zeros((4, 1), np.uint8), 1), (np.full((4, 8), 16, np.uint8), np.zeros((4, 1), np.uint8), 1),
                                (np.zeros((4, 8), np.int64), np.zeros((4, 1), np.uint8), 1), (np.zeros((4, 8), np.uint8), np.zeros((4, 1), np.uint8), 0),
                                (np.zeros(8, np.uint8), np.zeros(1, np.uint8), 1), (np.zeros((4, 8), np.uint8), np.zeros((4, 1), np.uint8), 2)):
        with pytest.raises(AghError):
            MxTensor.from_arrays(codes, scales, axis)
    assert tensor.MxTensor is MxTensor and Dense


def test_the_oracle():
    """The definition against hand-made blocks: the borders between codes, saturation, the scale of each power of two."""
    x = np.zeros((1, 32))
    x[0, :16] = [6, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5, 0.2500001, 0.7499999, 1.2500001, 1.7499999, 2.5000001, 3.4999999, 5.0000001, 7.99]
    x[0, 16:] = -x[0, :16]
    want = [6, 0, 1, 1, 2, 2, 4, 4, 0.5, 0.5, 1.5, 1.5, 3, 3, 6, 6]
    codes, scales = mxfp4.quantize(x)
    assert scales[0, 0] == 127 and mxfp4.values(codes, scales)[0].tolist() == want + [-w for w in want]
    for e in range(-149, 128):
        _, s = mxfp4.quantize(np.full((1, 1), np.ldexp(1.0, e)))
        assert s[0, 0] == max(0, e - 2 + 127)


# ---- on the GPU ----

SHAPES = [(1, 1), (1, 32), (3, 31), (16, 128), (17, 129), (64, 127), (65, 64), (5, 1001), (130, 300), (200, 33), (257, 259), (33, 530), (128, 256)]


@gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("shape", SHAPES)
def test_quantize(ag, dtype, shape):
    rng = np.random.default_rng(shape[0] * 1000 + shape[1])
    raw, x = as_type(some(rng, shape), dtype)
    t = ag.Tensor.from_array(raw)
    for axis, ref in ((1, x), (0, x.T)):
        codes, scales = mxfp4.quantize(ref)
        if axis == 0:
            codes, scales = codes.T, scales.T
        q = t.quantize_mxfp4(axis)
        got = q.into_arrays()
        assert q.shape == shape and np.array_equal(got[0], codes) and np.array_equal(got[1], scales)
        want = mxfp4.round_trip(ref)
        for out in ("f32", "bf16"):
            assert np.array_equal(values_of(q.dequantize(out)), want if axis == 1 else want.T)
            assert np.array_equal(values_of(q.t().dequantize(out)), want.T if axis == 1 else want)
        back = ag.MxTensor.from_arrays(*got, axis=axis)
        assert np.array_equal(values_of(back.dequantize("f32")), want if axis == 1 else want.T)


@gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_quantize_borders(ag, dtype):
    """Every border between two codes and its neighbours, under scales from the smallest to the largest, of both signs."""
    near = [b * (1 + d) for b in list(mxfp4.BETWEEN) + list(mxfp4.VALUES) + [7, 7.5] for d in (0, -2.0**-7, 2.0**-7, -2.0**-22, 2.0**-22)]
    block = np.zeros((len(near) + 30) // 31 * 32)
    for i, v in enumerate(near):
        block[i // 31 * 32 + 1 + i % 31] = v if i % 2 else -v
    block[::32] = 4
    x = np.concatenate([[np.ldexp(block, e)] for e in list(range(-151, -118)) + list(range(-8, 8)) + list(range(120, 126))])
    x = np.clip(x, -3.4028235e38, 3.4028235e38)
    raw, ref = as_type(x, dtype)
    ref = np.where(np.isfinite(ref), ref, np.inf)
    for view, axis in ((ag.Tensor.from_array(raw), 1), (ag.Tensor.from_array(np.ascontiguousarray(raw.T)).t(), 1)):
        got = view.quantize_mxfp4(axis).into_arrays()
        want = mxfp4.quantize(ref)
        assert np.array_equal(got[1], want[1])
        assert np.array_equal(got[0], want[0])


@gpu
def test_dequantize_every_code_and_scale(ag):
    """All codes under all scale bytes, by rows, by columns and into a strided matrix: exact in both types, subnormal values too."""
    codes = np.tile(np.arange(16, dtype=np.uint8), (256, 6))[:, :90]
    scales = np.repeat(np.arange(256, dtype=np.uint8)[:, None], 3, 1)
    want = mxfp4.values(codes, scales)
    want = np.where(np.abs(want) >= 2.0**128, np.copysign(np.inf, want), want)
    for q, ref in ((ag.MxTensor.from_arrays(codes, scales), want), (ag.MxTensor.from_arrays(codes.T, scales.T, axis=0), want.T)):
        for dtype in ("f32", "bf16"):
            assert np.array_equal(values_of(q.dequantize(dtype)), ref, equal_nan=True)
            assert np.array_equal(values_of(q.t().dequantize(dtype)), ref.T, equal_nan=True)
    wide = ag.Tensor.zeros((256 * 2, 90 * 3), "f32")
    q = ag.MxTensor.from_arrays(codes, scales)
    ag._ffi.check(ag.lib.agh_dequantize_mxfp4_f32(q.codes.ptr, q.scales.ptr, 256, 90, wide._ptr(), 5, 2 * 270, 3))
    got = wide.into_array().ravel()
    at = 5 + np.arange(256)[:, None] * 540 + np.arange(90)[None, :] * 3
    assert np.array_equal(got[at].astype(np.float64), want, equal_nan=True)
    got[at] = 0
    assert not got.any()


@gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_quantize_infinities_and_nan(ag, dtype):
    rng = np.random.default_rng(3)
    x = rng.standard_normal((20, 200))
    x[2, 5], x[3, 199], x[4, 64], x[19, 33] = np.inf, np.nan, -np.inf, np.nan
    raw, ref = as_type(x, dtype)
    q = ag.Tensor.from_array(raw).quantize_mxfp4()
    codes, scales = q.into_arrays()
    want = mxfp4.quantize(ref)
    assert np.array_equal(scales, want[1]) and (scales == 255).sum() == 4
    assert np.array_equal(values_of(q.dequantize("bf16")), mxfp4.values(*want), equal_nan=True)
    # a product: the rows with such a block are NaN, the others untouched
    w = as_type(rng.standard_normal((50, 200)), dtype)
    got = values_of(q.dot(ag.Tensor.from_array(w[0]).t().quantize_mxfp4(axis=0), dtype="f32"))
    bad = np.zeros(20, bool)
    bad[[2, 3, 4, 19]] = True
    assert np.isnan(got[bad]).all()
    check_product(got[~bad], mxfp4.round_trip(ref[~bad]), mxfp4.round_trip(w[1]), "f32")
    # relu keeps what is >= 0: NaN is not
    got = values_of(q.dot(ag.Tensor.from_array(w[0]).t().quantize_mxfp4(axis=0), relu=True, dtype="f32"))
    assert (got[bad] == 0).all()


@gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_quantize_views(ag, dtype):
    """Offsets, every second row or column, reversed rows, one row for all."""
    rng = np.random.default_rng(4)
    raw, x = as_type(rng.standard_normal((90, 77)), dtype)
    t = ag.Tensor.from_array(raw)
    for view, ref in ((t.slice_rows(3, 80), x[3:80]), (t.slice_rows(1, 90, 2), x[1:90:2]), (t.slice_rows(None, None, -1), x[::-1]), (t.t().slice_rows(5, 70, 3), x.T[5:70:3]),
                      (t.slice_rows(7, 8).broadcast((40, 77)), np.repeat(x[7:8], 40, 0)), (t.t().slice_rows(2, 60, 2).t(), x[:, 2:60:2])):
        for axis in (0, 1):
            want = mxfp4.round_trip(ref) if axis == 1 else mxfp4.round_trip(ref.T).T
            assert np.array_equal(values_of(view.quantize_mxfp4(axis).dequantize("f32")), want)


MNK = [(1, 1, 1), (1, 16, 32), (1, 4096, 96), (2, 33, 129), (16, 64, 128), (17, 5, 300), (33, 100, 64), (64, 64, 513), (100, 10, 84), (129, 257, 256), (300, 65, 1000),
       (257, 520, 40), (1, 1000, 5000), (31, 700, 2049)]


@gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("m,n,k", MNK)
def test_dot(ag, dtype, m, n, k):
    rng = np.random.default_rng(m * n + k)
    a = as_type(rng.standard_normal((m, k)) * np.exp2(rng.integers(-6, 6, (m, 1))), dtype)
    b = as_type(rng.standard_normal((k, n)), dtype)
    bias = as_type(rng.standard_normal(n) * 3, dtype)
    qa, qb = mxfp4.round_trip(a[1]), mxfp4.round_trip(b[1].T)
    ta, tb, tbias = ag.Tensor.from_array(a[0]).quantize_mxfp4(), ag.Tensor.from_array(b[0]).quantize_mxfp4(axis=0), ag.Tensor.from_array(bias[0])
    plain = ta.dot(tb, dtype=dtype)
    assert plain.shape == (m, n) and plain.dtype == dtype
    check_product(values_of(plain), qa, qb, dtype)
    fused = ta.dot(tb, bias=tbias, relu=True, dtype=dtype)
    check_product(values_of(fused), qa, qb, dtype, bias[1], True)
    # the layer quantises its input itself: the same bits
    layer = ag.Dense(ag.Tensor.from_array(b[0]), tbias).quantize_mxfp4()
    x = ag.Tensor.from_array(a[0])
    assert np.array_equal(layer.forward(x, relu=True).into_array(), fused.into_array())
    assert np.array_equal(ag.MxDense(tb).forward(x).into_array(), plain.into_array())
    # and a column-major input too
    xt = ag.Tensor.from_array(np.ascontiguousarray(a[0].T)).t()
    assert np.array_equal(layer.forward(xt, relu=True).into_array(), fused.into_array())


@gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("m,n,k", [(9, 7703, 1100), (16, 20001, 130), (1, 20001, 70), (45, 709, 3111), (300, 2390, 2500), (1000, 2900, 300), (4132, 1193, 47), (1813, 6715, 60),
                                   (4183, 3204, 894)])
def test_dot_every_tile(ag, dtype, m, n, k):
    """Sizes for which the wider tiles are chosen, in order 32x16, 16x32, 32x64, 128x128 and 256x256, ragged in every direction."""
    test_dot(ag, dtype, m, n, k)


@gpu
def test_dot_is_exact_where_f32_is(ag):
    """Integers as codes: every sum below 2^24, so every result equals the integer product, whatever the order."""
    rng = np.random.default_rng(8)
    for m, n, k in ((5, 70, 1000), (200, 300, 640), (1, 129, 4096)):
        a, b = rng.choice([-4, -3, -2, -1, 0, 1, 2, 3, 4], (m, k)), rng.choice([-4, -2, -1, 0, 1, 2, 3, 4], (n, k))
        a[:, ::32] = 4  # the scale 1 in every block
        b[:, ::32] = 4
        got = ag.Tensor.from_array(a.astype(np.float32)).quantize_mxfp4().dot(ag.Tensor.from_array(b.astype(np.float32)).quantize_mxfp4().t(), dtype="f32")
        assert np.array_equal(got.into_array(), (a @ b.T).astype(np.float32))


@gpu
def test_dot_scales_to_the_ends(ag):
    """Scale bytes from 0 to 254: products that f32 holds are right, those beyond it are infinities, those below it zero or subnormal."""
    scales = np.array([[0], [1], [64], [127], [190], [254]], np.uint8)
    codes = np.full((6, 32), 2, np.uint8)  # ones
    q = ag.MxTensor.from_arrays(codes, scales)
    got = q.dot(q.t(), dtype="f32").into_array().astype(np.float64)
    want = 32 * np.ldexp(1.0, scales.astype(int) - 127) * np.ldexp(1.0, scales.astype(int) - 127).T
    big, small = want >= 2.0**128, want < 2.0**-126
    assert np.array_equal(got[~big & ~small], want[~big & ~small])
    assert np.isinf(got[big]).all() and (np.abs(got[small]) <= 2.0**-126).all()


@gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_empty(ag, dtype):
    z = lambda r, c: ag.Tensor.zeros((r, c), dtype)  # noqa: E731
    assert z(0, 5).quantize_mxfp4().dequantize(dtype).shape == (0, 5)
    assert z(5, 0).quantize_mxfp4().dot(z(0, 4).quantize_mxfp4(axis=0), dtype=dtype).into_array().tolist() == [[0] * 4] * 5
    bias = as_type([1.5, -2, 0, 3], dtype)
    got = z(3, 0).quantize_mxfp4().dot(z(0, 4).quantize_mxfp4(axis=0), bias=ag.Tensor.from_array(bias[0]), relu=True, dtype=dtype)
    assert values_of(got).tolist() == [[1.5, 0, 0, 3]] * 3
    got = ag.Dense(z(0, 4), ag.Tensor.from_array(bias[0])).quantize_mxfp4().forward(z(2, 0))
    assert values_of(got).tolist() == [[1.5, -2, 0, 3]] * 2
    assert z(0, 7).quantize_mxfp4().dot(z(7, 4).quantize_mxfp4(axis=0), dtype=dtype).shape == (0, 4)


@gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("m,n,k", [(3, 40, 70), (70, 33, 200), (140, 300, 128)])
def test_strided_output_and_bias(ag, dtype, m, n, k):
    """c by columns and in a wider matrix, a bias of every second element: what lies between stays as it was."""
    rng = np.random.default_rng(9)
    a, b, bias = as_type(rng.standard_normal((m, k)), dtype), as_type(rng.standard_normal((n, k)), dtype), as_type(rng.standard_normal(2 * n), dtype)
    qa, qb = ag.Tensor.from_array(a[0]).quantize_mxfp4(), ag.Tensor.from_array(b[0]).quantize_mxfp4()
    tb = ag.Tensor.from_array(bias[0])
    want = values_of(qa.dot(qb.t(), bias=ag.Tensor.from_array(np.ascontiguousarray(bias[0][1::2])), dtype=dtype))
    fill = as_type(np.full((m + 2) * (n + 3), 7.0), dtype)[0]
    fn = getattr(ag.lib, f"agh_gemm_mxfp4_{dtype}")
    for rsc, csc, off in ((n + 3, 1, 1), (1, m + 2, 2), (-(n + 3), 1, (m - 1) * (n + 3) + 2)):
        out = ag.Tensor.from_array(fill)
        ag._ffi.check(fn(m, k, n, qa.codes.ptr, qa.scales.ptr, qb.codes.ptr, qb.scales.ptr, out._ptr(), off, rsc, csc, tb._ptr(), 1, 2, 0))
        got = values_of(out)
        at = off + np.arange(m)[:, None] * rsc + np.arange(n)[None, :] * csc
        assert np.array_equal(got[at], want)
        rest = np.ones(got.size, bool)
        rest[at.ravel()] = False
        assert (got[rest] == 7).all()


@gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("m,n,k", [(300, 2390, 2500), (1000, 2900, 300), (1813, 6715, 60), (1813, 6720, 60)])
def test_strided_output_of_wide_tiles(ag, dtype, m, n, k):
    test_strided_output_and_bias(ag, dtype, m, n, k)


@gpu
def test_refusals_of_the_library(ag):
    lib = ag.lib
    t = ag.Tensor.zeros((64, 64), "f32")
    q = t.quantize_mxfp4()
    c, s, x = q.codes.ptr, q.scales.ptr, t._ptr()
    for args, code in (((x, 0, 64, 1, -1, 64, c, s), -1), ((x, 0, 64, 1, 64, 2**31, c, s), -4), ((None, 0, 64, 1, 64, 64, c, s), -3), ((x, 0, 64, 1, 64, 64, None, s), -3),
                       ((x, 0, 64, 1, 64, 64, c + 8, s), -1), ((x, 0, 64, 1, 64, 64, c, s + 2), -1)):
        assert lib.agh_quantize_mxfp4_f32(*args) == code
    for args, code in (((c, s, 64, 64, None, 0, 64, 1), -3), ((c, s, 64, 64, x, 0, 0, 1), -1), ((c, s, 64, 64, x, 0, 64, 0), -1), ((c, None, 64, 64, x, 0, 64, 1), -3),
                       ((c, s, 64, -1, x, 0, 64, 1), -1)):
        assert lib.agh_dequantize_mxfp4_f32(*args) == code
    good = [64, 64, 64, c, s, c, s, x, 0, 64, 1, None, 0, 0, 0]
    for at, value, code in ((0, -1, -1), (1, 2**31, -4), (2, 2**31, -4), (3, None, -3), (6, None, -3), (3, c + 4, -1), (7, None, -3), (9, 0, -1), (10, 0, -1), (14, 2, -1)):
        assert lib.agh_gemm_mxfp4_f32(*good[:at], value, *good[at + 1:]) == code, at
    good = [64, 64, 64, x, 0, 64, 1, c, s, x, 0, 64, 1, None, 0, 0, 0]
    for at, value, code in ((0, -1, -1), (3, None, -3), (7, None, -3), (8, s + 1, -1), (9, None, -3), (11, 0, -1), (16, -1, -1)):
        assert lib.agh_dense_mxfp4_f32(*good[:at], value, *good[at + 1:]) == code, at
    assert values_of(t).tolist() == np.zeros((64, 64)).tolist()  # nothing was launched


@gpu
def test_capture_and_replay(ag):
    """A layer captured after an eager run, replayed with other inputs, larger eager calls (which outgrow the workspace) in between."""
    rng = np.random.default_rng(11)
    layers = {}
    for m, k, n in ((1, 300, 200), (200, 512, 700)):
        w = rng.standard_normal((k, n)).astype(np.float32)
        layer = ag.Dense(ag.Tensor.from_array(w)).quantize_mxfp4()
        x, y = ag.Tensor.zeros((m, k), "f32"), ag.Tensor.zeros((m, n), "f32")
        args = (m, k, n, x._ptr(), 0, k, 1, layer.weight.codes.ptr, layer.weight.scales.ptr, y._ptr(), 0, n, 1, None, 0, 0, 0)
        ag._ffi.check(ag.lib.agh_dense_mxfp4_f32(*args))
        ag._ffi.check(ag.lib.agh_sync())
        ag._ffi.check(ag.lib.agh_graph_begin())
        ag._ffi.check(ag.lib.agh_dense_mxfp4_f32(*args))
        g = C.c_void_p()
        ag._ffi.check(ag.lib.agh_graph_end(C.byref(g)))
        layers[m] = (layer, x, y, g)
    for i in range(4):
        new = {m: rng.standard_normal(x.shape).astype(np.float32) for m, (_, x, _, _) in layers.items()}
        for m, (layer, x, y, g) in layers.items():
            ag._ffi.check(ag.lib.agh_memcpy_h2d(x._ptr(), new[m].ctypes.data, new[m].nbytes))
            ag._ffi.check(ag.lib.agh_sync())
        for m, (layer, x, y, g) in layers.items():
            ag._ffi.check(ag.lib.agh_graph_launch(g))
        big = ag.Dense(ag.Tensor.zeros((4096, 64), "f32")).quantize_mxfp4().forward(ag.Tensor.zeros((2048 << i, 4096), "f32"))
        for m, (layer, x, y, g) in layers.items():
            assert np.array_equal(y.into_array(), layer.forward(ag.Tensor.from_array(new[m])).into_array()), (m, i)
        assert not big.into_array().any()
    for _, _, _, g in layers.values():
        ag._ffi.check(ag.lib.agh_graph_destroy(g))


@gpu
def test_two_streams(ag):
    """Layers in a branch and beside it: each stream has a workspace of its own."""
    rng = np.random.default_rng(12)
    layers = [ag.Dense(ag.Tensor.from_array(rng.standard_normal((1024, 512)).astype(np.float32))).quantize_mxfp4() for _ in range(2)]
    xs = [ag.Tensor.from_array(rng.standard_normal((300, 1024)).astype(np.float32)) for _ in range(2)]
    want = [layer.forward(x).into_array() for layer, x in zip(layers, xs)]
    for _ in range(5):
        with ag.branch():
            side = [layers[1].forward(xs[1]) for _ in range(4)]
        main = [layers[0].forward(xs[0]) for _ in range(4)]
        ag.join()
        assert all(np.array_equal(y.into_array(), want[0]) for y in main) and all(np.array_equal(y.into_array(), want[1]) for y in side)


@gpu
def test_codes_beyond_32_bits(ag):
    """140000 rows of 65536: codes behind 4 GiB.  The matrix is a view whose element (r, c) is r + c places into a short vector."""
    rng = np.random.default_rng(13)
    rows, k = 140000, 65536
    base = rng.standard_normal(rows + k).astype(np.float32)
    t = ag.Tensor(ag.Tensor.from_array(base).buffer, (rows, k), (1, 1), 0, "f32")
    q = t.quantize_mxfp4()
    assert q.codes.nbytes > 2**32
    x = ag.Tensor.from_array(rng.standard_normal((2, k)).astype(np.float32))
    got = values_of(x.quantize_mxfp4().dot(q.t(), dtype="f32"))
    a = mxfp4.round_trip(x.into_array().astype(np.float64))
    for r in (0, 1, 65535, 65536, 131071, 131072, 139998, 139999):
        check_product(got[:, r:r + 1], a, mxfp4.round_trip(base[None, r:r + k].astype(np.float64)), "f32")
    # and with the long matrix on the left
    got = values_of(q.dot(x.quantize_mxfp4().t(), dtype="f32"))
    for r in (0, 65536, 131072, 139999):
        check_product(got[r:r + 1], mxfp4.round_trip(base[None, r:r + k].astype(np.float64)), a, "f32")
