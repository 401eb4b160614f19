"""MXFP4 on inputs whose rows lie backwards, on top of each other or at odd places, in the launch that quantises its input itself and in the one before the
product; and values at the end of f32."""
import types

import numpy as np
import pytest

import mxfp4
from test_mx import ag, as_type, check_product, values_of  # noqa: F401

gpu = pytest.mark.gpu


@pytest.mark.parametrize("axis", [0, 1])
@pytest.mark.parametrize("shape", [(0, 5), (5, 0), (0, 0), (0, 40), (40, 0)])
def test_arrays_of_nothing(monkeypatch, shape, axis):
    """A matrix without rows or columns has codes of its shape and scales for none of its blocks, both ways; without a device."""
    from autograph_amd import MxTensor, tensor
    monkeypatch.setattr(tensor, "Buffer", lambda nbytes: types.SimpleNamespace(ptr=0, nbytes=nbytes))
    monkeypatch.setattr(tensor, "lib", types.SimpleNamespace(agh_memcpy_d2h=lambda *a: 0, agh_memcpy_h2d=lambda *a: 0, agh_sync=lambda: 0))
    blocks = tuple(-(-n // 32) if a == axis else n for a, n in enumerate(shape))
    assert tuple(a.shape for a in MxTensor.uninit(shape, axis).into_arrays()) == (shape, blocks)
    assert MxTensor.from_arrays(np.zeros(shape, np.uint8), np.zeros(blocks, np.uint8), axis).shape == shape


@gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("m,k,n", [(1, 40, 33), (5, 300, 200), (16, 1000, 700), (30, 129, 90), (64, 256, 256), (200, 300, 900), (700, 515, 1100)])
def test_dense_of_strided_rows(ag, dtype, m, k, n):  # noqa: F811
    """The bits of the quantiser and the product on a copy of the rows in standard layout, which are checked against 64 bits."""
    rng = np.random.default_rng(41)
    w = as_type(rng.standard_normal((k, n)), dtype)
    b = as_type(rng.standard_normal(n), dtype)
    tw, tb = ag.Tensor.from_array(w[0]), ag.Tensor.from_array(b[0])
    qw = tw.quantize_mxfp4(axis=0)
    pitch = k + 7
    store = as_type(rng.standard_normal(m * pitch + 11), dtype)
    ts = ag.Tensor.from_array(store[0])
    fn = getattr(ag.lib, f"agh_dense_mxfp4_{dtype}")
    rows, cols = np.arange(m)[:, None], np.arange(k)[None, :]
    # forwards at an odd place, backwards, one row for all, rows that overlap; and the same with the row itself backwards
    for off, rs in ((3, pitch), ((m - 1) * pitch + 5, -pitch), (1, 0), (2, 1)):
        for first, cs in ((off, 1), (off + k - 1, -1)):
            at = first + rows * rs + cols * cs
            assert at.min() >= 0 and at.max() < store[0].size
            want = ag.Tensor.from_array(np.ascontiguousarray(store[0][at])).quantize_mxfp4().dot(qw, bias=tb, relu=True, dtype=dtype)
            check_product(values_of(want), mxfp4.round_trip(store[1][at]), mxfp4.round_trip(w[1].T), dtype, b[1], True)
            y = ag.Tensor.uninit((m, n), dtype)
            ag._ffi.check(fn(m, k, n, ts._ptr(), first, rs, cs, qw.codes.ptr, qw.scales.ptr, y._ptr(), 0, n, 1, tb._ptr(), 0, 1, 1))
            assert np.array_equal(y.into_array(), want.into_array()), (off, rs, cs)


@gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_the_largest_numbers(ag, dtype):  # noqa: F811
    """What the quantiser makes of the largest numbers is finite in both types: a block's largest code is 6 * 2^125.  (Scale bytes 253 and 254 come from other quantisers only; what
    their codes stand for may be beyond f32, and is an infinity then.)"""
    largest = float(as_type(np.array([3.3895313892515355e38 if dtype == "bf16" else 3.4028234663852886e38]), dtype)[1][0])
    x = as_type(np.array([[largest, -largest] + [2.0**127] * 30, [-1.0] * 31 + [largest]]), dtype)
    q = ag.Tensor.from_array(x[0]).quantize_mxfp4()
    want = mxfp4.quantize(x[1])
    codes, scales = q.into_arrays()
    assert np.array_equal(codes, want[0]) and np.array_equal(scales, want[1]) and scales.max() == 252
    for to in ("f32", "bf16"):
        assert np.array_equal(values_of(q.dequantize(to)), mxfp4.values(*want)) and np.isfinite(values_of(q.dequantize(to))).all()
