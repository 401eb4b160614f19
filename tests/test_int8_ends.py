"""8-bit integers at the ends of f32: rows whose largest magnitude is f32's largest value, or so small that the scale loses its bits or is 0."""
import numpy as np
import pytest

import int8

pytestmark = pytest.mark.gpu
MOST = np.float32(3.4028235e38)
BELOW = np.float32(float.fromhex("0x1.020406p+121"))


@pytest.fixture(scope="module")
def ag():
    import autograph_amd as ag
    ag.Device(0)
    return ag


def quantised(ag, x):
    """By rows in each of the quantiser's ways: contiguous (1 and 4 rows a workgroup), and columns held, few of them and in shares."""
    t = ag.Tensor.from_array(x)
    many = ag.Tensor.from_array(np.tile(x, (600, 1)))
    yield t.quantize_int8().into_arrays()
    codes, scales = many.quantize_int8().into_arrays()
    yield codes[-len(x):], scales[-len(x):]
    for y in (x, np.pad(x, ((0, 0), (0, 9000)))):
        codes, scales = ag.Tensor.from_array(np.ascontiguousarray(y.T)).t().quantize_int8().into_arrays()
        yield codes[:, :x.shape[1]], scales


@pytest.mark.parametrize("k", [40, 200])
def test_the_largest_value(ag, k):
    """127 times the nearest f32 to a 127th of it is infinity; it comes back as a number, 2^-22 of its size away (half a step of the scale rounded, one step down, the product's half)."""
    x = np.random.default_rng(k).uniform(-1, 1, (4, k)).astype(np.float32) * MOST
    x[0, 3], x[1, k - 1], x[2, 0], x[3, 5] = MOST, -MOST, np.nextafter(MOST, np.float32(0)), MOST
    x[3, 6:] = 0
    want, nearest = int8.quantize(x)
    scales = np.where(np.abs(x).max(1) == MOST, BELOW, nearest)
    with np.errstate(over="ignore"):
        assert np.isinf(np.float32(127) * (MOST / np.float32(127))) and np.isfinite(np.float32(127) * BELOW) and nearest[2] == BELOW
    for codes, got in quantised(ag, x):
        assert np.array_equal(codes, want) and np.array_equal(got, scales)
    q = ag.Tensor.from_array(x).quantize_int8()
    back = q.dequantize("f32").into_array().astype(np.float64)
    assert np.isfinite(back).all() and abs(back[0, 3] / float(MOST) - 1) <= 2.0**-22 and abs(back[1, k - 1] / -float(MOST) - 1) <= 2.0**-22
    # through the products: one by one, in one launch with the quantiser (1 and 4 rows), times the identity in 8 bits (codes of 127 under the scale 1 / 127)
    eye = ag.Tensor.from_array(np.eye(k, dtype=np.float32)).quantize_int8(axis=0)
    v = want.astype(np.float64) * 127 * scales.astype(np.float64)[:, None] * float(np.float32(1) / np.float32(127))
    fits = np.abs(v) < float(MOST) * (1 - 2.0**-22)
    assert (~fits).any()
    for rows in (slice(0, 1), slice(0, 4)):
        t = ag.Tensor.from_array(x[rows])
        for got in (ag.I8Dense(eye).forward(t), t.quantize_int8().dot(eye, dtype="f32")):
            got = got.into_array().astype(np.float64)
            assert np.all((np.abs(got - v[rows]) <= 4 * 2.0**-24 * np.abs(v[rows]))[fits[rows]])


def test_the_smallest_values(ag):
    """Rows from 2^-149 up: codes as ever, the scale the f32 nearest to a 127th of the largest, 0 below 2^-143; values are code times scale."""
    tops = np.concatenate((np.arange(1, 300), 2**np.arange(8, 32))).astype(np.int64)
    x = np.zeros((len(tops), 70), np.float32)
    for i, t in enumerate(tops):
        x[i] = np.ldexp(np.random.default_rng(i).integers(-t, t + 1, 70).astype(np.float64), -149)
        x[i, i % 70] = np.ldexp(float(t), -149)
    want, scales = int8.quantize(x)
    assert (scales[:63] == 0).all() and (scales[63:] > 0).all() and want[:63].any() and float(x[62].max()) < 2.0**-143 <= float(x[63].max())
    for codes, got in quantised(ag, x):
        assert np.array_equal(codes, want) and np.array_equal(got, scales)
    back = ag.Tensor.from_array(x).quantize_int8().dequantize("f32").into_array()
    assert not back[:63].any() and np.all(np.abs(back - int8.values(want, scales)) <= 2.0**-24 * np.abs(back) + 2.0**-150)
