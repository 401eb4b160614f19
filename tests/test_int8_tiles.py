"""Every form of the 8-bit integer product's kernels against the definition (tests/int8.py, tests/gated.py): each tile forced at sizes ragged in every direction, and the tiles that
large products take by themselves.

Tolerances as in test_int8: sums are exact; their conversion, the scales' product, the product of both and the bias's addition are four roundings of 2^-24 each, the result half a
step of its type.  A gate's slope is at most 1.13, and gated.gate_error says what the gate adds."""
import re

import numpy as np
import pytest

import gated as gt
import int8
from test_int8 import STEP, as_type, check_product, values_of

gpu = pytest.mark.gpu
ACT = {"none": 0, "relu": 1, "silu": 2, "gelu": 3, "sigmoid": 4}


@pytest.fixture(scope="module")
def ag():
    import autograph_amd as ag
    ag.Device(0)
    return ag


def product(a, b):
    """int8.product by a product in 64-bit floats, which hold every whole sum below 2^53."""
    return (a[0].astype(np.float64) @ b[0].astype(np.float64).T) * a[1].astype(np.float64)[:, None] * b[1].astype(np.float64)


def check_gated(got, v, bias, activation, dtype):
    """v: the products' values in 64 bits, the gate's columns first"""
    n = v.shape[1] // 2
    h, size = (v, np.abs(v)) if bias is None else (v + bias, np.abs(v) + np.abs(bias))
    g, u = h[:, :n], h[:, n:]
    value, _ = gt.gate(g, activation)
    want = value * u
    tolerance = 4 * 2.0**-24 * (1.13 * size[:, :n] * np.abs(u) + size[:, n:] * np.abs(value)) + (gt.gate_error(g, activation) + STEP[dtype] * 1.02) * np.abs(want)
    off = np.abs(got - want)
    assert np.all(off <= tolerance * 1.001 + 1e-37), off.max()


class Result:
    """An m x n result inside a larger matrix of a value that no product here gives: by rows with a gap and at an odd offset, or by columns."""

    def __init__(self, ag, m, n, dtype, by_rows):
        self.ag, self.shape, self.dtype = ag, (m, n), dtype
        self.offset, self.rs, self.cs = (3, n + 5, 1) if by_rows else (7, 2, 2 * m + 1)
        self.size = self.offset + (m - 1) * self.rs + (n - 1) * self.cs + 1 + 64
        self.mark = as_type([-123456.0], dtype)
        self.tensor = ag.Tensor.from_array(np.full(self.size, self.mark[0][0]))

    def values(self):
        """The result's values; nothing beside them has been written."""
        got = values_of(self.tensor)
        at = self.offset + np.arange(self.shape[0])[:, None] * self.rs + np.arange(self.shape[1])[None, :] * self.cs
        out = got[at]
        got[at] = self.mark[1][0]
        assert (got == self.mark[1][0]).all()
        return out


def operands(rng, m, n, k, dtype):
    return (as_type(rng.standard_normal((m, k)) * np.exp2(rng.integers(-6, 6, (m, 1))), dtype), as_type(rng.standard_normal((k, n)) / np.sqrt(k), dtype),
            as_type(rng.standard_normal((n, 2)), dtype))


def test_no_kernel_that_nothing_launches():
    """A gated product of few rows takes one tile of each half a workgroup, never two: the library holds no kernel for that."""
    from autograph_amd import _ffi
    names = set(re.findall(rb"i8_rows_kernelI[ft]Lb([01])ELi(\d+)ELi(\d+)E", open(_ffi.lib._name, "rb").read()))
    assert names == {(b"0", rows, tiles) for rows, tiles in ((b"1", b"1"), (b"1", b"2"), (b"4", b"1"), (b"4", b"2"), (b"16", b"1"))} | {(b"1", rows, b"1") for rows in (b"1", b"4", b"16")}


# steps of 64 along k: 1, 3, 4, 5, 9, 11, 18 and 1, so that the four stages are filled in part, once, and several times with each remainder
SIZES = [(1, 1, 40), (17, 33, 190), (130, 70, 256), (257, 130, 300), (100, 515, 575), (300, 260, 650), (513, 257, 1100), (64, 64, 64)]


@gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("form", range(6))
def test_dot_every_form(ag, monkeypatch, form, dtype):
    """Plain, with bias and relu, and into rows with a gap at an odd offset and into columns, with a bias that has a stride; the layer on few rows gives the same bits."""
    monkeypatch.setenv("AGH_I8_FORM", str(form))
    call = getattr(ag.lib, f"agh_gemm_int8_{dtype}")
    for m, n, k in SIZES:
        a, b, bias = operands(np.random.default_rng(m * n + k), m, n, k, dtype)
        v = product(int8.quantize(a[1]), int8.quantize(b[1].T))
        qa, qb = ag.Tensor.from_array(a[0]).quantize_int8(), ag.Tensor.from_array(b[0]).quantize_int8(axis=0)
        check_product(values_of(qa.dot(qb, dtype=dtype)), v, dtype)
        tb = ag.Tensor.from_array(np.ascontiguousarray(bias[0][:, 1]))
        fused = qa.dot(qb, bias=tb, relu=True, dtype=dtype)
        check_product(values_of(fused), v, dtype, bias[1][:, 1], True)
        assert np.array_equal(ag.I8Dense(qb, tb).forward(ag.Tensor.from_array(a[0]), relu=True).into_array(), fused.into_array())
        strided = ag.Tensor.from_array(bias[0])
        for by_rows in (True, False):
            c = Result(ag, m, n, dtype, by_rows)
            ag._ffi.check(call(m, k, n, qa.codes.ptr, qa.scales.ptr, qb.codes.ptr, qb.scales.ptr, c.tensor._ptr(), c.offset, c.rs, c.cs, strided._ptr(), 1, 2, 1))
            assert np.array_equal(c.values(), values_of(fused)), (m, n, k, by_rows)


@gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("form", range(6))
def test_gated_every_form(ag, monkeypatch, form, dtype):
    monkeypatch.setenv("AGH_I8_FORM", str(form))
    call = getattr(ag.lib, f"agh_gated_dense_int8_{dtype}")
    for i, (m, n, k) in enumerate(SIZES):
        activation = gt.ACTIVATIONS[i % len(gt.ACTIVATIONS)]
        x, w, bias = operands(np.random.default_rng(m * n + k), m, 2 * n, k, dtype)
        v = product(int8.quantize(x[1]), int8.quantize(w[1].T))
        tx, tb = ag.Tensor.from_array(x[0]), ag.Tensor.from_array(np.ascontiguousarray(bias[0][:, 1]))
        layer = ag.GatedDense(ag.Tensor.from_array(w[0]), tb, activation).quantize_int8()
        y = layer.forward(tx)
        check_gated(values_of(y), v, bias[1][:, 1], activation, dtype)
        check_gated(values_of(ag.I8GatedDense(layer.gate, layer.up, None, activation).forward(tx)), v, None, activation, dtype)
        strided = ag.Tensor.from_array(bias[0])
        for by_rows in (True, False):
            c = Result(ag, m, n, dtype, by_rows)
            ag._ffi.check(call(m, k, n, tx._ptr(), 0, k, 1, layer.gate.codes.ptr, layer.gate.scales.ptr, layer.up.codes.ptr, layer.up.scales.ptr, c.tensor._ptr(), c.offset, c.rs, c.cs,
                               strided._ptr(), 1, 2, ACT[activation]))
            assert np.array_equal(c.values(), values_of(y)), (m, n, k, by_rows)


@gpu
def test_a_form_that_does_not_exist(ag, monkeypatch):
    q = ag.Tensor.zeros((20, 64), "f32").quantize_int8()
    monkeypatch.setenv("AGH_I8_FORM", "6")
    with pytest.raises(ag.AghError):
        q.dot(q.t(), dtype="f32")
    monkeypatch.delenv("AGH_I8_FORM")
    assert not q.dot(q.t(), dtype="f32").into_array().any()


@gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("m,n,k", [(1999, 1001, 2047), (3001, 2050, 650), (4099, 8200, 2000)])
def test_large_products(ag, dtype, m, n, k):
    """Sizes for which tiles of 128x64, 128x128 and 256x256 are the choice on 256 CUs (gated 64x128 for all three)."""
    rng = np.random.default_rng(n)
    x, w, bias = operands(rng, m, n, k, dtype)
    qx, qw = int8.quantize(x[1]), int8.quantize(w[1].T)
    v = product(qx, qw)
    tx, tw, tb = (ag.Tensor.from_array(t) for t in (x[0], w[0], np.ascontiguousarray(bias[0][:, 0])))
    layer = ag.Dense(tw, tb).quantize_int8()
    check_product(values_of(layer.forward(tx, relu=True)), v, dtype, bias[1][:, 0], True)
    if n % 2 == 0:
        gated = ag.GatedDense(tw, tb, "silu").quantize_int8()
        check_gated(values_of(gated.forward(tx)), v, bias[1][:, 0], "silu", dtype)


@gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_large_gated_product(ag, dtype):
    """Sizes for which the gated tile of 128x256 is the choice on 256 CUs."""
    m, n, k = 4096, 4096, 2048
    x, w, bias = operands(np.random.default_rng(1), m, 2 * n, k, dtype)
    layer = ag.GatedDense(ag.Tensor.from_array(w[0]), ag.Tensor.from_array(np.ascontiguousarray(bias[0][:, 0])), "gelu").quantize_int8()
    got = values_of(layer.forward(ag.Tensor.from_array(x[0])))
    rows = np.concatenate((np.arange(0, m, 7), np.arange(m - 20, m)))  # (the oracle's erfc is slow; every column, rows of every tile)
    v = product(tuple(t[rows] for t in int8.quantize(x[1])), int8.quantize(w[1].T))
    check_gated(got[rows], v, bias[1][:, 0], "gelu", dtype)
