"""Layer norm with one of its two parameters or neither: which gradients a layer returns, and what the kernels form without a weight."""
import types

import numpy as np
import pytest

from test_layer_norm import ag, as_type, backward, check_backward, make, values_of  # noqa: F401

gpu = pytest.mark.gpu


@pytest.mark.parametrize("has_weight,has_bias", [(True, True), (True, False), (False, True), (False, False)])
def test_what_the_layer_asks_for(monkeypatch, has_weight, has_bias):
    """Without a device: a gradient for each parameter that the layer has, and no other."""
    from autograph_amd import LayerNorm, tensor
    ptr = iter(range(1, 1000))
    monkeypatch.setattr(tensor, "Buffer", lambda nbytes: types.SimpleNamespace(ptr=next(ptr), nbytes=nbytes))
    made = []
    monkeypatch.setattr(tensor, "calls", types.SimpleNamespace(agh_layer_norm_backward_f32=lambda *a: made.append(a)))
    u = tensor.Tensor.uninit
    x, dy, v, s = u((4, 8), "f32"), u((4, 8), "f32"), u((8,), "f32"), u((4,), "f32")
    layer = LayerNorm(v if has_weight else None, u((8,), "f32") if has_bias else None)
    dx, dw, db = layer.backward(x, dy, s, s)
    (args,) = made
    assert (dx.shape, dw is not None, db is not None) == ((4, 8), has_weight, has_bias)
    assert [a is not None for a in args[:8]] == [True, True, has_weight, True, True, True, has_weight, has_bias]
    # of the tensor's own call: as the weight is there or not, unless it is said
    assert [t is not None for t in x.layer_norm_backward(dy, v, s, s)] == [True, True, True]
    assert [t is not None for t in x.layer_norm_backward(dy, None, s, s)] == [True, False, False]
    assert [t is not None for t in x.layer_norm_backward(dy, None, s, s, bias=True)] == [True, False, True]
    assert [t is not None for t in x.layer_norm_backward(dy, v, s, s, bias=False)] == [True, True, False]


@gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows,cols", [(12, 100), (300, 1000), (7, 9000), (3, 66000)])
def test_gradients_of_the_parameters_that_are_there(ag, dtype, rows, cols):  # noqa: F811
    rng = np.random.default_rng(31)
    x, w, b, dy = make(rng, rows, cols, dtype)
    tx, tw, tb, tdy = (ag.Tensor.from_array(v[0]) for v in (x, w, b, dy))
    for weight, bias in ((None, tb), (tw, None), (None, None), (tw, tb)):
        layer = ag.LayerNorm(weight, bias)
        _, mean, rstd = layer.forward_train(tx)
        dx, dw, db = layer.backward(tx, tdy, mean, rstd)
        assert (dw is None, db is None) == (weight is None, bias is None)
        m, r = values_of(mean), values_of(rstd)
        factor = w[1] if weight is not None else np.ones(cols)
        want = backward(x[1], dy[1], factor, m, r)
        # (what is absent is not compared: the wanted value stands in for it)
        check_backward([values_of(dx), want[1] if dw is None else values_of(dw), want[2] if db is None else values_of(db)], x[1], dy[1], factor, m, r, dtype)


@gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows,cols", [(12, 100), (300, 84), (500, 300), (300, 1000), (7, 2049), (7, 9000), (3, 66000)])
def test_both_gradients_without_a_weight(ag, dtype, rows, cols):  # noqa: F811
    """The library's entry forms all three with a null weight, which stands for ones."""
    rng = np.random.default_rng(32)
    x, _, _, dy = make(rng, rows, cols, dtype)
    tx, tdy = ag.Tensor.from_array(x[0]), ag.Tensor.from_array(dy[0])
    _, mean, rstd = tx.layer_norm(stats=True)
    out = [ag.Tensor.uninit(s, dtype) for s in ((rows, cols), (cols,), (cols,))]
    ag._ffi.check(getattr(ag.lib, f"agh_layer_norm_backward_{dtype}")(tx._ptr(), tdy._ptr(), None, mean._ptr(), rstd._ptr(), *[t._ptr() for t in out], rows, cols))
    check_backward([values_of(t) for t in out], x[1], dy[1], np.ones(cols), values_of(mean), values_of(rstd), dtype)


@gpu
def test_the_same_through_the_cpp_host_layer():
    import os
    import subprocess
    binary = os.path.join(os.path.dirname(os.path.abspath(__file__)), "cpp", "layer_norm_parameters_test")
    assert os.path.exists(binary), "tests/cpp/layer_norm_parameters_test has not been built (run __graft_entry__.build())"
    out = subprocess.run([binary, "gpu"], capture_output=True, text=True, timeout=120)
    assert out.returncode == 0 and "gpu ok" in out.stdout, out.stderr + out.stdout
