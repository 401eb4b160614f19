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
