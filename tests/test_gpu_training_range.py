"""The operators with a backward pass at the ends of their types' ranges, against the definition in 64 bits."""
import numpy as np
import pytest

import training_reference as R
from minml_amd import core as ml
from test_gpu_gated import space

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows", [2, 40, 64, 65, 200])
def test_an_infinite_gradient_of_the_gated_layer_stays_infinite(ctx, rows):
    """relu with both projections positive: d of that unit is +inf twice, and with both its rows of weights alike dx is an infinity of their signs, in its row alone; for any number of rows."""
    rng = np.random.default_rng(rows)
    features, hidden = 72, 40
    x, w = rng.standard_normal((rows, features)), rng.standard_normal((2, hidden, features)) / 8
    w[1, 7] = w[0, 7]
    p, dy = rng.standard_normal((rows, 2, hidden)), rng.standard_normal((rows, hidden))
    p[1, :, 7] = 2.0
    x, w, p, dy = (R.bits(a, "float16") for a in (x, w, p, dy))
    dy[1, 7] = 0x7c00
    X, W, P, DY = (ml.toDevice(ctx, a) for a in (x, w, p, dy))
    dx = ml.Tensor((rows, features), "float16")
    ml.gatedDenseBackward(ctx, X, W, P, DY, 0.0, dx, 0.0, None, None, "relu", space(ctx, X, W, True))
    got = R.numbers(dx.copyToHost(ctx))
    finite = [R.numbers(a) for a in (x, w, p, dy)]
    assert (np.abs(finite[1][0, 7]) > 0).all()
    assert np.array_equal(got[1], np.copysign(np.inf, finite[1][0, 7]))
    others = np.arange(rows) != 1
    args = finite[0][others], finite[1], finite[2][others], finite[3][others], "relu"
    assert R.worst(got[others], R.gated_gradients(*args)[0], R.gated_gradient_bounds(*args, "float16")[0]) <= 1
