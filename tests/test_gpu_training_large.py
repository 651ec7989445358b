"""The operators with a backward pass on tensors of more than 2^31 elements: places far into them are where they should be. Checked at sampled rows against the definition in 64 bits."""
import numpy as np
import pytest

import training_reference as R
from minml_amd import core as ml

pytestmark = pytest.mark.gpu


def at_rows(ctx, t, rows):
    """Rows of a tensor whose first dimension is the rows', on the host."""
    one = t.shape[1:]
    size = int(np.prod(one))
    return np.stack([t.view(one, r * size).copyToHost(ctx) for r in rows])


def test_layer_norm(ctx):
    """All rows but a few are zeros with no gradient, so the sums over 300 001 rows are those over the few."""
    rng = np.random.default_rng(1)
    rows, columns = 300001, 8192
    picked = [0, 150000, 262144, rows - 2, rows - 1]
    x, dy, out = (ml.Tensor((rows, columns), "float16") for _ in range(3))
    x.zeroall(ctx)
    dy.zeroall(ctx)
    xs, dys = (R.bits(rng.standard_normal((len(picked), columns)), "float16") for _ in range(2))
    for k, r in enumerate(picked):
        for t, a in ((x, xs), (dy, dys)):
            t.view((columns,), r * columns).copyFromHost(ctx, a[k])
    w = R.bits(1 + 0.1 * rng.standard_normal(columns), "float16")
    W, dw, db = ml.toDevice(ctx, w), ml.Tensor((columns,), "float32"), ml.Tensor((columns,), "float32")
    space = ml.Tensor((ml.layerNormGetWorkspaceSize(ctx, x),), "uint8")
    xf, wf, dyf = map(R.numbers, (xs, w, dys))
    ml.layerNormForward(ctx, x, W, None, out)
    assert R.worst(at_rows(ctx, out, picked), R.layer_norm(xf, wf, np.zeros(columns), 1e-5), R.layer_norm_bound(xf, wf, np.zeros(columns), 1e-5, "float16")) <= 1
    ml.layerNormBackward(ctx, x, W, dy, 0.0, out, 0.0, dw, db, space)
    want, bounds, sums = R.layer_norm_gradients(xf, wf, dyf, 1e-5), R.layer_norm_gradient_bounds(xf, wf, dyf, 1e-5, "float16"), R.layer_norm_gradient_bounds(xf, wf, dyf, 1e-5, "float32")
    assert R.worst(at_rows(ctx, out, picked), want[0], bounds[0]) <= 1
    assert R.worst(dw.copyToHost(ctx), want[1], sums[1]) <= 1 and R.worst(db.copyToHost(ctx), want[2], sums[2]) <= 1


def test_gated_dense(ctx):
    rng = np.random.default_rng(2)
    rows, features, hidden = 70001, 16, 16000
    picked = [0, 35000, 67109, rows - 1]
    x, w, b = (R.bits(a, "float16") for a in (rng.standard_normal((rows, features)), rng.standard_normal((2, hidden, features)) / 4, 0.3 * rng.standard_normal((2, hidden))))
    X, W, Bias = (ml.toDevice(ctx, a) for a in (x, w, b))
    y, kept, dx = ml.Tensor((rows, hidden), "float16"), ml.Tensor((rows, 2, hidden), "float16"), ml.Tensor((rows, features), "float16")
    space = ml.Tensor((max(ml.gatedDenseGetWorkspaceSize(ctx, X, W, k) for k in (False, True)),), "uint8")
    ml.gatedDenseForward(ctx, X, W, Bias, y, kept, "silu", space)
    xf, wf, bf = R.numbers(x)[picked], R.numbers(w), R.numbers(b)
    want, bound = R.gated(xf, wf, bf, "silu"), R.gated_bounds(xf, wf, bf, "silu", "float16")
    got = at_rows(ctx, kept, picked)
    assert R.worst(at_rows(ctx, y, picked), want[0], bound[0]) <= 1 and R.worst(got, want[1], bound[1]) <= 1
    ml.gatedDenseBackward(ctx, X, W, kept, y, 0.0, dx, 0.0, None, None, "silu", space)  # the gradient is the output, as of half its squares' sum
    args = xf, wf, R.numbers(got), R.numbers(at_rows(ctx, y, picked)), "silu"
    assert R.worst(at_rows(ctx, dx, picked), R.gated_gradients(*args)[0], R.gated_gradient_bounds(*args, "float16")[0]) <= 1


def test_cross_entropy(ctx):
    rng = np.random.default_rng(3)
    rows, features, classes = 40000, 16, 60000
    picked = [0, 17, 20000, 39999]
    x, w = (R.bits(a, "float16") for a in (rng.standard_normal((rows, features)), rng.standard_normal((classes, features)) / 2))
    targets = rng.integers(0, classes, rows).astype(np.int32)
    X, W, T = (ml.toDevice(ctx, a) for a in (x, w, targets))
    loss, lse, dx = ml.Tensor((rows,), "float32"), ml.Tensor((rows,), "float32"), ml.Tensor((rows, features), "float16")
    dloss = np.ones(rows, np.float32)
    space = ml.Tensor((ml.linearCrossEntropyGetWorkspaceSize(ctx, X, W, True),), "uint8")
    ml.linearCrossEntropyForward(ctx, X, W, None, T, loss, lse, space)
    ml.linearCrossEntropyBackward(ctx, X, W, None, T, lse, ml.toDevice(ctx, dloss), 0.0, dx, 0.0, None, None, space)
    args = R.numbers(x)[picked], R.numbers(w), np.zeros(classes), targets[picked]
    assert R.worst(loss.copyToHost(ctx)[picked], R.cross_entropy(*args)[0], R.cross_entropy_bounds(*args, "float16")[0]) <= 1
    args += (dloss[picked].astype(np.float64),)
    assert R.worst(at_rows(ctx, dx, picked), R.cross_entropy_gradients(*args)[0], R.cross_entropy_gradient_bounds(*args, "float16")[0]) <= 1


def test_loss_of_more_tiles_than_a_launch_has_threads_for(ctx):
    """2^21 + 3 rows and 2^18 classes are more than 2^23 tiles of 256 x 256; the two numbers that each leaves for a row are 17 GB."""
    rng = np.random.default_rng(4)
    rows, features, classes = 2 ** 21 + 3, 8, 2 ** 18
    picked = [0, 255, 256, 1234567, 2 ** 21 - 2048, 2 ** 21 - 2049, 2 ** 21 - 1, 2 ** 21, rows - 1]
    x, w = (R.bits(a, "float16") for a in (rng.standard_normal((rows, features)), rng.standard_normal((classes, features)) / 2))
    targets = rng.integers(0, classes, rows).astype(np.int32)
    X, W, T = (ml.toDevice(ctx, a) for a in (x, w, targets))
    loss, lse = ml.Tensor((rows,), "float32"), ml.Tensor((rows,), "float32")
    space = ml.Tensor((ml.linearCrossEntropyGetWorkspaceSize(ctx, X, W, False),), "uint8")
    ml.linearCrossEntropyForward(ctx, X, W, None, T, loss, lse, space)
    args = R.numbers(x)[picked], R.numbers(w), np.zeros(classes), targets[picked]
    want, bounds = R.cross_entropy(*args), R.cross_entropy_bounds(*args, "float16")
    losses = loss.copyToHost(ctx)
    assert R.worst(losses[picked], want[0], bounds[0]) <= 1 and R.worst(lse.copyToHost(ctx)[picked], want[1], bounds[1]) <= 1
    assert np.isfinite(losses).all() and (losses > 0).all()


def test_loss_of_more_rows_than_a_launch_has_wavefronts_for(ctx):
    """2^26 + 5 rows of zeros, three classes: the loss is that of the bias alone."""
    rows = 2 ** 26 + 5
    x, w = ml.Tensor((rows, 8), "float16"), ml.toDevice(ctx, R.bits(np.ones((3, 8)), "float16"))
    bias = np.array([0.0, 1.0, -2.0])
    targets, loss, lse = ml.Tensor((rows,), "int32"), ml.Tensor((rows,), "float32"), ml.Tensor((rows,), "float32")
    x.zeroall(ctx)
    targets.zeroall(ctx)
    loss.setall(ctx, -1.0)
    space = ml.Tensor((ml.linearCrossEntropyGetWorkspaceSize(ctx, x, w, False),), "uint8")
    ml.linearCrossEntropyForward(ctx, x, w, ml.toDevice(ctx, R.bits(bias, "float16")), targets, loss, lse, space)
    want = np.log(np.exp(bias).sum())
    # three exponentials, two additions, a logarithm and a difference: below 20 roundings of numbers up to 2
    assert np.abs(loss.copyToHost(ctx).astype(np.float64) - want).max() <= 40 * R.FP32
