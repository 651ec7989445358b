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


def gradient_bounds(x, w, p, dy, name):
    """As R.gated_gradient_bounds, for fp16 with the power of two that d is kept with: half a step of its smallest numbers is 2^-25 where the largest element is between 2^-3 and 2^15, and else 2^-25 of what the largest is
    2^14 of, at least."""
    a, slope = R.gate(p[:, 0], name)
    d = np.concatenate((dy * p[:, 1] * slope, dy * a), 1)
    off = np.concatenate((np.abs(dy * p[:, 1]) * (1 + np.abs(p[:, 0])), np.abs(dy) * (1 + np.abs(p[:, 0]))), 1) * 2 * R.GATE_ERROR["float16"] + 2 * R.FP32 * np.abs(d)
    top = np.abs(d).max()
    stored = off + R.STEP["float16"] * np.abs(d) + (2.0 ** -25 if 2.0 ** -3 <= top < 2.0 ** 15 else 2.0 ** -39 * top)
    dx, dw, db = R.gated_gradients(x, w, p, dy, name)
    flat = w.reshape(-1, w.shape[2])
    return (R.rounded(dx, "float16") + R.product_error(d, flat, "float16") + stored @ np.abs(flat),
            R.rounded(dw, "float32") + (R.product_error(d.T, x, "float16") + stored.T @ np.abs(x)).reshape(w.shape),
            R.rounded(db, "float32") + (off.sum(0) + (x.shape[0] + 80) * R.FP32 * np.abs(d).sum(0)).reshape(2, -1))


def worst_of_fp16(got, want, bound):
    """R.worst where results may pass the type's end: from 65520 on a value rounds to an infinity, and within the bound of that place both are right, the infinity and the last finite number."""
    got = R.numbers(got)
    near = np.abs(np.abs(want) - 65520) <= bound
    rounded_up = np.where(near, np.isinf(got), np.abs(want) >= 65520)
    return R.worst(got, np.where(rounded_up, np.copysign(np.inf, want), want), bound)


# of dy, of the other projection and of the weights: d beyond 65504 with a dx that is not; d at both sides of the limits of scaling; d among the subnormal numbers
SCALES = {"beyond": (2e4, 100.0, 1e-4), "at the upper limit": (2.0 ** 13, 2.0, 1.0), "usual": (1.0, 1.0, 0.1), "at the lower limit": (2.0 ** -5, 1.0, 0.1), "small": (2e-6, 1.0, 1.0), "smallest": (2.0 ** -23, 2.0 ** -12, 1.0)}


@pytest.mark.parametrize("rows", [1, 8, 64, 90, 700])
@pytest.mark.parametrize("scale", SCALES)
def test_gradients_of_the_gated_layer_of_any_size(ctx, scale, rows):
    """dx in fp16 and the sums in fp32, which have to keep their bits whatever size d has; what was in them is added."""
    rng = np.random.default_rng(rows)
    features, hidden = 72, 300
    of_dy, of_u, of_w = SCALES[scale]
    x, w = rng.standard_normal((rows, features)), of_w * rng.standard_normal((2, hidden, features))
    p, dy = rng.standard_normal((rows, 2, hidden)), of_dy * np.clip(rng.standard_normal((rows, hidden)), -3, 3)
    p[:, 1] *= of_u
    x, w, p, dy = (R.bits(a, "float16") for a in (x, w, p, dy))
    X, W, P, DY = (ml.toDevice(ctx, a) for a in (x, w, p, dy))
    args = [R.numbers(a) for a in (x, w, p, dy)] + ["silu"]
    wants, bounds = R.gated_gradients(*args), gradient_bounds(*args)
    old = np.ascontiguousarray(wants[1] / 4, np.float32)
    dx, dw, db = ml.Tensor((rows, features), "float16"), ml.toDevice(ctx, old), ml.Tensor((2, hidden), "float32")
    ml.gatedDenseBackward(ctx, X, W, P, DY, 0.0, dx, 0.0, None, None, "silu", space(ctx, X, W, True))
    assert worst_of_fp16(dx.copyToHost(ctx), wants[0], bounds[0]) <= 1
    ml.gatedDenseBackward(ctx, X, W, P, DY, 0.0, None, -1.0, dw, None, "silu", space(ctx, X, W, True))
    assert R.worst(dw.copyToHost(ctx), wants[1] - old.astype(np.float64), bounds[1] + 2 * R.rounded(old, "float32")) <= 1
    ml.gatedDenseBackward(ctx, X, W, P, DY, 0.0, None, 0.0, None, db, "silu", space(ctx, X, W, True))
    assert R.worst(db.copyToHost(ctx), wants[2], bounds[2]) <= 1


def test_one_infinite_row_has_no_say_in_the_scale_of_the_others(ctx):
    """Small gradients beside a row of infinities: dx of the other rows keeps the bits that it has without that row."""
    rng = np.random.default_rng(5)
    rows, features, hidden = 90, 64, 128
    x, w, p, dy = (R.bits(a, "float16") for a in (rng.standard_normal((rows, features)), rng.standard_normal((2, hidden, features)), rng.standard_normal((rows, 2, hidden)), 2e-4 * rng.standard_normal((rows, hidden))))
    dy[4] = 0
    results = []
    for bad in (False, True):
        if bad:
            dy[4, :9], dy[4, 9] = 0x7c00, 0x7e00
        X, W, P, DY = (ml.toDevice(ctx, a) for a in (x, w, p, dy))
        dx = ml.Tensor((rows, features), "float16")
        ml.gatedDenseBackward(ctx, X, W, P, DY, 0.0, dx, 0.0, None, None, "gelu", space(ctx, X, W, True))
        results.append(R.numbers(dx.copyToHost(ctx)))
    others = np.arange(rows) != 4
    assert np.array_equal(results[0][others], results[1][others]) and np.isnan(results[1][4]).all()


@pytest.mark.parametrize("dtype", ["float16", "float32"])
def test_slope_of_the_sigmoid_keeps_its_digits_on_both_sides(ctx, dtype):
    """db of one row with dy = u = 1 is the slope itself, e^-|g| / (1 + e^-|g|)^2, in fp32. Steps of 2^-24: the exponential 2 and, in fp16, the rounding of its argument, |g| and its scaling's |g|; 1 + e and its inverse 5, twice,
    and two products."""
    g = R.numbers(R.bits(np.concatenate([np.linspace(-20, 20, 401), [-60.0, 60.0]]), dtype))
    p = np.stack((g, np.ones_like(g)))[None]
    x, w = R.bits(np.ones((1, 8)), dtype), R.bits(np.ones((2, g.size, 8)), dtype)
    X, W, P, DY = (ml.toDevice(ctx, a) for a in (x, w, R.bits(p, dtype), R.bits(np.ones((1, g.size)), dtype)))
    db = ml.Tensor((2, g.size), "float32")
    ml.gatedDenseBackward(ctx, X, W, P, DY, 0.0, None, 0.0, None, db, "sigmoid", space(ctx, X, W, True))
    e = np.exp(-np.abs(g))
    want = e / (1 + e) ** 2
    steps = 14 + (2 * np.abs(g) if dtype == "float16" else 0)
    assert R.worst(db.copyToHost(ctx)[0], want, steps * R.FP32 * want) <= 1


# One rounding to fp16 is off by 2^-11 / sqrt 3 of a step's lower end, and 0.735 of that over numbers of any size: 2.07e-4 in norm. dx alone is rounded where what rounding leaves of d is kept; where d were rounded too, both would
# add up to 2.07e-4 sqrt 2 = 2.93e-4. Between the two:
ONE_ROUNDING = 2.45e-4


def off_in_norm(got, want):
    return np.linalg.norm(R.numbers(got) - want) / np.linalg.norm(want)


@pytest.mark.parametrize("rows,features,hidden", [(1, 2048, 700), (5, 1001, 129), (33, 1003, 513), (64, 520, 301)])
def test_dx_of_few_rows_of_the_gated_layer_has_no_rounding_of_d(ctx, rows, features, hidden):
    rng = np.random.default_rng(rows)
    x, w = rng.standard_normal((rows, features)), rng.standard_normal((2, hidden, features)) / np.sqrt(features)
    p, dy = rng.standard_normal((rows, 2, hidden)), rng.standard_normal((rows, hidden))
    x, w, p, dy = (R.bits(a, "float16") for a in (x, w, p, dy))
    X, W, P, DY = (ml.toDevice(ctx, a) for a in (x, w, p, dy))
    dx = ml.Tensor((rows, features), "float16")
    ml.gatedDenseBackward(ctx, X, W, P, DY, 0.0, dx, 0.0, None, None, "silu", space(ctx, X, W, True))
    assert off_in_norm(dx.copyToHost(ctx), R.gated_gradients(*[R.numbers(a) for a in (x, w, p, dy)], "silu")[0]) <= ONE_ROUNDING


DX_OF_LOSSES = [(*size, sharp, common) for size in [(1, 2048, 3000), (5, 1001, 400), (33, 1003, 777), (64, 333, 2001), (65, 256, 4000), (300, 3, 900), (700, 333, 2001)] for sharp in (False, True) for common in (0, 3, 10)]


@pytest.mark.parametrize("rows,features,classes,sharp,common", DX_OF_LOSSES + [(5000, 1100, 300, False, 10), (5000, 1100, 1500, False, 10), (9001, 20, 33, False, 3),
                                                                             (2100, 64, 70003, False, 10)])  # dx in one go on 256 x 256 and 128 x 128 tiles; in two pieces
def test_dx_of_the_cross_entropy_has_no_rounding_of_d(ctx, rows, features, classes, sharp, common):
    """For any number of rows and with weights whose rows have a large part in common, which the rounding of d would carry into dx: up to 2e-3 where it is ten times the rest. sharp: probabilities near 1 among the other
    classes, each of which is rounded, so that dx has two roundings after all."""
    rng = np.random.default_rng(100 + rows)
    x, w = (3.0 if sharp else 0.3) * rng.standard_normal((rows, features)), (rng.standard_normal((classes, features)) + common * rng.standard_normal(features)) / np.sqrt(features)
    targets, dloss = rng.integers(0, classes, rows).astype(np.int32), (rng.uniform(0.7, 1.3, rows) * np.sqrt(2)).astype(np.float32)
    targets[3::11] = -1
    x, w = R.bits(x, "float16"), R.bits(w, "float16")
    X, W, T, DL = (ml.toDevice(ctx, a) for a in (x, w, targets, dloss))
    old = R.bits(rng.standard_normal((rows, features)), "float16")
    loss, lse, dx, added = ml.Tensor((rows,), "float32"), ml.Tensor((rows,), "float32"), ml.Tensor((rows, features), "float16"), ml.toDevice(ctx, old)
    work = ml.Tensor((ml.linearCrossEntropyGetWorkspaceSize(ctx, X, W, True),), "uint8")
    work.setall(ctx, 0xff)
    ml.linearCrossEntropyForward(ctx, X, W, None, T, loss, lse, work)
    ml.linearCrossEntropyBackward(ctx, X, W, None, T, lse, DL, 0.0, dx, 0.0, None, None, work)
    want = R.cross_entropy_gradients(R.numbers(x), R.numbers(w), np.zeros(classes), targets, dloss.astype(np.float64))[0]
    assert off_in_norm(dx.copyToHost(ctx), want) <= (1.2 * np.sqrt(2) * 2.07e-4 if sharp else ONE_ROUNDING)
    assert (R.numbers(dx.copyToHost(ctx))[3::11] == 0).all()
    ml.linearCrossEntropyBackward(ctx, X, W, None, T, lse, DL, 0.5, added, 0.0, None, None, work)
    assert off_in_norm(added.copyToHost(ctx), want + 0.5 * R.numbers(old)) <= (1.2 * np.sqrt(2) * 2.07e-4 if sharp else ONE_ROUNDING)


@pytest.mark.parametrize("rows", [9, 90, 9000])
def test_one_infinite_loss_has_no_say_in_the_others_gradients(ctx, rows):
    """A row whose dloss is an infinity or no number, beside small ones: dx of the others keeps the bits that it has where that row has no gradient, also beside rows without a class and with NaN in their x."""
    rng = np.random.default_rng(rows)
    features, classes = 40, 300
    x, w = rng.standard_normal((rows, features)), rng.standard_normal((classes, features)) / 4
    targets, dloss = rng.integers(0, classes, rows).astype(np.int32), (1e-5 * rng.uniform(0.5, 1, rows)).astype(np.float32)
    targets[5] = -1
    x, w = R.bits(x, "float16"), R.bits(w, "float16")
    x[5] = 0x7e00
    W, T = ml.toDevice(ctx, w), ml.toDevice(ctx, targets)
    X = ml.toDevice(ctx, x)
    loss, lse = ml.Tensor((rows,), "float32"), ml.Tensor((rows,), "float32")
    work = ml.Tensor((ml.linearCrossEntropyGetWorkspaceSize(ctx, X, W, True),), "uint8")
    work.setall(ctx, 0xff)
    ml.linearCrossEntropyForward(ctx, X, W, None, T, loss, lse, work)
    results = []
    for value in (0.0, np.inf, np.nan):
        dloss[2] = value
        dx = ml.Tensor((rows, features), "float16")
        ml.linearCrossEntropyBackward(ctx, X, W, None, T, lse, ml.toDevice(ctx, dloss), 0.0, dx, 0.0, None, None, work)
        results.append(R.numbers(dx.copyToHost(ctx)))
    others = np.arange(rows) != 2
    assert np.isfinite(results[0]).all() and (results[0][[2, 5]] == 0).all() and (results[0][3] != 0).any()
    for got in results[1:]:
        assert np.array_equal(got[others], results[0][others]) and not np.isfinite(got[2]).any()
