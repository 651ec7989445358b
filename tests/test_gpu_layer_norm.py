"""Layer normalisation and its backward pass against the definition in 64 bits."""
import numpy as np
import pytest

import training_reference as R
from minml_amd import core as ml

pytestmark = pytest.mark.gpu
EPSILON = 1e-5


def tensors(ctx, rng, rows, columns, dtype, offset=0.0):
    x = R.bits(rng.standard_normal((rows, columns)) * np.exp(rng.standard_normal(columns) * 0.5) + offset, dtype)
    w, b, dy = (R.bits(a, dtype) for a in (1 + 0.1 * rng.standard_normal(columns), 0.1 * rng.standard_normal(columns), rng.standard_normal((rows, columns))))
    return x, w, b, dy


def workspace(ctx, x):
    return ml.Tensor((max(1, ml.layerNormGetWorkspaceSize(ctx, x)),), "uint8")


SIZES = [(1, 1), (3, 2), (1, 7), (5, 8), (17, 100), (225, 256), (64, 129), (33, 257), (5, 513), (7, 1001), (9, 2048), (4, 4096), (3, 5001), (2, 16384), (3, 16391), (2, 40000), (1500, 72),
         (5000, 40)]


@pytest.mark.parametrize("dtype", ["float16", "float32"])
@pytest.mark.parametrize("rows,columns", SIZES)
def test_forward_and_backward(ctx, rows, columns, dtype):
    rng = np.random.default_rng(rows * 1000003 + columns)
    x, w, b, dy = tensors(ctx, rng, rows, columns, dtype)
    X, W, Bias, DY = (ml.toDevice(ctx, a) for a in (x, w, b, dy))
    y, dx = ml.Tensor((rows, columns), dtype), ml.Tensor((rows, columns), dtype)
    dw, db = ml.Tensor((columns,), dtype), ml.Tensor((columns,), dtype)
    ml.layerNormForward(ctx, X, W, Bias, y, EPSILON)
    ml.layerNormBackward(ctx, X, W, DY, 0.0, dx, 0.0, dw, db, workspace(ctx, X), EPSILON)
    xf, wf, bf, dyf = map(R.numbers, (x, w, b, dy))
    assert R.worst(y.copyToHost(ctx), R.layer_norm(xf, wf, bf, EPSILON), R.layer_norm_bound(xf, wf, bf, EPSILON, dtype)) <= 1
    for got, want, bound in zip((dx, dw, db), R.layer_norm_gradients(xf, wf, dyf, EPSILON), R.layer_norm_gradient_bounds(xf, wf, dyf, EPSILON, dtype)):
        assert R.worst(got.copyToHost(ctx), want, bound) <= 1


@pytest.mark.parametrize("dtype", ["float16", "float32"])
@pytest.mark.parametrize("columns", [5, 96, 1000, 17000])
def test_gradients_are_added_to_what_was_there(ctx, columns, dtype):
    rng = np.random.default_rng(columns)
    x, w, _, dy = tensors(ctx, rng, 21, columns, dtype)
    old_x, old_w, old_b = (R.bits(rng.standard_normal(s), dtype) for s in ((21, columns), columns, columns))
    X, W, DY, dx = (ml.toDevice(ctx, a) for a in (x, w, dy, old_x))
    dw, db = (ml.toDevice(ctx, R.numbers(a).astype(np.float32)) for a in (old_w, old_b))  # in fp32 for both types
    ml.layerNormBackward(ctx, X, W, DY, 1.0, dx, 0.5, dw, db, workspace(ctx, X), EPSILON)
    xf, wf, dyf = map(R.numbers, (x, w, dy))
    want, bounds = R.layer_norm_gradients(xf, wf, dyf, EPSILON), R.layer_norm_gradient_bounds(xf, wf, dyf, EPSILON, dtype)
    sums = R.layer_norm_gradient_bounds(xf, wf, dyf, EPSILON, "float32")
    assert R.worst(dx.copyToHost(ctx), want[0] + R.numbers(old_x), bounds[0] + 2 * R.rounded(R.numbers(old_x), dtype)) <= 1
    for got, k, old in ((dw, 1, old_w), (db, 2, old_b)):
        assert R.worst(got.copyToHost(ctx), want[k] + 0.5 * R.numbers(old), sums[k] + 2 * R.rounded(R.numbers(old), "float32")) <= 1


@pytest.mark.parametrize("dtype", ["float16", "float32"])
def test_without_weights_and_with_some_gradients_only(ctx, dtype):
    rng = np.random.default_rng(5)
    x, _, _, dy = tensors(ctx, rng, 30, 200, dtype)
    X, DY = ml.toDevice(ctx, x), ml.toDevice(ctx, dy)
    xf, dyf, one, zero = R.numbers(x), R.numbers(dy), np.ones(200), np.zeros(200)
    y = ml.Tensor((30, 200), dtype)
    ml.layerNormForward(ctx, X, None, None, y)
    assert R.worst(y.copyToHost(ctx), R.layer_norm(xf, one, zero, EPSILON), R.layer_norm_bound(xf, one, zero, EPSILON, dtype)) <= 1
    want, bounds = R.layer_norm_gradients(xf, one, dyf, EPSILON), R.layer_norm_gradient_bounds(xf, one, dyf, EPSILON, dtype)
    for only in range(3):
        out = [ml.Tensor((30, 200) if k == 0 else (200,), dtype) if k == only else None for k in range(3)]
        ml.layerNormBackward(ctx, X, None, DY, 0.0, out[0], 0.0, out[1], out[2], workspace(ctx, X))
        assert R.worst(out[only].copyToHost(ctx), want[only], bounds[only]) <= 1


@pytest.mark.parametrize("dtype", ["float16", "float32"])
@pytest.mark.parametrize("columns", [3, 100, 1001, 16500])
def test_in_place_and_at_any_address(ctx, columns, dtype):
    """Results over their inputs, and tensors that begin one element into their memory, with what lies around them left as it was."""
    rng = np.random.default_rng(columns + 1)
    rows, size = 6, 6 * columns
    x, w, b, dy = tensors(ctx, rng, rows, columns, dtype)
    guard = R.bits(np.full(1, 7.0), dtype)
    shifted = lambda a: ml.toDevice(ctx, np.concatenate([guard, a.reshape(-1), guard])).view(a.shape, 1)
    X, W, Bias, DY = map(shifted, (x, w, b, dy))
    xf, wf, bf, dyf = map(R.numbers, (x, w, b, dy))
    dw, db = shifted(w), shifted(b)
    ml.layerNormBackward(ctx, X, W, DY, 0.0, DY, 0.0, dw, db, workspace(ctx, X), EPSILON)
    ml.layerNormForward(ctx, X, W, Bias, X, EPSILON)
    for got, want, bound in zip((DY, dw, db), R.layer_norm_gradients(xf, wf, dyf, EPSILON), R.layer_norm_gradient_bounds(xf, wf, dyf, EPSILON, dtype)):
        assert R.worst(got.copyToHost(ctx), want, bound) <= 1
    assert R.worst(X.copyToHost(ctx), R.layer_norm(xf, wf, bf, EPSILON), R.layer_norm_bound(xf, wf, bf, EPSILON, dtype)) <= 1
    for t in (X, DY, dw, db):
        whole = t._owner.copyToHost(ctx)
        assert whole[0] == guard[0] and whole[-1] == guard[0] and whole.size in (size + 2, columns + 2)


def test_far_mean_constant_rows_and_rows_that_are_not_finite(ctx):
    """The variance is taken about the mean; a row without variance stays finite; infinities and NaN stay in their row, and reach every column's sum."""
    rng = np.random.default_rng(9)
    x, w, b, dy = tensors(ctx, rng, 8, 300, "float32", offset=1000.0)
    x[1] = 3.5
    X, W, Bias, DY = (ml.toDevice(ctx, a) for a in (x, w, b, dy))
    y, dx = ml.Tensor((8, 300), "float32"), ml.Tensor((8, 300), "float32")
    ml.layerNormForward(ctx, X, W, Bias, y, EPSILON)
    ml.layerNormBackward(ctx, X, W, DY, 0.0, dx, 0.0, None, None, workspace(ctx, X), EPSILON)
    xf, wf, bf, dyf = map(R.numbers, (x, w, b, dy))
    assert R.worst(y.copyToHost(ctx), R.layer_norm(xf, wf, bf, EPSILON), R.layer_norm_bound(xf, wf, bf, EPSILON, "float32")) <= 1
    assert np.isfinite(dx.copyToHost(ctx)).all()
    assert R.worst(dx.copyToHost(ctx), R.layer_norm_gradients(xf, wf, dyf, EPSILON)[0], R.layer_norm_gradient_bounds(xf, wf, dyf, EPSILON, "float32")[0]) <= 1
    x[2, 7], x[4, 0] = np.inf, np.nan
    X.copyFromHost(ctx, x)
    z = ml.Tensor((8, 300), "float32")
    ml.layerNormForward(ctx, X, W, Bias, z, EPSILON)
    z, y = z.copyToHost(ctx), y.copyToHost(ctx)
    assert np.isnan(z[[2, 4]]).all() and np.array_equal(np.delete(z, [2, 4], 0), np.delete(y, [2, 4], 0))


def test_no_rows(ctx):
    """Nothing to sum: the gradients of the weights are what was there, times beta."""
    x, w = ml.Tensor((0, 64), "float16"), ml.toDevice(ctx, R.bits(np.ones(64), "float16"))
    dw, db = ml.toDevice(ctx, np.full(64, 3.0, np.float32)), ml.toDevice(ctx, R.bits(np.full(64, 5.0), "float16"))
    ml.layerNormForward(ctx, x, w, None, x)
    ml.layerNormBackward(ctx, x, w, x, 0.0, x, 0.5, dw, None, None)
    ml.layerNormBackward(ctx, x, w, x, 0.0, None, 0.0, None, db, None)
    assert (dw.copyToHost(ctx) == 1.5).all() and (R.numbers(db.copyToHost(ctx)) == 0).all()


def test_gradient_agrees_with_differences(ctx):
    """sum(y * dy) changes along a direction as the gradients say: central differences of the forward pass in fp32."""
    rng = np.random.default_rng(12)
    x, w, b, dy = tensors(ctx, rng, 12, 80, "float32")
    X, W, DY = (ml.toDevice(ctx, a) for a in (x, w, dy))
    dx, dw, db = ml.Tensor((12, 80), "float32"), ml.Tensor((80,), "float32"), ml.Tensor((80,), "float32")
    ml.layerNormBackward(ctx, X, W, DY, 0.0, dx, 0.0, dw, db, workspace(ctx, X), EPSILON)
    y = ml.Tensor((12, 80), "float32")

    def value(x, w, b):
        ml.layerNormForward(ctx, *(ml.toDevice(ctx, np.ascontiguousarray(a, np.float32)) for a in (x, w, b)), y, EPSILON)
        return float((y.copyToHost(ctx).astype(np.float64) * dy).sum())

    step = 2.0 ** -7
    for k, (at, gradient) in enumerate(((x, dx), (w, dw), (b, db))):
        direction = rng.choice([-1.0, 1.0], at.shape).astype(np.float32)
        ends = []
        for sign in (1, -1):
            args = [x, w, b]
            args[k] = at + sign * step * direction
            ends.append(value(*args))
        slope = (ends[0] - ends[1]) / (2 * step)
        want = float((gradient.copyToHost(ctx).astype(np.float64) * direction).sum())
        # 960 products of about 1, each off by some 2^-22, over 2 * 2^-7; and step^2 / 6 of a third derivative that is at most about 10 times the sum of |dx|
        assert abs(slope - want) <= 960 * 2.0 ** -22 / (2 * step) + step ** 2 / 6 * 10 * np.abs(gradient.copyToHost(ctx)).sum()


def test_recorded_pass_and_two_contexts(ctx):
    """A recorded backward pass gives the eager bits on every replay, also with another context's calls in between that have a workspace of their own."""
    rng = np.random.default_rng(13)
    x, w, _, dy = tensors(ctx, rng, 2000, 384, "float16")
    other = ml.Context(0)
    sets = []
    for c in (ctx, other):
        X, W, DY = (ml.toDevice(c, a) for a in (x, w, dy))
        out = ml.Tensor((2000, 384), "float16"), ml.Tensor((384,), "float16"), ml.Tensor((384,), "float32")
        space = workspace(c, X)
        sets.append((lambda c=c, X=X, W=W, DY=DY, out=out, space=space: ml.layerNormBackward(c, X, W, DY, 0.0, out[0], 0.0, out[1], out[2], space), out))
    sets[0][0]()
    eager = [t.copyToHost(ctx) for t in sets[0][1]]
    with ml.Graph.record(ctx, sets[0][0]) as graph:
        for _ in range(3):
            for t in sets[0][1]:
                t.zeroall(ctx)
            sets[1][0]()
            graph.launch()
            ctx.synchronize()
            other.synchronize()
            for _, out in sets:
                assert all(np.array_equal(t.copyToHost(ctx), e) for t, e in zip(out, eager))
    other.destroy()


@pytest.mark.parametrize("dtype", ["float16", "float32"])
@pytest.mark.parametrize("columns", [8200, 9001, 16384])
def test_several_long_rows_of_a_workgroup(ctx, columns, dtype):
    """More rows than workgroups, of lengths that 1024 threads hold in their registers; dx over dy."""
    rng = np.random.default_rng(columns)
    x, w, b, dy = tensors(ctx, rng, 1030, columns, dtype)
    X, W, DY = (ml.toDevice(ctx, a) for a in (x, w, dy))
    dw, db = ml.Tensor((columns,), "float32"), ml.Tensor((columns,), "float32")
    ml.layerNormBackward(ctx, X, W, DY, 0.0, DY, 0.0, dw, db, workspace(ctx, X), EPSILON)
    xf, wf, dyf = map(R.numbers, (x, w, dy))
    want, bounds, sums = R.layer_norm_gradients(xf, wf, dyf, EPSILON), R.layer_norm_gradient_bounds(xf, wf, dyf, EPSILON, dtype), R.layer_norm_gradient_bounds(xf, wf, dyf, EPSILON, "float32")
    assert R.worst(DY.copyToHost(ctx), want[0], bounds[0]) <= 1
    assert R.worst(dw.copyToHost(ctx), want[1], sums[1]) <= 1 and R.worst(db.copyToHost(ctx), want[2], sums[2]) <= 1
