"""The cross entropy over many classes and its gradients against the definition in 64 bits."""
import numpy as np
import pytest

import training_reference as R
from minml_amd import core as ml
from test_gpu_gated import check_guards, guarded

pytestmark = pytest.mark.gpu


def inputs(rng, rows, features, classes, dtype, ignored=0.1):
    x, w, b = rng.standard_normal((rows, features)), 2 * rng.standard_normal((classes, features)) / np.sqrt(features), 0.5 * rng.standard_normal(classes)
    targets = rng.integers(0, classes, rows)
    other = rng.random(rows) < ignored
    targets[other] = rng.choice([-1, -100, classes, classes + 5, 2 ** 31 - 1, -2 ** 31], int(other.sum()))
    return [R.bits(a, dtype) for a in (x, w, b)] + [targets.astype(np.int32), (rng.standard_normal(rows) * 3).astype(np.float32)]


def space(ctx, x, w, backward):
    t = ml.Tensor((max(1, ml.linearCrossEntropyGetWorkspaceSize(ctx, x, w, backward)),), "uint8")
    t.setall(ctx, 0xff)  # NaN in both types: nothing may be read before it was written
    return t


SIZES = [(1, 8, 1), (1, 64, 300), (3, 63, 20), (16, 200, 37), (17, 130, 16), (33, 72, 1000), (64, 333, 100), (65, 40, 513), (130, 65, 257), (300, 200, 130), (129, 1096, 24), (2, 2056, 70),
         (3500, 24, 3700), (513, 64, 8), (1, 16, 40001), (2, 8, 1100000), (9000, 8, 20)]


@pytest.mark.parametrize("dtype", ["float16", "float32"])
@pytest.mark.parametrize("rows,features,classes", SIZES)
def test_loss_and_gradients(ctx, rows, features, classes, dtype):
    rng = np.random.default_rng(rows * 10007 + features * 101 + classes)
    x, w, b, targets, dloss = inputs(rng, rows, features, classes, dtype)
    X, W, Bias = (guarded(ctx, a, dtype, np.nan) for a in (x, w, b))
    T, DL = ml.toDevice(ctx, targets), ml.toDevice(ctx, dloss)
    loss, lse = (guarded(ctx, np.zeros(rows, np.float32), "float32", 9.0) for _ in range(2))
    ml.linearCrossEntropyForward(ctx, X, W, Bias, T, loss, lse, space(ctx, X, W, False))
    xf, wf, bf = map(R.numbers, (x, w, b))
    want, bound = R.cross_entropy(xf, wf, bf, targets), R.cross_entropy_bounds(xf, wf, bf, targets, dtype)
    assert R.worst(loss.copyToHost(ctx), want[0], bound[0]) <= 1
    assert R.worst(lse.copyToHost(ctx), want[1], bound[1]) <= 1
    dx, dw, db = (guarded(ctx, R.bits(np.zeros(a.shape), dtype), dtype, 9.0) for a in (x, w, b))
    ml.linearCrossEntropyBackward(ctx, X, W, Bias, T, lse, DL, 0.0, dx, 0.0, dw, db, space(ctx, X, W, True))
    args = xf, wf, bf, targets, dloss.astype(np.float64)
    for got, exact, off in zip((dx, dw, db), R.cross_entropy_gradients(*args), R.cross_entropy_gradient_bounds(*args, dtype)):
        assert R.worst(got.copyToHost(ctx), exact, off) <= 1
        check_guards(ctx, got, 9.0)
    for t in (loss, lse):
        check_guards(ctx, t, 9.0)


def test_more_classes_than_one_piece_holds(ctx):
    """4100 rows in fp32: d of 17000 classes is more than 256 MB, so the classes are taken in two pieces, the second one smaller; the gradients are added to what was there."""
    rng = np.random.default_rng(2)
    x, w, b, targets, dloss = inputs(rng, 4100, 8, 17000, "float32")
    X, W, Bias, T, DL = (ml.toDevice(ctx, a) for a in (x, w, b, targets, dloss))
    work = space(ctx, X, W, True)
    assert work.sizeInBytes() < 4100 * 17000 * 4 + (4 << 20)
    loss, lse = ml.Tensor((4100,), "float32"), ml.Tensor((4100,), "float32")
    ml.linearCrossEntropyForward(ctx, X, W, Bias, T, loss, lse, work)
    olds = [rng.standard_normal(a.shape).astype(np.float32) for a in (x, w, b)]
    grads = [ml.toDevice(ctx, a) for a in olds]
    ml.linearCrossEntropyBackward(ctx, X, W, Bias, T, lse, DL, 0.5, grads[0], -1.0, grads[1], grads[2], work)
    args = [a.astype(np.float64) for a in (x, w, b)] + [targets, dloss.astype(np.float64)]
    for got, exact, off, old, beta in zip(grads, R.cross_entropy_gradients(*args), R.cross_entropy_gradient_bounds(*args, "float32"), olds, (0.5, -1.0, -1.0)):
        assert R.worst(got.copyToHost(ctx), exact + beta * old.astype(np.float64), off + 2 * R.rounded(old, "float32")) <= 1


@pytest.mark.parametrize("dtype", ["float16", "float32"])
def test_gradients_are_added_and_may_be_left_out(ctx, dtype):
    rng = np.random.default_rng(3)
    for rows, features, classes in ((90, 72, 400), (600, 33, 70)):
        x, w, b, targets, dloss = inputs(rng, rows, features, classes, dtype)
        olds = [R.bits(rng.standard_normal(a.shape), dtype) for a in (x, w, b)]
        X, W, Bias, T, DL = (ml.toDevice(ctx, a) for a in (x, w, b, targets, dloss))
        work = space(ctx, X, W, True)
        loss, lse = ml.Tensor((rows,), "float32"), ml.Tensor((rows,), "float32")
        ml.linearCrossEntropyForward(ctx, X, W, Bias, T, loss, lse, work)
        args = [R.numbers(a) for a in (x, w, b)] + [targets, dloss.astype(np.float64)]
        wants, bounds = R.cross_entropy_gradients(*args), R.cross_entropy_gradient_bounds(*args, dtype)
        for only in (None, 0, 1, 2):
            grads = [ml.toDevice(ctx, olds[0])] + [ml.toDevice(ctx, R.numbers(a).astype(np.float32)) for a in olds[1:]]
            given = [t if only in (None, k) else None for k, t in enumerate(grads)]
            ml.linearCrossEntropyBackward(ctx, X, W, Bias, T, lse, DL, -1.0, given[0], 0.5, given[1], given[2], work)
            for k, t in enumerate(grads):
                old = R.numbers(olds[k]) * (-1.0 if k == 0 else 0.5)
                if given[k] is None:
                    assert np.array_equal(R.numbers(t.copyToHost(ctx)), R.numbers(olds[k]))
                else:
                    assert R.worst(t.copyToHost(ctx), wants[k] + old, bounds[k] + 2 * R.rounded(old, dtype if k == 0 else "float32")) <= 1


@pytest.mark.parametrize("dtype", ["float16", "float32"])
@pytest.mark.parametrize("scale", [1e-30, 1e-6, 1.0, 1e4])
def test_gradients_of_losses_of_any_size(ctx, dtype, scale):
    """In fp16 the scaled d keeps probabilities of 1e-5 whatever the losses weigh; results that are themselves too small or large for the type are taken in fp32."""
    rng = np.random.default_rng(5)
    x, w, b, targets, dloss = inputs(rng, 100, 64, 5000, dtype)
    dloss *= scale
    X, W, Bias, T, DL = (ml.toDevice(ctx, a) for a in (x, w, b, targets, dloss))
    work = space(ctx, X, W, True)
    loss, lse = ml.Tensor((100,), "float32"), ml.Tensor((100,), "float32")
    ml.linearCrossEntropyForward(ctx, X, W, Bias, T, loss, lse, work)
    dw, db = ml.Tensor((5000, 64), "float32"), ml.Tensor((5000,), "float32")
    ml.linearCrossEntropyBackward(ctx, X, W, Bias, T, lse, DL, 0.0, None, 0.0, dw, db, work)
    args = [R.numbers(a) for a in (x, w, b)] + [targets, dloss.astype(np.float64)]
    wants, bounds = R.cross_entropy_gradients(*args), R.cross_entropy_gradient_bounds(*args, dtype)
    for got, k in ((dw, 1), (db, 2)):
        assert R.worst(got.copyToHost(ctx), wants[k], bounds[k]) <= 1


def test_large_logits_masks_and_infinities(ctx):
    """Logits of +-10000, classes that a bias of -inf or of the type's lowest value takes out, a row of NaN, and rows without any gradient."""
    rng = np.random.default_rng(6)
    for rows in (9, 90):
        x, w, b, targets, dloss = inputs(rng, rows, 64, 500, "float32")
        x[0] *= 10000
        b[100:200], b[200:250] = -np.inf, np.finfo(np.float32).min
        targets[:] = rng.integers(0, 100, rows)
        targets[5] = -1
        dloss[6] = 0
        X, W, Bias, T, DL = (ml.toDevice(ctx, a) for a in (x, w, b, targets, dloss))
        work = space(ctx, X, W, True)
        loss, lse = ml.Tensor((rows,), "float32"), ml.Tensor((rows,), "float32")
        ml.linearCrossEntropyForward(ctx, X, W, Bias, T, loss, lse, work)
        finite = b.astype(np.float64)
        finite[100:250] = -1e30  # the definition without infinities; the masked logits' own errors count for nothing
        xf, wf = x.astype(np.float64), w.astype(np.float64)
        inside = np.r_[0:100, 250:500]
        moved = np.searchsorted(inside, targets)
        moved[targets < 0] = -1
        args = xf, wf[inside], finite[inside], moved
        assert R.worst(loss.copyToHost(ctx), R.cross_entropy(*args)[0], R.cross_entropy_bounds(*args, "float32")[0]) <= 1
        dx, dw, db = ml.Tensor(x.shape, "float32"), ml.Tensor(w.shape, "float32"), ml.Tensor(b.shape, "float32")
        ml.linearCrossEntropyBackward(ctx, X, W, Bias, T, lse, DL, 0.0, dx, 0.0, dw, db, work)
        got = [t.copyToHost(ctx) for t in (dx, dw, db)]
        args += (dloss.astype(np.float64),)
        wants, bounds = R.cross_entropy_gradients(*args), R.cross_entropy_gradient_bounds(*args, "float32")
        for g, want, bound in zip((got[0], got[1][inside], got[2][inside]), wants, bounds):
            assert R.worst(g, want, bound) <= 1
        assert (got[1][100:250] == 0).all() and (got[2][100:250] == 0).all() and (got[0][5] == 0).all() and (got[0][6] == 0).all()
        # a logit of +inf, a row of -inf alone, NaN: in their rows only
        x2, b2 = np.zeros((rows, 64), np.float32), np.full(500, -np.inf, np.float32)
        x2[2, 0] = np.nan
        X2, Bias2 = ml.toDevice(ctx, x2), ml.toDevice(ctx, b2)
        ml.linearCrossEntropyForward(ctx, X2, W, Bias2, T, loss, lse, work)
        got = lse.copyToHost(ctx)
        assert np.isnan(got[2]) and (np.delete(got, 2) == -np.inf).all() and loss.copyToHost(ctx)[5] == 0
        b2[:], b2[7] = 0, np.inf
        Bias2.copyFromHost(ctx, b2)
        ml.linearCrossEntropyForward(ctx, X2, W, Bias2, T, loss, lse, work)
        got = lse.copyToHost(ctx)
        assert np.isnan(got[2]) and (np.delete(got, 2) == np.inf).all()


def test_no_rows(ctx):
    x, w = ml.Tensor((0, 64), "float16"), ml.toDevice(ctx, R.bits(np.ones((24, 64)), "float16"))
    t, f = ml.Tensor((0,), "int32"), ml.Tensor((0,), "float32")
    dw, db = ml.toDevice(ctx, np.full((24, 64), 3.0, np.float32)), ml.toDevice(ctx, R.bits(np.full(24, 5.0), "float16"))
    ml.linearCrossEntropyForward(ctx, x, w, None, t, f, f, None)
    ml.linearCrossEntropyBackward(ctx, x, w, None, t, f, f, 0.0, x, 0.5, dw, db, None)
    assert (dw.copyToHost(ctx) == 1.5).all() and (R.numbers(db.copyToHost(ctx)) == 2.5).all()


def test_gradient_agrees_with_differences(ctx):
    rng = np.random.default_rng(8)
    rows, features, classes = 80, 24, 150
    x, w, b, targets, dloss = inputs(rng, rows, features, classes, "float32")
    T, DL = ml.toDevice(ctx, targets), ml.toDevice(ctx, dloss)
    work = space(ctx, ml.toDevice(ctx, x), ml.toDevice(ctx, w), True)
    loss, lse = ml.Tensor((rows,), "float32"), ml.Tensor((rows,), "float32")

    def value(x, w, b):
        ml.linearCrossEntropyForward(ctx, *(ml.toDevice(ctx, np.ascontiguousarray(a, np.float32)) for a in (x, w, b)), T, loss, lse, work)
        return float((loss.copyToHost(ctx).astype(np.float64) * dloss).sum())

    value(x, w, b)
    grads = [ml.Tensor(a.shape, "float32") for a in (x, w, b)]
    ml.linearCrossEntropyBackward(ctx, ml.toDevice(ctx, x), ml.toDevice(ctx, w), ml.toDevice(ctx, b), T, lse, DL, 0.0, grads[0], 0.0, grads[1], grads[2], work)
    step = 2.0 ** -8
    for k, at in enumerate((x, w, b)):
        direction = rng.choice([-1.0, 1.0], at.shape).astype(np.float32)
        ends = []
        for sign in (1, -1):
            args = [x, w, b]
            args[k] = at + sign * step * direction
            ends.append(value(*args))
        want = float((grads[k].copyToHost(ctx).astype(np.float64) * direction).sum())
        # 80 losses of weight 3 or so, off by 2^-19 each; the third derivative of a log-sum-exp is at most the cube of the logits' spread along the direction, 12 here
        assert abs((ends[0] - ends[1]) / (2 * step) - want) <= np.abs(dloss).sum() * (2.0 ** -19 / step + step ** 2 / 6 * 12 ** 3)


@pytest.mark.parametrize("rows,features,classes", [(8, 512, 700), (200, 256, 3000)])
def test_recorded_pass_gives_the_eager_bits(ctx, rows, features, classes):
    rng = np.random.default_rng(9)
    x, w, b, targets, dloss = inputs(rng, rows, features, classes, "float16")
    other = ml.Context(0)
    passes = []
    for c in (ctx, other):
        X, W, Bias, T, DL = (ml.toDevice(c, a) for a in (x, w, b, targets, dloss))
        out = [ml.Tensor((rows,), "float32"), ml.Tensor((rows,), "float32")] + [ml.Tensor(a.shape, "float16") for a in (x, w, b)]
        work = space(c, X, W, True)

        def both(c=c, X=X, W=W, Bias=Bias, T=T, DL=DL, out=out, work=work):
            ml.linearCrossEntropyForward(c, X, W, Bias, T, out[0], out[1], work)
            ml.linearCrossEntropyBackward(c, X, W, Bias, T, out[1], DL, 0.0, out[2], 0.0, out[3], out[4], work)

        passes.append((both, out))
    passes[0][0]()
    eager = [t.copyToHost(ctx) for t in passes[0][1]]
    with ml.Graph.record(ctx, passes[0][0]) as graph:
        for _ in range(3):
            for t in passes[0][1]:
                t.zeroall(ctx)
            passes[1][0]()
            graph.launch()
            ctx.synchronize()
            other.synchronize()
            for _, out in passes:
                assert all(np.array_equal(t.copyToHost(ctx), e) for t, e in zip(out, eager))
    other.destroy()


def test_a_single_row_without_leading_dimensions(ctx):
    rng = np.random.default_rng(10)
    x, w, b, _, _ = inputs(rng, 1, 72, 300, "float16")
    results = []
    for lead in ((1,), ()):
        X, W, Bias = (ml.toDevice(ctx, a) for a in (x.reshape(lead + (72,)), w, b))
        T, DL = ml.toDevice(ctx, np.array([17], np.int32)), ml.toDevice(ctx, np.array([0.75], np.float32))
        loss, lse, dx = ml.Tensor((1,), "float32"), ml.Tensor((1,), "float32"), ml.Tensor(X.shape, "float16")
        work = space(ctx, X, W, True)
        ml.linearCrossEntropyForward(ctx, X, W, Bias, T, loss, lse, work)
        ml.linearCrossEntropyBackward(ctx, X, W, Bias, T, lse, DL, 0.0, dx, 0.0, None, None, work)
        results.append([t.copyToHost(ctx).reshape(-1) for t in (loss, lse, dx)])
    assert all(np.array_equal(a, c) for a, c in zip(*results)) and results[0][0][0] > 0
