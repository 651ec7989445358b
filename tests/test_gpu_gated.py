"""The gated dense layer and its backward pass against the definition in 64 bits."""
import numpy as np
import pytest

import training_reference as R
from minml_amd import core as ml

pytestmark = pytest.mark.gpu


def inputs(rng, rows, features, hidden, dtype):
    x = rng.standard_normal((rows, features))
    w, b = rng.standard_normal((2, hidden, features)) / np.sqrt(features), 0.3 * rng.standard_normal((2, hidden))
    p, dy = 1.5 * rng.standard_normal((rows, 2, hidden)), rng.standard_normal((rows, hidden))
    return [R.bits(a, dtype) for a in (x, w, b, p, dy)]


def space(ctx, x, w, backward):
    size = ml.gatedDenseGetWorkspaceSize(ctx, x, w, backward)
    t = ml.Tensor((max(1, size),), "uint8")
    t.setall(ctx, 0xff)  # NaN in both types: nothing may be read before it was written
    return t


def guarded(ctx, a, dtype, value):
    """The array as a device tensor with `value` on both sides of it, beginning 16 bytes into its memory."""
    pad = R.bits(np.full(16 // a.itemsize, value), dtype)
    return ml.toDevice(ctx, np.concatenate([pad, a.reshape(-1), pad])).view(a.shape, pad.size)


def check_guards(ctx, t, value):
    whole, n = R.numbers(t._owner.copyToHost(ctx)), t._owner.volume() - t.volume()
    assert (whole[:n // 2] == value).all() and (whole[-(n // 2):] == value).all()


FORWARD = [(1, 8, 1), (1, 64, 64), (3, 63, 20), (16, 200, 37), (17, 130, 16), (40, 333, 100), (64, 72, 257), (65, 40, 64), (130, 65, 65), (300, 200, 130), (129, 1096, 24), (1, 2056, 48),
           (70, 4104, 33), (3500, 24, 1900), (513, 64, 8)]


@pytest.mark.parametrize("dtype", ["float16", "float32"])
@pytest.mark.parametrize("rows,features,hidden", FORWARD)
def test_forward(ctx, rows, features, hidden, dtype):
    """Inputs with NaN beside them in memory: nothing outside a tensor reaches a result; and results that end where they should."""
    rng = np.random.default_rng(rows * 10007 + features * 101 + hidden)
    x, w, b, _, _ = inputs(rng, rows, features, hidden, dtype)
    X, W, Bias = (guarded(ctx, a, dtype, np.nan) for a in (x, w, b))
    name = R.GATES[(rows + features + hidden) % 4]
    y, kept = (guarded(ctx, R.bits(np.zeros(s), dtype), dtype, 9.0) for s in ((rows, hidden), (rows, 2, hidden)))
    ml.gatedDenseForward(ctx, X, W, Bias, y, kept, name, space(ctx, X, W, False))
    xf, wf, bf = map(R.numbers, (x, w, b))
    want, bound = R.gated(xf, wf, bf, name), R.gated_bounds(xf, wf, bf, name, dtype)
    assert R.worst(y.copyToHost(ctx), want[0], bound[0]) <= 1
    assert R.worst(kept.copyToHost(ctx), want[1], bound[1]) <= 1
    check_guards(ctx, y, 9.0)
    check_guards(ctx, kept, 9.0)


BACKWARD = [(1, 8, 1), (1, 200, 64), (3, 63, 20), (17, 130, 16), (65, 40, 64), (300, 200, 130), (129, 333, 257), (1030, 72, 24), (3500, 3600, 24), (33, 3600, 1800), (700, 16, 5), (4600, 4096, 1056)]


@pytest.mark.parametrize("dtype", ["float16", "float32"])
@pytest.mark.parametrize("rows,features,hidden", BACKWARD)
def test_backward(ctx, rows, features, hidden, dtype):
    rng = np.random.default_rng(rows * 10007 + features * 101 + hidden)
    x, w, b, p, dy = inputs(rng, rows, features, hidden, dtype)
    X, W, P, DY = (guarded(ctx, a, dtype, np.nan) for a in (x, w, p, dy))
    name = R.GATES[(rows + features) % 4]
    dx, dw, db = (guarded(ctx, R.bits(np.zeros(s), dtype), dtype, 9.0) for s in (x.shape, w.shape, b.shape))
    ml.gatedDenseBackward(ctx, X, W, P, DY, 0.0, dx, 0.0, dw, db, name, space(ctx, X, W, True))
    args = [R.numbers(a) for a in (x, w, p, dy)] + [name]
    for got, want, bound in zip((dx, dw, db), R.gated_gradients(*args), R.gated_gradient_bounds(*args, dtype)):
        assert R.worst(got.copyToHost(ctx), want, bound) <= 1
        check_guards(ctx, got, 9.0)


@pytest.mark.parametrize("dtype", ["float16", "float32"])
@pytest.mark.parametrize("name", R.GATES)
def test_every_gate_over_its_range(ctx, name, dtype):
    """Gate projections from -20 to 20 and the subnormal ones, through the few-rows kernel, the tiles and the backward pass."""
    g = np.concatenate([np.linspace(-20, 20, 240), [0.0, -0.0, 6e-8, -6e-8, 1e-5, -1e-5, 65000.0, -65000.0]])
    for rows in (2, 70):
        x = R.bits(np.ones((rows, 8)) * (np.arange(8) == 0), dtype)
        w = np.zeros((2, g.size, 8))
        w[0, :, 0], w[1, :, 0] = g, 0.75
        w = R.bits(w, dtype)
        X, W, y = ml.toDevice(ctx, x), ml.toDevice(ctx, w), ml.Tensor((rows, g.size), dtype)
        kept = ml.Tensor((rows, 2, g.size), dtype)
        ml.gatedDenseForward(ctx, X, W, None, y, kept, name, space(ctx, X, W, False))
        xf, wf, bf = R.numbers(x), R.numbers(w), np.zeros((2, g.size))
        bound = R.gated_bounds(xf, wf, bf, name, dtype)
        assert R.worst(y.copyToHost(ctx), R.gated(xf, wf, bf, name)[0], bound[0]) <= 1
        dy = R.bits(np.full((rows, g.size), 0.5), dtype)
        DY, db = ml.toDevice(ctx, dy), ml.Tensor((2, g.size), dtype)
        ml.gatedDenseBackward(ctx, X, W, kept, DY, 0.0, None, 0.0, None, db, name, space(ctx, X, W, True))
        args = xf, wf, R.numbers(kept.copyToHost(ctx)), R.numbers(dy), name
        assert R.worst(db.copyToHost(ctx), R.gated_gradients(*args)[2], R.gated_gradient_bounds(*args, dtype)[2]) <= 1


@pytest.mark.parametrize("dtype", ["float16", "float32"])
def test_gradients_are_added_and_may_be_left_out(ctx, dtype):
    rng = np.random.default_rng(3)
    for rows, features, hidden in ((90, 72, 40), (600, 33, 20)):
        x, w, b, p, dy = inputs(rng, rows, features, hidden, dtype)
        olds = [R.bits(rng.standard_normal(a.shape), dtype) for a in (x, w, b)]
        X, W, P, DY = (ml.toDevice(ctx, a) for a in (x, w, p, dy))
        work = space(ctx, X, W, True)
        args = [R.numbers(a) for a in (x, w, p, dy)] + ["silu"]
        wants, bounds, exact = R.gated_gradients(*args), R.gated_gradient_bounds(*args, dtype), R.gated_gradient_bounds(*args, "float32")
        stored = R.gated_gradient_bounds(*args, dtype)
        for only in (None, 0, 1, 2):
            grads = [ml.toDevice(ctx, olds[0])] + [ml.toDevice(ctx, R.numbers(a).astype(np.float32)) for a in olds[1:]]
            given = [t if only in (None, k) else None for k, t in enumerate(grads)]
            ml.gatedDenseBackward(ctx, X, W, P, DY, -1.0, given[0], 0.5, given[1], given[2], "silu", work)
            for k, t in enumerate(grads):
                old = R.numbers(olds[k]) * (-1.0 if k == 0 else 0.5)
                if given[k] is None:
                    assert np.array_equal(R.numbers(t.copyToHost(ctx)), R.numbers(olds[k]))
                else:
                    assert R.worst(t.copyToHost(ctx), wants[k] + old, bounds[k] + 2 * R.rounded(old, dtype if k == 0 else "float32")) <= 1


def test_rows_that_are_not_finite_stay_alone(ctx):
    rng = np.random.default_rng(4)
    for rows in (20, 200):
        x, w, b, _, _ = inputs(rng, rows, 136, 48, "float16")
        W, Bias = ml.toDevice(ctx, w), ml.toDevice(ctx, b)
        results = []
        for bad in (False, True):
            if bad:
                x[3, 5], x[rows - 1, 135] = 0x7c00, 0x7e00
            X, y = ml.toDevice(ctx, x), ml.Tensor((rows, 48), "float16")
            ml.gatedDenseForward(ctx, X, W, Bias, y, None, "gelu", space(ctx, X, W, False))
            results.append(R.numbers(y.copyToHost(ctx)))
        keep = [r for r in range(rows) if r not in (3, rows - 1)]
        assert np.array_equal(results[0][keep], results[1][keep]) and np.isnan(results[1][rows - 1]).all() and not np.isfinite(results[1][3]).all()


def test_no_rows(ctx):
    x, w = ml.Tensor((2, 0, 64), "float16"), ml.toDevice(ctx, R.bits(np.ones((2, 24, 64)), "float16"))
    y, p = ml.Tensor((2, 0, 24), "float16"), ml.Tensor((2, 0, 2, 24), "float16")
    dw, db = ml.toDevice(ctx, np.full((2, 24, 64), 3.0, np.float32)), ml.toDevice(ctx, R.bits(np.full((2, 24), 5.0), "float16"))
    ml.gatedDenseForward(ctx, x, w, None, y, p, "silu", None)
    ml.gatedDenseBackward(ctx, x, w, p, y, 0.0, x, 0.5, dw, db, "silu", space(ctx, x, w, True))
    assert (dw.copyToHost(ctx) == 1.5).all() and (R.numbers(db.copyToHost(ctx)) == 2.5).all()


def test_gradient_agrees_with_differences(ctx):
    """sum(y * dy) along a direction: central differences of the forward pass in fp32 against the backward pass of what it kept."""
    rng = np.random.default_rng(6)
    rows, features, hidden = 80, 40, 24
    x, w, b, _, dy = inputs(rng, rows, features, hidden, "float32")
    work = [space(ctx, ml.toDevice(ctx, x), ml.toDevice(ctx, w), k) for k in (False, True)]
    for name in ("sigmoid", "silu", "gelu"):
        y, kept = ml.Tensor((rows, hidden), "float32"), ml.Tensor((rows, 2, hidden), "float32")

        def value(x, w, b):
            ml.gatedDenseForward(ctx, *(ml.toDevice(ctx, np.ascontiguousarray(a, np.float32)) for a in (x, w, b)), y, kept, name, work[0])
            return float((y.copyToHost(ctx).astype(np.float64) * dy).sum())

        value(x, w, b)
        grads = [ml.Tensor(a.shape, "float32") for a in (x, w, b)]
        ml.gatedDenseBackward(ctx, ml.toDevice(ctx, x), ml.toDevice(ctx, w), kept, ml.toDevice(ctx, dy), 0.0, grads[0], 0.0, grads[1], grads[2], name, work[1])
        for k, at in enumerate((x, w, b)):
            direction = rng.choice([-1.0, 1.0], at.shape).astype(np.float32)
            step = 2.0 ** -10
            ends = []
            for sign in (1, -1):
                args = [x, w, b]
                args[k] = at + sign * step * direction
                ends.append(value(*args))
            want = float((grads[k].copyToHost(ctx).astype(np.float64) * direction).sum())
            # 1920 elements of y, each at most a few units and off by 2^-20, over 2 steps; the third derivative along the direction: projections move by at most 6 + 4 per unit step, cubed, over all elements
            assert abs((ends[0] - ends[1]) / (2 * step) - want) <= 1920 * 2.0 ** -20 / (2 * step) + step ** 2 / 6 * 1920 * 10 ** 3 * 4


@pytest.mark.parametrize("rows,features,hidden", [(8, 512, 256), (200, 2048, 64), (1000, 200, 96)])
def test_recorded_pass_gives_the_eager_bits(ctx, rows, features, hidden):
    """Forward and backward in one graph, replayed with eager passes of another context between."""
    rng = np.random.default_rng(7)
    x, w, b, _, dy = inputs(rng, rows, features, hidden, "float16")
    other = ml.Context(0)
    passes = []
    for c in (ctx, other):
        X, W, Bias, DY = (ml.toDevice(c, a) for a in (x, w, b, dy))
        out = [ml.Tensor(s, "float16") for s in ((rows, hidden), (rows, 2, hidden), x.shape, w.shape, b.shape)]
        work = [space(c, X, W, k) for k in (False, True)]

        def both(c=c, X=X, W=W, Bias=Bias, DY=DY, out=out, work=work):
            ml.gatedDenseForward(c, X, W, Bias, out[0], out[1], "silu", work[0])
            ml.gatedDenseBackward(c, X, W, out[1], DY, 0.0, out[2], 0.0, out[3], out[4], "silu", work[1])

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
