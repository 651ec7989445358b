"""The distillation of a teacher's top logits and its gradients against the definition in 64 bits."""
import numpy as np
import pytest

import training_reference as R
import vocabulary_reference as V
from minml_amd import core as ml
from test_gpu_gated import check_guards, guarded

pytestmark = pytest.mark.gpu


def inputs(rng, rows, features, classes, count, dtype, logits_dtype=None, ignored=0.1):
    """A student that leans towards what its teacher names; some places name no class, some classes stand twice, some rows have none."""
    x, w, b = rng.standard_normal((rows, features)), 2 * rng.standard_normal((classes, features)) / np.sqrt(features), 0.5 * rng.standard_normal(classes)
    named = rng.integers(0, classes, (rows, count))
    logits = 3 * rng.standard_normal((rows, count))
    x += 1.5 * w[named[:, 0]]
    other = rng.random(named.shape) < ignored
    named[other] = rng.choice([-1, -100, classes, classes + 5, 2 ** 31 - 1, -2 ** 31], int(other.sum()))
    logits[rng.random(logits.shape) < 0.05] = -np.inf
    named[rng.random(rows) < 0.1] = -1
    logits = R.bits(logits, logits_dtype or dtype)
    unused = (named < 0) | (named >= classes)
    logits[unused] = rng.choice(R.bits(np.array([np.nan, np.inf, -np.inf, 5.0]), logits_dtype or dtype), int(unused.sum()))
    return [R.bits(a, dtype) for a in (x, w, b)] + [named.astype(np.int32), logits, (rng.standard_normal(rows) * 3).astype(np.float32)]


def space(ctx, x, w, count, backward):
    return V.workspace(ctx, ml.linearDistillationGetWorkspaceSize(ctx, x, w, count, backward))


class Distillation:
    """Both calls with everything around them, NaN beside the inputs."""

    def __init__(self, ctx, x, w, b, named, logits, temperature, dtype):
        self.ctx, self.temperature, self.dtype = ctx, temperature, dtype
        self.rows, self.count = named.shape
        self.X, self.W, self.B = (guarded(ctx, a, dtype, np.nan) for a in (x, w, b))
        self.named, self.logits = ml.toDevice(ctx, named), guarded(ctx, logits, "float16" if logits.dtype == np.uint16 else "float32", np.nan)
        self.loss, self.lse = (guarded(ctx, np.full(self.rows, np.nan, np.float32), "float32", 9.0) for _ in range(2))
        self.log_p = guarded(ctx, np.full(named.shape, np.nan, np.float32), "float32", 9.0)
        work = space(ctx, self.X, self.W, self.count, False)
        ml.linearDistillationForward(ctx, self.X, self.W, self.B, self.named, self.logits, temperature, self.loss, self.lse, self.log_p, work)
        V.check_workspace(ctx, work)
        for t in (self.loss, self.lse, self.log_p):
            check_guards(ctx, t, 9.0)

    def backward(self, dloss, dx, dw, db, beta=0.0, beta_weights=0.0):
        work = space(self.ctx, self.X, self.W, self.count, True)
        ml.linearDistillationBackward(self.ctx, self.X, self.W, self.B, self.named, self.logits, self.temperature, self.lse, self.log_p, ml.toDevice(self.ctx, dloss), beta, dx, beta_weights, dw, db, work)
        V.check_workspace(self.ctx, work)

    def gradients(self, dloss):
        out = [guarded(self.ctx, R.bits(np.full(t.shape, np.nan), self.dtype), self.dtype, 9.0) for t in (self.X, self.W, self.B)]
        self.backward(dloss, *out)
        for t in out:
            check_guards(self.ctx, t, 9.0)
        return [t.copyToHost(self.ctx) for t in out]


def check(ctx, data, temperature, dtype):
    x, w, b, named, logits, dloss = data
    step = Distillation(ctx, x, w, b, named, logits, temperature, dtype)
    args = [R.numbers(a) for a in (x, w, b)] + [named, R.numbers(logits), float(np.float32(temperature))]
    for got, want, off in zip((step.loss, step.lse, step.log_p), V.distillation(*args), V.distillation_bounds(*args, dtype)):
        assert R.worst(got.copyToHost(ctx), want, off + 1e-30) <= 1
    args.append(dloss.astype(np.float64))
    for got, want, off in zip(step.gradients(dloss), V.distillation_gradients(*args), V.distillation_gradient_bounds(*args, dtype)):
        assert R.worst(got, want, off) <= 1


SIZES = [(1, 8, 1, 1), (1, 64, 300, 5), (3, 63, 20, 40), (16, 200, 37, 8), (17, 130, 16, 16), (33, 72, 1000, 64), (64, 333, 100, 3), (65, 40, 513, 100), (130, 65, 257, 256), (300, 200, 130, 17),
         (129, 1096, 24, 2), (2, 2056, 70, 1), (3500, 24, 3700, 9), (513, 64, 8, 300), (1, 16, 40001, 1024), (2, 8, 300000, 33), (9000, 8, 20, 4), (257, 48, 3000, 65), (24, 1021, 9000, 12), (17, 1024, 9000, 5), (7, 4100, 333, 11), (5, 5, 2000, 6), (8, 515, 5003, 30), (9, 256, 4000, 8), (2, 16384, 40, 3), (4, 1, 70, 9)]


@pytest.mark.parametrize("dtype", ["float16", "float32"])
@pytest.mark.parametrize("rows,features,classes,count", SIZES)
def test_loss_and_gradients(ctx, rows, features, classes, count, dtype):
    rng = np.random.default_rng(rows * 10007 + features * 101 + classes + count)
    check(ctx, inputs(rng, rows, features, classes, count, dtype), (1.0, 2.0, 0.7)[(rows + count) % 3], dtype)


@pytest.mark.parametrize("dtype", ["float16", "float32"])
@pytest.mark.parametrize("rows,features,classes,count", [(6819, 48, 838, 66), (3001, 160, 2000, 40), (1200, 96, 3000, 20), (700, 256, 5000, 100)])
def test_many_tiles_at_once(ctx, rows, features, classes, count, dtype):
    """More tiles than the units take at a time, which keeps the wavefronts of a workgroup apart: what one lays down for a tile's end may not be where another still reads the product's operands, whose chunks are even in number."""
    rng = np.random.default_rng(rows)
    check(ctx, inputs(rng, rows, features, classes, count, dtype), 2.0, dtype)


def test_logits_of_the_teacher_in_fp32(ctx):
    rng = np.random.default_rng(1)
    for rows, features, classes, count in ((5, 64, 700, 12), (200, 40, 400, 30)):
        check(ctx, inputs(rng, rows, features, classes, count, "float16", "float32"), 3.0, "float16")


def test_more_classes_than_one_piece_holds(ctx):
    """4100 rows in fp32: d of 17000 classes is more than 256 MB, so the classes are taken in two pieces, the second one smaller, and a row's lie in both; the gradients are added to what was there."""
    rng = np.random.default_rng(2)
    x, w, b, named, logits, dloss = inputs(rng, 4100, 8, 17000, 20, "float32")
    step = Distillation(ctx, x, w, b, named, logits, 2.0, "float32")
    olds = [rng.standard_normal(a.shape).astype(np.float32) for a in (x, w, b)]
    grads = [ml.toDevice(ctx, a) for a in olds]
    step.backward(dloss, *grads, 0.5, -1.0)
    args = [a.astype(np.float64) for a in (x, w, b)] + [named, logits.astype(np.float64), 2.0, dloss.astype(np.float64)]
    for got, exact, off, old, beta in zip(grads, V.distillation_gradients(*args), V.distillation_gradient_bounds(*args, "float32"), olds, (0.5, -1.0, -1.0)):
        assert R.worst(got.copyToHost(ctx), exact + beta * old.astype(np.float64), off + 2 * R.rounded(old, "float32")) <= 1


def test_more_classes_than_one_piece_holds_of_few_rows(ctx):
    """A piece has 524288 classes at most; the rows' low parts lie behind d's rows in both."""
    check(ctx, inputs(np.random.default_rng(12), 20, 8, 530000, 9, "float16"), 2.0, "float16")


@pytest.mark.parametrize("dtype", ["float16", "float32"])
def test_gradients_are_added_and_may_be_left_out(ctx, dtype):
    rng = np.random.default_rng(3)
    for rows, features, classes, count in ((6, 72, 400, 10), (3, 33, 90, 7), (90, 72, 400, 10), (600, 33, 70, 20)):
        x, w, b, named, logits, dloss = inputs(rng, rows, features, classes, count, dtype)
        olds = [R.bits(rng.standard_normal(a.shape), dtype) for a in (x, w, b)]
        step = Distillation(ctx, x, w, b, named, logits, 2.0, dtype)
        args = [R.numbers(a) for a in (x, w, b)] + [named, R.numbers(logits), 2.0, dloss.astype(np.float64)]
        wants, bounds = V.distillation_gradients(*args), V.distillation_gradient_bounds(*args, dtype)
        for only in (None, 0, 1, 2):
            grads = [ml.toDevice(ctx, olds[0])] + [ml.toDevice(ctx, R.numbers(a).astype(np.float32)) for a in olds[1:]]
            given = [t if only in (None, k) else None for k, t in enumerate(grads)]
            step.backward(dloss, *given, -1.0, 0.5)
            for k, t in enumerate(grads):
                old = R.numbers(olds[k]) * (-1.0 if k == 0 else 0.5)
                if given[k] is None:
                    assert np.array_equal(R.numbers(t.copyToHost(ctx)), R.numbers(olds[k]))
                else:
                    assert R.worst(t.copyToHost(ctx), wants[k] + old, bounds[k] + 2 * R.rounded(old, dtype if k == 0 else "float32")) <= 1


@pytest.mark.parametrize("dtype", ["float16", "float32"])
@pytest.mark.parametrize("scale", [1e-30, 1e-6, 1e4])
def test_gradients_of_losses_of_any_size(ctx, dtype, scale):
    rng = np.random.default_rng(5)
    x, w, b, named, logits, dloss = inputs(rng, 100, 64, 5000, 32, dtype)
    dloss *= scale
    step = Distillation(ctx, x, w, b, named, logits, 2.0, dtype)
    dw, db = ml.Tensor((5000, 64), "float32"), ml.Tensor((5000,), "float32")
    step.backward(dloss, None, dw, db)
    args = [R.numbers(a) for a in (x, w, b)] + [named, R.numbers(logits), 2.0, dloss.astype(np.float64)]
    wants, bounds = V.distillation_gradients(*args), V.distillation_gradient_bounds(*args, dtype)
    for got, k in ((dw, 1), (db, 2)):
        assert R.worst(got.copyToHost(ctx), wants[k], bounds[k]) <= 1


@pytest.mark.parametrize("dtype", ["float16", "float32"])
def test_a_teacher_that_the_student_agrees_with(ctx, dtype):
    """The teacher's classes are the student's best, with the student's logits and all of its mass but 1e-4: p and q are close everywhere, and so small differences of theirs are all there is."""
    rng = np.random.default_rng(7)
    rows, features, classes, count = 200, 64, 600, 32
    x, w, b = (R.bits(a, dtype) for a in (rng.standard_normal((rows, features)), rng.standard_normal((classes, features)) / 8, 0.1 * rng.standard_normal(classes)))
    z = R.numbers(x) @ R.numbers(w).T + R.numbers(b)
    named = np.argsort(-z, 1)[:, :count].astype(np.int32)
    b2 = R.numbers(b) - 12
    taken = np.zeros(classes, bool)
    taken[named] = True
    b = R.bits(np.where(taken, R.numbers(b), b2), dtype)
    z = R.numbers(x) @ R.numbers(w).T + R.numbers(b)
    logits = np.take_along_axis(z, named, 1).astype(np.float32)
    check(ctx, [x, w, b, named, logits, np.full(rows, 2.0, np.float32)], 1.0, dtype)


def test_one_class_of_the_teacher_is_the_cross_entropy(ctx):
    """A teacher that is sure of one class at temperature 1: the cross entropy's loss, and its gradients as far as their roundings go."""
    rng = np.random.default_rng(8)
    for rows in (20, 150):
        x, w, b, named, logits, dloss = inputs(rng, rows, 64, 900, 1, "float16")
        logits[np.isneginf(R.numbers(logits))] = 0
        step = Distillation(ctx, x, w, b, named, logits, 1.0, "float16")
        loss, lse = ml.Tensor((rows,), "float32"), ml.Tensor((rows,), "float32")
        work = ml.Tensor((ml.linearCrossEntropyGetWorkspaceSize(ctx, step.X, step.W, True),), "uint8")
        T = ml.toDevice(ctx, named.reshape(-1))
        ml.linearCrossEntropyForward(ctx, step.X, step.W, step.B, T, loss, lse, work)
        assert np.array_equal(lse.copyToHost(ctx), step.lse.copyToHost(ctx)) and np.allclose(loss.copyToHost(ctx), step.loss.copyToHost(ctx), rtol=2e-7, atol=0)
        other = [ml.Tensor(t.shape, "float16") for t in (step.X, step.W, step.B)]
        ml.linearCrossEntropyBackward(ctx, step.X, step.W, step.B, T, lse, ml.toDevice(ctx, dloss), 0.0, other[0], 0.0, other[1], other[2], work)
        args = [R.numbers(a) for a in (x, w, b)] + [named, R.numbers(logits), 1.0, dloss.astype(np.float64)]
        for got, same, off in zip(step.gradients(dloss), other, V.distillation_gradient_bounds(*args, "float16")):
            assert (np.abs(R.numbers(got) - R.numbers(same.copyToHost(ctx))) <= 2 * off).all()


@pytest.mark.parametrize("common", [0, 10])
@pytest.mark.parametrize("rows,features,classes,count,ignored", [(40, 512, 2000, 24, 0.1), (300, 200, 900, 64, 0.1), (1100, 96, 300, 1, 0.1), (1500, 1024, 256, 40, 0.1), (600, 333, 500, 16, 0.99)])
def test_fp16_gradients_are_off_by_their_roundings_alone(ctx, rows, features, classes, count, ignored, common):
    """Teachers and students that are sure of nothing, so that no class has most of d, also where the rows of W have much in common: dx is as far off as random roundings are. The sum over rows x features (20480 at least) and,
    for d, rows x as many classes as are likely, is within a tenth of what is expected."""
    rng = np.random.default_rng(rows + common)
    x, w, b, named, logits, _ = inputs(rng, rows, features, classes, count, "float16", ignored=ignored)
    w, logits = R.bits(R.numbers(w) + common * 2 / np.sqrt(features) * rng.standard_normal(features), "float16"), R.bits(np.where(np.isneginf(R.numbers(logits)), -np.inf, R.numbers(logits) / 3), "float16")
    dloss = rng.uniform(0.5, 1, rows).astype(np.float32) * rng.choice([-1, 1], rows).astype(np.float32)
    step = Distillation(ctx, x, w, b, named, logits, 2.0, "float16")
    args = [R.numbers(a) for a in (x, w, b)] + [named, R.numbers(logits), 2.0, dloss.astype(np.float64)]
    error = np.linalg.norm(R.numbers(step.gradients(dloss)[0]) - V.distillation_gradients(*args)[0])
    assert error <= 1.1 * V.distillation_input_noise(*args)


@pytest.mark.parametrize("common", [0, 10])
@pytest.mark.parametrize("rows,features,classes,count", [(9, 512, 2000, 24), (33, 333, 500, 16), (64, 200, 3001, 40), (17, 1024, 300, 1)])
def test_fp16_gradients_of_few_rows_are_off_by_their_own_roundings_alone(ctx, rows, features, classes, count, common):
    """Up to 64 rows what rounding leaves of d takes part in both products: dx and dW are as far off as rounding them makes them, a twelfth of a spacing squared for each element, of 4608 elements or more (a tenth is four
    standard deviations and more)."""
    rng = np.random.default_rng(rows + common)
    x, w, b, named, logits, dloss = inputs(rng, rows, features, classes, count, "float16")
    w = R.bits(R.numbers(w) + common * 2 / np.sqrt(features) * rng.standard_normal(features), "float16")
    step = Distillation(ctx, x, w, b, named, logits, 2.0, "float16")
    args = [R.numbers(a) for a in (x, w, b)] + [named, R.numbers(logits), 2.0, dloss.astype(np.float64)]
    for got, want in zip(step.gradients(dloss)[:2], V.distillation_gradients(*args)):
        assert np.linalg.norm(R.numbers(got) - want) <= 1.1 * np.sqrt((V.spacing(want) ** 2).sum() / 12)


def test_rows_without_a_teacher_and_without_gradient(ctx):
    rng = np.random.default_rng(9)
    for rows in (9, 90):
        x, w, b, named, logits, dloss = inputs(rng, rows, 64, 500, 6, "float32", ignored=0)
        named[2], logits[3], dloss[4] = -1, -np.inf, 0
        step = Distillation(ctx, x, w, b, named, logits, 2.0, "float32")
        loss, log_p = step.loss.copyToHost(ctx), step.log_p.copyToHost(ctx)
        assert loss[2] == 0 and loss[3] == 0 and (log_p[2:4] == 0).all() and np.isfinite(step.lse.copyToHost(ctx)).all()
        dx = step.gradients(dloss)[0]
        assert (dx[2:5] == 0).all() and np.isfinite(dx).all()


def test_masked_classes_and_infinities(ctx):
    """Classes that a bias of -inf or of the type's lowest value takes out of the student: no gradient where the teacher does not name them, an infinite loss where it does; a row of NaN stays in its row."""
    rng = np.random.default_rng(10)
    for rows in (9, 90):
        x, w, b, named, logits, dloss = inputs(rng, rows, 64, 500, 6, "float32", ignored=0)
        named[:], logits[:] = rng.permuted(np.tile(np.arange(100), (rows, 1)), axis=1)[:, :6], rng.standard_normal(logits.shape)
        b[100:200], b[200:250] = -np.inf, np.finfo(np.float32).min
        step = Distillation(ctx, x, w, b, named, logits, 2.0, "float32")
        inside = np.r_[0:100, 250:500]
        args = [x.astype(np.float64), w[inside].astype(np.float64), b[inside].astype(np.float64), named, logits.astype(np.float64), 2.0]
        assert R.worst(step.loss.copyToHost(ctx), V.distillation(*args)[0], V.distillation_bounds(*args, "float32")[0]) <= 1
        dx, dw, db = step.gradients(dloss)
        args.append(dloss.astype(np.float64))
        for got, want, off in zip((dx, dw[inside], db[inside]), V.distillation_gradients(*args), V.distillation_gradient_bounds(*args, "float32")):
            assert R.worst(got, want, off) <= 1
        assert (dw[100:250] == 0).all() and (db[100:250] == 0).all()
        named[1, 2], x[3] = 150, np.nan
        step = Distillation(ctx, x, w, b, named, logits, 2.0, "float32")
        loss = step.loss.copyToHost(ctx)
        assert loss[1] == np.inf and np.isnan(loss[3]) and np.isfinite(np.delete(loss, [1, 3])).all() and step.log_p.copyToHost(ctx)[1, 2] == -np.inf


def test_no_rows(ctx):
    X, W, named, logits = ml.Tensor((0, 16), "float32"), ml.toDevice(ctx, np.ones((20, 16), np.float32)), ml.Tensor((0, 3), "int32"), ml.Tensor((0, 3), "float32")
    none = ml.Tensor((0,), "float32")
    ml.linearDistillationForward(ctx, X, W, None, named, logits, 1.0, none, none, logits, None)
    dw = ml.toDevice(ctx, np.full((20, 16), 4.0, np.float32))
    ml.linearDistillationBackward(ctx, X, W, None, named, logits, 1.0, none, logits, none, 0.0, None, 0.5, dw, None, None)
    assert (dw.copyToHost(ctx) == 2).all()


def test_the_same_bits_every_time(ctx):
    """What several threads add to the sums of a column is added in whole numbers: no order changes it."""
    rng = np.random.default_rng(11)
    x, w, b, named, logits, dloss = inputs(rng, 700, 64, 40, 60, "float16")
    step = Distillation(ctx, x, w, b, named, logits, 2.0, "float16")
    first = step.gradients(dloss)
    for _ in range(3):
        assert all(np.array_equal(a, b) for a, b in zip(first, step.gradients(dloss)))


@pytest.mark.parametrize("dtype,logits_dtype", [("float16", "float16"), ("float16", "float32"), ("float32", "float32")])
@pytest.mark.parametrize("rows", [3, 20, 130])
def test_probabilities_of_the_teacher_at_a_small_temperature(ctx, rows, dtype, logits_dtype):
    """Logits of about 20 at a temperature of 0.01: v / t is about 2000, whose rounding to fp32 would take 6e-5 of a probability, but only v - max v counts. The student's logits are zeros, and no class is named twice, so db
    is what all rows have of it, 1 / 4000 each, less the one probability of the teacher."""
    rng = np.random.default_rng(rows)
    classes, count, temperature = 4000, 20, float(np.float32(0.01))
    named = rng.permutation(classes)[:rows * count].reshape(rows, count).astype(np.int32)
    logits = R.bits(20 + 0.05 * rng.random((rows, count)), logits_dtype)
    x, w, b = (R.bits(a, dtype) for a in (rng.standard_normal((rows, 16)), np.zeros((classes, 16)), np.zeros(classes)))
    step = Distillation(ctx, x, w, b, named, logits, temperature, dtype)
    db = ml.Tensor((classes,), "float32")
    step.backward(np.ones(rows, np.float32), None, None, db)
    dense, q, _ = V.teacher(named, R.numbers(logits), classes, temperature)
    # v - max v is exact (both are between 16 and 32); the quotient, up to 6, is rounded once; 24 roundings for the exponential, the sum's joins and the division; the sum's additions
    relative = R.FP32 * (6 + 24 + count / 32)
    p = rows / classes
    # the student's: lse is 8.3, rounded, the hardware's exponential takes 8.3 log2(e) in fp32: below 2^-18
    assert R.worst(db.copyToHost(ctx), (p - dense.sum(0)) / temperature, (dense.sum(0) * (relative + 4 * R.FP32) + p * 2.0 ** -18) / temperature) <= 1
    log_q = np.log(q)
    loss = (q * (log_q + np.log(classes))).sum(1)
    assert R.worst(step.loss.copyToHost(ctx), loss, (relative + 24 * R.FP32) * (q * (np.abs(log_q) + np.log(classes) + 1)).sum(1)) <= 1


@pytest.mark.parametrize("rows", [3, 20, 130])
def test_a_temperature_that_makes_infinities(ctx, rows):
    """At 1e-38 a logit of 5 over it is none of fp32, and one of -5 is no -inf that does not count: the teacher is sure of its best class, or of both."""
    rng = np.random.default_rng(rows)
    classes = 300
    named, logits = np.array([[7, 8, 9], [10, -1, -1], [20, 30, 40]], np.int32), np.array([[4, 5, -5], [-5, 9, 9], [7, 7, 6]], np.float32)
    named, logits = (np.tile(a, (rows // 3 + 1, 1))[:rows] for a in (named, logits))
    x, w, b = rng.standard_normal((rows, 16)).astype(np.float32), np.zeros((classes, 16), np.float32), np.zeros(classes, np.float32)
    step = Distillation(ctx, x, w, b, named, logits, 1e-38, "float32")
    want = np.tile(np.log(classes) - np.array([0, 0, np.log(2)]), rows // 3 + 1)[:rows]
    # logarithms below 8 and sums of them
    assert R.worst(step.loss.copyToHost(ctx), want, np.full(rows, 32 * R.FP32)) <= 1
    assert R.worst(step.log_p.copyToHost(ctx), np.where(named >= 0, -np.log(classes), 0), np.full(named.shape, 32 * R.FP32)) <= 1


def test_more_rows_than_a_launch_has_wavefronts_for(ctx):
    """2^26 + 5 rows of zeros and three classes: the student's distribution is that of the bias alone, the teacher's is all of class 0, which it names twice; a few rows have a teacher of their own. dx is checked at them, and db,
    which is a sum of equal numbers but for them, over all."""
    rows, classes, features = 2 ** 26 + 5, 3, 8
    picked = {0: (1, 2), 4: (2, -1), 2 ** 22 + 3: (0, 1), 2 ** 26 - 1: (1, 1), 2 ** 26: (2, 1), rows - 1: (-1, 1)}
    x, named, logits = ml.Tensor((rows, features), "float16"), ml.Tensor((rows, 2), "int32"), ml.Tensor((rows, 2), "float16")
    for t in (x, named, logits):
        t.zeroall(ctx)
    for row, c in picked.items():
        named.view((2,), 2 * row).copyFromHost(ctx, np.array(c, np.int32))
    w, bias = R.bits(np.arange(24).reshape(classes, features) / 16, "float16"), np.array([0.0, 1.0, -2.0])
    W, B = ml.toDevice(ctx, w), ml.toDevice(ctx, R.bits(bias, "float16"))
    loss, lse, log_p, dloss, dx, db = (ml.Tensor(s, d) for s, d in (((rows,), "float32"), ((rows,), "float32"), ((rows, 2), "float32"), ((rows,), "float32"), ((rows, features), "float16"), ((classes,), "float32")))
    dloss.setall(ctx, 1.0)
    work = ml.Tensor((ml.linearDistillationGetWorkspaceSize(ctx, x, W, 2, True),), "uint8")
    ml.linearDistillationForward(ctx, x, W, B, named, logits, 1.0, loss, lse, log_p, work)
    ml.linearDistillationBackward(ctx, x, W, B, named, logits, 1.0, lse, log_p, dloss, 0.0, dx, 0.0, None, db, work)
    p = np.exp(bias) / np.exp(bias).sum()
    losses, log_ps = loss.copyToHost(ctx), log_p.copyToHost(ctx)
    total, others = rows * p, np.ones(rows, bool)
    total[0] -= rows - len(picked)
    for row, c in picked.items():
        q = np.zeros(classes)
        for v in c:
            if v >= 0:
                q[v] += 1 / (np.array(c) >= 0).sum()
        total -= q
        others[row] = False
        want = sum(v * (np.log(v) - np.log(p[k])) for k, v in enumerate(q) if v > 0)
        assert abs(losses[row] - want) <= 40 * R.FP32  # as for the cross entropy of as many rows
        assert np.abs(log_ps[row] - np.array([np.log(p[v]) if v >= 0 else 0 for v in c])).max() <= 40 * R.FP32
        # d of up to 1 in fp16, three of them times weights up to 1.5, and the result's rounding
        assert np.abs(R.numbers(dx.view((features,), row * features).copyToHost(ctx)) - (p - q) @ R.numbers(w)).max() <= 4 * 3 * R.STEP["float16"]
    assert np.abs(losses[others] + np.log(p[0])).max() <= 40 * R.FP32 and np.abs(log_ps[others] - np.log(p[0])).max() <= 40 * R.FP32
    # a row's p is 2^-18 off at most (the hardware's exponential, lse), the sums of 128 and of 2^19 tiles, in eighths, go through below 2^17 additions of numbers that are equal but for few
    assert np.abs(db.copyToHost(ctx) - total).max() <= rows * (2.0 ** -18 + 2 ** 17 * R.FP32)
