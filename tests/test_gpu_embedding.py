"""The embedding and its table's gradient against the definition in 64 bits."""
import numpy as np
import pytest

import training_reference as R
import vocabulary_reference as V
from minml_amd import core as ml
from test_gpu_gated import check_guards, guarded

pytestmark = pytest.mark.gpu

# one token to more than one workgroup sorts at once and more than one of its digits; tables of one row, of one digit of the sort and of two; rows below, at and beyond a vector
SIZES = [(1, 1, 1), (1, 7, 3), (3, 2, 8), (5, 300, 7), (63, 2, 5), (64, 1, 9), (65, 300, 16), (129, 40, 4096), (1000, 17, 40), (2047, 2048, 13), (4096, 50, 24), (4097, 3000, 33), (9000, 2, 260),
         (20000, 70000, 8), (70001, 1023, 12), (3001, 5, 2056), (70, 3, 9000), (300000, 5, 4), (4000, 1, 24), (3501, 400, 16), (6001, 1500, 24), (8193, 2049, 9), (12000, 130000, 16)]


def tokens_of(rng, rows, classes, ignored=0.1):
    """Often few classes have most of the tokens; some tokens are no class."""
    tokens = np.minimum((np.exp(rng.random(rows) * np.log(classes + 1.0)) - 1).astype(np.int64), classes - 1)
    other = rng.random(rows) < ignored
    tokens[other] = rng.choice([-1, -100, classes, classes + 5, 2 ** 31 - 1, -2 ** 31], int(other.sum()))
    return tokens.astype(np.int32)


def space(ctx, tokens, table):
    return V.workspace(ctx, ml.embeddingGetWorkspaceSize(ctx, tokens, table))


@pytest.mark.parametrize("dtype", ["float16", "float32"])
@pytest.mark.parametrize("rows,classes,features", SIZES)
def test_forward(ctx, rows, classes, features, dtype):
    rng = np.random.default_rng(rows * 10007 + classes * 101 + features)
    tokens, table = tokens_of(rng, rows, classes), R.bits(rng.standard_normal((classes, features)), dtype)
    scale = float(np.float32(np.sqrt(features)))
    y = guarded(ctx, R.bits(np.zeros((rows, features)), dtype), dtype, 9.0)
    ml.embeddingForward(ctx, ml.toDevice(ctx, tokens), guarded(ctx, table, dtype, np.nan), scale, y)
    want = V.embedding(tokens, R.numbers(table), scale)
    got = y.copyToHost(ctx)
    assert R.worst(got, want, V.embedding_bound(want, dtype)) <= 1
    assert (R.numbers(got)[(tokens < 0) | (tokens >= classes)] == 0).all()
    check_guards(ctx, y, 9.0)


@pytest.mark.parametrize("dtype,out", [("float16", "float16"), ("float16", "float32"), ("float32", "float32")])
@pytest.mark.parametrize("rows,classes,features", SIZES)
def test_gradient(ctx, rows, classes, features, dtype, out):
    """Written over NaN, and added to what was there; rows of the gradient without a class hold NaN, which reaches nothing."""
    rng = np.random.default_rng(rows * 10009 + classes * 103 + features)
    tokens, dy = tokens_of(rng, rows, classes), R.bits(rng.standard_normal((rows, features)), dtype)
    outside = (tokens < 0) | (tokens >= classes)
    dy[outside] = R.bits(np.full((1, features), np.nan), dtype)
    T, DY = ml.toDevice(ctx, tokens), guarded(ctx, dy, dtype, np.nan)
    exact, weighted = V.embedding_gradient(tokens, np.where(outside[:, None], 0, R.numbers(dy)), classes, 0.5)
    old = R.bits(rng.standard_normal((classes, features)), out)
    for beta in (0.0, 1.0, -0.75):
        dtable = guarded(ctx, R.bits(np.full(old.shape, np.nan), out) if beta == 0 else old, out, 9.0)
        work = space(ctx, T, dtable)
        ml.embeddingBackward(ctx, T, DY, 0.5, beta, dtable, work)
        V.check_workspace(ctx, work)
        kept = beta * R.numbers(old)
        assert R.worst(dtable.copyToHost(ctx), exact + kept, V.embedding_gradient_bound(exact, weighted, kept, out)) <= 1
        check_guards(ctx, dtable, 9.0)


def test_rows_that_no_token_names(ctx):
    """beta 1 leaves them as they are to the last bit, infinities and NaN among them; beta 0 makes zeros of them."""
    tokens = np.array([3, -1, 3, 9, 12], np.int32)
    old = np.full((11, 9), 7.0, np.float32)
    old[0], old[5] = np.nan, -np.inf
    T, DY = ml.toDevice(ctx, tokens), ml.toDevice(ctx, np.ones((5, 9), np.float32))
    for beta in (1.0, 0.0):
        dtable = ml.toDevice(ctx, old)
        ml.embeddingBackward(ctx, T, DY, 2.0, beta, dtable, space(ctx, T, dtable))
        want = beta * np.nan_to_num(old, nan=0, neginf=0) if beta == 0 else old.copy()
        want[3], want[9] = want[3] + 4, want[9] + 2
        assert np.array_equal(dtable.copyToHost(ctx), want, equal_nan=True)


def test_no_tokens(ctx):
    T, DY = ml.Tensor((0,), "int32"), ml.Tensor((0, 6), "float32")
    for beta, want in ((0.0, 0.0), (0.5, 4.0)):
        dtable = ml.toDevice(ctx, np.full((4, 6), 8.0, np.float32))
        ml.embeddingBackward(ctx, T, DY, 1.0, beta, dtable, None)
        assert (dtable.copyToHost(ctx) == want).all()
    ml.embeddingForward(ctx, T, dtable, 1.0, DY)
    # tokens that are all none of the table's
    T = ml.toDevice(ctx, np.full(5000, -1, np.int32))
    DY = ml.toDevice(ctx, np.full((5000, 6), np.nan, np.float32))
    ml.embeddingBackward(ctx, T, DY, 1.0, 0.0, dtable, space(ctx, T, dtable))
    assert (dtable.copyToHost(ctx) == 0).all()


def test_the_same_bits_every_time(ctx):
    rng = np.random.default_rng(4)
    for rows, classes, features in ((4000, 30, 40), (60000, 300, 24)):
        T, DY = ml.toDevice(ctx, tokens_of(rng, rows, classes)), ml.toDevice(ctx, rng.standard_normal((rows, features)).astype(np.float32))
        results = []
        for _ in range(3):
            dtable = ml.Tensor((classes, features), "float32")
            ml.embeddingBackward(ctx, T, DY, 1.0, 0.0, dtable, space(ctx, T, dtable))
            results.append(dtable.copyToHost(ctx))
        assert all(np.array_equal(results[0], r) for r in results)


@pytest.mark.parametrize("dtype", ["float16", "float32"])
def test_tensors_that_begin_at_any_element(ctx, dtype):
    rng = np.random.default_rng(6)
    for rows, classes, features in ((50, 20, 24), (50, 20, 33), (700, 3, 2050)):
        tokens, dy = tokens_of(rng, rows, classes), R.bits(rng.standard_normal((rows, features)), dtype)
        table = R.bits(rng.standard_normal((classes, features)), dtype)
        shifted = lambda a: ml.toDevice(ctx, np.concatenate([a.reshape(-1)[:1], a.reshape(-1)])).view(a.shape, 1)
        T, y, dtable = shifted(tokens), shifted(dy), shifted(table)
        ml.embeddingForward(ctx, T, shifted(table), 3.0, y)
        want = V.embedding(tokens, R.numbers(table), 3.0)
        assert R.worst(y.copyToHost(ctx), want, V.embedding_bound(want, dtype)) <= 1
        ml.embeddingBackward(ctx, T, shifted(dy), 1.0, 0.0, dtable, space(ctx, T, dtable))
        exact, weighted = V.embedding_gradient(tokens, R.numbers(dy), classes, 1.0)
        assert R.worst(dtable.copyToHost(ctx), exact, V.embedding_gradient_bound(exact, weighted, 0 * exact, dtype)) <= 1
        assert R.numbers(dtable._owner.copyToHost(ctx))[0] == R.numbers(table).reshape(-1)[0]


# classes of up to 100000 rows; more tokens than the sort keeps in registers, with one digit, two and, of 2^22 classes and more, three
WHOLE = [(1, 7, 3), (65, 300, 16), (2047, 2048, 13), (9000, 2, 260), (3001, 5, 2056), (12000, 130000, 16), (70001, 1023, 12), (70001, 5000, 8), (66000, 2048, 1), (200000, 60000, 4), (300000, 5, 4), (9000, 4200000, 1), (90000, 5000000, 3)]


@pytest.mark.parametrize("dtype,out", [("float16", "float16"), ("float16", "float32"), ("float32", "float32")])
@pytest.mark.parametrize("rows,classes,features", WHOLE)
def test_gradient_of_whole_numbers(ctx, rows, classes, features, dtype, out):
    """Rows of whole numbers from 1 to 7, of either sign, times 2^-8, whose sums are exact in 32 bits in any order: a row that is left out, taken twice or added to another class changes every column of its class. In fp16 what
    is left is one rounding to nearest."""
    rng = np.random.default_rng(rows * 10037 + classes * 107 + features)
    tokens = tokens_of(rng, rows, classes)
    dy = rng.integers(1, 8, (rows, features)) * rng.choice([-1, 1], (rows, features), p=[0.3, 0.7])
    kept = (tokens >= 0) & (tokens < classes)
    total = np.zeros((classes, features), np.int64)
    np.add.at(total, tokens[kept], dy[kept])
    old = rng.integers(-8, 9, total.shape)
    assert np.abs(total).max() + 8 < 2 ** 24
    T, DY = ml.toDevice(ctx, tokens), guarded(ctx, R.bits(dy, dtype), dtype, np.nan)
    for beta in (0.0, 1.0):
        dtable = guarded(ctx, R.bits(np.full(old.shape, np.nan) if beta == 0 else old / 256, out), out, 9.0)
        work = space(ctx, T, dtable)
        ml.embeddingBackward(ctx, T, DY, 2.0 ** -8, beta, dtable, work)
        V.check_workspace(ctx, work)
        assert np.array_equal(R.numbers(dtable.copyToHost(ctx)), R.numbers(R.bits((total + int(beta) * old) / 256, out)))
        check_guards(ctx, dtable, 9.0)
